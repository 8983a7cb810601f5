// Attention of each query over the key blocks that were chosen for it (64 keys to a block), the choice itself, and the
// gradients.
//
//   keys[b][h][j]    = mean of block j's valid keys                         (dm_block_keys)
//   blocks[b][h][i]  = the `top` blocks of the highest q_i . keys_j         (dm_block_select)
//   p_it             = softmax over the valid keys t of query i's blocks of scale * q_i . k_t
//   out_i            = sum_t p_it v_t                                       (dm_block_attention_fwd)
//   delta_i          = do_i . out_i,  ds_it = p_it (do_i . v_t - delta_i) scale
//   dq_i = sum_t ds_it k_t,  dk_t = sum_i ds_it q_i,  dv_t = sum_i p_it do_i  (dm_block_attention_bwd)
//
// Query heads share key heads (Hq = G Hkv). The ROWS of a (sample, key head) are its G Lq queries, r = i G + g: they all
// read the same keys and values. delta is taken from out and what out's rounding lost (out_lo): where a query's weight lies on
// few keys, ds is a small difference of do . v and delta, and the rounding of out alone would be as large. No kernel adds with float atomics: results do not depend on scheduling.
#include "dm_common.h"

namespace {

constexpr int BLK = 64;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct Rows {          // a [B][L][H][D] tensor by element strides, D contiguous
  const bf16_t* p;
  long sb, sl, sh;
};

struct Args {
  Rows q, k, v;
  const bf16_t *o, *o_lo, *go;   // forward output, what its rounding lost, its gradient: [B][Lq][Hq][D]
  bf16_t *out, *out_lo, *dq, *dk, *dv;
  long dqb, dql, dqh, dkb, dkl, dkh, dvb, dvl, dvh;
  float *lse, *delta;
  const int* blocks;
  const int* k_len;
  unsigned long long* mask;
  int B, Lq, Lk, Hq, Hkv, G, top, nblk;
  float scale;
};

__device__ __forceinline__ int valid_keys(const int* k_len, int b, int Lk) {
  return k_len ? min(max(k_len[b], 0), Lk) : Lk;
}

// x of the lane whose number differs in bit log2(O), or (O = 4, 8, once smaller distances are reduced) of a lane that
// holds that lane's value: sums and maxima over lane groups without LDS traffic
template <int O>
__device__ __forceinline__ float lane_xor(float x) {
  const int v = __builtin_bit_cast(int, x);
  int r;
  if constexpr (O == 1) r = __builtin_amdgcn_update_dpp(v, v, 0xB1, 0xF, 0xF, false);        // quad_perm [1,0,3,2]
  else if constexpr (O == 2) r = __builtin_amdgcn_update_dpp(v, v, 0x4E, 0xF, 0xF, false);   // quad_perm [2,3,0,1]
  else if constexpr (O == 4) r = __builtin_amdgcn_update_dpp(v, v, 0x141, 0xF, 0xF, false);  // row_half_mirror
  else r = __builtin_amdgcn_update_dpp(v, v, 0x140, 0xF, 0xF, false);                        // row_mirror
  return __builtin_bit_cast(float, r);
}
template <int LPR>   // sum over groups of LPR <= 8 neighbouring lanes
__device__ __forceinline__ float group_sum(float x) {
  if constexpr (LPR > 1) x += lane_xor<1>(x);
  if constexpr (LPR > 2) x += lane_xor<2>(x);
  if constexpr (LPR > 4) x += lane_xor<4>(x);
  return x;
}
template <int LPR>   // over the lanes l, l + LPR, l + 2 LPR ...
__device__ __forceinline__ float across_max(float x) {
#pragma unroll
  for (int o = LPR; o < 64; o <<= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
  return x;
}
template <int LPR>
__device__ __forceinline__ float across_sum(float x) {
#pragma unroll
  for (int o = LPR; o < 64; o <<= 1) x += __shfl_xor(x, o, 64);
  return x;
}

// ---------------------------------------------------------------------------------------------------------------
// One summary per block: the mean of its valid keys. Summed in 64 bits (64 bf16 values of ordinary spread add up
// exactly, so the order does not matter) and rounded to fp32 and then bf16: the summary is only a score's operand, and
// as bf16 its products with q are exact in 64-bit sums too, which makes the choice of blocks independent of batch, tile and order.
// A workgroup holds one block of up to 512 features (8 a lane) of all heads, its threads splitting the 64 keys.
__global__ __launch_bounds__(256) void block_keys_kernel(Rows k, const int* __restrict__ k_len, bf16_t* __restrict__ keys, int Lk, int Hkv,
                                                         int D, int nblk, int vt) {
  __shared__ double part[256][8];
  const int j = blockIdx.x, b = blockIdx.z, tid = threadIdx.x;
  const int vl = tid & (vt - 1), phase = tid / vt, phases = 256 / vt;
  const int f = (blockIdx.y * vt + vl) * 8;
  const bool live = f < Hkv * D;
  const int h = live ? f / D : 0, d = live ? f - h * D : 0;
  const int n = min(valid_keys(k_len, b, Lk) - j * BLK, BLK);
  double s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (live) {
    const bf16_t* p = k.p + b * k.sb + (long)j * BLK * k.sl + h * k.sh + d;
#pragma unroll 4
    for (int t = phase; t < n; t += phases) {
      const bf16x8_t x = *(const bf16x8_t*)(p + t * k.sl);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] += (double)(float)x[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) part[tid][e] = s[e];
  __syncthreads();
  if (phase == 0 && live) {
    bf16x8_t y;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      double t = part[vl][e];
      for (int w = 1; w < phases; ++w) t += part[w * vt + vl][e];
      y[e] = (bf16_t)(float)(n > 0 ? t / n : 0.0);
    }
    *(bf16x8_t*)(keys + (((long)b * Hkv + h) * nblk + j) * D + d) = y;
  }
}

// ---------------------------------------------------------------------------------------------------------------
// The `top` blocks of a query, one wave a query: scores in 64 bits, lane by lane, once for every block taken (the best
// one behind the last taken in the order "higher score, then lower block"), so any number of blocks works.
template <int D>
__global__ __launch_bounds__(256) void block_select_kernel(Rows q, const bf16_t* __restrict__ keys, const int* __restrict__ k_len,
                                                           int* __restrict__ blocks, int Lq, int Lk, int Hq, int G, int top, int nblk,
                                                           long rows) {
  const int lane = threadIdx.x & 63;
  const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int i = row % Lq, h = (row / Lq) % Hq, b = row / ((long)Lq * Hq);
  const int have = (valid_keys(k_len, b, Lk) + BLK - 1) / BLK;
  const bf16_t* qp = q.p + b * q.sb + i * q.sl + h * q.sh;
  const bf16_t* kp = keys + ((long)b * (Hq / G) + h / G) * nblk * (long)D;
  double last = INFINITY;
  int last_j = -1;
  int mine = 0x7fffffff;           // lane t: the t-th block taken
  for (int t = 0; t < top && t < have; ++t) {
    double best = -INFINITY;
    int best_j = 0x7fffffff;
    for (int j = lane; j < have; j += 64) {
      double s = 0;
      for (int d = 0; d < D; d += 8) {
        const bf16x8_t x = *(const bf16x8_t*)(qp + d), y = *(const bf16x8_t*)(kp + (long)j * D + d);
#pragma unroll
        for (int e = 0; e < 8; ++e) s += (double)(float)x[e] * (double)(float)y[e];
      }
      if (s != s) s = -INFINITY;
      const bool open = s < last || (s == last && j > last_j);
      if (open && (best_j == 0x7fffffff || s > best)) { best = s; best_j = j; }   // j ascends: ties keep the lower
    }
    for (int o = 32; o > 0; o >>= 1) {
      const double s = __shfl_xor(best, o, 64);
      const int j = __shfl_xor(best_j, o, 64);
      if (j != 0x7fffffff && (best_j == 0x7fffffff || s > best || (s == best && j < best_j))) { best = s; best_j = j; }
    }
    last = best;
    last_j = best_j;
    if (lane == t) mine = best_j;
  }
  int rank = 0;   // ascending order of the blocks taken
  for (int t = 0; t < top; ++t) {
    const int other = __shfl(mine, t, 64);
    rank += other < mine || (other == mine && t < lane);
  }
  if (lane < top) blocks[row * top + rank] = mine == 0x7fffffff ? -1 : mine;
}

// ---------------------------------------------------------------------------------------------------------------
// Which rows chose a block, as bits: mask[b][hkv][group of 64 rows][block]. A set, whatever the order of the list and
// however often it names a block; numbers outside 0 .. nblk-1 name none.
constexpr int MASK_CHUNK = 2048;
__global__ __launch_bounds__(256) void block_mask_kernel(const int* __restrict__ blocks, unsigned long long* __restrict__ mask, int Lq,
                                                         int Hq, int G, int top, int nblk, int ngroups) {
  __shared__ unsigned long long word[MASK_CHUNK];
  const int rg = blockIdx.x, bh = blockIdx.y, tid = threadIdx.x;
  const int Hkv = Hq / G, b = bh / Hkv, hk = bh - b * Hkv;
  const long rows = (long)Lq * G;
  for (int j0 = 0; j0 < nblk; j0 += MASK_CHUNK) {
    const int n = min(MASK_CHUNK, nblk - j0);
    for (int j = tid; j < n; j += 256) word[j] = 0;
    __syncthreads();
    for (int e = tid; e < 64 * top; e += 256) {
      const int rr = e / top, t = e - rr * top;
      const long r = (long)rg * 64 + rr;
      if (r >= rows) break;
      const long i = r / G;
      const int h = hk * G + (int)(r - i * G);
      const int j = blocks[(((long)b * Hq + h) * Lq + i) * top + t];
      if (j >= j0 && j < j0 + n) atomicOr(&word[j - j0], 1ull << rr);
    }
    __syncthreads();
    for (int j = tid; j < n; j += 256) mask[((long)bh * ngroups + rg) * nblk + j0 + j] = word[j];
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------------------------
// One query a workgroup: its blocks are dealt to the waves, whose partial results are joined through LDS. A block's keys
// and values are read as whole rows, D/8 lanes a row with 16 bytes each; the lanes that hold a key's features also hold
// the same features of its value, so a weight never moves between lanes. (The form for few queries.)
template <int D, int NW>
__global__ __launch_bounds__(NW * 64) void attend_row_kernel(Args a) {
  constexpr int LPR = D / 8, KPI = 64 / LPR, NI = BLK / KPI;
  __shared__ float so[NW][D];
  __shared__ float sm[NW], sl[NW];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long row = blockIdx.x;
  const int i = row % a.Lq, h = (row / a.Lq) % a.Hq, b = row / ((long)a.Lq * a.Hq), hk = h / a.G;
  const int n = valid_keys(a.k_len, b, a.Lk);
  const int c = (lane % LPR) * 8, key = lane / LPR;
  float q[8];
  dm_unpack8(*(const bf16x8_t*)(a.q.p + b * a.q.sb + i * a.q.sl + h * a.q.sh + c), q);
  const bf16_t* kp = a.k.p + b * a.k.sb + hk * a.k.sh + c;
  const bf16_t* vp = a.v.p + b * a.v.sb + hk * a.v.sh + c;
  const int listed = lane < a.top ? a.blocks[row * a.top + lane] : -1;
  const float sc = a.scale * LOG2E;
  float m = -INFINITY, l = 0.f, o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  for (int t = wave; t < a.top; t += NW) {
    const int j = __builtin_amdgcn_readlane(listed, t);
    if (j < 0 || j >= a.nblk) continue;
    if (__ballot(listed == j) & ((1ull << t) - 1)) continue;   // named before
    const int n0 = n - j * BLK;
    if (n0 <= 0) continue;
    const bf16x8_t none = {};
    bf16x8_t kk[NI], vv[NI];
#pragma unroll
    for (int u = 0; u < NI; ++u) {
      const long pos = (long)j * BLK + u * KPI + key;
      kk[u] = u * KPI + key < n0 ? *(const bf16x8_t*)(kp + pos * a.k.sl) : none;
      vv[u] = u * KPI + key < n0 ? *(const bf16x8_t*)(vp + pos * a.v.sl) : none;
    }
    float s[NI], mx = m;
#pragma unroll
    for (int u = 0; u < NI; ++u) {
      float x[8], d = 0.f;
      dm_unpack8(kk[u], x);
#pragma unroll
      for (int e = 0; e < 8; ++e) d += q[e] * x[e];
      d = group_sum<LPR>(d) * sc;
      s[u] = u * KPI + key < n0 ? d : -INFINITY;
      mx = fmaxf(mx, s[u]);
    }
    mx = across_max<LPR>(mx);
    const float base = mx == -INFINITY ? 0.f : mx, alpha = __builtin_amdgcn_exp2f(m - base);
    m = mx;
    l *= alpha;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] *= alpha;
#pragma unroll
    for (int u = 0; u < NI; ++u) {
      const float p = __builtin_amdgcn_exp2f(s[u] - base);
      float x[8];
      dm_unpack8(vv[u], x);
      l += p;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] += p * x[e];
    }
  }
  l = across_sum<LPR>(l);
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = across_sum<LPR>(o[e]);
  if (lane < LPR) {
#pragma unroll
    for (int e = 0; e < 8; ++e) so[wave][c + e] = o[e];
  }
  if (lane == 0) { sm[wave] = m; sl[wave] = l; }
  __syncthreads();
  if (threadIdx.x < D) {
    float mx = -INFINITY, lt = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) mx = fmaxf(mx, sm[w]);
    const float base = mx == -INFINITY ? 0.f : mx;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = __builtin_amdgcn_exp2f(sm[w] - base);
      lt += sl[w] * f;
      x += so[w][threadIdx.x] * f;
    }
    const long at = (((long)b * a.Lq + i) * a.Hq + h) * D + threadIdx.x;
    const float y = lt == 0.f ? 0.f : x / lt;
    const bf16_t hi = (bf16_t)y;
    a.out[at] = hi;
    if (a.out_lo) a.out_lo[at] = (bf16_t)(y - (float)hi);
    if (threadIdx.x == 0 && a.lse) a.lse[row] = lt == 0.f ? -INFINITY : mx * LN2 + logf(lt);
  }
}

// dq of one query a wave, and delta for the kernel behind
template <int D>
__global__ __launch_bounds__(256) void dq_row_kernel(Args a, long rows) {
  constexpr int LPR = D / 8, KPI = 64 / LPR, NI = BLK / KPI;
  const int lane = threadIdx.x & 63;
  const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int i = row % a.Lq, h = (row / a.Lq) % a.Hq, b = row / ((long)a.Lq * a.Hq), hk = h / a.G;
  const int n = valid_keys(a.k_len, b, a.Lk);
  const int c = (lane % LPR) * 8, key = lane / LPR;
  const long orow = (((long)b * a.Lq + i) * a.Hq + h) * D + c;
  float q[8], go[8], oo[8], lo[8], delta = 0.f, dq[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  dm_unpack8(*(const bf16x8_t*)(a.q.p + b * a.q.sb + i * a.q.sl + h * a.q.sh + c), q);
  dm_unpack8(*(const bf16x8_t*)(a.go + orow), go);
  dm_unpack8(*(const bf16x8_t*)(a.o + orow), oo);
  dm_unpack8(*(const bf16x8_t*)(a.o_lo + orow), lo);
#pragma unroll
  for (int e = 0; e < 8; ++e) delta += go[e] * (oo[e] + lo[e]);
  delta = group_sum<LPR>(delta);
  const float lse = a.lse[row], sc = a.scale * LOG2E, ls = lse * LOG2E;
  if (lane == 0) a.delta[row] = delta;
  const int listed = lane < a.top ? a.blocks[row * a.top + lane] : -1;
  if (lse != -INFINITY) {
    for (int t = 0; t < a.top; ++t) {
      const int j = __builtin_amdgcn_readlane(listed, t);
      if (j < 0 || j >= a.nblk) continue;
      if (__ballot(listed == j) & ((1ull << t) - 1)) continue;
      const int n0 = n - j * BLK;
      if (n0 <= 0) continue;
      const bf16_t* kp = a.k.p + b * a.k.sb + hk * a.k.sh + (long)j * BLK * a.k.sl + c;
      const bf16_t* vp = a.v.p + b * a.v.sb + hk * a.v.sh + (long)j * BLK * a.v.sl + c;
#pragma unroll
      for (int u = 0; u < NI; ++u) {
        const int pos = u * KPI + key;
        if (pos < n0) {
          float x[8], y[8], s = 0.f, dp = 0.f;
          dm_unpack8(*(const bf16x8_t*)(kp + pos * a.k.sl), x);
          dm_unpack8(*(const bf16x8_t*)(vp + pos * a.v.sl), y);
#pragma unroll
          for (int e = 0; e < 8; ++e) { s += q[e] * x[e]; dp += go[e] * y[e]; }
          s = group_sum<LPR>(s) * sc;
          dp = group_sum<LPR>(dp);
          const float ds = __builtin_amdgcn_exp2f(s - ls) * (dp - delta) * a.scale;
#pragma unroll
          for (int e = 0; e < 8; ++e) dq[e] += ds * x[e];
        }
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) dq[e] = across_sum<LPR>(dq[e]);
  if (lane < LPR) *(bf16x8_t*)(a.dq + b * a.dqb + i * a.dql + h * a.dqh + c) = dm_pack8(dq);
}

// dk and dv of one block a workgroup: its keys and values stay in registers, the rows that chose it are dealt to the
// waves, whose sums are added in wave order
template <int D>
__global__ __launch_bounds__(256) void dkv_row_kernel(Args a, int ngroups) {
  constexpr int LPR = D / 8, KPI = 64 / LPR, NI = BLK / KPI;
  __shared__ float acc[2][BLK][D];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int j = blockIdx.x, bh = blockIdx.y, b = bh / a.Hkv, hk = bh - b * a.Hkv;
  const int n0 = valid_keys(a.k_len, b, a.Lk) - j * BLK;
  const int c = (lane % LPR) * 8, key = lane / LPR;
  const float sc = a.scale * LOG2E;
  const bf16_t* kp = a.k.p + b * a.k.sb + hk * a.k.sh + (long)j * BLK * a.k.sl + c;
  const bf16_t* vp = a.v.p + b * a.v.sb + hk * a.v.sh + (long)j * BLK * a.v.sl + c;
  const bf16x8_t none = {};
  bf16x8_t kk[NI], vv[NI];
  float dk[NI][8], dv[NI][8];
#pragma unroll
  for (int u = 0; u < NI; ++u) {
    const int pos = u * KPI + key;
    kk[u] = pos < n0 ? *(const bf16x8_t*)(kp + pos * a.k.sl) : none;
    vv[u] = pos < n0 ? *(const bf16x8_t*)(vp + pos * a.v.sl) : none;
#pragma unroll
    for (int e = 0; e < 8; ++e) dk[u][e] = dv[u][e] = 0.f;
  }
  for (int rg = wave; rg < ngroups; rg += 4) {
    const unsigned long long w = a.mask[((long)bh * ngroups + rg) * a.nblk + j];
    unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)w), hi = __builtin_amdgcn_readfirstlane((unsigned)(w >> 32));
    unsigned long long bits = ((unsigned long long)hi << 32) | lo;
    if (n0 <= 0) bits = 0;
    while (bits) {
      const long r = (long)rg * 64 + __builtin_ctzll(bits);
      bits &= bits - 1;
      const long i = r / a.G;
      const int h = hk * a.G + (int)(r - i * a.G);
      const long row = ((long)b * a.Hq + h) * a.Lq + i;
      const float lse = a.lse[row], ls = lse * LOG2E, delta = a.delta[row];
      if (lse == -INFINITY) continue;
      float q[8], go[8];
      dm_unpack8(*(const bf16x8_t*)(a.q.p + b * a.q.sb + i * a.q.sl + h * a.q.sh + c), q);
      dm_unpack8(*(const bf16x8_t*)(a.go + (((long)b * a.Lq + i) * a.Hq + h) * D + c), go);
#pragma unroll
      for (int u = 0; u < NI; ++u) {
        float x[8], y[8], s = 0.f, dp = 0.f;
        dm_unpack8(kk[u], x);
        dm_unpack8(vv[u], y);
#pragma unroll
        for (int e = 0; e < 8; ++e) { s += q[e] * x[e]; dp += go[e] * y[e]; }
        s = group_sum<LPR>(s) * sc;
        dp = group_sum<LPR>(dp);
        const float p = __builtin_amdgcn_exp2f(s - ls), ds = p * (dp - delta) * a.scale;
#pragma unroll
        for (int e = 0; e < 8; ++e) { dk[u][e] += ds * q[e]; dv[u][e] += p * go[e]; }
      }
    }
  }
  for (int w = 0; w < 4; ++w) {
    if (wave == w) {
#pragma unroll
      for (int u = 0; u < NI; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float* pk = &acc[0][u * KPI + key][c + e];
          float* pv = &acc[1][u * KPI + key][c + e];
          *pk = (w ? *pk : 0.f) + dk[u][e];
          *pv = (w ? *pv : 0.f) + dv[u][e];
        }
    }
    __syncthreads();
  }
  const int in = min(BLK, a.Lk - j * BLK);
  for (int e = threadIdx.x; e < BLK * D / 8; e += 256) {
    const int t = e / LPR, d = (e % LPR) * 8;
    if (t >= in) break;
    const long pos = (long)j * BLK + t;
    const bool live = t < n0;   // positions behind the last valid key: zero
    float f[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) f[x] = live ? acc[0][t][d + x] : 0.f;
    *(bf16x8_t*)(a.dk + b * a.dkb + pos * a.dkl + hk * a.dkh + d) = dm_pack8(f);
#pragma unroll
    for (int x = 0; x < 8; ++x) f[x] = live ? acc[1][t][d + x] : 0.f;
    *(bf16x8_t*)(a.dv + b * a.dvb + pos * a.dvl + hk * a.dvh + d) = dm_pack8(f);
  }
}

bool aligned(const void* p) { return p && ((uintptr_t)p & 15) == 0; }

int check_desc(const char* who, const dm_block_desc* d) {
  DM_REQUIRE(d, DM_ERR_ARG, "%s: null descriptor", who);
  DM_REQUIRE(d->B > 0 && d->Lq > 0 && d->Lk > 0 && d->Hq > 0 && d->Hkv > 0, DM_ERR_SHAPE, "%s: B, Lq, Lk, Hq and Hkv must be positive", who);
  DM_REQUIRE(d->Hq % d->Hkv == 0, DM_ERR_SHAPE, "%s: %d query heads do not share %d key heads evenly", who, d->Hq, d->Hkv);
  DM_REQUIRE(d->D == 8 || d->D == 16 || d->D == 32 || d->D == 64, DM_ERR_SHAPE, "%s: head dim %d (8, 16, 32 and 64 are covered)", who, d->D);
  DM_REQUIRE(d->top > 0 && d->top <= 64, DM_ERR_SHAPE, "%s: top %d (1 to 64 blocks a query)", who, d->top);
  DM_REQUIRE((long)d->B * d->Hq * d->Lq <= 0x7fffffffL && (long)d->B * d->Hkv <= 65535 && (long)d->Lq * (d->Hq / d->Hkv) <= 0x7fffffffL,
             DM_ERR_SHAPE, "%s: more than 2^31-1 queries or 65535 (sample, key head) pairs", who);
  return DM_OK;
}
int check_strides(const char* who, const char* name, const long* s) {
  for (int i = 0; i < 3; ++i)
    DM_REQUIRE(s[i] % 8 == 0, DM_ERR_ARG, "%s: strides of %s must be multiples of 8 elements (rows are read 16 bytes at a time)", who, name);
  return DM_OK;
}
int blocks_of(const dm_block_desc* d) { return (d->Lk + BLK - 1) / BLK; }
int groups_of(const dm_block_desc* d) { return dm_cdiv((long)d->Lq * (d->Hq / d->Hkv), 64); }

Rows rows_of(const void* p, const long* s) { return Rows{(const bf16_t*)p, s[0], s[1], s[2]}; }

Args args_of(const dm_block_desc* d) {
  Args a = {};
  a.B = d->B; a.Lq = d->Lq; a.Lk = d->Lk; a.Hq = d->Hq; a.Hkv = d->Hkv; a.G = d->Hq / d->Hkv; a.top = d->top;
  a.nblk = blocks_of(d);
  a.scale = d->scale;
  return a;
}

#define BY_HEAD_DIM(D_, CALL)                      \
  switch (D_) {                                    \
    case 8: { constexpr int HD = 8; CALL; } break;   \
    case 16: { constexpr int HD = 16; CALL; } break; \
    case 32: { constexpr int HD = 32; CALL; } break; \
    default: { constexpr int HD = 64; CALL; } break; \
  }

}  // namespace

extern "C" int dm_block_keys(const dm_block_desc* d, const void* k, const int* k_len, void* keys, void* stream) {
  const char* who = "dm_block_keys";
  int rc = check_desc(who, d);
  if (rc) return rc;
  DM_REQUIRE(aligned(k) && aligned(keys), DM_ERR_ARG, "%s: null or misaligned pointer", who);
  if ((rc = check_strides(who, "k", d->k_stride))) return rc;
  const int vecs = d->Hkv * d->D / 8;
  DM_REQUIRE(d->B <= 65535 && dm_cdiv(vecs, 64) <= 65535, DM_ERR_SHAPE, "%s: batch or heads too large", who);
  int vt = 1;
  while (vt < 64 && vt < vecs) vt <<= 1;
  hipLaunchKernelGGL(block_keys_kernel, dim3(blocks_of(d), dm_cdiv(vecs, vt), d->B), dim3(256), 0, (hipStream_t)stream,
                     rows_of(k, d->k_stride), k_len, (bf16_t*)keys, d->Lk, d->Hkv, d->D, blocks_of(d), vt);
  DM_CHECK_LAUNCH();
  return DM_OK;
}

extern "C" int dm_block_select(const dm_block_desc* d, const void* q, const void* keys, const int* k_len, int* blocks, void* stream) {
  const char* who = "dm_block_select";
  int rc = check_desc(who, d);
  if (rc) return rc;
  DM_REQUIRE(aligned(q) && aligned(keys) && blocks, DM_ERR_ARG, "%s: null or misaligned pointer", who);
  if ((rc = check_strides(who, "q", d->q_stride))) return rc;
  const long rows = (long)d->B * d->Hq * d->Lq;
  BY_HEAD_DIM(d->D, hipLaunchKernelGGL((block_select_kernel<HD>), dim3(dm_cdiv(rows, 4)), dim3(256), 0, (hipStream_t)stream,
                                       rows_of(q, d->q_stride), (const bf16_t*)keys, k_len, blocks, d->Lq, d->Lk, d->Hq,
                                       d->Hq / d->Hkv, d->top, blocks_of(d), rows));
  DM_CHECK_LAUNCH();
  return DM_OK;
}

extern "C" size_t dm_block_attention_mask_bytes(const dm_block_desc* d, int for_backward) {
  if (check_desc("dm_block_attention_mask_bytes", d) || !for_backward) return 0;
  return (size_t)d->B * d->Hkv * groups_of(d) * blocks_of(d) * 8;
}

extern "C" int dm_block_attention_fwd(const dm_block_desc* d, const void* q, const void* k, const void* v, const int* blocks,
                                      const int* k_len, void* out, void* out_lo, float* lse, void* mask, void* stream) {
  const char* who = "dm_block_attention_fwd";
  int rc = check_desc(who, d);
  if (rc) return rc;
  DM_REQUIRE(aligned(q) && aligned(k) && aligned(v) && aligned(out) && blocks, DM_ERR_ARG, "%s: null or misaligned pointer", who);
  if ((rc = check_strides(who, "q", d->q_stride)) || (rc = check_strides(who, "k", d->k_stride)) ||
      (rc = check_strides(who, "v", d->v_stride)))
    return rc;
  Args a = args_of(d);
  a.q = rows_of(q, d->q_stride); a.k = rows_of(k, d->k_stride); a.v = rows_of(v, d->v_stride);
  a.blocks = blocks; a.k_len = k_len; a.out = (bf16_t*)out; a.out_lo = (bf16_t*)out_lo; a.lse = lse;
  hipStream_t st = (hipStream_t)stream;
  if (mask) {
    hipLaunchKernelGGL(block_mask_kernel, dim3(groups_of(d), d->B * d->Hkv), dim3(256), 0, st, blocks, (unsigned long long*)mask, d->Lq,
                       d->Hq, a.G, d->top, a.nblk, groups_of(d));
    DM_CHECK_LAUNCH();
  }
  const long rows = (long)d->B * d->Hq * d->Lq;
  BY_HEAD_DIM(d->D, hipLaunchKernelGGL((attend_row_kernel<HD, 4>), dim3((unsigned)rows), dim3(256), 0, st, a));
  DM_CHECK_LAUNCH();
  return DM_OK;
}

extern "C" size_t dm_block_attention_bwd_ws_bytes(const dm_block_desc* d) {
  if (check_desc("dm_block_attention_bwd_ws_bytes", d)) return 0;
  return (size_t)d->B * d->Hq * d->Lq * 4;
}

extern "C" int dm_block_attention_bwd(const dm_block_desc* d, const void* q, const void* k, const void* v, const int* blocks,
                                      const int* k_len, const void* mask, const void* out, const void* out_lo, const float* lse, const void* dout,
                                      void* dq, void* dk, void* dv, void* ws, size_t ws_bytes, void* stream) {
  const char* who = "dm_block_attention_bwd";
  int rc = check_desc(who, d);
  if (rc) return rc;
  DM_REQUIRE(aligned(q) && aligned(k) && aligned(v) && aligned(out) && aligned(out_lo) && aligned(dout) && aligned(dq) && aligned(dk) && aligned(dv) &&
                 aligned(mask) && blocks && lse, DM_ERR_ARG, "%s: null or misaligned pointer", who);
  DM_REQUIRE(aligned(ws) && ws_bytes >= dm_block_attention_bwd_ws_bytes(d), DM_ERR_ARG, "%s: workspace of %zu bytes is too small or misaligned", who, ws_bytes);
  const struct { const char* n; const long* s; } all[] = {{"q", d->q_stride}, {"k", d->k_stride}, {"v", d->v_stride},
                                                          {"dq", d->dq_stride}, {"dk", d->dk_stride}, {"dv", d->dv_stride}};
  for (const auto& x : all)
    if ((rc = check_strides(who, x.n, x.s))) return rc;
  Args a = args_of(d);
  a.q = rows_of(q, d->q_stride); a.k = rows_of(k, d->k_stride); a.v = rows_of(v, d->v_stride);
  a.o = (const bf16_t*)out; a.o_lo = (const bf16_t*)out_lo; a.go = (const bf16_t*)dout;
  a.blocks = blocks; a.k_len = k_len; a.mask = (unsigned long long*)mask;
  a.lse = const_cast<float*>(lse); a.delta = (float*)ws;
  a.dq = (bf16_t*)dq; a.dk = (bf16_t*)dk; a.dv = (bf16_t*)dv;
  a.dqb = d->dq_stride[0]; a.dql = d->dq_stride[1]; a.dqh = d->dq_stride[2];
  a.dkb = d->dk_stride[0]; a.dkl = d->dk_stride[1]; a.dkh = d->dk_stride[2];
  a.dvb = d->dv_stride[0]; a.dvl = d->dv_stride[1]; a.dvh = d->dv_stride[2];
  hipStream_t st = (hipStream_t)stream;
  const long rows = (long)d->B * d->Hq * d->Lq;
  BY_HEAD_DIM(d->D, hipLaunchKernelGGL((dq_row_kernel<HD>), dim3(dm_cdiv(rows, 4)), dim3(256), 0, st, a, rows));
  DM_CHECK_LAUNCH();
  BY_HEAD_DIM(d->D, hipLaunchKernelGGL((dkv_row_kernel<HD>), dim3(a.nblk, d->B * d->Hkv), dim3(256), 0, st, a, groups_of(d)));
  DM_CHECK_LAUNCH();
  return DM_OK;
}
