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

extern int g_dm_block_pool;

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

// ---------------------------------------------------------------------------------------------------------------
// The matrix-core form. A workgroup owns a POOL of P rows of one (sample, key head) and walks the blocks that any of
// them chose, in order. A block's keys and values are staged in LDS once for the pool; the pool's rows that chose it
// are packed into tiles of 16, so that a matrix instruction works on 16 rows that all want the block however the choices are
// scattered (16 neighbouring rows would share few blocks: with 8 of 64 chosen at random a tile of neighbours has to
// visit 56). A tile is dealt to a wave; what a row accumulates (its output, maximum and sum, or its dq) lives in LDS in fp32, because
// the next block packs it into another tile. Rows of one block are disjoint and blocks are separated by barriers, so
// a row's sums run in block order: the same bits every time.
//
// Products are formed transposed, S^T = K Q^T: a lane then holds 4 keys x 4 tiles of ONE row (lane & 15), the row's
// maximum and sum are two lane swaps away, and exp(S^T) is in the register layout that the second product takes as its
// right operand (its left operand, V^T or K^T, is read by transposing LDS reads in the same order of keys).
template <int D>
struct Geo {
  static constexpr int DV = D < 16 ? 16 : D;           // features of a row in LDS, zeros behind D
  static constexpr int ROWB = DV * 2, KV_BYTES = BLK * ROWB;
  static constexpr int KS = D <= 16 ? 1 : D / 32;      // matrix instructions (of 16 or 32 features) to a score
  static constexpr int DT = DV / 16;                   // 16-feature tiles of a row
  static constexpr int OC = DV / 4;                    // 16-byte pieces of an fp32 row
};
// Byte offset of 16-byte piece c of bf16 row r: 32-byte units are exchanged by row such that both the 16-byte reads (16
// rows, one piece) and the transposing reads (4 groups of 4 rows, one unit) meet every bank equally often.
template <int D>
__device__ __forceinline__ int lds_at(int r, int c) {
  if constexpr (D == 64) return r * 128 + (((((c >> 1) ^ (r & 3)) << 1) | (c & 1)) << 4);
  else if constexpr (D == 32) return r * 64 + (((((c >> 1) ^ ((r >> 1) & 1)) << 1) | (c & 1)) << 4);
  else return r * 32 + (c << 4);
}
// float offset of 4-feature piece c of fp32 row r
template <int D>
__device__ __forceinline__ int acc_at(int r, int c) {
  if constexpr (D == 64) return r * 64 + ((c ^ (r & 15)) << 2);
  else if constexpr (D == 32) return r * 32 + ((c ^ (r & 7)) << 2);
  else return r * 16 + (c << 2);
}

// 4 consecutive rows (row0 + 4 (lane >> 4) ...) of one feature (16 dt + (lane & 15)) for every lane
template <int D>
__device__ __forceinline__ bf16x4_t read_tr(const char* base, int row0, int dt, int lane) {
  typedef __attribute__((address_space(3))) bf16x4_t* lds_ptr;
  const int i = lane & 15, row = row0 + 4 * (lane >> 4) + (i >> 2);
  return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_ptr)(base + lds_at<D>(row, dt * 2 + ((i >> 1) & 1)) + (i & 1) * 8));
}
__device__ __forceinline__ bf16x8_t join4(bf16x4_t a, bf16x4_t b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

// operand of a product over features: the row's KS pieces of 8 (or, up to 16 features, its piece of 4)
template <int D>
struct Frag {
  bf16x8_t x[Geo<D>::KS];
  // p: the row, g = lane >> 4
  __device__ __forceinline__ void load(const bf16_t* p, int g) {
    if constexpr (D <= 16) {
      const bf16x4_t z = {}, v = D == 16 || g < 2 ? *(const bf16x4_t*)(p + g * 4) : z;
      x[0] = join4(v, z);
    } else {
#pragma unroll
      for (int s = 0; s < Geo<D>::KS; ++s) x[s] = *(const bf16x8_t*)(p + s * 32 + g * 8);
    }
  }
  // waits for the operand here and not behind younger loads (the compiler counts loads in order, and across branches all of them)
  __device__ __forceinline__ void arrived() {
#pragma unroll
    for (int s = 0; s < Geo<D>::KS; ++s) asm volatile("" : "+v"(x[s]));
  }
  __device__ __forceinline__ void negate() {
    typedef __attribute__((ext_vector_type(4))) unsigned bits_t;
#pragma unroll
    for (int s = 0; s < Geo<D>::KS; ++s) x[s] = __builtin_bit_cast(bf16x8_t, __builtin_bit_cast(bits_t, x[s]) ^ 0x80008000u);
  }
  __device__ __forceinline__ void zero() {
    const bf16x8_t z = {};
#pragma unroll
    for (int s = 0; s < Geo<D>::KS; ++s) x[s] = z;
  }
  __device__ __forceinline__ void from_lds(const char* base, int row, int g) {
    if constexpr (D <= 16) {
      const bf16x4_t z = {};
      x[0] = join4(*(const bf16x4_t*)(base + lds_at<D>(row, g >> 1) + (g & 1) * 8), z);
    } else {
#pragma unroll
      for (int s = 0; s < Geo<D>::KS; ++s) x[s] = *(const bf16x8_t*)(base + lds_at<D>(row, s * 4 + g));
    }
  }
};
template <int D>
__device__ __forceinline__ f32x4_t dot_frag(const Frag<D>& a, const Frag<D>& b) {
  f32x4_t c = {0.f, 0.f, 0.f, 0.f};
  if constexpr (D <= 16) {
    typedef __attribute__((ext_vector_type(4))) short half_t;
    const bf16x4_t a4 = __builtin_shufflevector(a.x[0], a.x[0], 0, 1, 2, 3), b4 = __builtin_shufflevector(b.x[0], b.x[0], 0, 1, 2, 3);
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(half_t, a4), __builtin_bit_cast(half_t, b4), c, 0, 0, 0);
  } else {
#pragma unroll
    for (int s = 0; s < Geo<D>::KS; ++s) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.x[s], b.x[s], c, 0, 0, 0);
    return c;
  }
}
// over the lanes l, l ^ 16, l ^ 32, l ^ 48 (the lanes that hold one row)
__device__ __forceinline__ float row_max(float x) {
  unsigned u = __builtin_bit_cast(unsigned, x);
  auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  x = fmaxf(__builtin_bit_cast(float, (unsigned)a[0]), __builtin_bit_cast(float, (unsigned)a[1]));
  u = __builtin_bit_cast(unsigned, x);
  a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__builtin_bit_cast(float, (unsigned)a[0]), __builtin_bit_cast(float, (unsigned)a[1]));
}
__device__ __forceinline__ float row_sum(float x) {
  unsigned u = __builtin_bit_cast(unsigned, x);
  auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  x = __builtin_bit_cast(float, (unsigned)a[0]) + __builtin_bit_cast(float, (unsigned)a[1]);
  u = __builtin_bit_cast(unsigned, x);
  a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __builtin_bit_cast(float, (unsigned)a[0]) + __builtin_bit_cast(float, (unsigned)a[1]);
}

// ---------------------------------------------------------------------------------------------------------------
// The choice of blocks. Scores are compared as 64-bit sums; two ways to get there:
//
// exact_top: one query a wave, all scores in 64 bits, EXACT_CHUNK blocks at a time beside the best of the earlier ones. A
// score becomes an unsigned number of the same order (NaN: that of -infinity), 0 stands for a block already taken.
constexpr int EXACT_CHUNK = 512;
template <int O>
__device__ __forceinline__ unsigned lane_xor_u(unsigned x) {   // as lane_xor, and O = 16, 32 (whole-wave reductions)
  if constexpr (O == 16) { auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false); return (threadIdx.x & 16) ? r[0] : r[1]; }
  else if constexpr (O == 32) { auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false); return (threadIdx.x & 32) ? r[0] : r[1]; }
  else return __builtin_bit_cast(unsigned, lane_xor<O>(__builtin_bit_cast(float, x)));
}
template <int O>
__device__ __forceinline__ void take_best(unsigned long long& key, int& j) {
  const unsigned long long k = (unsigned long long)lane_xor_u<O>((unsigned)(key >> 32)) << 32 | lane_xor_u<O>((unsigned)key);
  const int i = (int)lane_xor_u<O>((unsigned)j);
  if (k > key || (k == key && i < j)) { key = k; j = i; }
}
constexpr int NO_BLOCK = 0x7fffffff;

// lane t's return value: the t-th block taken, or NO_BLOCK
template <int D>
__device__ int exact_top(const bf16_t* qp, const bf16_t* kp, int have, int top, unsigned long long* buf, int lane) {
  unsigned long long won = 0;    // lane t: the t-th best of the chunks so far
  int won_j = NO_BLOCK;
  for (int c0 = 0; c0 < have; c0 += EXACT_CHUNK) {
    const int n = min(EXACT_CHUNK, have - c0);
    for (int x = lane; x < n; x += 64) {
      double s = 0;
#pragma unroll 2
      for (int d = 0; d < D; d += 8) {
        const bf16x8_t a = *(const bf16x8_t*)(qp + d), b = *(const bf16x8_t*)(kp + (long)(c0 + x) * D + d);
#pragma unroll
        for (int e = 0; e < 8; ++e) s += (double)(float)a[e] * (double)(float)b[e];
      }
      s = s == s ? s + 0.0 : -INFINITY;   // (-0 and 0 are equal)
      const unsigned long long u = __builtin_bit_cast(unsigned long long, s);
      buf[x] = (u >> 63) ? ~u : u | 0x8000000000000000ull;
    }
    unsigned long long next = 0;
    int next_j = NO_BLOCK;
    for (int t = 0; t < top; ++t) {
      unsigned long long key = won;
      int j = won_j;
      for (int x = lane; x < n; x += 64)
        if (buf[x] > key) { key = buf[x]; j = c0 + x; }   // (earlier chunks have the lower numbers: ties stay with them)
      take_best<1>(key, j);
      take_best<2>(key, j);
      take_best<4>(key, j);
      take_best<8>(key, j);
      take_best<16>(key, j);
      take_best<32>(key, j);
      if (!key) break;
      if (lane == t) { next = key; next_j = j; }
      if (won_j == j) won = 0;
      if (j >= c0 && ((j - c0) & 63) == lane) buf[j - c0] = 0;   // (a lane reads only what it wrote)
    }
    won = next;
    won_j = next_j;
  }
  return won_j;
}
// the blocks taken, in ascending order, -1 behind
__device__ __forceinline__ void write_taken(int* to, int taken, int top, int lane) {
  int rank = 0;
  for (int t = 0; t < top; ++t) {
    const int other = __builtin_amdgcn_readlane(taken, t);
    rank += other < taken || (other == taken && t < lane);
  }
  if (lane < top) to[rank] = taken == NO_BLOCK ? -1 : taken;
}

template <int D>
__global__ __launch_bounds__(256) void block_select_row_kernel(Rows q, const bf16_t* __restrict__ keys, const int* __restrict__ k_len,
                                                               int* __restrict__ blocks, int Lq, int Lk, int Hq, int G, int top,
                                                               int nblk, long rows) {
  __shared__ unsigned long long buf[4][EXACT_CHUNK];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long row = (long)blockIdx.x * 4 + wave;
  if (row >= rows) return;
  const int i = row % Lq, h = (row / Lq) % Hq, b = row / ((long)Lq * Hq);
  const int have = (valid_keys(k_len, b, Lk) + BLK - 1) / BLK;
  const int taken = exact_top<D>(q.p + b * q.sb + i * q.sl + h * q.sh, keys + ((long)b * (Hq / G) + h / G) * nblk * (long)D, have, top, buf[wave], lane);
  write_taken(blocks + row * top, taken, top, lane);
}

// The screening kernel: 16 rows a wave. Scores come from the matrix cores in fp32, off by at most
//   eps = max(D, 16) 2^-23 |q| max |key| + 2^-118
// (exact products, at most that many additions each off by one unit of the sum of absolute terms, which |q| |key| bounds; 2^-118, here and under
// the roots, covers products too small for fp32; the factor 1.016 the roundings of the norms themselves). With T the (top)-th and U the (top + 1)-th best of them, T - U > 2 eps says that
// the fp32 scores order these two as 64-bit ones would, and the choice is the scores above U. Rows where that fails, and waves
// that meet an infinity or NaN, are decided by exact_top.
//   Every lane keeps the K best of the blocks it sees (a row's blocks are dealt to 4 lanes, neighbouring blocks to
// different ones), sorted, one v_med3 a place and score. K is about twice the fair share (top + 1) / 4: a lane that may have
// dropped one that counts sends its row to exact_top as well. A second pass over the same scores writes the choice in order.
template <int D, int K>
__global__ __launch_bounds__(256) void block_select_kernel(Rows q, const bf16_t* __restrict__ keys, const int* __restrict__ k_len,
                                                           int* __restrict__ blocks, int Lq, int Lk, int Hkv, int G, int top, int nblk) {
  constexpr int EXACT_FLOATS = EXACT_CHUNK * 2, LIST_FLOATS = 2 * K * 64;
  __shared__ __attribute__((aligned(16))) float scratch[4][EXACT_FLOATS > LIST_FLOATS ? EXACT_FLOATS : LIST_FLOATS];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, bh = blockIdx.y, b = bh / Hkv, hk = bh - b * Hkv;
  const long rows = (long)Lq * G, r0 = ((long)blockIdx.x * 4 + wave) * 16;
  if (r0 >= rows) return;   // (waves are independent: no barriers)
  const long r = min(r0 + (lane & 15), rows - 1);
  const bool in = r0 + (lane & 15) < rows;
  const unsigned i = G == 1 ? (unsigned)r : (unsigned)r / (unsigned)G;
  const int h = hk * G + (int)((unsigned)r - i * (unsigned)G), Hq = Hkv * G;
  int* to = blocks + (((long)b * Hq + h) * Lq + i) * top;
  const int have = (valid_keys(k_len, b, Lk) + BLK - 1) / BLK;
  if (have <= top) {   // every block
    if (in)
      for (int t = g; t < top; t += 4) to[t] = t < have ? t : -1;
    return;
  }
  const bf16_t* kp = keys + (long)bh * nblk * D;
  const bf16_t* qp = q.p + b * q.sb + (long)i * q.sl + h * q.sh;
  Frag<D> qf;
  qf.load(qp, g);
  float qq = 0.f;
#pragma unroll
  for (int s = 0; s < Geo<D>::KS; ++s)
#pragma unroll
    for (int e = 0; e < 8; ++e) qq += (float)qf.x[s][e] * (float)qf.x[s][e];
  qq = row_sum(qq);
  const int mine = 4 * (lane & 3) + ((lane & 15) >> 2);   // the block of a chunk of 16 that this lane fetches; it gets the scores of 4 e + g
  float best[K];
#pragma unroll
  for (int x = 0; x < K; ++x) best[x] = -INFINITY;
  unsigned kk = 0;   // the largest |key|^2, by its bits: a NaN is larger than any number
  for (int c = 0; c < have; c += 16) {
    Frag<D> kf;
    kf.load(kp + (long)min(c + mine, have - 1) * D, g);
    const f32x4_t s = dot_frag<D>(kf, qf), n = dot_frag<D>(kf, kf);
    const float d01 = (lane & 1) ? n[1] : n[0], d23 = (lane & 1) ? n[3] : n[2], d = (lane & 2) ? d23 : d01;
    if (g == ((lane & 15) >> 2)) kk = max(kk, __builtin_bit_cast(unsigned, d) & 0x7fffffffu);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = c + 4 * e + g < have ? s[e] : -INFINITY;
#pragma unroll
      for (int p = K - 1; p > 0; --p) best[p] = __builtin_amdgcn_fmed3f(best[p - 1], best[p], x);
      best[0] = fmaxf(best[0], x);
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) kk = max(kk, (unsigned)__shfl_xor((int)kk, o, 64));
  // two lanes' lists become one of 2 K (values of the other lane in order: the j-th takes place j or a later one)
  float two[2 * K];
#pragma unroll
  for (int x = 0; x < K; ++x) { two[x] = best[x]; two[K + x] = -INFINITY; }
#pragma unroll
  for (int x = 0; x < K; ++x) {
    const float y = __builtin_bit_cast(float, lane_xor_u<16>(__builtin_bit_cast(unsigned, best[x])));
#pragma unroll
    for (int p = K + x; p > x; --p) two[p] = __builtin_amdgcn_fmed3f(two[p - 1], two[p], y);
    two[x] = fmaxf(two[x], y);
  }
  // the m-th best of two sorted lists: max over i of min(a_i, b_(m - i)), counted from 1, a_0 = b_0 = infinity
  float* lists = scratch[wave];
#pragma unroll
  for (int x = 0; x < 2 * K; ++x) lists[x * 64 + lane] = two[x];
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  float T = -INFINITY, U = -INFINITY;
#pragma unroll
  for (int x = 0; x <= 2 * K; ++x) {
    const float a = x == 0 ? INFINITY : two[x == 0 ? 0 : x - 1];
    const int m = top - x;
    auto other = [&](int y) { return y == 0 ? INFINITY : y > 0 && y <= 2 * K ? lists[(y - 1) * 64 + (lane ^ 32)] : -INFINITY; };
    T = fmaxf(T, fminf(a, other(m)));
    U = fmaxf(U, fminf(a, other(m + 1)));
  }
  const float eps2 = 2.f * ((D < 16 ? 16 : D) * 0x1.04p-23f * __builtin_sqrtf(qq + 0x1p-118f) * __builtin_sqrtf(__builtin_bit_cast(float, kk) + 0x1p-118f) + 0x1p-118f);
  bool clear = T - U > eps2;                                            // (false if anything is NaN or infinite)
  if (K < top + 1) {
    const float last = best[K - 1], l16 = fmaxf(last, __builtin_bit_cast(float, lane_xor_u<16>(__builtin_bit_cast(unsigned, last))));
    const float l32 = fmaxf(l16, __builtin_bit_cast(float, lane_xor_u<32>(__builtin_bit_cast(unsigned, l16))));
    clear = clear && (l32 == -INFINITY || U > l32);                     // what a lane dropped is not above its last
  }
  clear = clear && kk < 0x7f800000u && qq < INFINITY;
  int count = 0;
  for (int c = 0; c < have; c += 16) {
    Frag<D> kf;
    kf.load(kp + (long)min(c + mine, have - 1) * D, g);
    const f32x4_t s = dot_frag<D>(kf, qf);
    unsigned bits = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + 4 * e + g < have && s[e] > U) bits |= 1u << (4 * e + g);
    unsigned all = bits | lane_xor_u<16>(bits);
    all |= lane_xor_u<32>(all);
    if (clear && in) {
      while (bits) {
        const int x = __builtin_ctz(bits);
        bits &= bits - 1;
        to[count + __builtin_popcount(all & ((1u << x) - 1))] = c + x;
      }
    }
    count += __builtin_popcount(all);
  }
  unsigned long long open = __ballot(!clear && in && g == 0);
  while (open) {   // rows that 32 bits cannot decide
    const int x = __builtin_ctzll(open);
    open &= open - 1;
    const unsigned ri = __builtin_amdgcn_readlane(i, x);
    const int rh = __builtin_amdgcn_readlane(h, x);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int taken = exact_top<D>(q.p + b * q.sb + (long)ri * q.sl + rh * q.sh, kp, have, top, (unsigned long long*)scratch[wave], lane);
    write_taken(blocks + (((long)b * Hq + rh) * Lq + ri) * top, taken, top, lane);
  }
}

// The walk over a pool's blocks: which come next, the rows that chose each (packed into `list`, one wave a group of 64
// rows), and the staging of keys and values.
template <int D, int P>
struct Walk {
  static constexpr int NG = P / 64;                 // groups of 64 rows = waves
  static constexpr int PIECES = 2 * BLK * D / 8;    // 16-byte pieces of a block's keys and values
  static constexpr int PER = (PIECES + P - 1) / P;
  const Args& a;
  const int bh, b, hk, rg0, ngroups, tid, lane, wave, n, nb;
  unsigned short (*list)[P];
  unsigned long long bits = 0, mine = 0;
  int base = 0, next0 = 0, pre = 0, tot = 0;
  bf16x8_t kv[PER];
  const bf16_t* src[PER];   // this thread's pieces of block 0, the distance of a block, their place in LDS
  long step[PER];
  int key[PER], to[PER];
  struct Hit { int j, n; };

  __device__ __forceinline__ Walk(const Args& a_, int bh_, int tile, int ngroups_, unsigned short (*l)[P])
      : a(a_), bh(bh_), b(bh_ / a_.Hkv), hk(bh_ - (bh_ / a_.Hkv) * a_.Hkv), rg0(tile * NG), ngroups(ngroups_), tid(threadIdx.x),
        lane(threadIdx.x & 63), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), n(valid_keys(a_.k_len, bh_ / a_.Hkv, a_.Lk)),
        nb((n + BLK - 1) / BLK), list(l) {
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int e = u * P + tid, half = e >= PIECES / 2 ? 1 : 0, x = e - half * (PIECES / 2), t = x / (D / 8), c = x % (D / 8);
      const Rows& r = half ? a.v : a.k;
      src[u] = r.p + b * r.sb + t * r.sl + hk * r.sh + c * 8;
      step[u] = BLK * r.sl;
      key[u] = e < PIECES ? t : 0x40000000;   // (no piece: behind every valid key)
      to[u] = half * Geo<D>::KV_BYTES + lds_at<D>(t, c);
    }
  }

  // The next block that a row of the pool chose (j < 0: none) and its rows, into list[buf]. Lane x looks at block base + x.
  __device__ __forceinline__ Hit advance(int buf) {
    while (!bits) {
      if (next0 >= nb) return Hit{-1, 0};
      base = next0;
      next0 += 64;
      pre = tot = 0;
      mine = 0;
      const int j = base + lane;
#pragma unroll
      for (int x = 0; x < NG; ++x) {
        const unsigned long long w = j < nb && rg0 + x < ngroups ? a.mask[((long)bh * ngroups + rg0 + x) * a.nblk + j] : 0;
        if (x == wave) { mine = w; pre = tot; }
        tot += __builtin_popcountll(w);
      }
      bits = __ballot(tot > 0);
    }
    const int x = __builtin_ctzll(bits);
    bits &= bits - 1;
    const unsigned lo = __builtin_amdgcn_readlane((unsigned)mine, x), hi = __builtin_amdgcn_readlane((unsigned)(mine >> 32), x);
    const int first = __builtin_amdgcn_readlane(pre, x);
    const int rank = __builtin_amdgcn_mbcnt_hi(hi, __builtin_amdgcn_mbcnt_lo(lo, 0));
    if (((lane < 32 ? lo : hi) >> (lane & 31)) & 1) list[buf][first + rank] = (unsigned short)(wave * 64 + lane);
    return Hit{base + x, __builtin_amdgcn_readlane(tot, x)};
  }

  // a row's place in a [..][positions][heads][D] tensor, in units of 8 features from the sample's first (0 behind the last row)
  __device__ __forceinline__ unsigned offset(int row, long sl, long sh) const {
    if (row_index(row) >= (long)a.Lq * a.G) return 0;
    long i;
    int h;
    place(row, i, h);
    return (unsigned)((i * sl + h * sh) >> 3);
  }
  __device__ __forceinline__ long row_index(int row) const { return (long)rg0 * 64 + row; }
  // position and head of a row
  __device__ __forceinline__ void place(int row, long& i, int& h) const {
    const unsigned r = (unsigned)row_index(row);
    if (a.G == 1) { i = r; h = hk; }
    else { const unsigned q = r / (unsigned)a.G; i = q; h = hk * a.G + (int)(r - q * a.G); }
  }

  __device__ __forceinline__ void fetch(int j) {   // block j's keys and values into registers
    const bf16x8_t none = {};
    const int left = n - j * BLK;
#pragma unroll
    for (int u = 0; u < PER; ++u) kv[u] = key[u] < left ? *(const bf16x8_t*)(src[u] + j * step[u]) : none;
  }
  __device__ __forceinline__ void stage(char* kvbuf) const {
    const bf16x8_t none = {};
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      if (PIECES < P * PER && key[u] >= 0x40000000) continue;
      *(bf16x8_t*)(kvbuf + to[u]) = kv[u];
      if constexpr (D == 8) *(bf16x8_t*)(kvbuf + to[u] + 16) = none;
    }
  }
};

__device__ __forceinline__ bool pool_of(int nbh, int ntiles, int& bh, int& tile) {
  if ((nbh & 7) == 0) dm_xcd_tile(blockIdx.x, ntiles, bh, tile);   // one head's pools on one XCD: its keys and values stay in that L2
  else { bh = blockIdx.x / ntiles; tile = blockIdx.x % ntiles; }
  return bh < nbh;
}

template <int D, int P>
__global__ __launch_bounds__(P) void attend_pool_kernel(Args a, int ngroups, int ntiles) {
  using GE = Geo<D>;
  __shared__ __attribute__((aligned(16))) char kbuf[2 * GE::KV_BYTES];
  char* const vbuf = kbuf + GE::KV_BYTES;
  __shared__ __attribute__((aligned(16))) float acc[P * GE::DV];
  __shared__ unsigned rowoff[P];          // a row's place in q, in units of 8 features from the sample's first
  __shared__ float sm[P], sl[P], sr[P];   // maximum, sum of the weights, sum of the weights as rounded
  __shared__ unsigned short list[3][P];
  int bh, tile;
  if (!pool_of(a.B * a.Hkv, ntiles, bh, tile)) return;
  Walk<D, P> w(a, bh, tile, ngroups, list);
  const int lane = w.lane, g = lane >> 4;
  const float sc = a.scale * LOG2E, asc = fabsf(sc);   // (the sign of the scale goes to q: a maximum is scaled by the amount)
  auto cur = w.advance(0);
  typename Walk<D, P>::Hit nxt{-1, 0};
  if (cur.j >= 0) {
    nxt = w.advance(1);
    w.fetch(cur.j);
    w.stage(kbuf);
  }
  const f32x4_t zero4 = {0.f, 0.f, 0.f, 0.f};
  const bf16_t one = (bf16_t)1.f;
  const bf16x8_t ones = {one, one, one, one, one, one, one, one};
  for (int e = w.tid; e < P * GE::OC; e += P) *(f32x4_t*)(acc + e * 4) = zero4;
  rowoff[w.tid] = w.offset(w.tid, a.q.sl, a.q.sh);
  sm[w.tid] = -INFINITY;
  sl[w.tid] = sr[w.tid] = 0.f;
  __syncthreads();

  const bf16_t* const qbase = a.q.p + w.b * a.q.sb;
  auto load_q = [&](Frag<D>& f, const unsigned short* ls, int t, int count) {
    const int li = t * 16 + (lane & 15);
    f.load(qbase + (size_t)rowoff[ls[li < count ? li : t * 16]] * 8, g);
    if (sc < 0.f) f.negate();
  };
  Frag<D> qf, qn;
  qf.zero();
  qn.zero();
  if (cur.j >= 0 && w.wave * 16 < cur.n) load_q(qf, list[0], w.wave, cur.n);
  qf.arrived();
  int buf = 0;
  while (cur.j >= 0) {
    const int b1 = buf == 2 ? 0 : buf + 1, b2 = b1 == 2 ? 0 : b1 + 1;
    typename Walk<D, P>::Hit nn{-1, 0};
    if (nxt.j >= 0) {
      w.fetch(nxt.j);
      nn = w.advance(b2);
      if (w.wave * 16 < nxt.n) load_q(qn, list[b1], w.wave, nxt.n);
    }
    const int n0 = w.n - cur.j * BLK;   // valid keys from this block on
    for (int t = w.wave; t * 16 < cur.n; t += P / 64) {
      if (t != w.wave) {
        load_q(qf, list[buf], t, cur.n);
        qf.arrived();
      }
      const int li = t * 16 + (lane & 15);
      const bool live = li < cur.n;
      const int row = list[buf][live ? li : t * 16];
      float s[16];
      {
        Frag<D> kf[4];
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) kf[kt].from_lds(kbuf, kt * 16 + (lane & 15), g);
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) *(f32x4_t*)(s + kt * 4) = dot_frag<D>(kf[kt], qf);
      }
      // everything else that the tile reads from LDS is under way before the softmax
      const float m_old = sm[row], l_old = sl[row], r_sum = sr[row];
      f32x4_t o[GE::DT];
      bf16x4_t vt[GE::DT][4];
#pragma unroll
      for (int dt = 0; dt < GE::DT; ++dt) {
        o[dt] = *(const f32x4_t*)(acc + acc_at<D>(row, dt * 4 + g));
#pragma unroll
        for (int u = 0; u < 4; ++u) vt[dt][u] = read_tr<D>(vbuf, u * 16, dt, lane);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (n0 < BLK) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if ((e >> 2) * 16 + g * 4 + (e & 3) >= n0) s[e] = -INFINITY;
      }
      float mx = s[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
      const float m_new = fmaxf(m_old, row_max(mx) * asc), at = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = __builtin_amdgcn_exp2f(m_old - at);
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(s[e] * asc - at);
      if (n0 < BLK) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if ((e >> 2) * 16 + g * 4 + (e & 3) >= n0) s[e] = 0.f;   // (a scale of zero times -infinity is no zero)
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) sum += s[e];
      sum = row_sum(sum);
      // The weights are rounded to bf16 as the matrix instruction's operand. The output is divided by the sum of the
      // ROUNDED weights (one more product, with ones), so that it stays an average of values: a rounding then counts only
      // with the value's distance from the output. The saved statistic is of the unrounded ones.
      bf16x8_t p[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) p[u] = dm_pack8(s + u * 8);
      const float r_old = r_sum * alpha;
      f32x4_t rs = {r_old, r_old, r_old, r_old};
#pragma unroll
      for (int u = 0; u < 2; ++u) rs = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, p[u], rs, 0, 0, 0);
      if (live && g == 0) {
        sl[row] = l_old * alpha + sum;
        sr[row] = rs[0];
        sm[row] = m_new;
      }
#pragma unroll
      for (int dt = 0; dt < GE::DT; ++dt) {
        f32x4_t c = o[dt];
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e] *= alpha;
#pragma unroll
        for (int u = 0; u < 2; ++u) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(join4(vt[dt][2 * u], vt[dt][2 * u + 1]), p[u], c, 0, 0, 0);
        if (live) *(f32x4_t*)(acc + acc_at<D>(row, dt * 4 + g)) = c;
      }
    }
    __syncthreads();
    if (nxt.j >= 0) w.stage(kbuf);
    __syncthreads();
    cur = nxt;
    nxt = nn;
    qf = qn;
    qf.arrived();
    buf = b1;
  }
  constexpr int PC = D / 8;
  for (int e = w.tid; e < P * PC; e += P) {
    const int row = e / PC, c = e % PC;
    if (w.row_index(row) >= (long)a.Lq * a.G) break;
    long i;
    int h;
    w.place(row, i, h);
    const float l = sl[row], inv = 1.0f / sr[row];
    float f[8], lo[8];
    *(f32x4_t*)f = *(const f32x4_t*)(acc + acc_at<D>(row, c * 2));
    *(f32x4_t*)(f + 4) = *(const f32x4_t*)(acc + acc_at<D>(row, c * 2 + 1));
#pragma unroll
    for (int x = 0; x < 8; ++x) f[x] = l == 0.f ? 0.f : f[x] * inv;
    const bf16x8_t y = dm_pack8(f);
    const long at = (((long)w.b * a.Lq + i) * a.Hq + h) * D + c * 8;
    *(bf16x8_t*)(a.out + at) = y;
    if (a.out_lo) {
#pragma unroll
      for (int x = 0; x < 8; ++x) lo[x] = f[x] - (float)y[x];
      *(bf16x8_t*)(a.out_lo + at) = dm_pack8(lo);
    }
    if (a.lse && c == 0) a.lse[((long)w.b * a.Hq + h) * a.Lq + i] = l == 0.f ? -INFINITY : sm[row] * LN2 + logf(l);
  }
}

// dq of a pool, and delta for the kernel behind. dq gathers p (dp - delta) k; the scale is applied once at the end.
template <int D, int P>
__global__ __launch_bounds__(P) void dq_pool_kernel(Args a, int ngroups, int ntiles) {
  using GE = Geo<D>;
  __shared__ __attribute__((aligned(16))) char kbuf[2 * GE::KV_BYTES];
  char* const vbuf = kbuf + GE::KV_BYTES;
  __shared__ __attribute__((aligned(16))) float acc[P * GE::DV];
  __shared__ unsigned rowoff[P];          // a row's place in q, in units of 8 features from the sample's first
  __shared__ unsigned gooff[P];           // ... and in the output's gradient
  __shared__ float s_lse[P], s_delta[P];
  __shared__ unsigned short list[3][P];
  int bh, tile;
  if (!pool_of(a.B * a.Hkv, ntiles, bh, tile)) return;
  Walk<D, P> w(a, bh, tile, ngroups, list);
  const int lane = w.lane, g = lane >> 4;
  const float sc = a.scale * LOG2E;
  auto cur = w.advance(0);
  typename Walk<D, P>::Hit nxt{-1, 0};
  if (cur.j >= 0) {
    nxt = w.advance(1);
    w.fetch(cur.j);
    w.stage(kbuf);
  }
  const f32x4_t zero4 = {0.f, 0.f, 0.f, 0.f};
  for (int e = w.tid; e < P * GE::OC; e += P) *(f32x4_t*)(acc + e * 4) = zero4;
  rowoff[w.tid] = w.offset(w.tid, a.q.sl, a.q.sh);
  gooff[w.tid] = w.offset(w.tid, (long)a.Hq * D, D);
  constexpr int PC = D / 8;
  for (int e = w.tid; e < P * PC; e += P) {   // (a row's PC lanes are neighbours: P is a multiple of PC)
    const int row = e / PC, c = e % PC;
    const bool in = w.row_index(row) < (long)a.Lq * a.G;
    long i = 0;
    int h = 0;
    if (in) w.place(row, i, h);
    const long at = (((long)w.b * a.Lq + i) * a.Hq + h) * D + c * 8, lrow = ((long)w.b * a.Hq + h) * a.Lq + i;
    float go[8], o[8], lo[8], delta = 0.f;
    if (in) {
      dm_unpack8(*(const bf16x8_t*)(a.go + at), go);
      dm_unpack8(*(const bf16x8_t*)(a.o + at), o);
      dm_unpack8(*(const bf16x8_t*)(a.o_lo + at), lo);
#pragma unroll
      for (int x = 0; x < 8; ++x) delta += go[x] * (o[x] + lo[x]);
    }
    delta = group_sum<PC>(delta);
    if (c == 0) {
      const float lse = in ? a.lse[lrow] : 0.f;
      s_delta[row] = delta;
      s_lse[row] = lse == -INFINITY ? INFINITY : lse * LOG2E;   // no key: every weight becomes zero
      if (in) a.delta[lrow] = delta;
    }
  }
  __syncthreads();

  const bf16_t* const qbase = a.q.p + w.b * a.q.sb;
  const bf16_t* const obase = a.go + (long)w.b * a.Lq * a.Hq * D;
  auto load_rows = [&](Frag<D>& fq, Frag<D>& fo, const unsigned short* ls, int t, int count) {
    const int li = t * 16 + (lane & 15), row = ls[li < count ? li : t * 16];
    fq.load(qbase + (size_t)rowoff[row] * 8, g);
    fo.load(obase + (size_t)gooff[row] * 8, g);
  };
  Frag<D> qf, qn, of, on;
  qf.zero(); qn.zero(); of.zero(); on.zero();
  if (cur.j >= 0 && w.wave * 16 < cur.n) load_rows(qf, of, list[0], w.wave, cur.n);
  qf.arrived();
  of.arrived();
  int buf = 0;
  while (cur.j >= 0) {
    const int b1 = buf == 2 ? 0 : buf + 1, b2 = b1 == 2 ? 0 : b1 + 1;
    typename Walk<D, P>::Hit nn{-1, 0};
    if (nxt.j >= 0) {
      w.fetch(nxt.j);
      nn = w.advance(b2);
      if (w.wave * 16 < nxt.n) load_rows(qn, on, list[b1], w.wave, nxt.n);
    }
    const int n0 = w.n - cur.j * BLK;
    for (int t = w.wave; t * 16 < cur.n; t += P / 64) {
      if (t != w.wave) {
        load_rows(qf, of, list[buf], t, cur.n);
        qf.arrived();
        of.arrived();
      }
      const int li = t * 16 + (lane & 15);
      const bool live = li < cur.n;
      const int row = list[buf][live ? li : t * 16];
      const float lse = s_lse[row], delta = s_delta[row];
      float ds[16];
      Frag<D> kf[4], vf[4];
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) {
        kf[kt].from_lds(kbuf, kt * 16 + (lane & 15), g);
        vf[kt].from_lds(vbuf, kt * 16 + (lane & 15), g);
      }
      f32x4_t s[4], dp[4];
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) {
        s[kt] = dot_frag<D>(kf[kt], qf);
        dp[kt] = dot_frag<D>(vf[kt], of);
      }
      f32x4_t o[GE::DT];
      bf16x4_t kt_[GE::DT][4];
#pragma unroll
      for (int dt = 0; dt < GE::DT; ++dt) {
        o[dt] = *(const f32x4_t*)(acc + acc_at<D>(row, dt * 4 + g));
#pragma unroll
        for (int u = 0; u < 4; ++u) kt_[dt][u] = read_tr<D>(kbuf, u * 16, dt, lane);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) ds[kt * 4 + e] = __builtin_amdgcn_exp2f(s[kt][e] * sc - lse) * (dp[kt][e] - delta);
      if (n0 < BLK) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if ((e >> 2) * 16 + g * 4 + (e & 3) >= n0) ds[e] = 0.f;
      }
      bf16x8_t p[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) p[u] = dm_pack8(ds + u * 8);
#pragma unroll
      for (int dt = 0; dt < GE::DT; ++dt) {
        f32x4_t c = o[dt];
#pragma unroll
        for (int u = 0; u < 2; ++u) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(join4(kt_[dt][2 * u], kt_[dt][2 * u + 1]), p[u], c, 0, 0, 0);
        if (live) *(f32x4_t*)(acc + acc_at<D>(row, dt * 4 + g)) = c;
      }
    }
    __syncthreads();
    if (nxt.j >= 0) w.stage(kbuf);
    __syncthreads();
    cur = nxt;
    nxt = nn;
    qf = qn;
    of = on;
    qf.arrived();
    of.arrived();
    buf = b1;
  }
  for (int e = w.tid; e < P * PC; e += P) {
    const int row = e / PC, c = e % PC;
    if (w.row_index(row) >= (long)a.Lq * a.G) break;
    long i;
    int h;
    w.place(row, i, h);
    float f[8];
    *(f32x4_t*)f = *(const f32x4_t*)(acc + acc_at<D>(row, c * 2));
    *(f32x4_t*)(f + 4) = *(const f32x4_t*)(acc + acc_at<D>(row, c * 2 + 1));
#pragma unroll
    for (int x = 0; x < 8; ++x) f[x] *= a.scale;
    *(bf16x8_t*)(a.dq + w.b * a.dqb + i * a.dql + h * a.dqh + c * 8) = dm_pack8(f);
  }
}

// dk and dv of one block, four waves. The rows that chose it are packed into a list, 4096 rows at a time, and dealt to the
// waves in tiles of 32; every wave sums all 64 keys over its own rows in registers, and the four sums are added in wave
// order. Scores are formed as S = Q K^T here: a lane holds 4 rows x 2 tiles of ONE key, which is the layout that dv =
// P^T dO and dk = dS^T Q take as their left operand; the right operands are the tile's rows, read transposed from the wave's own LDS.
constexpr int LIST = 4096;
template <int D>
__global__ __launch_bounds__(256, 2) void dkv_kernel(Args a, int ngroups) {
  using GE = Geo<D>;
  constexpr int TILE_BYTES = 32 * GE::ROWB;
  __shared__ __attribute__((aligned(16))) char kbuf[GE::KV_BYTES], vbuf[GE::KV_BYTES];
  __shared__ __attribute__((aligned(16))) char rows[4][2][TILE_BYTES];    // q and do of a wave's tile; at the end the sums
  __shared__ __attribute__((aligned(16))) float stat[4][2][32];           // lse, delta
  __shared__ unsigned short list[LIST];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4;
  const int j = blockIdx.x, bh = blockIdx.y, b = bh / a.Hkv, hk = bh - b * a.Hkv;
  const int n0 = valid_keys(a.k_len, b, a.Lk) - j * BLK;
  const float sc = a.scale * LOG2E;
  const bf16x8_t none = {};
  if (n0 > 0) {
    for (int e = tid; e < 2 * BLK * D / 8; e += 256) {
      const int half = e >= BLK * D / 8 ? 1 : 0, p = e - half * (BLK * D / 8), t = p / (D / 8), c = p % (D / 8);
      const Rows& s = half ? a.v : a.k;
      char* to = half ? vbuf : kbuf;
      *(bf16x8_t*)(to + lds_at<D>(t, c)) = t < n0 ? *(const bf16x8_t*)(s.p + b * s.sb + ((long)j * BLK + t) * s.sl + hk * s.sh + c * 8) : none;
      if constexpr (D == 8) *(bf16x8_t*)(to + lds_at<D>(t, 1)) = none;
    }
  }
  f32x4_t dk[4][GE::DT], dv[4][GE::DT];
#pragma unroll
  for (int kt = 0; kt < 4; ++kt)
#pragma unroll
    for (int dt = 0; dt < GE::DT; ++dt) dk[kt][dt] = dv[kt][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  char *qb = rows[wave][0], *ob = rows[wave][1];
  float *st_lse = stat[wave][0], *st_delta = stat[wave][1];
  for (int rg0 = 0; rg0 < ngroups && n0 > 0; rg0 += LIST / 64) {
    const unsigned long long word = rg0 + lane < ngroups ? a.mask[((long)bh * ngroups + rg0 + lane) * a.nblk + j] : 0;
    int inc = __builtin_popcountll(word);
    const int own = inc;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int up = __shfl_up(inc, o, 64);
      if (lane >= o) inc += up;
    }
    const int count = __builtin_amdgcn_readlane(inc, 63), before = inc - own;
    __syncthreads();   // the list's last use is over
    for (int x = wave; x < LIST / 64; x += 4) {
      const unsigned lo = __builtin_amdgcn_readlane((unsigned)word, x), hi = __builtin_amdgcn_readlane((unsigned)(word >> 32), x);
      const int first = __builtin_amdgcn_readlane(before, x);
      const int rank = __builtin_amdgcn_mbcnt_hi(hi, __builtin_amdgcn_mbcnt_lo(lo, 0));
      if (((lane < 32 ? lo : hi) >> (lane & 31)) & 1) list[first + rank] = (unsigned short)(x * 64 + lane);
    }
    __syncthreads();
    for (int t = wave; t * 32 < count; t += 4) {
      // a lane's two rows: 16 mt + (lane & 15)
      Frag<D> qf[2], of[2];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const int li = t * 32 + mt * 16 + (lane & 15);
        qf[mt].zero();
        of[mt].zero();
        float lse = INFINITY, delta = 0.f;
        if (li < count) {
          const unsigned r = (unsigned)(rg0 * 64 + list[li]);
          const unsigned i = a.G == 1 ? r : r / (unsigned)a.G;
          const int h = hk * a.G + (int)(r - i * a.G);
          const long lrow = ((long)b * a.Hq + h) * a.Lq + i;
          qf[mt].load(a.q.p + b * a.q.sb + (long)i * a.q.sl + h * a.q.sh, g);
          of[mt].load(a.go + (((long)b * a.Lq + i) * a.Hq + h) * D, g);
          lse = a.lse[lrow];
          lse = lse == -INFINITY ? INFINITY : lse * LOG2E;
          delta = a.delta[lrow];
        }
        const int row = mt * 16 + (lane & 15);
        if (g == 0) { st_lse[row] = lse; st_delta[row] = delta; }
        if constexpr (D <= 16) {
          *(bf16x4_t*)(qb + lds_at<D>(row, g >> 1) + (g & 1) * 8) = __builtin_shufflevector(qf[mt].x[0], qf[mt].x[0], 0, 1, 2, 3);
          *(bf16x4_t*)(ob + lds_at<D>(row, g >> 1) + (g & 1) * 8) = __builtin_shufflevector(of[mt].x[0], of[mt].x[0], 0, 1, 2, 3);
        } else {
#pragma unroll
          for (int s = 0; s < GE::KS; ++s) {
            *(bf16x8_t*)(qb + lds_at<D>(row, s * 4 + g)) = qf[mt].x[s];
            *(bf16x8_t*)(ob + lds_at<D>(row, s * 4 + g)) = of[mt].x[s];
          }
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the wave's own writes, read by its other lanes
      bf16x8_t qt[GE::DT], ot[GE::DT];
#pragma unroll
      for (int dt = 0; dt < GE::DT; ++dt) {
        qt[dt] = join4(read_tr<D>(qb, 0, dt, lane), read_tr<D>(qb, 16, dt, lane));
        ot[dt] = join4(read_tr<D>(ob, 0, dt, lane), read_tr<D>(ob, 16, dt, lane));
      }
      f32x4_t lse4[2], delta4[2];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        lse4[mt] = *(const f32x4_t*)(st_lse + mt * 16 + g * 4);
        delta4[mt] = *(const f32x4_t*)(st_delta + mt * 16 + g * 4);
      }
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) {
        Frag<D> kf, vf;
        kf.from_lds(kbuf, kt * 16 + (lane & 15), g);
        vf.from_lds(vbuf, kt * 16 + (lane & 15), g);
        float p[8], ds[8];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          const f32x4_t s = dot_frag<D>(qf[mt], kf), dp = dot_frag<D>(of[mt], vf);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            p[mt * 4 + e] = __builtin_amdgcn_exp2f(s[e] * sc - lse4[mt][e]);
            ds[mt * 4 + e] = p[mt * 4 + e] * (dp[e] - delta4[mt][e]);
          }
        }
        const bf16x8_t pt = dm_pack8(p), dst = dm_pack8(ds);
#pragma unroll
        for (int dt = 0; dt < GE::DT; ++dt) {
          dv[kt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pt, ot[dt], dv[kt][dt], 0, 0, 0);
          dk[kt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(dst, qt[dt], dk[kt][dt], 0, 0, 0);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }
  // the four waves' sums, in wave order: [key][feature] fp32 in the tiles' memory (4 x 2 x 32 rows hold 64 rows twice)
  float* sum = (float*)&rows[0][0][0];
  constexpr int HALF = BLK * GE::DV;
  for (int x = 0; x < 4; ++x) {
    __syncthreads();
    if (wave == x) {
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int dt = 0; dt < GE::DT; ++dt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int at = (kt * 16 + g * 4 + e) * GE::DV + dt * 16 + (lane & 15);
            sum[at] = (x ? sum[at] : 0.f) + dk[kt][dt][e];
            sum[HALF + at] = (x ? sum[HALF + at] : 0.f) + dv[kt][dt][e];
          }
    }
  }
  __syncthreads();
  const int in = min(BLK, a.Lk - j * BLK);
  for (int e = tid; e < BLK * D / 8; e += 256) {
    const int t = e / (D / 8), d = (e % (D / 8)) * 8;
    if (t >= in) break;
    const long pos = (long)j * BLK + t;
    const bool live = t < n0;   // positions behind the last valid key: zero
    float f[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) f[x] = live ? sum[t * GE::DV + d + x] * a.scale : 0.f;
    *(bf16x8_t*)(a.dk + b * a.dkb + pos * a.dkl + hk * a.dkh + d) = dm_pack8(f);
#pragma unroll
    for (int x = 0; x < 8; ++x) f[x] = live ? sum[HALF + t * GE::DV + d + x] : 0.f;
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
// rows are addressed inside a sample by 32-bit numbers of 8 features
int check_span(const char* who, const dm_block_desc* d) {
  const long* s = d->q_stride;
  for (int i = 0; i < 3; ++i) DM_REQUIRE(s[i] >= 0, DM_ERR_ARG, "%s: negative stride of q", who);
  DM_REQUIRE((d->Lq - 1) * s[1] + (d->Hq - 1) * s[2] < (1L << 35) && (long)d->Lq * d->Hq * d->D < (1L << 35), DM_ERR_SHAPE,
             "%s: a sample of q spans more than 2^35 elements", who);
  return DM_OK;
}
int blocks_of(const dm_block_desc* d) { return (d->Lk + BLK - 1) / BLK; }
// Rows of a pool (0: one query a workgroup). Large pools fill tiles better and read keys and values less often; small ones
// give more workgroups where there are few rows.
int pool_rows(const dm_block_desc* d) {
  if (g_dm_block_pool) return g_dm_block_pool == 1 ? 0 : g_dm_block_pool;
  const long rows = (long)d->Lq * (d->Hq / d->Hkv), heads = (long)d->B * d->Hkv;
  if (rows < 16) return 0;
  return heads * dm_cdiv(rows, 512) >= 256 ? 512 : 128;
}
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
  const int G = d->Hq / d->Hkv, n = blocks_of(d), top = d->top;
  const long rows = (long)d->B * d->Hq * d->Lq, shared = (long)d->Lq * G;
  hipStream_t st = (hipStream_t)stream;
  if (shared < 16) {
    BY_HEAD_DIM(d->D, hipLaunchKernelGGL((block_select_row_kernel<HD>), dim3(dm_cdiv(rows, 4)), dim3(256), 0, st, rows_of(q, d->q_stride),
                                         (const bf16_t*)keys, k_len, blocks, d->Lq, d->Lk, d->Hq, G, top, n, rows));
  } else {
    const dim3 grid(dm_cdiv(shared, 64), d->B * d->Hkv);
#define GO(K) BY_HEAD_DIM(d->D, hipLaunchKernelGGL((block_select_kernel<HD, K>), grid, dim3(256), 0, st, rows_of(q, d->q_stride), \
                                                   (const bf16_t*)keys, k_len, blocks, d->Lq, d->Lk, d->Hkv, G, top, n))
    if (top <= 4) GO(5) else if (top <= 11) GO(8) else if (top <= 19) GO(12) else if (top <= 35) GO(20) else GO(36)
#undef GO
  }
  DM_CHECK_LAUNCH();
  return DM_OK;
}

extern "C" size_t dm_block_attention_mask_bytes(const dm_block_desc* d, int for_backward) {
  if (check_desc("dm_block_attention_mask_bytes", d) || (!for_backward && !pool_rows(d))) return 0;
  return (size_t)d->B * d->Hkv * groups_of(d) * blocks_of(d) * 8;
}

extern "C" int dm_block_attention_fwd(const dm_block_desc* d, const void* q, const void* k, const void* v, const int* blocks,
                                      const int* k_len, void* out, void* out_lo, float* lse, void* mask, void* stream) {
  const char* who = "dm_block_attention_fwd";
  int rc = check_desc(who, d);
  if (rc) return rc;
  DM_REQUIRE(aligned(q) && aligned(k) && aligned(v) && aligned(out) && blocks, DM_ERR_ARG, "%s: null or misaligned pointer", who);
  if ((rc = check_strides(who, "q", d->q_stride)) || (rc = check_strides(who, "k", d->k_stride)) ||
      (rc = check_strides(who, "v", d->v_stride)) || (rc = check_span(who, d)))
    return rc;
  Args a = args_of(d);
  a.q = rows_of(q, d->q_stride); a.k = rows_of(k, d->k_stride); a.v = rows_of(v, d->v_stride);
  a.blocks = blocks; a.k_len = k_len; a.out = (bf16_t*)out; a.out_lo = (bf16_t*)out_lo; a.lse = lse; a.mask = (unsigned long long*)mask;
  hipStream_t st = (hipStream_t)stream;
  const int pool = pool_rows(d), tiles = pool ? dm_cdiv((long)d->Lq * a.G, pool) : 0;
  DM_REQUIRE(aligned(mask) || (!mask && !pool), DM_ERR_ARG, "%s: this shape needs a mask (dm_block_attention_mask_bytes), 16-byte aligned", who);
  if (mask) {
    hipLaunchKernelGGL(block_mask_kernel, dim3(groups_of(d), d->B * d->Hkv), dim3(256), 0, st, blocks, (unsigned long long*)mask, d->Lq,
                       d->Hq, a.G, d->top, a.nblk, groups_of(d));
    DM_CHECK_LAUNCH();
  }
  const long rows = (long)d->B * d->Hq * d->Lq;
  const dim3 grid(d->B * d->Hkv * tiles);
  switch (pool) {
    case 0: BY_HEAD_DIM(d->D, hipLaunchKernelGGL((attend_row_kernel<HD, 4>), dim3((unsigned)rows), dim3(256), 0, st, a)); break;
    case 128: BY_HEAD_DIM(d->D, hipLaunchKernelGGL((attend_pool_kernel<HD, 128>), grid, dim3(128), 0, st, a, groups_of(d), tiles)); break;
    case 256: BY_HEAD_DIM(d->D, hipLaunchKernelGGL((attend_pool_kernel<HD, 256>), grid, dim3(256), 0, st, a, groups_of(d), tiles)); break;
    default: BY_HEAD_DIM(d->D, hipLaunchKernelGGL((attend_pool_kernel<HD, 512>), grid, dim3(512), 0, st, a, groups_of(d), tiles)); break;
  }
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
  if ((rc = check_span(who, d))) return rc;
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
  const int pool = pool_rows(d), tiles = pool ? dm_cdiv((long)d->Lq * a.G, pool) : 0;
  const dim3 grid(d->B * d->Hkv * tiles);
  switch (pool) {
    case 0: BY_HEAD_DIM(d->D, hipLaunchKernelGGL((dq_row_kernel<HD>), dim3(dm_cdiv(rows, 4)), dim3(256), 0, st, a, rows)); break;
    case 128: BY_HEAD_DIM(d->D, hipLaunchKernelGGL((dq_pool_kernel<HD, 128>), grid, dim3(128), 0, st, a, groups_of(d), tiles)); break;
    case 256: BY_HEAD_DIM(d->D, hipLaunchKernelGGL((dq_pool_kernel<HD, 256>), grid, dim3(256), 0, st, a, groups_of(d), tiles)); break;
    default: BY_HEAD_DIM(d->D, hipLaunchKernelGGL((dq_pool_kernel<HD, 512>), grid, dim3(512), 0, st, a, groups_of(d), tiles)); break;
  }
  DM_CHECK_LAUNCH();
  BY_HEAD_DIM(d->D, hipLaunchKernelGGL((dkv_kernel<HD>), dim3(a.nblk, d->B * d->Hkv), dim3(256), 0, st, a, groups_of(d)));
  DM_CHECK_LAUNCH();
  return DM_OK;
}
