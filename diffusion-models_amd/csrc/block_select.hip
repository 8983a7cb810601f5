// The choice of key blocks: one summary per block of 64 keys, and for every query the blocks whose summaries it scores highest.
//
//   keys[b][h][j]   = mean of block j's valid keys              (dm_block_keys)
//   blocks[b][h][i] = the `top` blocks of the highest q_i . keys_j (dm_block_select)
//
// Query heads share key heads (Hq = G Hkv). The ROWS of a (sample, key head) are its G Lq queries, r = i G + g.
#include "block_common.h"

namespace {

// ---------------------------------------------------------------------------------------------------------------
// One summary per block: the mean of its valid keys. Summed in 64 bits (64 bf16 values of ordinary spread add up
// exactly, so the order does not matter) and rounded to fp32 and then bf16: the summary is only a score's operand, and
// as bf16 its products with q are exact in 64-bit sums too, which makes the choice of blocks independent of batch, tile and order.
// A workgroup holds one block of up to 512 features (8 a lane) of all heads, its threads splitting the 64 keys: rows of all heads are
// read whole. Bound by HBM (2 x 16384 keys of 8 x 64 features, 33.6 MB: 9.7 us, 3.5 TB/s).
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
#pragma unroll 8
    for (int t = phase; t < n; t += phases) {
      const bf16x8_t x = *(const bf16x8_t*)(p + t * k.sl);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] += (double)(float)x[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) part[tid][e] = s[e];
  __syncthreads();
  for (int o = tid; o < vt * 8; o += 256) {   // a thread a feature
    const int to = blockIdx.y * vt * 8 + o, head = to / D;
    if (to >= Hkv * D) break;
    double t = part[o >> 3][o & 7];
    for (int w = 1; w < phases; ++w) t += part[w * vt + (o >> 3)][o & 7];
    keys[(((long)b * Hkv + head) * nblk + j) * D + (to - head * D)] = (bf16_t)(float)(n > 0 ? t / n : 0.0);
  }
}

// ---------------------------------------------------------------------------------------------------------------
// The choice of blocks. Scores are compared as 64-bit sums; two ways to get there:
//
// exact_top: a query at a time, all scores in 64 bits, EXACT_CHUNK blocks at a time beside the best of the earlier ones. A
// score becomes an unsigned number of the same order (NaN: that of -infinity), 0 stands for a block already taken.
constexpr int EXACT_CHUNK = 256;
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

// The `top` best of what the wave's lanes hold (PER candidates a lane, and one more, won / won_j), best first: the t-th goes to
// lane t's won / won_j.
template <int PER>
__device__ __forceinline__ void keep_best(unsigned long long (&score)[PER], const int (&place)[PER], int top, int lane,
                                          unsigned long long& won, int& won_j) {
  unsigned long long next = 0;
  int next_j = NO_BLOCK;
  for (int t = 0; t < top; ++t) {
    unsigned long long key = won;
    int j = won_j;
#pragma unroll
    for (int u = 0; u < PER; ++u)
      if (score[u] > key || (score[u] == key && place[u] < j)) { key = score[u]; j = place[u]; }
    take_best<1>(key, j);
    take_best<2>(key, j);
    take_best<4>(key, j);
    take_best<8>(key, j);
    take_best<16>(key, j);
    take_best<32>(key, j);
    if (!key) break;
    if (lane == t) { next = key; next_j = j; }
    if (won_j == j) won = 0;
#pragma unroll
    for (int u = 0; u < PER; ++u)
      if (place[u] == j) score[u] = 0;
  }
  won = next;
  won_j = next_j;
}

// The `top` best of the chunks first, first + step ... of a query's blocks; lane x scores blocks c0 + x, c0 + x + 64 ... of a chunk.
template <int D>
__device__ void exact_top(const bf16_t* qp, const bf16_t* kp, int have, int top, int lane, int first, int step, unsigned long long& won,
                          int& won_j) {
  constexpr int PER = EXACT_CHUNK / 64;
  won = 0;
  won_j = NO_BLOCK;
  for (int c0 = first * EXACT_CHUNK; c0 < have; c0 += step * EXACT_CHUNK) {
    double s[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) s[u] = 0;
#pragma unroll 1
    for (int d = 0; d < D; d += 8) {
      const bf16x8_t a = *(const bf16x8_t*)(qp + d);
      double q[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e] = (double)(float)a[e];
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        if (c0 + u * 64 >= have) break;
        const bf16x8_t b = *(const bf16x8_t*)(kp + (long)min(c0 + u * 64 + lane, have - 1) * D + d);
#pragma unroll
        for (int e = 0; e < 8; ++e) s[u] += q[e] * (double)(float)b[e];
      }
    }
    unsigned long long score[PER];
    int place[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const double x = s[u] == s[u] ? s[u] + 0.0 : -INFINITY;   // (-0 and 0 are equal)
      const unsigned long long v = __builtin_bit_cast(unsigned long long, x);
      place[u] = c0 + u * 64 + lane;
      score[u] = place[u] >= have ? 0 : (v >> 63) ? ~v : v | 0x8000000000000000ull;
    }
    keep_best<PER>(score, place, top, lane, won, won_j);
  }
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

// NW waves a query: its chunks are dealt to them, and one wave takes the best of theirs
template <int D, int NW>
__global__ __launch_bounds__(NW == 1 ? 256 : NW * 64) void block_select_row_kernel(Rows q, const bf16_t* __restrict__ keys,
                                                                                    const int* __restrict__ k_len, int* __restrict__ blocks,
                                                                                    int Lq, int Lk, int Hq, int G, int top, int nblk, long rows) {
  __shared__ unsigned long long score[NW][64];
  __shared__ int place[NW][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long row = NW == 1 ? dm_block_index() * 4 + wave : dm_block_index();
  if (row >= rows) return;
  const int i = row % Lq, h = (row / Lq) % Hq, b = row / ((long)Lq * Hq);
  const int have = (valid_keys(k_len, b, Lk) + BLK - 1) / BLK;
  unsigned long long won;
  int taken;
  exact_top<D>(q.p + b * q.sb + i * q.sl + h * q.sh, keys + ((long)b * (Hq / G) + h / G) * nblk * (long)D, have, top, lane, NW == 1 ? 0 : wave, NW,
               won, taken);
  if (NW > 1) {
    score[wave][lane] = won;
    place[wave][lane] = taken;
    __syncthreads();
    if (wave) return;
    unsigned long long s[NW];
    int p[NW];
#pragma unroll
    for (int w = 0; w < NW; ++w) { s[w] = score[w][lane]; p[w] = place[w][lane]; }
    won = 0;
    taken = NO_BLOCK;
    keep_best<NW>(s, p, top, lane, won, taken);
  }
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
// dropped one that counts sends its row to exact_top as well. A second pass over the same scores writes the choice in order, a word
// of 32 blocks at a time. Bound by the VALU: 12 places and 64 scores a lane are 768 of the 3100 instructions a wave issues for 16 of 256 blocks,
// the second pass 900, the merge of four lists 600, rows decided by exact_top (0.5 % at 64 features) 200. 2 x 8 heads of 16384 queries: 147 us;
// 16 x 16 heads of 1024 queries, 4 of 16 blocks of 8 features: 18.5 us. K = 10 there: a lane overflows in 0.9 % of the rows, 255 us.
template <int D, int K>
__global__ __launch_bounds__(256) void block_select_kernel(Rows q, const bf16_t* __restrict__ keys, const int* __restrict__ k_len,
                                                           int* __restrict__ blocks, int Lq, int Lk, int Hkv, int G, int top, int nblk) {
  constexpr int LIST_FLOATS = 2 * K * 64, CHOICE_FLOATS = 16 * 64;
  __shared__ __attribute__((aligned(16))) float scratch[4][CHOICE_FLOATS > LIST_FLOATS ? CHOICE_FLOATS : LIST_FLOATS];
  __shared__ __attribute__((aligned(16))) char kbuf[2][Geo<D>::KV_BYTES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, bh = blockIdx.y, b_ = bh / Hkv, hk = bh - b_ * Hkv;
  const long rows = (long)Lq * G, r0 = ((long)blockIdx.x * 4 + wave) * 16;
  const long r = min(r0 + (lane & 15), rows - 1);   // (waves behind the last row work on it and write nothing)
  const bool in = r0 + (lane & 15) < rows;
  const unsigned i = G == 1 ? (unsigned)r : (unsigned)r / (unsigned)G;
  const int h = hk * G + (int)((unsigned)r - i * (unsigned)G), Hq = Hkv * G;
  int* to = blocks + (((long)b_ * Hq + h) * Lq + i) * top;
  const int have = (valid_keys(k_len, b_, Lk) + BLK - 1) / BLK;
  if (have <= top) {   // every block
    if (in)
      for (int t = g; t < top; t += 4) to[t] = t < have ? t : -1;
    return;
  }
  const bf16_t* kp = keys + (long)bh * nblk * D;
  const bf16_t* qp = q.p + b_ * q.sb + (long)i * q.sl + h * q.sh;
  Frag<D> qf;
  qf.load(qp, g);
  float qq = 0.f;
#pragma unroll
  for (int s = 0; s < Geo<D>::KS; ++s)
#pragma unroll
    for (int e = 0; e < Frag<D>::W; ++e) qq += (float)qf.x[s][e] * (float)qf.x[s][e];
  qq = row_sum(qq);
  const int mine = 4 * (lane & 3) + ((lane & 15) >> 2);   // the block of a chunk of 16 that this lane fetches; it gets the scores of 4 e + g
  float best[K];
#pragma unroll
  for (int x = 0; x < K; ++x) best[x] = -INFINITY;
  unsigned kk = 0;   // the largest |key|^2, by its bits: a NaN is larger than any number
  // The summaries pass through LDS, 64 at a time in two buffers, for the four waves (fetched by every wave for itself they were 1 GB
  // of L2 traffic at 128x128 images: 180 us against 170).
  constexpr int PER = (BLK * D / 8 + 255) / 256;
  bf16x8_t piece[PER];
  auto fetch = [&](int c0) {
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int e = u * 256 + threadIdx.x;
      if (e < BLK * D / 8) piece[u] = *(const bf16x8_t*)(kp + (long)min(c0 + e / (D / 8), have - 1) * D + e % (D / 8) * 8);
    }
  };
  auto stage = [&](char* to) {
    const bf16x8_t none = {};
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int e = u * 256 + threadIdx.x, t = e / (D / 8), x = e % (D / 8);
      if (e < BLK * D / 8) {
        *(bf16x8_t*)(to + lds_at<D>(t, x)) = piece[u];
        if constexpr (D == 8) *(bf16x8_t*)(to + lds_at<D>(t, 1)) = none;
      }
    }
  };
  Frag<D> kf;
  fetch(0);
  for (int c = 0; c < have; c += 16) {
    const char* const kb = kbuf[(c >> 6) & 1];
    if ((c & 63) == 0) {
      stage(kbuf[(c >> 6) & 1]);
      if (c + 64 < have) fetch(c + 64);
      __syncthreads();
    }
    kf.from_lds(kb, (c & 63) + mine, g);
    f32x4_t s = dot_frag<D>(kf, qf);
    const f32x4_t n = dot_frag<D>(kf, kf);
    const float d01 = (lane & 1) ? n[1] : n[0], d23 = (lane & 1) ? n[3] : n[2], d = (lane & 2) ? d23 : d01;
    if (g == ((lane & 15) >> 2)) kk = max(kk, __builtin_bit_cast(unsigned, d) & 0x7fffffffu);
    if (c + 16 > have) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c + 4 * e + g >= have) s[e] = -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
#pragma unroll
      for (int p = K - 1; p > 0; --p) best[p] = __builtin_amdgcn_fmed3f(best[p - 1], best[p], s[e]);
      best[0] = __builtin_amdgcn_fmed3f(best[0], s[e], INFINITY);   // (the larger of two, in one instruction)
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
  float T = -INFINITY, U = -INFINITY, b[2 * K + 2];   // b[x]: the other list's (top + 1 - x)-th
#pragma unroll
  for (int x = 0; x < 2 * K + 2; ++x) b[x] = lists[min(max(top - x, 0), 2 * K - 1) * 64 + (lane ^ 32)];
#pragma unroll
  for (int x = 0; x < 2 * K + 2; ++x) b[x] = top + 1 - x == 0 ? INFINITY : top + 1 - x > 0 && top + 1 - x <= 2 * K ? b[x] : -INFINITY;
#pragma unroll
  for (int x = 0; x <= 2 * K; ++x) {
    const float a = x == 0 ? INFINITY : two[x == 0 ? 0 : x - 1];
    T = fmaxf(T, fminf(a, b[x + 1]));
    U = fmaxf(U, fminf(a, b[x]));
  }
  const float eps2 = 2.f * ((D < 16 ? 16 : D) * 0x1.04p-23f * __builtin_sqrtf(qq + 0x1p-118f) * __builtin_sqrtf(__builtin_bit_cast(float, kk) + 0x1p-118f) + 0x1p-118f);
  bool clear = T - U > eps2;                                            // (false if anything is NaN or infinite)
  if (K < top + 1) {
    const float last = best[K - 1], l16 = fmaxf(last, __builtin_bit_cast(float, lane_xor_u<16>(__builtin_bit_cast(unsigned, last))));
    const float l32 = fmaxf(l16, __builtin_bit_cast(float, lane_xor_u<32>(__builtin_bit_cast(unsigned, l16))));
    clear = clear && (l32 == -INFINITY || U > l32);                     // what a lane dropped is not above its last
  }
  clear = clear && kk < 0x7f800000u && qq < INFINITY;
  // the choice in order into LDS (a row of `top` numbers a query), from there to memory by whole rows
  int* const chosen = (int*)scratch[wave] + (lane & 15) * top;
  fetch(0);
  __syncthreads();   // (every wave is done with the buffers of the first pass, and this one with its lists)
  int count = 0;
  for (int c = 0; c < have; c += 32) {   // a word of 32 blocks at a time
    const char* const kb = kbuf[(c >> 6) & 1];
    if ((c & 63) == 0) {
      stage(kbuf[(c >> 6) & 1]);
      if (c + 64 < have) fetch(c + 64);
      __syncthreads();
    }
    unsigned bits = 0;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      kf.from_lds(kb, (c & 63) + half * 16 + mine, g);
      const f32x4_t s = dot_frag<D>(kf, qf);
#pragma unroll
      for (int e = 0; e < 4; ++e) bits |= s[e] > U ? 1u << (half * 16 + 4 * e) : 0u;
    }
    bits <<= g;
    if (c + 32 > have) bits &= (1u << (have - c)) - 1;
    if (!__ballot(bits != 0)) continue;
    unsigned all = bits | lane_xor_u<16>(bits);
    all |= lane_xor_u<32>(all);
    if (!clear) bits = 0;
    while (bits) {
      const unsigned bit = bits & -bits;
      chosen[count + __builtin_popcount(all & (bit - 1))] = c + __builtin_ctz(bits);
      bits ^= bit;
    }
    count += __builtin_popcount(all);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  {
    const int x = lane >> 2;   // four lanes a query
    int* const row = blocks + (((long)b_ * Hq + __shfl(h, x, 64)) * Lq + __shfl((int)i, x, 64)) * top;
    const bool ok = (__ballot(clear && in) >> x) & 1;
    for (int t = lane & 3; ok && t < top; t += 4) row[t] = ((int*)scratch[wave])[x * top + t];
  }
  unsigned long long open = __ballot(!clear && in && g == 0);
  while (open) {   // rows that 32 bits cannot decide
    const int x = __builtin_ctzll(open);
    open &= open - 1;
    const unsigned ri = __builtin_amdgcn_readlane(i, x);
    const int rh = __builtin_amdgcn_readlane(h, x);
    unsigned long long won;
    int taken;
    exact_top<D>(q.p + b_ * q.sb + (long)ri * q.sl + rh * q.sh, kp, have, top, lane, 0, 1, won, taken);
    write_taken(blocks + (((long)b_ * Hq + rh) * Lq + ri) * top, taken, top, lane);
  }
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
  if ((rc = check_strides(who, "q", d->q_stride)) || (rc = check_pool(who, d))) return rc;
  const int G = d->Hq / d->Hkv, n = blocks_of(d), top = d->top;
  const long rows = (long)d->B * d->Hq * d->Lq, shared = (long)d->Lq * G;
  hipStream_t st = (hipStream_t)stream;
  // Every query by itself, or 16 a wave behind the screen (the results are the same). Measured (us, by itself / 16 a wave), 64 features:
  //   2048 queries  top 8 of 64 blocks 12 / 14   top 16 of 256 26 / 43    top 8 of 512 96 / 44   top 16 of 1025 172 / 118
  //    512 queries  top 8 of 64 blocks 12 / 14   top 16 of 256 18 / 43    top 8 of 512 32 / 44   top 16 of 1025 56 / 111
  //   8192 queries  top 8 of 64 blocks 28 / 20   top 16 of 256 74 / 45    top 8 of 512 343 / 62  top 16 of 1025 637 / 173
  // and by itself one wave a query up to 256 blocks, 16 beyond (one query a head, 1025 blocks: 69 us with one, 31 with 16).
  const bool alone = d->pool ? d->pool == 1 : rows <= (n <= EXACT_CHUNK ? 2048 : 1024);
  if (alone) {
    if (n <= EXACT_CHUNK)
      BY_HEAD_DIM(d->D, hipLaunchKernelGGL((block_select_row_kernel<HD, 1>), dm_grid(dm_cdiv(rows, 4)), dim3(256), 0, st, rows_of(q, d->q_stride),
                                           (const bf16_t*)keys, k_len, blocks, d->Lq, d->Lk, d->Hq, G, top, n, rows))
    else
      BY_HEAD_DIM(d->D, hipLaunchKernelGGL((block_select_row_kernel<HD, 16>), dm_grid(rows), dim3(1024), 0, st, rows_of(q, d->q_stride),
                                           (const bf16_t*)keys, k_len, blocks, d->Lq, d->Lk, d->Hq, G, top, n, rows))
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
