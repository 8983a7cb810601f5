// Attention of each query over the key blocks that were chosen for it (64 keys to a block), and its gradients.
//
//   p_it             = softmax over the valid keys t of query i's blocks of scale * q_i . k_t
//   out_i            = sum_t p_it v_t                                       (dm_block_attention_fwd)
//   delta_i          = do_i . out_i,  ds_it = p_it (do_i . v_t - delta_i) scale
//   dq_i = sum_t ds_it k_t,  dk_t = sum_i ds_it q_i,  dv_t = sum_i p_it do_i  (dm_block_attention_bwd)
//
// Query heads share key heads (Hq = G Hkv). The ROWS of a (sample, key head) are its G Lq queries, r = i G + g: they all
// read the same keys and values. delta is taken from out and what out's rounding lost (out_lo): where a query's weight lies on
// few keys, ds is a small difference of do . v and delta, and the rounding of out alone would be as large. No kernel adds with float
// atomics: results do not depend on scheduling.
#include "block_common.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct Args {
  Rows q, k, v;
  const bf16_t *o, *o_lo, *go;   // forward output, what its rounding lost, its gradient: [B][Lq][Hq][D]
  bf16_t *out, *out_lo, *dq, *dk, *dv;
  long dqb, dql, dqh, dkb, dkl, dkh, dvb, dvl, dvh;
  float *lse, *delta;
  const int* blocks;
  const int* k_len;
  const int* offs;             // the plan (block_plan_kernel)
  const unsigned short* rows;
  float* part;                 // of a pool whose blocks are split: its slices' sums, [slice][row of the call][D], and statistics behind
  f32x4_t* part_stat;
  float* key_part;             // of blocks whose rows are split: the slices' dk and dv, [slice][sample, key head][block][2][64][D]
  int B, Lq, Lk, Hq, Hkv, G, top, nblk, pools, slices, row_slices, near;
  float scale;
};

// ---------------------------------------------------------------------------------------------------------------
// NW waves a query: its blocks are dealt to them and their partial results joined through LDS (NW = 4 where a sample has few
// queries, else 1). A block's keys and values are read as whole rows, D/8 lanes a row with 16 bytes each, the next block's
// while this one is computed; the lanes that hold a key's features also hold the same features of its value, so a
// weight never moves between lanes.
// Bound by the latency of a query's chain of blocks where the queries are few (2 x 32 heads with one query, 16 of 1025 blocks of 64
// features: 13 us for 16.8 MB, 1.3 TB/s), by the caches' traffic where they are many, which is where the pools take over.
template <int D, int NW>
__global__ __launch_bounds__(256) void attend_row_kernel(Args a, long rows) {
  constexpr int LPR = D / 8, KPI = 64 / LPR, NI = BLK / KPI;
  __shared__ float so[4][D], sm[4], sl[4];
  const int lane = threadIdx.x & 63, w4 = threadIdx.x >> 6, wave = w4 % NW;
  const long row = dm_block_index() * (4 / NW) + w4 / NW;
  if (row >= rows) return;   // (all of a query's waves)
  const int i = row % a.Lq, h = (row / a.Lq) % a.Hq, b = row / ((long)a.Lq * a.Hq), hk = h / a.G;
  const int n = valid_keys(a.k_len, b, a.Lk);
  const int c = (lane % LPR) * 8, key = lane / LPR;
  const bf16x8_t q = *(const bf16x8_t*)(a.q.p + b * a.q.sb + i * a.q.sl + h * a.q.sh + c);
  const bf16_t* kp = a.k.p + b * a.k.sb + hk * a.k.sh + c;
  const bf16_t* vp = a.v.p + b * a.v.sb + hk * a.v.sh + c;
  const int listed = lane < a.top ? a.blocks[row * a.top + lane] : -1;
  // which of the listed blocks count: in range, with a valid key, and not named before
  bool first = listed >= 0 && listed < a.nblk && listed * BLK < n;
  for (int t = 0; t < a.top - 1; ++t) first = first && !(t < lane && __builtin_amdgcn_readlane(listed, t) == listed);
  unsigned long long todo = __ballot(first);
  if (NW > 1) {   // every NW-th of them
    unsigned long long left = todo, own = 0;
    for (int x = 0; left; ++x) {
      const unsigned long long bit = left & -left;
      if (x % NW == wave) own |= bit;
      left ^= bit;
    }
    todo = own;
  }
  const float sc = a.scale * LOG2E;
  const bf16x8_t none = {};
  bf16x8_t kk[NI], vv[NI];
  auto load = [&](int j) {
#pragma unroll
    for (int u = 0; u < NI; ++u) {
      const int t = u * KPI + key;
      const long pos = (long)j * BLK + t;
      const bool in = j * BLK + t < n;
      kk[u] = in ? *(const bf16x8_t*)(kp + pos * a.k.sl) : none;
      vv[u] = in ? *(const bf16x8_t*)(vp + pos * a.v.sl) : none;
    }
  };
  auto take = [&]() {
    const int t = __builtin_ctzll(todo);
    todo &= todo - 1;
    return __builtin_amdgcn_readlane(listed, t);
  };
  float m = -INFINITY, l = 0.f, o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  int j = -1;
  if (todo) load(j = take());
  while (j >= 0) {
    const int n0 = n - j * BLK;
    float s[NI], mx = m;
#pragma unroll
    for (int u = 0; u < NI; ++u) {
      const float d = group_sum<LPR>(dot8(q, kk[u], 0.f)) * sc;
      s[u] = u * KPI + key < n0 ? d : -INFINITY;
      mx = fmaxf(mx, s[u]);
    }
    bf16x8_t v[NI];
#pragma unroll
    for (int u = 0; u < NI; ++u) v[u] = vv[u];
    j = -1;
    if (todo) load(j = take());
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
      dm_unpack8(v[u], x);
      l += p;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] += p * x[e];
    }
  }
  l = across_sum<LPR>(l);
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = across_sum<LPR>(o[e]);
  if (NW > 1) {
    if (lane < LPR) {
#pragma unroll
      for (int e = 0; e < 8; ++e) so[wave][c + e] = o[e];
    }
    if (lane == 0) { sm[wave] = m; sl[wave] = l; }
    __syncthreads();
    if (wave) return;
    float mt = -INFINITY, f[NW];
#pragma unroll
    for (int w = 0; w < NW; ++w) mt = fmaxf(mt, sm[w]);
    const float base = mt == -INFINITY ? 0.f : mt;
    l = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      f[w] = __builtin_amdgcn_exp2f(sm[w] - base);
      l += sl[w] * f[w];
    }
    m = mt;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      o[e] = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) o[e] += so[w][c + e] * f[w];
    }
  }
  if (lane < LPR) {
    float lo[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = l == 0.f ? 0.f : o[e] / l;
    const bf16x8_t y = dm_pack8(o);
    const long at = (((long)b * a.Lq + i) * a.Hq + h) * D + c;
    *(bf16x8_t*)(a.out + at) = y;
    if (a.out_lo) {
#pragma unroll
      for (int e = 0; e < 8; ++e) lo[e] = o[e] - (float)y[e];
      *(bf16x8_t*)(a.out_lo + at) = dm_pack8(lo);
    }
    if (a.lse && lane == 0) a.lse[row] = l == 0.f ? -INFINITY : m * LN2 + logf(l);
  }
}

// dq of one query a wave, and delta for the kernel behind. Bound by the caches, which every query reads its blocks from (2 x 4 heads x 200
// queries, 16 of 256 blocks of 64 features: 61 us for 419 MB, 6.9 TB/s)
template <int D>
__global__ __launch_bounds__(256) void dq_row_kernel(Args a, long rows) {
  constexpr int LPR = D / 8, KPI = 64 / LPR, NI = BLK / KPI;
  const int lane = threadIdx.x & 63;
  const long row = dm_block_index() * 4 + (threadIdx.x >> 6);
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
// The matrix-core form. A workgroup owns a POOL of 512 rows of one (sample, key head) and visits the blocks that any of
// them chose, in order. The pool's rows that chose a block are packed into tiles of 16, so that a matrix instruction works on 16
// rows that all want the block however the choices are scattered (16 neighbouring rows would share few blocks: with 8 of 64
// chosen at random a tile of neighbours has to visit 56). What a row accumulates (its output and statistics, or its dq) lives in LDS in
// fp32, because the next block packs it into another tile. The rows of one block are disjoint and blocks are separated by
// a barrier, so a row's sums run in block order: the same bits every time.
//
// The lists of rows are made once for all passes (block_plan_kernel). A block's keys and values are staged in LDS for all waves,
// one block ahead. A wave's tiles are a sequence of their own that runs ahead of the visits: while a tile is computed, the rows of the
// wave's next one are on their way from global memory straight into matrix operands, and the row numbers of the one
// behind that.
//
// What bounds it is the latency of a visit: with 8 of 64 blocks a pool has 4 or 5 tiles a visit, one to a wave, so LDS reads, two
// products, 16 exponentials a lane, the write-back and a barrier stand one behind the other (of 1.5 us with 64 features: LDS reads of K 0.17,
// of V and sums 0.16, exponentials 0.15, second product and write-back 0.2, staging and barriers 0.3). 4 x 8 heads of 4096 queries and
// 64 features, 8 of 64 blocks: 95 us, 0.18 PFLOP/s and 0.75 TB/s. Measured and slower: keys fetched straight into
// operands, so that only V needs LDS (134 us against 116 then: every wave gathers the block by 64-byte pieces); two tiles of a wave
// at once (110 against 99: registers, hence fewer waves); 10 or 12 waves a pool (103 .. 105 against 102).
//
// Products are formed transposed, S^T = K Q^T: a lane then holds 4 keys x 4 tiles of ONE row (lane & 15), the row's
// maximum and sum are two lane swaps away, and exp(S^T) is in the register layout that the second product takes as its
// right operand (its left operand, V^T or K^T, is read by transposing LDS reads in the same order of keys).

constexpr int POOL = 512, MAX_SLICES = 8;

// offs[b][hkv][pool][0 .. nblk]: where the rows of a block begin in rows[b][hkv][pool][512 top] (numbers inside the pool,
// ascending). A set: a block that a query names twice counts once, numbers outside 0 .. nblk-1 name none.
// A thread is a row. It sets its bit in the words of its blocks; after the counts' prefix sums a row's place in a block's list is the
// block's start + the bits of earlier words + those of earlier lanes. Four barriers for 256 blocks: 8 us for 256 pools, 8 of 64 blocks.
constexpr int PLAN_CHUNK = 256;   // blocks at a time
__global__ __launch_bounds__(POOL) void block_plan_kernel(const int* __restrict__ blocks, int* __restrict__ offs,
                                                          unsigned short* __restrict__ rows, int Lq, int Hq, int G, int top, int nblk,
                                                          int pools) {
  constexpr int P = POOL, NG = P / 64;
  __shared__ unsigned long long word[NG][PLAN_CHUNK];
  __shared__ int place[NG][PLAN_CHUNK], wsum[4];
  const int pool = blockIdx.x, bh = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int Hkv = Hq / G, b = bh / Hkv, hk = bh - b * Hkv;
  const long r0 = (long)pool * P;
  const bool in = r0 + tid < (long)Lq * G;
  const unsigned r = (unsigned)(r0 + tid), i = G == 1 ? r : r / (unsigned)G;
  const int* const named = blocks + (((long)b * Hq + hk * G + (int)(r - i * (unsigned)G)) * Lq + i) * top;
  int* const of = offs + ((long)bh * pools + pool) * (nblk + 1);
  unsigned short* const out = rows + ((long)bh * pools + pool) * ((long)P * top);
  int base = 0;
  for (int j0 = 0; j0 < nblk; j0 += PLAN_CHUNK) {
    const int n = min(PLAN_CHUNK, nblk - j0);
    for (int e = tid; e < PLAN_CHUNK * NG; e += P) (&word[0][0])[e] = 0;
    __syncthreads();
    if (in) {
#pragma unroll 8
      for (int t = 0; t < top; ++t) {
        const int j = named[t] - j0;
        if (j >= 0 && j < n) atomicOr(&word[wave][j], 1ull << lane);
      }
    }
    __syncthreads();
    int count = 0, before = 0;
    if (tid < PLAN_CHUNK) {
#pragma unroll
      for (int x = 0; x < NG; ++x) count += __builtin_popcountll(word[x][tid]);
      int inc = count;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(inc, o, 64);
        if (lane >= o) inc += up;
      }
      if (lane == 63) wsum[wave] = inc;
      before = inc - count;
    }
    __syncthreads();
    if (tid < PLAN_CHUNK) {
      before += base;
#pragma unroll
      for (int w = 0; w < 3; ++w) before += w < wave ? wsum[w] : 0;
      if (tid < n) of[j0 + tid] = before;
#pragma unroll
      for (int x = 0; x < NG; ++x) {
        place[x][tid] = before;
        before += __builtin_popcountll(word[x][tid]);
      }
    }
    base += wsum[0] + wsum[1] + wsum[2] + wsum[3];
    __syncthreads();
    if (in) {
#pragma unroll 8
      for (int t = 0; t < top; ++t) {
        const int j = named[t] - j0;
        if (j >= 0 && j < n)   // (a block named twice: the same place and row again)
          out[place[wave][j] + __builtin_popcountll(word[wave][j] & ((1ull << lane) - 1))] = (unsigned short)tid;
      }
    }
    __syncthreads();
  }
  if (tid == 0) of[nblk] = base;
}

// The blocks of a pool that more than `least` rows chose, in order: 64 at a time, lane x knows block base + x.
struct Hit { int j, start, n; };   // block (-1: no more), its rows' place in the list, their number
struct Visits {
  const int* offs;
  int nb, lane, base = 0, next0, start = 0, count = 0;
  unsigned long long bits = 0;
  __device__ __forceinline__ Visits(const int* o, int first, int nb_, int lane_) : offs(o), nb(nb_), lane(lane_), next0(first) {}
  __device__ __forceinline__ Hit next(int least) {
    while (__builtin_expect(!bits, 0)) {
      if (next0 >= nb) return Hit{-1, 0, 0};
      base = next0;
      next0 += 64;
      const int j = base + lane, s = j < nb ? offs[j] : 0, e = j < nb ? offs[j + 1] : 0;
      start = s;
      count = e - s;
      bits = __ballot(count > least);
    }
    const int x = __builtin_ctzll(bits);
    bits &= bits - 1;
    return Hit{base + x, __builtin_amdgcn_readlane(start, x), __builtin_amdgcn_readlane(count, x)};
  }
};

// One pool's place, its waves' tiles and the staging of the operand that is read transposed.
template <int D>
struct Pool {
  static constexpr int P = POOL, NW = P / 64;
  static constexpr int PIECES = 2 * BLK * D / 8, PER = (PIECES + P - 1) / P;   // 16-byte pieces of a block's keys and values
  // two buffers where they fit beside what the rows accumulate (all but 512 rows of 64 features)
  static constexpr int KV = 2 * Geo<D>::KV_BYTES, BUFS = P * (Geo<D>::DV * 4 + 24) + 2 * KV <= 160 * 1024 ? 2 : 1;
  struct Tile { int j, start, n, t; };
  const Args& a;
  int bh, b, hk, pool, slice, n, lo, nb, lane, wave, l15, g;   // (blocks lo .. nb - 1 of the pool's are this workgroup's)
  const unsigned short* rows;
  Visits mine;
  bf16x8_t piece[PER];
  const bf16_t* src[PER];   // this thread's pieces of block 0, the distance of a block
  long step[PER];
  int left = 0;             // valid keys from the fetched block on
  // which of keys and values a wave's piece u is of, and whether it has one (the same for all lanes: no branch by lane)
  __device__ __forceinline__ int half(int u) const { return u * P + wave * 64 >= PIECES / 2 ? 1 : 0; }
  static __device__ __forceinline__ int key(int u) {   // the key of piece u (for a sample's last block alone: not kept in a register)
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    return (u * P + tid) % (PIECES / 2) / (D / 8);
  }
  __device__ __forceinline__ bool has(int u) const { return PIECES % P == 0 || u * P + wave * 64 < PIECES; }

  __device__ __forceinline__ Pool(const Args& a_, int bh_, int pool_, int slice_)
      : a(a_), bh(bh_), b(bh_ / a_.Hkv), hk(bh_ - (bh_ / a_.Hkv) * a_.Hkv), pool(pool_), slice(slice_), n(valid_keys(a_.k_len, bh_ / a_.Hkv, a_.Lk)),
        lo(share(n, slice_, a_.slices)), nb(share(n, slice_ + 1, a_.slices)), lane(threadIdx.x & 63),
        wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), l15(threadIdx.x & 15),
        g((threadIdx.x & 63) >> 4), rows(a_.rows + ((long)bh_ * a_.pools + pool_) * ((long)P * a_.top)),
        mine(offsets(a_, bh_, pool_), lo, nb, threadIdx.x & 63) {
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int x = (u * P + threadIdx.x) % (PIECES / 2), t = x / (D / 8), c = x % (D / 8);
      const Rows& r = half(u) ? a.v : a.k;
      src[u] = r.p + b * r.sb + t * r.sl + hk * r.sh + c * 8;
      step[u] = BLK * r.sl;
    }
  }
  static __device__ __forceinline__ int share(int n, int slice, int slices) {   // where a slice's blocks begin
    return (int)((long)((n + BLK - 1) / BLK) * slice / slices);
  }
  static __device__ __forceinline__ const int* offsets(const Args& a, int bh, int pool) {
    return a.offs + ((long)bh * a.pools + pool) * (a.nblk + 1);
  }
  // Block j's keys and values into registers. Behind the valid keys the last one is read, and becomes zeros on its way into LDS: a
  // load that a branch may replace by zeros makes the compiler wait for the loads before it.
  __device__ __forceinline__ void fetch(int j) {
    left = n - j * BLK;
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const bf16_t* at = src[u] + j * step[u];
      if (__builtin_expect(left < BLK, 0)) at -= (long)max(key(u) - (left - 1), 0) * (step[u] / BLK);
      if (has(u)) piece[u] = *(const bf16x8_t*)at;
    }
  }
  __device__ __forceinline__ void stage(char* buf) {   // keys, then values
    const bf16x8_t none = {};
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int x = (u * P + threadIdx.x) % (PIECES / 2), t = x / (D / 8), c = x % (D / 8);
      if (has(u)) {
        if (__builtin_expect(left < BLK, 0)) piece[u] = key(u) < left ? piece[u] : none;
        *(bf16x8_t*)(buf + half(u) * Geo<D>::KV_BYTES + lds_at<D>(t, c)) = piece[u];
        if constexpr (D == 8) *(bf16x8_t*)(buf + half(u) * Geo<D>::KV_BYTES + lds_at<D>(t, 1)) = none;
      }
    }
  }

  // the tile that this wave computes behind `it` (start with Tile{}); j = -1: none
  __device__ __forceinline__ Tile next(const Tile& it) {
    if (__builtin_expect((it.t + NW) * 16 < it.n, 0)) return Tile{it.j, it.start, it.n, it.t + NW};
    const Hit h = mine.next(wave * 16);
    return Tile{h.j, h.start, h.n, wave};
  }
  // A lane's row of a tile. Behind the last one row P, which belongs to nobody: a tile's sums are written back without a
  // branch by lane, so that the compiler may interleave the products of its features.
  __device__ __forceinline__ int row_of(const Tile& it) const {
    const int li = it.t * 16 + l15;
    return li < it.n ? rows[it.start + li] : P;
  }

  __device__ __forceinline__ long row_index(int row) const { return (long)pool * P + row; }
  __device__ __forceinline__ bool inside(int row) const { return row_index(row) < (long)a.Lq * a.G; }
  __device__ __forceinline__ void place(int row, long& i, int& h) const {   // position and head of a row
    const unsigned r = (unsigned)row_index(row), q = a.G == 1 ? r : r / (unsigned)a.G;
    i = q;
    h = hk * a.G + (int)(r - q * a.G);
  }
  // each(e) for the scores of keys n0 and behind. (The place is hidden from the compiler, which would
  // otherwise keep every lane's keys in registers and compare them at every visit, also of whole blocks.)
  template <typename F>
  __device__ __forceinline__ void behind(int n0, F&& each) const {
    if (__builtin_expect(n0 < BLK, 0)) {
      int mine0 = n0 - g * 4;
      asm volatile("" : "+v"(mine0));
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if ((e >> 2) * 16 + (e & 3) >= mine0) each(e);
    }
  }
  // a row's place in a [..][positions][heads][D] tensor, in units of 8 features from the sample's first (0 behind the last row)
  __device__ __forceinline__ unsigned offset(int row, long sl, long sh) const {
    if (!inside(row)) return 0;
    long i;
    int h;
    place(row, i, h);
    return (unsigned)i * (unsigned)(sl >> 3) + (unsigned)h * (unsigned)(sh >> 3);
  }
};

// Workgroup `id` of `each` to a (sample, key head): which one, and which of its `each`. The workgroups of a head go to one XCD, whose L2
// then holds its keys and values, and so do those of `near` neighbouring heads, side by side: narrow heads share cache lines (8 of
// 8 features in 128 bytes), which 8 XCDs would otherwise fetch once each (8 x 64 heads of 1024 queries and 8 features: dq 125 -> 87 us).
__device__ __forceinline__ bool head_of_block(const Args& a, long id, int each, int& bh, int& part) {
  const int nbh = a.B * a.Hkv, units = nbh / a.near, wide = each * a.near;
  long unit, in;
  if ((units & 7) == 0) {
    const long local = id >> 3;
    unit = local / wide * 8 + (id & 7);
    in = local % wide;
  } else {
    unit = id / wide;
    in = id % wide;
  }
  part = (int)(in / a.near);
  bh = (int)(unit * a.near + in % a.near);
  return unit < units;
}
__device__ __forceinline__ bool pool_of_block(const Args& a, int& bh, int& pool, int& slice) {
  if (!head_of_block(a, blockIdx.x, a.pools * a.slices, bh, pool)) return false;
  slice = a.slices == 1 ? 0 : pool / a.pools;
  pool -= slice * a.pools;
  return true;
}
// where a slice's sums of a row begin (`row` counts the call's rows: (sample, position, head))
__device__ __forceinline__ long part_row(const Args& a, int slice, long row) { return (long)slice * ((long)a.B * a.Lq * a.Hq) + row; }

// 8 features of a row's output, what their rounding lost and the row's statistic, from its sums f and its `stat`
template <int D>
__device__ __forceinline__ void write_out(const Args& a, float (&f)[8], const f32x4_t& st, long row, int c, long lrow) {
  const float inv = 1.0f / st[2];
#pragma unroll
  for (int x = 0; x < 8; ++x) f[x] = st[2] == 0.f ? 0.f : f[x] * inv;
  const bf16x8_t y = dm_pack8(f);
  *(bf16x8_t*)(a.out + row * D + c * 8) = y;
  if (a.out_lo) {
#pragma unroll
    for (int x = 0; x < 8; ++x) f[x] -= (float)y[x];
    *(bf16x8_t*)(a.out_lo + row * D + c * 8) = dm_pack8(f);
  }
  if (a.lse && c == 0) a.lse[lrow] = st[2] == 0.f ? -INFINITY : st[0] * LN2 + logf(st[1]);
}

// KEEP: for a backward call. The weights are the matrix instruction's operands in bf16: for an output alone rounded, and the output is
// divided by the sum of the ROUNDED weights (one more product, with ones), so that it stays an average of values and a rounding
// counts only with the value's distance from the output. With KEEP as a pair, the rounded weight and what the rounding lost (2^-17),
// and the output is divided by the weights' own sum: delta is taken from it, and would pass its error on to every ds of the row (111 us
// for the call above).
template <int D, bool KEEP>
__global__ __launch_bounds__(POOL, D == 8 ? 5 : D == 16 ? 6 : 2) void attend_pool_kernel(Args a) {
  using GE = Geo<D>;
  using PL = Pool<D>;
  constexpr int P = POOL;
  __shared__ __attribute__((aligned(16))) char kv[PL::BUFS][PL::KV];
  __shared__ __attribute__((aligned(16))) float acc[(P + 1) * GE::DV];
  __shared__ __attribute__((aligned(16))) f32x4_t stat[P + 1];   // maximum, sum of the weights (KEEP), what the output is divided by
  __shared__ unsigned rowoff[P + 1];
  int bh, pool, slice;
  if (!pool_of_block(a, bh, pool, slice)) return;
  PL w(a, bh, pool, slice);
  const int tid = threadIdx.x, lane = w.lane, g = w.g;
  const float sc = a.scale * LOG2E, asc = fabsf(sc);   // (the sign of the scale goes to q: a maximum is scaled by the amount)
  const bf16_t one = (bf16_t)1.f;
  const bf16x8_t ones = {one, one, one, one, one, one, one, one};
  const f32x4_t zero4 = {0.f, 0.f, 0.f, 0.f};
  Visits visits(PL::offsets(a, bh, pool), w.lo, w.nb, lane);
  Hit cur = visits.next(0);
  if (cur.j >= 0) {
    w.fetch(cur.j);
    w.stage(kv[0]);
  }
  for (int e = tid; e < P * GE::OC; e += P) *(f32x4_t*)(acc + e * 4) = zero4;
  rowoff[tid] = w.offset(tid, a.q.sl, a.q.sh);
  stat[tid] = f32x4_t{-INFINITY, 0.f, 0.f, 0.f};
  if (tid < GE::OC) *(f32x4_t*)(acc + (P * GE::OC + tid) * 4) = zero4;
  if (tid == 0) {
    rowoff[P] = 0;
    stat[P] = zero4;
  }
  __syncthreads();

  const bf16_t* const qbase = a.q.p + w.b * a.q.sb;
  Frag<D> qf;
  typename PL::Tile it = w.next(typename PL::Tile{}), it1 = w.next(it);
  int row = w.row_of(it), row1 = w.row_of(it1);
  qf.load(qbase + (size_t)rowoff[row] * 8, g);
  qf.arrived();
  int buf = 0;
  while (cur.j >= 0) {
    const Hit nxt = visits.next(0);
    if (nxt.j >= 0) w.fetch(nxt.j);
    const char *const kb = kv[buf], *const vb = kb + GE::KV_BYTES;
    while (it.j == cur.j) {
      const unsigned off1 = rowoff[row1];   // (LDS answers in order: asked for behind the reads below, the next rows would go out late)
      Frag<D> kf[4];
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) kf[kt].from_lds(kb, kt * 16 + w.l15, g);
      const typename PL::Tile it2 = w.next(it1);
      const int row2 = w.row_of(it2);
      if (sc < 0.f) qf.negate();
      __builtin_amdgcn_sched_barrier(0);
      float s[16];
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) *(f32x4_t*)(s + kt * 4) = dot_frag<D>(kf[kt], qf);
      // the next tile's rows and what this one reads from LDS are under way before the softmax
      qf.load(qbase + (size_t)off1 * 8, g);
      f32x4_t st = stat[row], o[GE::DT];
      bf16x4_t vt[GE::DT][4];
#pragma unroll
      for (int dt = 0; dt < GE::DT; ++dt) {
        o[dt] = *(const f32x4_t*)(acc + acc_at<D>(row, dt * 4 + g));
#pragma unroll
        for (int u = 0; u < 4; ++u) vt[dt][u] = read_tr<D>(vb, u * 16, dt, lane);
      }
      __builtin_amdgcn_sched_barrier(0);
      const int n0 = w.n - cur.j * BLK;   // valid keys from this block on
      w.behind(n0, [&](int e) { s[e] = -INFINITY; });
      float mx[4];
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) mx[kt] = fmaxf(fmaxf(s[kt * 4], s[kt * 4 + 1]), fmaxf(s[kt * 4 + 2], s[kt * 4 + 3]));
      const float m_new = fmaxf(st[0], row_max(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]))) * asc), at = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = __builtin_amdgcn_exp2f(st[0] - at);
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(s[e] * asc - at);
      w.behind(n0, [&](int e) { s[e] = 0.f; });   // (a scale of zero times -infinity is no zero)
      float sum = 0.f;
      if (KEEP) {
        float part[4];
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) part[kt] = (s[kt * 4] + s[kt * 4 + 1]) + (s[kt * 4 + 2] + s[kt * 4 + 3]);
        sum = st[1] * alpha + row_sum((part[0] + part[1]) + (part[2] + part[3]));
      }
      bf16x8_t p[2], lost[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        p[u] = dm_pack8(s + u * 8);
        if (KEEP) {
#pragma unroll
          for (int e = 0; e < 8; ++e) s[u * 8 + e] -= (float)p[u][e];
          lost[u] = dm_pack8(s + u * 8);
        }
      }
      const float r_old = st[2] * alpha;
      f32x4_t rs = {r_old, r_old, r_old, r_old};
#pragma unroll
      for (int dt = 0; dt < GE::DT; ++dt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[dt][e] *= alpha;
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int dt = 0; dt < GE::DT; ++dt) {
          const bf16x8_t values = join4(vt[dt][2 * u], vt[dt][2 * u + 1]);
          o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(values, p[u], o[dt], 0, 0, 0);
          if (KEEP) o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(values, lost[u], o[dt], 0, 0, 0);
        }
        if (!KEEP) rs = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, p[u], rs, 0, 0, 0);
      }
#pragma unroll
      for (int dt = 0; dt < GE::DT; ++dt) *(f32x4_t*)(acc + acc_at<D>(row, dt * 4 + g)) = o[dt];
      stat[row] = f32x4_t{m_new, sum, KEEP ? sum : rs[0], 0.f};   // (four lanes, the same values)
      it = it1;
      row = row1;
      it1 = it2;
      row1 = row2;
      qf.arrived();
    }
    if (PL::BUFS == 2) buf ^= 1;
    else __syncthreads();
    if (nxt.j >= 0) w.stage(kv[buf]);
    __syncthreads();
    cur = nxt;
  }
  constexpr int PC = D / 8;
  for (int e = tid; e < P * PC; e += P) {
    const int r = e / PC, c = e % PC;
    if (!w.inside(r)) break;
    long i;
    int h;
    w.place(r, i, h);
    const f32x4_t st = stat[r];
    float f[8];
    *(f32x4_t*)f = *(const f32x4_t*)(acc + acc_at<D>(r, c * 2));
    *(f32x4_t*)(f + 4) = *(const f32x4_t*)(acc + acc_at<D>(r, c * 2 + 1));
    const long at = ((long)w.b * a.Lq + i) * a.Hq + h;
    if (a.slices == 1) {
      write_out<D>(a, f, st, at, c, ((long)w.b * a.Hq + h) * a.Lq + i);
    } else {
      const long p = part_row(a, w.slice, at);
      *(f32x4_t*)(a.part + p * D + c * 8) = *(const f32x4_t*)f;
      *(f32x4_t*)(a.part + p * D + c * 8 + 4) = *(const f32x4_t*)(f + 4);
      if (c == 0) a.part_stat[p] = st;
    }
  }
}

// The slices of a split pool become one: their sums, brought to a common maximum, in the order of the slices. (4 or 5 us for 13320 rows
// of 32 features, 8 slices: 17 MB, 3.4 TB/s.)
template <int D>
__global__ __launch_bounds__(256) void attend_join_kernel(Args a) {
  constexpr int PC = D / 8;
  const long e = dm_block_index() * 256 + threadIdx.x, at = e / PC;
  const int c = (int)(e % PC);
  if (at >= (long)a.B * a.Lq * a.Hq) return;
  f32x4_t st[MAX_SLICES];
  float m = -INFINITY;
#pragma unroll
  for (int s = 0; s < MAX_SLICES; ++s)
    if (s < a.slices) st[s] = a.part_stat[part_row(a, s, at)];
#pragma unroll
  for (int s = 0; s < MAX_SLICES; ++s)
    if (s < a.slices) m = fmaxf(m, st[s][0]);
  const float base = m == -INFINITY ? 0.f : m;
  float f[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  f32x4_t all = {m, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < MAX_SLICES; ++s)
    if (s < a.slices) {
      const float* p = a.part + part_row(a, s, at) * D + c * 8;
      const f32x4_t x = *(const f32x4_t*)p, y = *(const f32x4_t*)(p + 4);
      const float by = __builtin_amdgcn_exp2f(st[s][0] - base);
      all[1] += st[s][1] * by;
      all[2] += st[s][2] * by;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        f[k] += x[k] * by;
        f[k + 4] += y[k] * by;
      }
    }
  const long h = at % a.Hq, i = at / a.Hq % a.Lq, b = at / ((long)a.Hq * a.Lq);
  write_out<D>(a, f, all, at, c, (b * a.Hq + h) * a.Lq + i);
}
template <int D>
__global__ __launch_bounds__(256) void dq_join_kernel(Args a) {
  constexpr int PC = D / 8;
  const long e = dm_block_index() * 256 + threadIdx.x, at = e / PC;
  const int c = (int)(e % PC);
  if (at >= (long)a.B * a.Lq * a.Hq) return;
  float f[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int s = 0; s < MAX_SLICES; ++s)
    if (s < a.slices) {
      const float* p = a.part + part_row(a, s, at) * D + c * 8;
      const f32x4_t x = *(const f32x4_t*)p, y = *(const f32x4_t*)(p + 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        f[k] += x[k];
        f[k + 4] += y[k];
      }
    }
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] *= a.scale;
  const long h = at % a.Hq, i = at / a.Hq % a.Lq, b = at / ((long)a.Hq * a.Lq);
  *(bf16x8_t*)(a.dq + b * a.dqb + i * a.dql + h * a.dqh + c * 8) = dm_pack8(f);
}

// dq of a pool, and delta for the kernel behind. dq gathers p (dp - delta) k; the scale is applied once at the end. Bound as the
// forward kernel is, with one product more in a visit (the call above: 117 us).
template <int D>
__global__ __launch_bounds__(POOL) void dq_pool_kernel(Args a) {
  using GE = Geo<D>;
  using PL = Pool<D>;
  constexpr int P = POOL;
  __shared__ __attribute__((aligned(16))) char kv[PL::BUFS][PL::KV];
  __shared__ __attribute__((aligned(16))) float acc[(P + 1) * GE::DV];
  __shared__ f32x2_t stat[P + 1];   // lse, -delta (the products of do and v start from it)
  __shared__ unsigned rowoff[P + 1], gooff[P + 1];
  int bh, pool, slice;
  if (!pool_of_block(a, bh, pool, slice)) return;
  PL w(a, bh, pool, slice);
  const int tid = threadIdx.x, lane = w.lane, g = w.g;
  const float sc = a.scale * LOG2E;
  const f32x4_t zero4 = {0.f, 0.f, 0.f, 0.f};
  Visits visits(PL::offsets(a, bh, pool), w.lo, w.nb, lane);
  Hit cur = visits.next(0);
  if (cur.j >= 0) {
    w.fetch(cur.j);
    w.stage(kv[0]);
  }
  for (int e = tid; e < P * GE::OC; e += P) *(f32x4_t*)(acc + e * 4) = zero4;
  rowoff[tid] = w.offset(tid, a.q.sl, a.q.sh);
  gooff[tid] = w.offset(tid, (long)a.Hq * D, D);
  if (tid < GE::OC) *(f32x4_t*)(acc + (P * GE::OC + tid) * 4) = zero4;
  if (tid == 0) {
    rowoff[P] = gooff[P] = 0;
    stat[P] = f32x2_t{INFINITY, 0.f};
  }
  constexpr int PC = D / 8;
  for (int e = tid; e < P * PC; e += P) {   // (a row's PC lanes are neighbours: P is a multiple of PC)
    const int r = e / PC, c = e % PC;
    const bool in = w.inside(r);
    long i = 0;
    int h = 0;
    if (in) w.place(r, i, h);
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
      stat[r] = f32x2_t{lse == -INFINITY ? INFINITY : lse * LOG2E, -delta};   // no key: every weight becomes zero
      if (in && w.slice == 0) a.delta[lrow] = delta;
    }
  }
  __syncthreads();

  const bf16_t* const qbase = a.q.p + w.b * a.q.sb;
  const bf16_t* const obase = a.go + (long)w.b * a.Lq * a.Hq * D;
  Frag<D> qf, of;
  auto load = [&](unsigned at_q, unsigned at_o) {
    qf.load(qbase + (size_t)at_q * 8, g);
    of.load(obase + (size_t)at_o * 8, g);
  };
  auto arrived = [&]() {
    qf.arrived();
    of.arrived();
  };
  typename PL::Tile it = w.next(typename PL::Tile{}), it1 = w.next(it);
  int row = w.row_of(it), row1 = w.row_of(it1);
  load(rowoff[row], gooff[row]);
  arrived();
  int buf = 0;
  while (cur.j >= 0) {
    const Hit nxt = visits.next(0);
    if (nxt.j >= 0) w.fetch(nxt.j);
    const char *const kb = kv[buf], *const vb = kb + GE::KV_BYTES;
    while (it.j == cur.j) {
      const unsigned off1 = rowoff[row1], off2 = gooff[row1];   // (first, as in the forward kernel)
      const f32x2_t st = stat[row];
      Frag<D> kf[4], vf[4];
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) {
        kf[kt].from_lds(kb, kt * 16 + w.l15, g);
        vf[kt].from_lds(vb, kt * 16 + w.l15, g);
      }
      const typename PL::Tile it2 = w.next(it1);
      const int row2 = w.row_of(it2);
      __builtin_amdgcn_sched_barrier(0);
      f32x4_t s[4], dp[4];
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) {
        s[kt] = dot_frag<D>(kf[kt], qf);
        dp[kt] = dot_frag<D>(vf[kt], of, f32x4_t{st[1], st[1], st[1], st[1]});
      }
      load(off1, off2);
      f32x4_t o[GE::DT];
      bf16x4_t tr[GE::DT][4];
#pragma unroll
      for (int dt = 0; dt < GE::DT; ++dt) {
        o[dt] = *(const f32x4_t*)(acc + acc_at<D>(row, dt * 4 + g));
#pragma unroll
        for (int u = 0; u < 4; ++u) tr[dt][u] = read_tr<D>(kb, u * 16, dt, lane);
      }
      __builtin_amdgcn_sched_barrier(0);
      float ds[16];
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) ds[kt * 4 + e] = __builtin_amdgcn_exp2f(s[kt][e] * sc - st[0]) * dp[kt][e];
      w.behind(w.n - cur.j * BLK, [&](int e) { ds[e] = 0.f; });
      // ds sums to zero over a row's keys, so what its keys have in common cancels in dq: rounded to bf16 it would not, by 2^-9 of
      // the common part. Two bf16 operands, the rounded ds and what the rounding lost, keep 2^-17.
      bf16x8_t p[2], lost[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        p[u] = dm_pack8(ds + u * 8);
#pragma unroll
        for (int e = 0; e < 8; ++e) ds[u * 8 + e] -= (float)p[u][e];
        lost[u] = dm_pack8(ds + u * 8);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int dt = 0; dt < GE::DT; ++dt) {
          const bf16x8_t keys = join4(tr[dt][2 * u], tr[dt][2 * u + 1]);
          o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(keys, p[u], o[dt], 0, 0, 0);
          o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(keys, lost[u], o[dt], 0, 0, 0);
        }
#pragma unroll
      for (int dt = 0; dt < GE::DT; ++dt) *(f32x4_t*)(acc + acc_at<D>(row, dt * 4 + g)) = o[dt];
      it = it1;
      row = row1;
      it1 = it2;
      row1 = row2;
      arrived();
    }
    if (PL::BUFS == 2) buf ^= 1;
    else __syncthreads();
    if (nxt.j >= 0) w.stage(kv[buf]);
    __syncthreads();
    cur = nxt;
  }
  for (int e = tid; e < P * PC; e += P) {
    const int r = e / PC, c = e % PC;
    if (!w.inside(r)) break;
    long i;
    int h;
    w.place(r, i, h);
    float f[8];
    *(f32x4_t*)f = *(const f32x4_t*)(acc + acc_at<D>(r, c * 2));
    *(f32x4_t*)(f + 4) = *(const f32x4_t*)(acc + acc_at<D>(r, c * 2 + 1));
    if (a.slices == 1) {
#pragma unroll
      for (int x = 0; x < 8; ++x) f[x] *= a.scale;
      *(bf16x8_t*)(a.dq + w.b * a.dqb + i * a.dql + h * a.dqh + c * 8) = dm_pack8(f);
    } else {
      float* p = a.part + part_row(a, w.slice, ((long)w.b * a.Lq + i) * a.Hq + h) * D + c * 8;
      *(f32x4_t*)p = *(const f32x4_t*)f;
      *(f32x4_t*)(p + 4) = *(const f32x4_t*)(f + 4);
    }
  }
}

__device__ __forceinline__ void write_keys(const Args& a, float (&dk)[8], const float (&dv)[8], int b, int hk, long pos, int d) {
#pragma unroll
  for (int x = 0; x < 8; ++x) dk[x] *= a.scale;
  *(bf16x8_t*)(a.dk + b * a.dkb + pos * a.dkl + hk * a.dkh + d) = dm_pack8(dk);
  *(bf16x8_t*)(a.dv + b * a.dvb + pos * a.dvl + hk * a.dvh + d) = dm_pack8(dv);
}

// dk and dv of one block, four waves. The rows that chose it are packed into a list, 4096 rows at a time, and dealt to the
// waves in tiles of 32; every wave sums all 64 keys over its own rows in registers, and the four sums are added in wave
// order. Scores are formed as S = Q K^T here: a lane holds 4 rows x 2 tiles of ONE key, which is the layout that dv =
// P^T dO and dk = dS^T Q take as their left operand; the right operands are the tile's rows, read transposed from the wave's own LDS.
// Bound by registers with 64 features (the sums of 64 keys take 128; 2 waves a SIMD) and by the latency of a tile's chain: 121 us for 4 x 8
// heads of 4096 queries and keys, 8 of 64 blocks, 0.43 PFLOP/s issued; 107 us for 8 x 64 heads of 1024 and 8 features, 4 of 16. (p and
// ds rounded once: 107 and 87 us. Pairs with 32 keys at a time: 148 and 138, registers spilled.) Where blocks are few, their rows are dealt
// to up to 8 workgroups, pool by pool, and joined by dkv_join_kernel (row_slices_of).
constexpr int LIST = 4096;
template <int D>
__global__ __launch_bounds__(256, D <= 16 ? 4 : D == 32 ? 3 : 2) void dkv_kernel(Args a) {
  using GE = Geo<D>;
  constexpr int TILE_BYTES = 32 * GE::ROWB;
  __shared__ __attribute__((aligned(16))) char kbuf[GE::KV_BYTES], vbuf[GE::KV_BYTES];
  __shared__ __attribute__((aligned(16))) char rows[4][2][TILE_BYTES];    // q and do of a wave's tile; at the end the sums
  __shared__ __attribute__((aligned(16))) float stat[4][2][32];           // lse, -delta
  __shared__ unsigned short list[LIST];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4;
  int j, bh;
  if (!head_of_block(a, dm_block_index(), a.nblk * a.row_slices, bh, j)) return;
  const int slice = j / a.nblk, p_first = (int)((long)a.pools * slice / a.row_slices), p_end = (int)((long)a.pools * (slice + 1) / a.row_slices);
  j -= slice * a.nblk;
  const int b = bh / a.Hkv, hk = bh - b * a.Hkv;
  const int n0 = valid_keys(a.k_len, b, a.Lk) - j * BLK;
  const float sc = a.scale * LOG2E;
  // The chain of loads at the start (where the block's rows lie in the lists, the rows, their q and do) and the keys and values
  // beside it decide the time of a short list: the first one goes out first.
  constexpr int per = LIST / POOL;    // pools whose rows fit the list
  int start = 0, own = 0;
  auto find = [&](int p0) {           // lane x: the rows of pool p0 + x
    const bool has = lane < per && p0 + lane < p_end;
    const int* at = a.offs + ((long)bh * a.pools + p0 + lane) * (a.nblk + 1) + j;
    start = has ? at[0] : 0;
    own = has ? at[1] - start : 0;
  };
  if (n0 > 0) {
    find(p_first);
    constexpr int PER = (2 * BLK * D / 8 + 255) / 256;
    const bf16x8_t none = {};
    bf16x8_t x[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int e = u * 256 + tid, half = e >= BLK * D / 8 ? 1 : 0, p = e - half * (BLK * D / 8), t = p / (D / 8), c = p % (D / 8);
      const Rows& s = half ? a.v : a.k;
      x[u] = e < 2 * BLK * D / 8 && t < n0 ? *(const bf16x8_t*)(s.p + b * s.sb + ((long)j * BLK + t) * s.sl + hk * s.sh + c * 8) : none;
    }
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int e = u * 256 + tid, half = e >= BLK * D / 8 ? 1 : 0, p = e - half * (BLK * D / 8), t = p / (D / 8), c = p % (D / 8);
      char* to = half ? vbuf : kbuf;
      if (e < 2 * BLK * D / 8) {
        *(bf16x8_t*)(to + lds_at<D>(t, c)) = x[u];
        if constexpr (D == 8) *(bf16x8_t*)(to + lds_at<D>(t, 1)) = none;
      }
    }
  }
  f32x4_t dk[4][GE::DT], dv[4][GE::DT];
#pragma unroll
  for (int kt = 0; kt < 4; ++kt)
#pragma unroll
    for (int dt = 0; dt < GE::DT; ++dt) dk[kt][dt] = dv[kt][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const unsigned q8l = (unsigned)(a.q.sl >> 3), q8h = (unsigned)(a.q.sh >> 3);
  const bf16_t *const qbase = a.q.p + b * a.q.sb, *const obase = a.go + (long)b * a.Lq * a.Hq * D;
  const float *const lbase = a.lse + (long)b * a.Hq * a.Lq, *const dbase = a.delta + (long)b * a.Hq * a.Lq;
  char *qb = rows[wave][0], *ob = rows[wave][1];
  float *st_lse = stat[wave][0], *st_delta = stat[wave][1];
  for (int p0 = p_first; p0 < p_end && n0 > 0; p0 += per) {
    if (p0 > p_first) find(p0);
    int inc = own;
#pragma unroll
    for (int o = 1; o < per; o <<= 1) {
      const int up = __shfl_up(inc, o, 64);
      if (lane >= o) inc += up;
    }
    const int count = __builtin_amdgcn_readlane(inc, per - 1), before = inc - own;
    __syncthreads();   // the list's last use is over
    for (int x = wave; x < per && p0 + x < p_end; x += 4) {
      const int s = __builtin_amdgcn_readlane(start, x), m = __builtin_amdgcn_readlane(own, x), to = __builtin_amdgcn_readlane(before, x);
      const unsigned short* from = a.rows + ((long)bh * a.pools + p0 + x) * ((long)POOL * a.top) + s;
      for (int e = lane; e < m; e += 64) list[to + e] = (unsigned short)(x * POOL + from[e]);
    }
    __syncthreads();
    // a lane's two rows of a tile, 16 mt + (lane & 15), as operands; behind the last row zeros, with a weight of zero
    Frag<D> qf[2], of[2];
    float lse[2], delta[2];
    auto load = [&](int t) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const int li = t * 32 + mt * 16 + (lane & 15);
        qf[mt].zero();
        of[mt].zero();
        lse[mt] = -INFINITY;
        delta[mt] = 0.f;
        if (li < count) {
          const unsigned r = (unsigned)(p0 * POOL + list[li]);
          const unsigned i = a.G == 1 ? r : r / (unsigned)a.G;
          const int h = hk * a.G + (int)(r - i * a.G);
          // (32-bit places inside the sample, in units of 8 features: check_span)
          qf[mt].load(qbase + (size_t)(i * q8l + (unsigned)h * q8h) * 8, g);
          of[mt].load(obase + (size_t)((i * (unsigned)a.Hq + (unsigned)h) * (D / 8)) * 8, g);
          const unsigned at = (unsigned)h * (unsigned)a.Lq + i;
          lse[mt] = lbase[at];
          delta[mt] = dbase[at];
        }
      }
    };
    if (wave * 32 < count) load(wave);
    for (int t = wave; t * 32 < count; t += 4) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const int row = mt * 16 + (lane & 15);
        if (g == 0) {
          st_lse[row] = lse[mt] == -INFINITY ? INFINITY : lse[mt] * LOG2E;   // (also a row without a key: every weight is zero)
          st_delta[row] = -delta[mt];
        }
        qf[mt].to_lds(qb, row, g);
        of[mt].to_lds(ob, row, g);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the wave's own writes, read by its other lanes
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) {   // 16 keys at a time (more would not leave registers for the next rows)
        Frag<D> kf, vf;
        kf.from_lds(kbuf, kt * 16 + (lane & 15), g);
        vf.from_lds(vbuf, kt * 16 + (lane & 15), g);
        float p[8], ds[8];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          const f32x4_t ls = *(const f32x4_t*)(st_lse + mt * 16 + g * 4), de = *(const f32x4_t*)(st_delta + mt * 16 + g * 4);
          const f32x4_t s = dot_frag<D>(qf[mt], kf), dp = dot_frag<D>(of[mt], vf, de);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            p[mt * 4 + e] = __builtin_amdgcn_exp2f(s[e] * sc - ls[e]);
            ds[mt * 4 + e] = p[mt * 4 + e] * dp[e];
          }
        }
        if (kt == 3 && (t + 4) * 32 < count) load(t + 4);   // on its way during the last products
        // p and ds as pairs of operands, rounded to bf16 and what that lost: weights of one size are rounded one way in every row, an error
        // that their sum over rows would keep
        const bf16x8_t ph = dm_pack8(p), dh = dm_pack8(ds);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          p[e] -= (float)ph[e];
          ds[e] -= (float)dh[e];
        }
        const bf16x8_t pl = dm_pack8(p), dl = dm_pack8(ds);
#pragma unroll
        for (int dt = 0; dt < GE::DT; ++dt) {
          const bf16x8_t qt = join4(read_tr<D>(qb, 0, dt, lane), read_tr<D>(qb, 16, dt, lane));
          const bf16x8_t ot = join4(read_tr<D>(ob, 0, dt, lane), read_tr<D>(ob, 16, dt, lane));
          dv[kt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ph, ot, dv[kt][dt], 0, 0, 0);
          dk[kt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(dh, qt, dk[kt][dt], 0, 0, 0);
          dv[kt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pl, ot, dv[kt][dt], 0, 0, 0);
          dk[kt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(dl, qt, dk[kt][dt], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);   // (the next keys' products would be begun before these are done, and spill)
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }
  // The four waves' sums in a fixed order, dk beginning with wave 0 and dv with wave 2 so that two waves work at a time, in the tiles'
  // memory (4 x 2 x 32 rows hold the 64 keys twice in fp32) and in the order of the accumulator registers.
  float* const sum = (float*)&rows[0][0][0];
  constexpr int HALF = BLK * GE::DV;
  auto add = [&](float* to, const f32x4_t (&x)[4][GE::DT], bool first) {
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int dt = 0; dt < GE::DT; ++dt) {
        f32x4_t* at = (f32x4_t*)(to + ((kt * GE::DT + dt) * 64 + lane) * 4);
        *at = first ? x[kt][dt] : *at + x[kt][dt];
      }
  };
#pragma unroll 1
  for (int x = 0; x < 4; ++x) {
    __syncthreads();
    if (wave == x) add(sum, dk, x == 0);
    if (wave == (x ^ 2)) add(sum + HALF, dv, x == 0);
  }
  __syncthreads();
  const int in = min(BLK, a.Lk - j * BLK);
  for (int e = tid; e < BLK * D / 8; e += 256) {
    const int t = e / (D / 8), d = (e % (D / 8)) * 8;
    if (t >= in) break;
    const long pos = (long)j * BLK + t;
    const bool live = t < n0;   // positions behind the last valid key: zero
    const int place = (((t >> 4) * GE::DT + (d >> 4)) * 64 + ((t >> 2) & 3) * 16 + (d & 15)) * 4 + (t & 3);
    float f[8], h[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      f[x] = live ? sum[place + x * 4] : 0.f;
      h[x] = live ? sum[HALF + place + x * 4] : 0.f;
    }
    if (a.row_slices == 1) {
      write_keys(a, f, h, b, hk, pos, d);
    } else {
      float* to = a.key_part + ((((long)slice * a.B * a.Hkv + bh) * a.nblk + j) * 2 * BLK + t) * D + d;
      *(f32x4_t*)to = *(const f32x4_t*)f;
      *(f32x4_t*)(to + 4) = *(const f32x4_t*)(f + 4);
      *(f32x4_t*)(to + BLK * D) = *(const f32x4_t*)h;
      *(f32x4_t*)(to + BLK * D + 4) = *(const f32x4_t*)(h + 4);
    }
  }
}

// dk and dv of blocks whose rows were split, in the order of the slices
template <int D>
__global__ __launch_bounds__(256) void dkv_join_kernel(Args a) {
  constexpr int PC = D / 8;
  const long e = dm_block_index() * 256 + threadIdx.x, at = e / PC;   // (sample, key head), key
  const int d = (int)(e % PC) * 8;
  const long bh = at / a.Lk, pos = at - bh * a.Lk;
  if (bh >= (long)a.B * a.Hkv) return;
  float f[8] = {0, 0, 0, 0, 0, 0, 0, 0}, h[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int s = 0; s < MAX_SLICES; ++s)
    if (s < a.row_slices) {
      const float* p = a.key_part + ((((long)s * a.B * a.Hkv + bh) * a.nblk + pos / BLK) * 2 * BLK + pos % BLK) * D + d;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        f[k] += p[k];
        h[k] += p[BLK * D + k];
      }
    }
  write_keys(a, f, h, (int)(bh / a.Hkv), (int)(bh % a.Hkv), pos, d);
}

// rows are addressed inside a sample by 32-bit numbers of 8 features
int check_span(const char* who, const dm_block_desc* d) {
  const long* s = d->q_stride;
  for (int i = 0; i < 3; ++i) DM_REQUIRE(s[i] >= 0, DM_ERR_ARG, "%s: negative stride of q", who);
  DM_REQUIRE((d->Lq - 1) * s[1] + (d->Hq - 1) * s[2] < (1L << 35) && (long)d->Lq * d->Hq * d->D < (1L << 35), DM_ERR_SHAPE,
             "%s: a sample of q spans more than 2^35 elements", who);
  return check_pool(who, d);
}
// Whether the rows are taken in pools on the matrix cores or one query a workgroup, and in how many slices a pool's blocks are dealt to
// workgroups (joined by attend_join_kernel and dq_join_kernel) where pools alone would leave CUs idle. A pool's time is the
// number of its visits (its blocks) times what a visit takes from barrier to barrier, however few rows want the block: 0.9 us up to
// 16 features, 1.05 us with 32, 1.5 us with 64 (256 pools run at a time, twice as many up to 16 features); a slice's sums cross
// memory twice (3 TB/s); a query's time is 0.3 ns + 0.5 .. 0.8 ns a block over the whole chip, a quarter less where little of it is
// in use. Measured, a forward call on its own (us): one query a workgroup / pools unsplit / as the rule splits them
//   8 heads x 256 queries, 8 of 64 blocks       D 8  16 / 57 / 25       D 64  25 / 84 / 28
//   4 x 8 heads x 256 queries, 8 of 64          D 8  40 / 57 / 27       D 64  74 / 85 / 31
//   4 x 8 heads x 1024 queries, 4 of 16         D 8  70 / 28 / 28       D 64  132 / 41 / 40
//   2 x 8 heads x 2048 queries, 8 of 128        D 8  139 / 103 / 44     D 64  243 / 160 / 91
//   4 x 8 heads x 4096 queries, 8 of 64         D 8  507 / 66 / 58      D 64  893 / 103 / 95
//   2 heads of 4 x 200 queries, 16 of 256       D 8  15 / 191 / 45      D 64  41 / 309 / 57
// (Pools of 128 and 256 rows, which occupy more CUs where there are few rows, were never faster by more than 5 %.)
struct Form { bool pool; int slices; };
Form form_of(const dm_block_desc* d) {
  if (d->pool) return Form{d->pool == POOL, 1};
  // The forms round differently, and a sample's result must not depend on the batch it is in: they are priced for a batch that is
  // assumed, slices for 4 samples and single queries for 8. (What that costs other batches, us, as chosen / the best form: 8 heads x 256
  // queries, 8 of 64 blocks of 64 features, 1 sample 28 / 25, 64 samples 342 / 176; 2 heads of 4 x 333, 7 of 65 of 32 features, 80 samples 247 / 134.)
  const double rows = (double)d->Lq * (d->Hq / d->Hkv), most = (rows < POOL ? rows : POOL) * d->top;
  const double at_once = d->D <= 16 ? 512 : 256, visit = d->D <= 16 ? 900 : d->D == 32 ? 1050 : 1500;
  const double visits = most < blocks_of(d) ? most : blocks_of(d);
  auto pool_ns = [&](double samples, int s) {
    const double heads = samples * d->Hkv, pools = heads * dm_cdiv((long)rows, POOL);
    const double rounds = (double)(long)((pools * s + at_once - 1) / at_once), moved = s > 1 ? heads * rows * s * (d->D * 4 + 16) * 2 : 0;
    return (s > 1 ? 14000.0 : 8000.0) + rounds * visits / s * visit + moved / 3000;
  };
  Form f = {true, 1};
  for (int s = 2; s <= MAX_SLICES; s *= 2)
    if (pool_ns(4, s) < pool_ns(4, f.slices)) f.slices = s;
  f.pool = 8 * d->Hkv * rows * (0.3 + d->top * (0.46 + 0.005 * d->D)) > 1.25 * pool_ns(8, f.slices);
  return f;
}
// In how many slices the rows of a block are dealt to workgroups for dk and dv, priced for 4 samples as above: 256 CUs hold 2 workgroups
// with 64 features, 3 with 32, 4 with fewer; one takes 5 us + 2.5 us for 128 rows. (A training call, unsplit / split, us, host included: 8 heads
// of 16384 queries and 77 keys of 64 features 370 / 144; 32 such samples of 4096 queries, for which a split is not needed, 625 / 691.)
int row_slices_of(const dm_block_desc* d) {
  const double rows = (double)d->Lq * (d->Hq / d->Hkv), named = rows * d->top / blocks_of(d), each = named < rows ? named : rows;
  const double groups = 4.0 * d->Hkv * blocks_of(d), at_once = 256 * (d->D == 64 ? 2 : d->D == 32 ? 3 : 4);
  const int pools = dm_cdiv((long)rows, POOL);
  auto ns = [&](int s) {
    const double rounds = (double)(long)((groups * s + at_once - 1) / at_once);
    return rounds * (5000 + each / s / 128 * 2500) + (s > 1 ? 6000 + groups * s * BLK * d->D * 16 / 3000 : 0);
  };
  int best = 1;
  for (int s = 2; s <= MAX_SLICES && s <= pools; s *= 2)
    if (ns(s) < ns(best)) best = s;
  return best;
}
size_t key_part_bytes(const dm_block_desc* d, int slices) { return (size_t)slices * d->B * d->Hkv * blocks_of(d) * 2 * BLK * d->D * 4; }
// The plan's pools (made for the backward pass also where the forward takes one query a workgroup), and its parts
struct PlanLayout { int pools; size_t offs, bytes; };
PlanLayout plan_of(const dm_block_desc* d) {
  PlanLayout p;
  p.pools = dm_cdiv((long)d->Lq * (d->Hq / d->Hkv), POOL);
  const size_t all = (size_t)d->B * d->Hkv * p.pools;
  p.offs = (all * (blocks_of(d) + 1) * 4 + 15) / 16 * 16;
  p.bytes = p.offs + all * POOL * d->top * 2;
  return p;
}

Args args_of(const dm_block_desc* d) {
  Args a = {};
  a.B = d->B; a.Lq = d->Lq; a.Lk = d->Lk; a.Hq = d->Hq; a.Hkv = d->Hkv; a.G = d->Hq / d->Hkv; a.top = d->top;
  a.nblk = blocks_of(d);
  a.pools = plan_of(d).pools;
  a.scale = d->scale;
  a.slices = a.row_slices = 1;
  // neighbouring heads that share cache lines, as many as leave every XCD some
  for (a.near = 64 / d->D; a.near > 1 && (d->Hkv % a.near || (long)d->B * d->Hkv / a.near % 8); a.near /= 2) {}
  return a;
}

}  // namespace

extern "C" size_t dm_block_attention_plan_bytes(const dm_block_desc* d, int for_backward) {
  const char* who = "dm_block_attention_plan_bytes";
  if (check_desc(who, d) || check_span(who, d) || (!for_backward && !form_of(d).pool)) return 0;
  return plan_of(d).bytes;
}

extern "C" size_t dm_block_attention_fwd_ws_bytes(const dm_block_desc* d) {
  const char* who = "dm_block_attention_fwd_ws_bytes";
  if (check_desc(who, d) || check_span(who, d)) return 0;
  const Form f = form_of(d);
  return f.pool && f.slices > 1 ? (size_t)f.slices * d->B * d->Hq * d->Lq * (d->D * 4 + 16) : 0;
}

extern "C" int dm_block_attention_fwd(const dm_block_desc* d, const void* q, const void* k, const void* v, const int* blocks,
                                      const int* k_len, void* out, void* out_lo, float* lse, void* plan, void* ws, size_t ws_bytes, void* stream) {
  const char* who = "dm_block_attention_fwd";
  int rc = check_desc(who, d);
  if (rc) return rc;
  DM_REQUIRE(aligned(q) && aligned(k) && aligned(v) && aligned(out) && blocks, DM_ERR_ARG, "%s: null or misaligned pointer", who);
  if ((rc = check_strides(who, "q", d->q_stride)) || (rc = check_strides(who, "k", d->k_stride)) ||
      (rc = check_strides(who, "v", d->v_stride)) || (rc = check_span(who, d)))
    return rc;
  Args a = args_of(d);
  a.q = rows_of(q, d->q_stride); a.k = rows_of(k, d->k_stride); a.v = rows_of(v, d->v_stride);
  a.blocks = blocks; a.k_len = k_len; a.out = (bf16_t*)out; a.out_lo = (bf16_t*)out_lo; a.lse = lse;
  hipStream_t st = (hipStream_t)stream;
  const Form form = form_of(d);
  const bool pool = form.pool;
  DM_REQUIRE(aligned(plan) || (!plan && !pool), DM_ERR_ARG, "%s: this shape needs a plan (dm_block_attention_plan_bytes), 16-byte aligned", who);
  const size_t need = dm_block_attention_fwd_ws_bytes(d);
  DM_REQUIRE(!need || (aligned(ws) && ws_bytes >= need), DM_ERR_ARG, "%s: workspace of %zu bytes is too small or misaligned (%zu)", who, ws_bytes, need);
  if (plan) {
    const PlanLayout p = plan_of(d);
    int* offs = (int*)plan;
    unsigned short* rows = (unsigned short*)((char*)plan + p.offs);
    a.offs = offs; a.rows = rows;
    hipLaunchKernelGGL(block_plan_kernel, dim3(p.pools, d->B * d->Hkv), dim3(POOL), 0, st, blocks, offs, rows, d->Lq, d->Hq, a.G, d->top, a.nblk, p.pools);
    DM_CHECK_LAUNCH();
  }
  const long rows = (long)d->B * d->Hq * d->Lq;
  if (pool) {
    a.slices = form.slices;
    if (a.slices > 1) {
      a.part = (float*)ws;
      a.part_stat = (f32x4_t*)(a.part + a.slices * rows * d->D);
    }
    const dim3 grid(d->B * d->Hkv * a.pools * a.slices);
    if (lse || out_lo) BY_HEAD_DIM(d->D, hipLaunchKernelGGL((attend_pool_kernel<HD, true>), grid, dim3(POOL), 0, st, a))
    else BY_HEAD_DIM(d->D, hipLaunchKernelGGL((attend_pool_kernel<HD, false>), grid, dim3(POOL), 0, st, a))
    if (a.slices > 1) {
      DM_CHECK_LAUNCH();
      BY_HEAD_DIM(d->D, hipLaunchKernelGGL((attend_join_kernel<HD>), dm_grid((rows * (HD / 8) + 255) / 256), dim3(256), 0, st, a))
    }
  }
  else if ((long)d->Hq * d->Lq < 512) BY_HEAD_DIM(d->D, hipLaunchKernelGGL((attend_row_kernel<HD, 4>), dm_grid(rows), dim3(256), 0, st, a, rows))
  else BY_HEAD_DIM(d->D, hipLaunchKernelGGL((attend_row_kernel<HD, 1>), dm_grid(dm_cdiv(rows, 4)), dim3(256), 0, st, a, rows))
  DM_CHECK_LAUNCH();
  return DM_OK;
}

// (delta first in the workspace, slices' sums behind it)
static size_t delta_bytes(size_t rows) { return (rows * 4 + 15) / 16 * 16; }

extern "C" size_t dm_block_attention_bwd_ws_bytes(const dm_block_desc* d) {
  const char* who = "dm_block_attention_bwd_ws_bytes";
  if (check_desc(who, d) || check_pool(who, d)) return 0;
  const Form f = form_of(d);
  const size_t rows = (size_t)d->B * d->Hq * d->Lq;
  const int k = row_slices_of(d);
  const size_t queries = f.pool && f.slices > 1 ? f.slices * rows * d->D * 4 : 0, keys = k > 1 ? key_part_bytes(d, k) : 0;
  return delta_bytes(rows) + (queries > keys ? queries : keys);   // (one after the other in the same memory)
}

extern "C" int dm_block_attention_bwd(const dm_block_desc* d, const void* q, const void* k, const void* v, const int* blocks,
                                      const int* k_len, const void* plan, const void* out, const void* out_lo, const float* lse,
                                      const void* dout, void* dq, void* dk, void* dv, void* ws, size_t ws_bytes, void* stream) {
  const char* who = "dm_block_attention_bwd";
  int rc = check_desc(who, d);
  if (rc) return rc;
  DM_REQUIRE(aligned(q) && aligned(k) && aligned(v) && aligned(out) && aligned(out_lo) && aligned(dout) && aligned(dq) && aligned(dk) &&
                 aligned(dv) && aligned(plan) && blocks && lse, DM_ERR_ARG, "%s: null or misaligned pointer", who);
  DM_REQUIRE(aligned(ws) && ws_bytes >= dm_block_attention_bwd_ws_bytes(d), DM_ERR_ARG, "%s: workspace of %zu bytes is too small or misaligned", who, ws_bytes);
  const struct { const char* n; const long* s; } all[] = {{"q", d->q_stride}, {"k", d->k_stride}, {"v", d->v_stride},
                                                          {"dq", d->dq_stride}, {"dk", d->dk_stride}, {"dv", d->dv_stride}};
  for (const auto& x : all)
    if ((rc = check_strides(who, x.n, x.s))) return rc;
  if ((rc = check_span(who, d))) return rc;
  const PlanLayout p = plan_of(d);
  Args a = args_of(d);
  a.q = rows_of(q, d->q_stride); a.k = rows_of(k, d->k_stride); a.v = rows_of(v, d->v_stride);
  a.o = (const bf16_t*)out; a.o_lo = (const bf16_t*)out_lo; a.go = (const bf16_t*)dout;
  a.blocks = blocks; a.k_len = k_len; a.offs = (const int*)plan; a.rows = (const unsigned short*)((const char*)plan + p.offs);
  a.lse = const_cast<float*>(lse); a.delta = (float*)ws;
  a.dq = (bf16_t*)dq; a.dk = (bf16_t*)dk; a.dv = (bf16_t*)dv;
  a.dqb = d->dq_stride[0]; a.dql = d->dq_stride[1]; a.dqh = d->dq_stride[2];
  a.dkb = d->dk_stride[0]; a.dkl = d->dk_stride[1]; a.dkh = d->dk_stride[2];
  a.dvb = d->dv_stride[0]; a.dvl = d->dv_stride[1]; a.dvh = d->dv_stride[2];
  hipStream_t st = (hipStream_t)stream;
  const long rows = (long)d->B * d->Hq * d->Lq;
  const Form form = form_of(d);
  if (form.pool) {
    a.slices = form.slices;
    a.part = (float*)((char*)ws + delta_bytes(rows));
    BY_HEAD_DIM(d->D, hipLaunchKernelGGL((dq_pool_kernel<HD>), dim3(d->B * d->Hkv * a.pools * a.slices), dim3(POOL), 0, st, a))
    if (a.slices > 1) {
      DM_CHECK_LAUNCH();
      BY_HEAD_DIM(d->D, hipLaunchKernelGGL((dq_join_kernel<HD>), dm_grid((rows * (HD / 8) + 255) / 256), dim3(256), 0, st, a))
    }
  }
  else BY_HEAD_DIM(d->D, hipLaunchKernelGGL((dq_row_kernel<HD>), dm_grid(dm_cdiv(rows, 4)), dim3(256), 0, st, a, rows))
  DM_CHECK_LAUNCH();
  a.row_slices = row_slices_of(d);
  a.key_part = (float*)((char*)ws + delta_bytes(rows));
  BY_HEAD_DIM(d->D, hipLaunchKernelGGL((dkv_kernel<HD>), dm_grid((long)a.nblk * a.row_slices * d->B * d->Hkv), dim3(256), 0, st, a));
  if (a.row_slices > 1) {
    DM_CHECK_LAUNCH();
    BY_HEAD_DIM(d->D, hipLaunchKernelGGL((dkv_join_kernel<HD>), dm_grid(((long)d->B * d->Hkv * d->Lk * (HD / 8) + 255) / 256), dim3(256), 0, st, a));
  }
  DM_CHECK_LAUNCH();
  return DM_OK;
}
