// Rows of an embedding table by token, scaled, and the table's gradient.
//
//   out[i]     = scale * table[token_i]
//   dtable[t] += scale * sum of dout[i] over the i with token_i = t, in ascending order of i inside chunks of the sorted
//                tokens, chunk by chunk (never by float atomics: the same bits every time)
//
// Both directions only move data: forward reads a row and writes a row per token, the gradient reads dout once and writes every
// row that some token names. The gradient sorts the (token, i) pairs by token (stable radix sort, 8 bits a pass), so
// that a row's terms are neighbours, and cuts the SORTED order into equal chunks: a token that makes up half of the
// batch costs no more than as many rare ones.
#include "dm_common.h"

namespace {

constexpr int TILE = 2048;      // keys a workgroup sorts at a time: 4 waves x 8 rounds x 64 lanes
constexpr int RADIX = 256;
constexpr int SCAN_TILES = 256;   // with / without the kernel of that name: 262144 tokens 99 / 95 us, 1048576 129 / 131, 4194304 331 / 520

// number of threads that share a row of `vecs` vectors: a power of two, so that a workgroup holds whole rows
int threads_per_row(int vecs) {
  int t = 1;
  while (t < 256 && t < vecs) t <<= 1;
  return t;
}

template <typename T, int V> struct Vec;
template <typename T, int V> using Raw = T __attribute__((ext_vector_type(V)));   // as it lies in memory
template <> struct Vec<float, 4> {
  static __device__ __forceinline__ void load(const float* p, float* f) { *(f32x4_t*)f = *(const f32x4_t*)p; }
  static __device__ __forceinline__ void store(float* p, const float* f) { *(f32x4_t*)p = *(const f32x4_t*)f; }
};
template <> struct Vec<float, 8> {
  static __device__ __forceinline__ void load(const float* p, float* f) { *(f32x4_t*)f = *(const f32x4_t*)p; *(f32x4_t*)(f + 4) = *(const f32x4_t*)(p + 4); }
  static __device__ __forceinline__ void store(float* p, const float* f) { *(f32x4_t*)p = *(const f32x4_t*)f; *(f32x4_t*)(p + 4) = *(const f32x4_t*)(f + 4); }
};
template <> struct Vec<bf16_t, 8> {
  static __device__ __forceinline__ void load(const bf16_t* p, float* f) { dm_unpack8(*(const bf16x8_t*)p, f); }
  static __device__ __forceinline__ void store(bf16_t* p, const float* f) { *(bf16x8_t*)p = dm_pack8(f); }
};
template <> struct Vec<float, 1> {
  static __device__ __forceinline__ void load(const float* p, float* f) { *f = *p; }
  static __device__ __forceinline__ void store(float* p, const float* f) { *p = *f; }
};
template <> struct Vec<bf16_t, 4> {
  static __device__ __forceinline__ void load(const bf16_t* p, float* f) {
    const bf16x4_t v = *(const bf16x4_t*)p;
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = (float)v[e];
  }
  static __device__ __forceinline__ void store(bf16_t* p, const float* f) {
    bf16x4_t v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (bf16_t)f[e];
    *(bf16x4_t*)p = v;
  }
};
template <> struct Vec<bf16_t, 1> {
  static __device__ __forceinline__ void load(const bf16_t* p, float* f) { *f = (float)*p; }
  static __device__ __forceinline__ void store(bf16_t* p, const float* f) { *p = (bf16_t)*f; }
};

// A thread copies V features of U rows: the U rows' loads are in flight together. Bound by HBM: 131072 rows of 1024 in bf16 87 us, which
// is 5.4 TB/s of what it moves (some rows from the caches); 19712 rows of 512 7.6 us; 256 rows 2.5 us, a launch.
template <typename T, int V, int U>
__global__ __launch_bounds__(256) void token_embed_kernel(const float* __restrict__ table, const int64_t* __restrict__ tokens,
                                                          T* __restrict__ out, long n, long rows, int width, float scale, int tpr) {
  const int per = 256 / tpr;
  const long i0 = dm_block_index() * (per * U) + threadIdx.x / tpr;
  const float* src[U];
  bool live[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long i = i0 + (long)u * per;
    const int64_t t = i < n ? tokens[i] : -1;
    live[u] = t >= 0 && t < rows;
    src[u] = table + (live[u] ? t : 0) * (long)width;
  }
  for (int e = (threadIdx.x & (tpr - 1)) * V; e < width; e += tpr * V) {
    float f[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) Vec<float, V>::load(src[u] + e, f[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long i = i0 + (long)u * per;
#pragma unroll
      for (int x = 0; x < V; ++x) f[u][x] = live[u] ? f[u][x] * scale : 0.f;
      if (i < n) Vec<T, V>::store(out + i * (long)width + e, f[u]);
    }
  }
}

// A token's sort key: the token itself, or `rows` (sorted behind every token) where it has no gradient
__device__ __forceinline__ unsigned key_of(const int64_t* tokens, long i, long rows, long padding) {
  const int64_t t = tokens[i];
  return t < 0 || t >= rows || t == padding ? (unsigned)rows : (unsigned)t;
}

// counts of a pass's digit in every tile
template <bool FIRST>
__global__ __launch_bounds__(256) void sort_count_kernel(const int64_t* __restrict__ tokens, const unsigned* __restrict__ key_in,
                                                         unsigned* __restrict__ counts, long n, long rows, long padding, int shift) {
  __shared__ unsigned c[RADIX];
  const int t = blockIdx.x, tid = threadIdx.x;
  c[tid] = 0;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < TILE / 256; ++u) {
    const long i = (long)t * TILE + u * 256 + tid;
    if (i < n) atomicAdd(&c[((FIRST ? key_of(tokens, i, rows, padding) : key_in[i]) >> shift) & (RADIX - 1)], 1u);
  }
  __syncthreads();
  counts[(long)t * RADIX + tid] = c[tid];
}

// The counts become the number of that digit's keys in earlier tiles, and their sums stand behind the last tile: a thread is a
// digit of a quarter of the tiles. (Up to SCAN_TILES tiles every workgroup of the pass adds them up by itself.)
__global__ __launch_bounds__(1024) void sort_scan_kernel(unsigned* __restrict__ counts, int tiles) {
  __shared__ unsigned sum[4][RADIX];
  const int digit = threadIdx.x & (RADIX - 1), part = threadIdx.x / RADIX, per = (tiles + 3) / 4;
  const int first = part * per, end = min(first + per, tiles);
  unsigned s = 0;
#pragma unroll 16
  for (int t = first; t < end; ++t) s += counts[(long)t * RADIX + digit];
  sum[part][digit] = s;
  __syncthreads();
  s = 0;
  for (int p = 0; p < part; ++p) s += sum[p][digit];
#pragma unroll 16
  for (int t = first; t < end; ++t) {
    const unsigned c = counts[(long)t * RADIX + digit];
    counts[(long)t * RADIX + digit] = s;
    s += c;
  }
  if (part == 3) counts[(long)tiles * RADIX + digit] = s;
}

// One stable pass: a key's place is (keys of smaller digits) + (keys of its digit in earlier tiles, waves and lanes).
// Inside a wave the lanes of one digit find each other with 8 ballots.
template <bool FIRST>
__global__ __launch_bounds__(256) void sort_pass_kernel(const int64_t* __restrict__ tokens, const unsigned* __restrict__ key_in,
                                                        const unsigned* __restrict__ idx_in, unsigned* __restrict__ key_out,
                                                        unsigned* __restrict__ idx_out, const unsigned* __restrict__ counts, long n,
                                                        long rows, long padding, int tiles, int scanned, int shift) {
  __shared__ unsigned base[RADIX], wcount[4][RADIX];
  const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
#pragma unroll
  for (int w = 0; w < 4; ++w) wcount[w][tid] = 0;
  unsigned before = 0, total = 0;
  if (scanned) {
    before = counts[(long)t * RADIX + tid];
    total = counts[(long)tiles * RADIX + tid];
  } else {
#pragma unroll 8
    for (int x = 0; x < tiles; ++x) {
      const unsigned c = counts[(long)x * RADIX + tid];
      total += c;
      before += x < t ? c : 0;
    }
  }
  base[tid] = total;
  __syncthreads();
  for (int o = 1; o < RADIX; o <<= 1) {   // inclusive sums over the digits
    const unsigned v = tid >= o ? base[tid - o] : 0;
    __syncthreads();
    base[tid] += v;
    __syncthreads();
  }
  const unsigned start = base[tid] - total + before;
  constexpr int ROUNDS = TILE / 256;
  unsigned key[ROUNDS], idx[ROUNDS], rank[ROUNDS];
#pragma unroll
  for (int u = 0; u < ROUNDS; ++u) {
    const long i = (long)t * TILE + wave * (TILE / 4) + u * 64 + lane;
    const bool in = i < n;
    if constexpr (FIRST) {
      key[u] = in ? key_of(tokens, i, rows, padding) : 0;
      idx[u] = (unsigned)i;
    } else {
      key[u] = in ? key_in[i] : 0;
      idx[u] = in ? idx_in[i] : 0;
    }
    const unsigned d = (key[u] >> shift) & (RADIX - 1);
    unsigned long long same = __ballot(in);
#pragma unroll
    for (int bit = 0; bit < 8; ++bit) {
      const bool one = (d >> bit) & 1;
      const unsigned long long m = __ballot(one);
      same &= one ? m : ~m;
    }
    const int lower = __builtin_amdgcn_mbcnt_hi((unsigned)(same >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)same, 0));
    const unsigned have = wcount[wave][d];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // every lane has read before one of them writes, and the next round reads that
    rank[u] = have + lower;
    if (in && lower == 0) wcount[wave][d] = have + __builtin_popcountll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  __syncthreads();
  {   // the wave counts become places
    unsigned s = start;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const unsigned c = wcount[w][tid];
      wcount[w][tid] = s;
      s += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < ROUNDS; ++u) {
    const long i = (long)t * TILE + wave * (TILE / 4) + u * 64 + lane;
    if (i >= n) continue;
    const unsigned to = wcount[wave][(key[u] >> shift) & (RADIX - 1)] + rank[u];
    key_out[to] = key[u];
    idx_out[to] = idx[u];
  }
}

// A table of zeros, for rows that no token names: workgroup `group` of `groups` with T threads. Bound by HBM's writes.
constexpr int CLEAR = 4;   // 16-byte pieces a thread
template <int T>
__device__ __forceinline__ void clear(float* __restrict__ to, long n, long vecs, long group, long groups) {
  const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < CLEAR; ++u) {
    const long i = (group * CLEAR + u) * T + threadIdx.x;
    if (i < vecs) ((f32x4_t*)to)[i] = zero;
  }
  for (long i = vecs * 4 + group * T + threadIdx.x; i < n; i += groups * T) to[i] = 0.f;
}
__global__ __launch_bounds__(256) void clear_kernel(float* __restrict__ to, long n, long vecs) {
  clear<256>(to, n, vecs, dm_block_index(), (long)gridDim.x * gridDim.y);
}

// The whole sort of a small call in one launch: the same passes, by one workgroup in LDS. The others clear the table meanwhile.
constexpr int SMALL = 8192;
__global__ __launch_bounds__(1024) void sort_small_kernel(const int64_t* __restrict__ tokens, unsigned* __restrict__ key_out,
                                                          unsigned* __restrict__ idx_out, int n, long rows, long padding, int passes,
                                                          float* __restrict__ table, long floats, long vecs) {
  if (dm_block_index() > 0) {
    clear<1024>(table, floats, vecs, dm_block_index() - 1, (long)gridDim.x * gridDim.y - 1);
    return;
  }
  __shared__ unsigned skey[SMALL];
  __shared__ unsigned short sidx[SMALL], wcount[16][RADIX];
  __shared__ unsigned wsum[4];
  constexpr int ROUNDS = SMALL / 1024;
  const int span = (n + 1023) / 1024 * 64;   // a wave's neighbouring keys
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, first = wave * span + lane, rounds = span / 64;
  unsigned key[ROUNDS], idx[ROUNDS], rank[ROUNDS];
#pragma unroll
  for (int u = 0; u < ROUNDS; ++u) {
    const int i = first + u * 64;
    if (u >= rounds) break;
    key[u] = i < n ? key_of(tokens, i, rows, padding) : 0;
    idx[u] = i;
  }
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = 8 * pass;
    for (int x = tid; x < 16 * RADIX / 2; x += 1024) ((unsigned*)&wcount[0][0])[x] = 0;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < ROUNDS; ++u) {
      if (u >= rounds) break;
      const bool in = first + u * 64 < n;
      const unsigned d = (key[u] >> shift) & (RADIX - 1);
      unsigned long long same = __ballot(in);
#pragma unroll
      for (int bit = 0; bit < 8; ++bit) {
        const bool one = (d >> bit) & 1;
        const unsigned long long m = __ballot(one);
        same &= one ? m : ~m;
      }
      const int lower = __builtin_amdgcn_mbcnt_hi((unsigned)(same >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)same, 0));
      const unsigned have = wcount[wave][d];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // as in the pass above
      rank[u] = have + lower;
      if (in && lower == 0) wcount[wave][d] = (unsigned short)(have + __builtin_popcountll(same));
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    __syncthreads();
    unsigned total = 0, inc = 0;
    if (tid < RADIX) {
#pragma unroll
      for (int w = 0; w < 16; ++w) total += wcount[w][tid];
      inc = total;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const unsigned up = __shfl_up(inc, o, 64);
        if (lane >= o) inc += up;
      }
      if (lane == 63) wsum[wave] = inc;
    }
    __syncthreads();
    if (tid < RADIX) {
      unsigned at = inc - total;
#pragma unroll
      for (int w = 0; w < 3; ++w) at += w < wave ? wsum[w] : 0;
#pragma unroll
      for (int w = 0; w < 16; ++w) {
        const unsigned c = wcount[w][tid];
        wcount[w][tid] = (unsigned short)at;   // (places are below 8192)
        at += c;
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < ROUNDS; ++u) {
      if (u >= rounds || first + u * 64 >= n) break;
      const unsigned to = wcount[wave][(key[u] >> shift) & (RADIX - 1)] + rank[u];
      skey[to] = key[u];
      sidx[to] = (unsigned short)idx[u];
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < ROUNDS; ++u) {
      const int i = first + u * 64;
      if (u >= rounds) break;
      key[u] = i < n ? skey[i] : 0;
      idx[u] = i < n ? sidx[i] : 0;
    }
  }
#pragma unroll
  for (int u = 0; u < ROUNDS; ++u) {
    const int i = first + u * 64;
    if (u < rounds && i < n) {
      key_out[i] = key[u];
      idx_out[i] = idx[u];
    }
  }
}

// Sums of runs of equal keys inside one chunk of the sorted order. A run that lies inside the chunk goes to its row; the
// part of a run that began before the chunk, and the part of one that goes on behind it, are left in part[chunk][0 / 1].
// `chunk` <= MAX_CHUNK neighbouring positions a group of tpr threads, U rows' loads in flight at a time. Bound by HBM: the rows are read
// once, in the sorted order (131072 rows of 1024 in bf16, 50000 of the table: 100 us for 268 + 110 MB, 3.8 TB/s).
constexpr int MAX_CHUNK = 64;
template <int V>
__device__ __forceinline__ void finish_row(float* to, const float* s, float scale, int accumulate) {
  float g[V];
  if (accumulate) Vec<float, V>::load(to, g);
#pragma unroll
  for (int x = 0; x < V; ++x) g[x] = accumulate ? g[x] + s[x] * scale : s[x] * scale;
  Vec<float, V>::store(to, g);
}
template <typename T, int V>
__global__ __launch_bounds__(256) void run_sum_kernel(const T* __restrict__ dout, const unsigned* __restrict__ key,
                                                      const unsigned* __restrict__ idx, float* __restrict__ dtable, float* __restrict__ part,
                                                      long n, unsigned rows, int width, float scale, int tpr, int chunk, int accumulate) {
  // the keys of the workgroup's chunks and of one position on either side; 256 / tpr chunks of at most 64, or of 16 (small calls)
  __shared__ unsigned skey[4096 + 2], sidx[4096];
  const int per = 256 / tpr, all = per * chunk;
  const long first = (long)blockIdx.x * all;
  for (int x = threadIdx.x; x < all + 2; x += 256) {
    const long p = first + x - 1;
    skey[x] = p >= 0 && p < n ? key[p] : 0xffffffffu;   // (no key: keys are at most `rows` < 2^31)
    if (x >= 1 && x <= all) sidx[x - 1] = p < n ? idx[p] : 0;
  }
  __syncthreads();
  const int c = threadIdx.x / tpr, p0 = c * chunk, p1 = (int)min((long)(p0 + chunk), n - first);
  const int e = (blockIdx.y * tpr + (threadIdx.x & (tpr - 1))) * V;
  if (p0 >= p1 || e >= width) return;
  constexpr int U = 8;
  float s[V];
#pragma unroll
  for (int x = 0; x < V; ++x) s[x] = 0.f;
  bool began = skey[p0] != skey[p0 + 1];   // the current run began in this chunk
  for (int p = p0; p < p1; p += U) {
    if (skey[p + 1] >= rows) break;        // only positions without a gradient follow
    T raw[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (p + u < p1) *(Raw<T, V>*)raw[u] = *(const Raw<T, V>*)(dout + (long)sidx[p + u] * width + e);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (p + u >= p1) break;
      const unsigned k = skey[p + u + 1];
      if (k >= rows) break;
#pragma unroll
      for (int x = 0; x < V; ++x) s[x] += (float)raw[u][x];
      const bool ends = skey[p + u + 2] != k;
      if (ends || p + u + 1 >= p1) {
        if (began && ends) finish_row<V>(dtable + (long)k * width + e, s, scale, accumulate);
        else Vec<float, V>::store(part + (((long)blockIdx.x * per + c) * 2 + (began ? 1 : 0)) * (long)width + e, s);
#pragma unroll
        for (int x = 0; x < V; ++x) s[x] = 0.f;
        began = true;
      }
    }
  }
}

// A run that goes on behind the chunk it began in: its parts, chunk by chunk
template <int V>
__global__ __launch_bounds__(256) void run_join_kernel(const unsigned* __restrict__ key, const float* __restrict__ part,
                                                       float* __restrict__ dtable, long n, unsigned rows, int width, float scale, int tpr,
                                                       int chunk, int accumulate) {
  const long c = (long)blockIdx.x * (256 / tpr) + threadIdx.x / tpr;
  const int e = (blockIdx.y * tpr + (threadIdx.x & (tpr - 1))) * V;
  const long p0 = c * chunk, p1 = p0 + chunk;
  if (p1 >= n || e >= width) return;
  const unsigned k = key[p1 - 1];
  if (k >= rows || key[p1] != k) return;
  if (key[p0] == k && p0 > 0 && key[p0 - 1] == k) return;   // began before this chunk
  long lo = c + 1, hi = (n + chunk - 1) / chunk;            // the first chunk behind that does not begin with the run
  while (lo < hi) {
    const long mid = (lo + hi) / 2;
    if (key[mid * chunk] == k) lo = mid + 1;
    else hi = mid;
  }
  float s[V];
  Vec<float, V>::load(part + (c * 2 + 1) * (long)width + e, s);
  constexpr int U = 16;
  for (long x = c + 1; x < lo; x += U) {
    float f[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (x + u < lo) Vec<float, V>::load(part + (x + u) * 2 * (long)width + e, f[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (x + u < lo) {
#pragma unroll
        for (int y = 0; y < V; ++y) s[y] += f[u][y];
      }
  }
  finish_row<V>(dtable + (long)k * width + e, s, scale, accumulate);
}

// positions of the sorted order that a group of threads sums: 16 where there are few, so that they fill the chip (backward with 512
// features, 16 / 64 a group: 32768 tokens 50 / 58 us, 65536 66 / 63, 131072 98 / 79)
int chunk_of(long n) { return n >= 65536 ? MAX_CHUNK : 16; }

// (at least 4 threads a row: a workgroup's chunks, 256 / threads of them, fit its LDS)
int sum_threads(int vecs) { return threads_per_row(vecs) < 4 ? 4 : threads_per_row(vecs); }

struct Plan {   // parts of the workspace, in bytes
  long tiles, chunks;
  int passes;
  size_t key[2], idx[2], counts, part, total;
};
Plan plan_of(long n, long rows, int width) {
  Plan p;
  p.tiles = (n + TILE - 1) / TILE;
  const int chunk = chunk_of(n);
  p.chunks = (n + chunk - 1) / chunk;
  p.passes = 1;
  while (p.passes < 4 && (rows >> (8 * p.passes)) != 0) ++p.passes;
  size_t at = 0;
  auto take = [&](size_t bytes) { const size_t here = at; at += (bytes + 255) / 256 * 256; return here; };
  for (int i = 0; i < 2; ++i) { p.key[i] = take(n * 4); p.idx[i] = take(n * 4); }
  p.counts = take((size_t)(p.tiles + 1) * RADIX * 4);
  p.part = take((size_t)p.chunks * 2 * width * 4);
  p.total = at;
  return p;
}

int check_embed(const char* who, long n, long rows, int width) {
  DM_REQUIRE(n >= 0 && n < 0x7fffffffL, DM_ERR_SHAPE, "%s: %ld tokens (up to 2^31-2)", who, n);
  DM_REQUIRE(rows > 0 && rows < 0x7fffffffL, DM_ERR_SHAPE, "%s: %ld rows (1 to 2^31-2)", who, rows);
  DM_REQUIRE(width > 0 && width <= 65536, DM_ERR_SHAPE, "%s: width %d (1 to 65536)", who, width);
  return DM_OK;
}
// features a thread handles at a time: 16 bytes of the bf16 side, or of fp32; 1 where rows or bases are not aligned
int vectors(int width, const void* a, const void* b, int bf16) {
  if (width % 4 || (((uintptr_t)a | (uintptr_t)b) & 15)) return 1;
  return bf16 && width % 8 == 0 ? 8 : 4;
}

}  // namespace

extern "C" int dm_token_embed(const float* table, const int64_t* tokens, void* out, int out_bf16, long n, long rows, int width,
                              float scale, void* stream) {
  const char* who = "dm_token_embed";
  int rc = check_embed(who, n, rows, width);
  if (rc) return rc;
  if (n == 0) return DM_OK;
  DM_REQUIRE(table && tokens && out, DM_ERR_ARG, "%s: null pointer", who);
  const int V = vectors(width, table, out, out_bf16);
  const int tpr = threads_per_row(width / V);
  const int U = n / (256 / tpr) >= 8192 ? 4 : 1;   // 4 rows a thread once that leaves 8 workgroups a CU (131072 rows of 1024: 100 -> 97 us)
  const dim3 grid = dm_grid(dm_cdiv(n, 256 / tpr * U)), block(256);
  hipStream_t st = (hipStream_t)stream;
#define GO(T, V, U) hipLaunchKernelGGL((token_embed_kernel<T, V, U>), grid, block, 0, st, table, tokens, (T*)out, n, rows, width, scale, tpr)
#define GO_U(T, V) do { if (U == 4) GO(T, V, 4); else GO(T, V, 1); } while (0)
  if (out_bf16) { if (V == 8) GO_U(bf16_t, 8); else if (V == 4) GO_U(bf16_t, 4); else GO_U(bf16_t, 1); }
  else { if (V == 4) GO_U(float, 4); else GO_U(float, 1); }
#undef GO_U
#undef GO
  DM_CHECK_LAUNCH();
  return DM_OK;
}

extern "C" size_t dm_token_embed_bwd_ws_bytes(long n, long rows, int width) {
  if (check_embed("dm_token_embed_bwd_ws_bytes", n, rows, width)) return 0;
  return plan_of(n, rows, width).total;
}

extern "C" int dm_token_embed_bwd(const void* dout, int dout_bf16, const int64_t* tokens, float* dtable, long n, long rows, int width,
                                  float scale, long padding, int accumulate, void* ws, size_t ws_bytes, void* stream) {
  const char* who = "dm_token_embed_bwd";
  int rc = check_embed(who, n, rows, width);
  if (rc) return rc;
  DM_REQUIRE(accumulate >= 0 && accumulate <= 2, DM_ERR_ARG, "%s: accumulate is 0, 1 or 2, not %d", who, accumulate);
  if (n == 0 && accumulate != 2) return DM_OK;
  DM_REQUIRE(n > 0, DM_ERR_SHAPE, "%s: no tokens to write a table from", who);
  DM_REQUIRE(dout && tokens && dtable, DM_ERR_ARG, "%s: null pointer", who);
  const Plan p = plan_of(n, rows, width);
  DM_REQUIRE(ws && ((uintptr_t)ws & 15) == 0 && ws_bytes >= p.total, DM_ERR_ARG, "%s: workspace of %zu bytes is too small or misaligned (%zu)", who, ws_bytes, p.total);
  char* w = (char*)ws;
  unsigned *key[2] = {(unsigned*)(w + p.key[0]), (unsigned*)(w + p.key[1])}, *idx[2] = {(unsigned*)(w + p.idx[0]), (unsigned*)(w + p.idx[1])};
  unsigned* counts = (unsigned*)(w + p.counts);
  float* part = (float*)(w + p.part);
  hipStream_t st = (hipStream_t)stream;
  const dim3 block(256), tiles(p.tiles);
  const int scan = p.tiles > SCAN_TILES;
  const long floats = accumulate == 2 ? rows * width : 0, vecs = ((uintptr_t)dtable & 15) ? 0 : floats / 4;
  if (floats && n > SMALL) {
    hipLaunchKernelGGL(clear_kernel, dm_grid(floats / (4 * 256 * CLEAR) + 1), block, 0, st, dtable, floats, vecs);
    DM_CHECK_LAUNCH();
  }
  // one workgroup up to 8192 tokens (backward with 320 features, in one launch / in two a pass: 4999 tokens 26 / 35 us, 8192 32 / 37)
  if (n <= SMALL) {
    hipLaunchKernelGGL(sort_small_kernel, dm_grid(floats ? floats / (4 * 1024 * CLEAR) + 2 : 1), dim3(1024), 0, st, tokens,
                       key[(p.passes - 1) & 1], idx[(p.passes - 1) & 1], (int)n, rows, padding, p.passes, dtable, floats, vecs);
    DM_CHECK_LAUNCH();
  }
  for (int i = 0; i < p.passes && n > SMALL; ++i) {
    const unsigned *ki = key[(i + 1) & 1], *ii = idx[(i + 1) & 1];
    unsigned *ko = key[i & 1], *io = idx[i & 1];
    if (i == 0) hipLaunchKernelGGL((sort_count_kernel<true>), tiles, block, 0, st, tokens, nullptr, counts, n, rows, padding, 0);
    else hipLaunchKernelGGL((sort_count_kernel<false>), tiles, block, 0, st, nullptr, ki, counts, n, rows, padding, 8 * i);
    DM_CHECK_LAUNCH();
    if (scan) {
      hipLaunchKernelGGL(sort_scan_kernel, dim3(1), dim3(1024), 0, st, counts, (int)p.tiles);
      DM_CHECK_LAUNCH();
    }
    if (i == 0) hipLaunchKernelGGL((sort_pass_kernel<true>), tiles, block, 0, st, tokens, nullptr, nullptr, ko, io, counts, n, rows, padding, (int)p.tiles, scan, 0);
    else hipLaunchKernelGGL((sort_pass_kernel<false>), tiles, block, 0, st, nullptr, ki, ii, ko, io, counts, n, rows, padding, (int)p.tiles, scan, 8 * i);
    DM_CHECK_LAUNCH();
  }
  const unsigned *sk = key[(p.passes - 1) & 1], *si = idx[(p.passes - 1) & 1];
  const int V = vectors(width, dout, dtable, dout_bf16), tpr = sum_threads(width / V), chunk = chunk_of(n);
  const dim3 grid(dm_cdiv(p.chunks, 256 / tpr), dm_cdiv(width / V, tpr));
#define GO(T, V) hipLaunchKernelGGL((run_sum_kernel<T, V>), grid, block, 0, st, (const T*)dout, sk, si, dtable, part, n, (unsigned)rows, width, scale, tpr, chunk, accumulate == 1)
  if (dout_bf16) { if (V == 8) GO(bf16_t, 8); else if (V == 4) GO(bf16_t, 4); else GO(bf16_t, 1); }
  else { if (V == 4) GO(float, 4); else GO(float, 1); }
#undef GO
  DM_CHECK_LAUNCH();
  if (p.chunks > 1) {
    const int W = V == 1 ? 1 : 4, t = sum_threads(width / W);   // (the parts are fp32 whatever dout is)
    const dim3 jgrid(dm_cdiv(p.chunks, 256 / t), dm_cdiv(width / W, t));
    if (W == 4) hipLaunchKernelGGL((run_join_kernel<4>), jgrid, block, 0, st, sk, part, dtable, n, (unsigned)rows, width, scale, t, chunk, accumulate == 1);
    else hipLaunchKernelGGL((run_join_kernel<1>), jgrid, block, 0, st, sk, part, dtable, n, (unsigned)rows, width, scale, t, chunk, accumulate == 1);
    DM_CHECK_LAUNCH();
  }
  return DM_OK;
}
