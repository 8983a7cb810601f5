// What the kernels that choose key blocks (block_select.hip) and those that attend to them (block_attention.hip) share:
// tensors by strides, operands of the matrix instructions, sums over lanes, argument checks.
#pragma once
#include "dm_common.h"

namespace {

constexpr int BLK = 64;   // keys of a block

struct Rows {          // a [B][L][H][D] tensor by element strides, D contiguous
  const bf16_t* p;
  long sb, sl, sh;
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
template <int O>   // lane distance 16 or 32: the other half's value
__device__ __forceinline__ float half_xor(float x) {
  const unsigned u = __builtin_bit_cast(unsigned, x);
  if constexpr (O == 16) { auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false); return __builtin_bit_cast(float, (unsigned)((threadIdx.x & 16) ? r[0] : r[1])); }
  else { auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false); return __builtin_bit_cast(float, (unsigned)((threadIdx.x & 32) ? r[0] : r[1])); }
}
template <int LPR>   // over groups of LPR <= 8 lanes, each of which holds one value in all its lanes
__device__ __forceinline__ float across_max(float x) {
  if constexpr (LPR < 2) x = fmaxf(x, lane_xor<1>(x));
  if constexpr (LPR < 4) x = fmaxf(x, lane_xor<2>(x));
  if constexpr (LPR < 8) x = fmaxf(x, lane_xor<4>(x));
  x = fmaxf(x, lane_xor<8>(x));
  x = fmaxf(x, half_xor<16>(x));
  return fmaxf(x, half_xor<32>(x));
}
// c + the products of 8 features, exact in fp32 but for the sum's roundings
__device__ __forceinline__ float dot8(const bf16x8_t& a, const bf16x8_t& b, float c) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    typedef __attribute__((ext_vector_type(2))) __bf16 pair_t;
    const pair_t x = {a[e], a[e + 1]}, y = {b[e], b[e + 1]};
    c = __builtin_amdgcn_fdot2_f32_bf16(x, y, c, false);
  }
  return c;
}
template <int LPR>
__device__ __forceinline__ float across_sum(float x) {
#pragma unroll
  for (int o = LPR; o < 64; o <<= 1) x += __shfl_xor(x, o, 64);
  return x;
}

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
  else return r * 16 + ((c ^ ((r >> 2) & 3)) << 2);
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
template <int D> struct Piece { typedef bf16x8_t type; typedef __attribute__((ext_vector_type(4))) unsigned bits; };
template <> struct Piece<8> { typedef bf16x4_t type; typedef __attribute__((ext_vector_type(2))) unsigned bits; };
template <> struct Piece<16> : Piece<8> {};
template <int D>
struct Frag {
  static constexpr int W = D <= 16 ? 4 : 8;
  typedef typename Piece<D>::type piece_t;
  piece_t x[Geo<D>::KS];
  // p: the row, g = lane >> 4
  __device__ __forceinline__ void load(const bf16_t* p, int g) {
#pragma unroll
    for (int s = 0; s < Geo<D>::KS; ++s) {
      const piece_t none = {};
      x[s] = D >= 16 || g < 2 ? *(const piece_t*)(p + s * 32 + g * W) : none;
    }
  }
  static __device__ __forceinline__ int place(int row, int s, int g) {   // byte offset of a lane's piece in an LDS row
    return D <= 16 ? lds_at<D>(row, g >> 1) + (g & 1) * 8 : lds_at<D>(row, s * 4 + g);
  }
  __device__ __forceinline__ void from_lds(const char* base, int row, int g) {
#pragma unroll
    for (int s = 0; s < Geo<D>::KS; ++s) x[s] = *(const piece_t*)(base + place(row, s, g));
  }
  __device__ __forceinline__ void to_lds(char* base, int row, int g) const {
#pragma unroll
    for (int s = 0; s < Geo<D>::KS; ++s) *(piece_t*)(base + place(row, s, g)) = x[s];
  }
  // waits for the operand here and not behind younger loads (the compiler counts loads in order, and across branches all of them)
  __device__ __forceinline__ void arrived() {
#pragma unroll
    for (int s = 0; s < Geo<D>::KS; ++s) asm volatile("" : "+v"(x[s]));
  }
  __device__ __forceinline__ void negate() {
#pragma unroll
    for (int s = 0; s < Geo<D>::KS; ++s) x[s] = __builtin_bit_cast(piece_t, __builtin_bit_cast(typename Piece<D>::bits, x[s]) ^ 0x80008000u);
  }
  __device__ __forceinline__ void zero() {
    const piece_t none = {};
#pragma unroll
    for (int s = 0; s < Geo<D>::KS; ++s) x[s] = none;
  }
};
template <int D>
__device__ __forceinline__ f32x4_t dot_frag(const Frag<D>& a, const Frag<D>& b, f32x4_t c = f32x4_t{0.f, 0.f, 0.f, 0.f}) {
  if constexpr (D <= 16) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4_t, a.x[0]), __builtin_bit_cast(s16x4_t, b.x[0]), c, 0, 0, 0);
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

bool aligned(const void* p) { return p && ((uintptr_t)p & 15) == 0; }

[[maybe_unused]] int check_desc(const char* who, const dm_block_desc* d) {
  DM_REQUIRE(d, DM_ERR_ARG, "%s: null descriptor", who);
  DM_REQUIRE(d->B > 0 && d->Lq > 0 && d->Lk > 0 && d->Hq > 0 && d->Hkv > 0, DM_ERR_SHAPE, "%s: B, Lq, Lk, Hq and Hkv must be positive", who);
  DM_REQUIRE(d->Hq % d->Hkv == 0, DM_ERR_SHAPE, "%s: %d query heads do not share %d key heads evenly", who, d->Hq, d->Hkv);
  DM_REQUIRE(d->D == 8 || d->D == 16 || d->D == 32 || d->D == 64, DM_ERR_SHAPE, "%s: head dim %d (8, 16, 32 and 64 are covered)", who, d->D);
  DM_REQUIRE(d->top > 0 && d->top <= 64, DM_ERR_SHAPE, "%s: top %d (1 to 64 blocks a query)", who, d->top);
  DM_REQUIRE(d->Lk < (1 << 30) - BLK, DM_ERR_SHAPE, "%s: 2^30 keys and more are not covered", who);
  DM_REQUIRE((long)d->B * d->Hq * d->Lq <= 0x7fffffffL && (long)d->B * d->Hkv <= 65535 && (long)d->Lq * (d->Hq / d->Hkv) < (1L << 30),
             DM_ERR_SHAPE, "%s: more than 2^31-1 queries, 2^30 of one key head or 65535 (sample, key head) pairs", who);
  return DM_OK;
}
[[maybe_unused]] int check_strides(const char* who, const char* name, const long* s) {
  for (int i = 0; i < 3; ++i)
    DM_REQUIRE(s[i] % 8 == 0, DM_ERR_ARG, "%s: strides of %s must be multiples of 8 elements (rows are read 16 bytes at a time)", who, name);
  return DM_OK;
}
[[maybe_unused]] int check_pool(const char* who, const dm_block_desc* d) {
  DM_REQUIRE(d->pool == 0 || d->pool == 1 || d->pool == 512, DM_ERR_ARG, "%s: pool is 0, 1 or 512, not %d", who, d->pool);
  return DM_OK;
}
int blocks_of(const dm_block_desc* d) { return (d->Lk + BLK - 1) / BLK; }

Rows rows_of(const void* p, const long* s) { return Rows{(const bf16_t*)p, s[0], s[1], s[2]}; }

#define BY_HEAD_DIM(D_, CALL)                      \
  switch (D_) {                                    \
    case 8: { constexpr int HD = 8; CALL; } break;   \
    case 16: { constexpr int HD = 16; CALL; } break; \
    case 32: { constexpr int HD = 32; CALL; } break; \
    default: { constexpr int HD = 64; CALL; } break; \
  }

}  // namespace
