// Blocks of 64 rows in 8 bits: a head's block shares an fp32 scale, codes are e4m3 (mote_relation.h has the format
// and the layout of a page).
//
// A page of P2 lies [Dp / 16][64 rows][16 dims], so that lane r of a wave holds row r and its whole score is a sum
// of its own; one of I~ lies [Dp dims][64 rows], so that a lane holds 16 rows of one dim and the weighted sum over
// rows ends inside a quad. Both are read in 1 KB pieces without a gap.
#pragma once

#include "params.hpp"
#include "stream.hpp"
#include "wave_uint.hpp"

namespace mote {

constexpr int kPage8 = 64;                // rows of a block
constexpr float kTop8 = 448.0f;           // the largest e4m3 value
constexpr float kSmall8 = 0x1p-112f;      // a smaller maximum stores zeros (448 / max would overflow)
constexpr int kMaxChunks8 = 8;            // 16-dim chunks of a row: D <= 128
constexpr int kPitchT = kPage8 + 4;       // LDS bytes between dims of a block that is being transposed
constexpr int kBlockLds8 = 16 * kMaxChunks8 * kPitchT;  // LDS that store_block8 needs

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(2))) float f32x2;

// values 0, 1 (HI false) or 2, 3 (true) of a word of codes
template <bool HI>
__device__ __forceinline__ f32x2 codes8_f32(uint32_t w) {
  return __builtin_amdgcn_cvt_pk_f32_fp8(int(w), HI);
}
template <bool HI>
__device__ __forceinline__ bf16x2 codes8_bf16(uint32_t w) {  // exact: e4m3 has four significant bits
  return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI);
}
__device__ __forceinline__ uint32_t encode8(float a, float b, float c, float d) {  // nearest, ties to even
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
}

// N elements (16-byte pieces) of a 16-byte aligned row
template <int N, typename T>
__device__ __forceinline__ void load_values(const T* p, float* x) {
  constexpr int PER = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < N / PER; ++i) {
    const Chunk c = load_chunk(p + i * PER);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 2) {
        x[i * 8 + 2 * j] = __uint_as_float(c.w[j] << 16);
        x[i * 8 + 2 * j + 1] = __uint_as_float(c.w[j] & 0xffff0000u);
      } else {
        x[i * 4 + j] = __uint_as_float(c.w[j]);
      }
    }
  }
}

// A block of 64 rows to its page in 8 bits, by a workgroup of 256 threads (all of them here). A thread holds up to
// two pieces of 16 dims of a row, taken by load(row, chunk, x). The maximum goes over the bits of |x|: as unsigned
// integers they order as the magnitudes do, with infinities and NaNs on top. TRANSPOSED: the layout of I~, turned
// in LDS (`bytes`, kBlockLds8); `top` is four words of LDS.
template <int C, bool TRANSPOSED, typename Load>
__device__ __forceinline__ void store_block8(Load load, uint8_t* page, float* scale, uint32_t* top, uint8_t* bytes) {
  constexpr int ITEMS = (kPage8 * C + 255) / 256;
  const int tid = threadIdx.x;
  float x[ITEMS][16];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int it = tid + 256 * i, row = it / C, ch = it % C;
#pragma unroll
    for (int j = 0; j < 16; ++j) x[i][j] = 0.f;
    if (it < kPage8 * C) load(row, ch, x[i]);
#pragma unroll
    for (int j = 0; j < 16; ++j) m = max(m, __float_as_uint(x[i][j]) & 0x7fffffffu);
  }
  m = wave_umax(m);
  if ((tid & 63) == 0) top[tid >> 6] = m;
  __syncthreads();
  m = max(max(top[0], top[1]), max(top[2], top[3]));
  const float t = __uint_as_float(m);
  const bool finite = m < 0x7f800000u, live = finite && t >= kSmall8;
  const float inv = live ? __fdiv_rn(kTop8, t) : 0.f;
  if (tid == 0) *scale = live ? __fdiv_rn(t, kTop8) : finite ? 0.f : __builtin_nanf("");
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int it = tid + 256 * i, row = it / C, ch = it % C;
    if (it >= kPage8 * C) break;
    Chunk c;
#pragma unroll
    for (int j = 0; j < 4; ++j)  // the products reach 448 (1 + 2^-22), which is 448
      c.w[j] = live ? encode8(x[i][4 * j] * inv, x[i][4 * j + 1] * inv, x[i][4 * j + 2] * inv, x[i][4 * j + 3] * inv) : 0u;
    if constexpr (!TRANSPOSED) {
      store_chunk(page + ch * (16 * kPage8) + row * 16, c);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) bytes[(ch * 16 + j) * kPitchT + row] = uint8_t(c.w[j / 4] >> (8 * (j % 4)));
    }
  }
  if constexpr (TRANSPOSED) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int it = tid + 256 * i;
      if (it >= kPage8 * C) break;
      const uint32_t* src = reinterpret_cast<const uint32_t*>(bytes + (it / 4) * kPitchT + (it % 4) * 16);
      Chunk c;
#pragma unroll
      for (int j = 0; j < 4; ++j) c.w[j] = src[j];
      store_chunk(page + it * 16, c);
    }
  }
}

inline int chunks8(int D) { return (D + 15) / 16; }

// what a launcher checks of a cache in 8 bits: pointers, alignment, strides, sizes
inline const char* bad_cache8(const mote_cache8& c, int B, int H, int D, int elem_bytes) {
  if (!c.p2 || !c.p2_scale || !c.info || !c.info_scale || !c.p2_tail || !c.info_tail || !c.table) return "null pointer";
  if (c.pages < 1 || c.blocks < 1 || c.blocks > (1 << 24)) return "bad sizes of the pool or the table";
  const int64_t page = int64_t(kPage8) * 16 * chunks8(D);
  const uintptr_t codes = reinterpret_cast<uintptr_t>(c.p2) | reinterpret_cast<uintptr_t>(c.info);
  const uintptr_t tails = reinterpret_cast<uintptr_t>(c.p2_tail) | reinterpret_cast<uintptr_t>(c.info_tail);
  if (codes % 16 || c.codes_sp % 16) return "pages must start on 16-byte boundaries";
  if (tails % 16 || (B > 1 && c.tail_sb * elem_bytes % 16)) return "tails must start on 16-byte boundaries";
  if (c.pages > 1 && (c.codes_sp < H * page || c.scale_sp < H)) return "pages lie over one another";
  if (B > 1 && (c.tail_sb < int64_t(H) * kPage8 * D || c.table_sb < c.blocks)) return "sequences lie over one another";
  return nullptr;
}

}  // namespace mote
