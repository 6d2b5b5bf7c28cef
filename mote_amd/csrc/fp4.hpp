// Values in 4 bits: groups of 32 share a bf16 scale, codes are e2m1 (mote_relation.h has the format).
//
// Four lanes of a quad hold one group of a row while it is encoded, eight values (an octet) each. The
// group's maximum goes over the bits of |x|: as unsigned integers they order as the magnitudes do, with
// infinities and NaNs on top, so one comparison finds the groups that have no scale.
#pragma once

#include <algorithm>
#include <cstdlib>
#include <limits>

#include "stream.hpp"

namespace mote {

constexpr int kGroup4 = 32;            // values per scale
constexpr float kTiny4 = 0x1p-126f;    // a smaller scale stores zeros (its inverse would overflow)
constexpr bf16_t kNanScale4 = 0x7fc0;

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(2))) float f32x2;

// byte i (0..3) of a code word: values 2 i and 2 i + 1
template <int I>
__device__ __forceinline__ bf16x2 codes_bf16(uint32_t w) {
  return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, I);
}
template <int I>
__device__ __forceinline__ f32x2 codes_f32(uint32_t w) {
  return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, I);
}

__device__ __forceinline__ uint32_t quad_umax(uint32_t m) {
  m = max(m, uint32_t(__builtin_amdgcn_mov_dpp(int(m), kDppXor1, 0xF, 0xF, false)));
  return max(m, uint32_t(__builtin_amdgcn_mov_dpp(int(m), kDppXor2, 0xF, 0xF, false)));
}

// max / 6 as a division rounds it, in three instructions for a division's ten: one step on the remainder, which
// fma holds exactly (equal to max / 6 for every float from 2^-125 on; smaller ones have no scale).
__device__ __forceinline__ float sixth4(float top) {
  constexpr float r = 1.0f / 6.0f;
  const float t = top * r;
  return __builtin_fmaf(__builtin_fmaf(-6.0f, t, top), r, t);
}
// 1 / scale as a division rounds it, for normal bf16 scales up to 2^126: one Newton step on the hardware's
// reciprocal (1 ulp; right from 2 ulps off, for every bf16)
__device__ __forceinline__ float inverse4(float s) {
  const float r = __builtin_amdgcn_rcpf(s);
  return __builtin_fmaf(__builtin_fmaf(-s, r, 1.0f), r, r);
}

// The quad's group in 4 bits: this lane's eight codes, and the group's scale. All four lanes must be here
// (lanes past the head dim with zeros, or with values of the group, their codes dropped). Rounding points: the
// scale once to bf16 (a wider one would cost more than it gains: codes are 2^-2 apart), the inverse and the
// products in fp32. Products reach 6 (1 + 2^-8), where the scale was rounded down, and convert to 6.
__device__ __forceinline__ uint32_t encode4(const float (&x)[8], bf16_t& scale) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[j]) & 0x7fffffffu);
  top = quad_umax(top);
  const bool finite = top < 0x7f800000u;
  bf16_t sb = f2bf(sixth4(__uint_as_float(finite ? top : 0u)));
  if (bf2f(sb) < kTiny4) sb = 0;
  const float inv = sb ? inverse4(bf2f(sb)) : 0.f;
  scale = finite ? sb : kNanScale4;
  uint32_t w = 0;  // v_cvt_scalef32_pk_fp4_f32 rounds to nearest, ties to the even code
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0] * inv, x[1] * inv, 1.0f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2] * inv, x[3] * inv, 1.0f, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4] * inv, x[5] * inv, 1.0f, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6] * inv, x[7] * inv, 1.0f, 3);
  return finite ? w : 0u;
}

__device__ __forceinline__ void decode4(uint32_t w, float s, float (&x)[8]) {
  const f32x2 a = codes_f32<0>(w), b = codes_f32<1>(w), c = codes_f32<2>(w), d = codes_f32<3>(w);
  x[0] = a.x * s; x[1] = a.y * s; x[2] = b.x * s; x[3] = b.y * s;
  x[4] = c.x * s; x[5] = c.y * s; x[6] = d.x * s; x[7] = d.y * s;
}

// eight elements of a 16-byte aligned row
template <bool STREAM, typename T>
__device__ __forceinline__ void load_octet(const T* p, float (&x)[8]) {
  if constexpr (sizeof(T) == 2) {
    const Chunk c = load_chunk_as<STREAM>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[2 * j] = __uint_as_float(c.w[j] << 16);
      x[2 * j + 1] = __uint_as_float(c.w[j] & 0xffff0000u);
    }
  } else {
    const Chunk a = load_chunk_as<STREAM>(p), b = load_chunk_as<STREAM>(p + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = __uint_as_float(a.w[j]);
      x[4 + j] = __uint_as_float(b.w[j]);
    }
  }
}
// what a launcher checks of a cache in 4 bits: null pointers, alignment
inline const char* bad_cache4(const mote_cache4& c) {
  if (!c.p2 || !c.p2_scale || !c.info || !c.info_scale) return "null pointer";
  const uintptr_t codes = reinterpret_cast<uintptr_t>(c.p2) | reinterpret_cast<uintptr_t>(c.info);
  const uintptr_t scales = reinterpret_cast<uintptr_t>(c.p2_scale) | reinterpret_cast<uintptr_t>(c.info_scale);
  if (codes % 16 || c.codes_sb % 16 || c.codes_sh % 16 || scales % 2) return "codes must start on 16-byte boundaries";
  return nullptr;
}
// and of one that it writes: every sequence and head has rows of its own
inline const char* shared_cache4(const mote_cache4& c, int64_t B, int64_t H, int64_t capacity, int64_t groups) {
  auto apart = [&](int64_t sb, int64_t sh, int64_t block) {
    sb = B > 1 ? std::abs(sb) : std::numeric_limits<int64_t>::max();
    sh = H > 1 ? std::abs(sh) : std::numeric_limits<int64_t>::max();
    const bool by_head = sh < sb;
    const int64_t low = std::min(sb, sh), high = std::max(sb, sh), n = by_head ? H : B;
    if (B <= 1 && H <= 1) return true;
    if (low < block) return false;
    return B <= 1 || H <= 1 || (high - block) / low >= n - 1;
  };
  if (!apart(c.codes_sb, c.codes_sh, capacity * 16 * groups) || !apart(c.scale_sb, c.scale_sh, capacity * groups))
    return "sequences or heads share rows";
  return nullptr;
}

}  // namespace mote
