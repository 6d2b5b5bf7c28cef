// 16-byte accesses with the non-temporal hint, for data that no cache holds until its next use: stores of
// results larger than the L2s (which then keep what is read again), loads of a cache larger than the
// Infinity Cache.
#pragma once

#include "common.hpp"

namespace mote {

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

__device__ __forceinline__ void store_stream(void* p, const Chunk& c) {
  __builtin_nontemporal_store(__builtin_bit_cast(u32x4, c), reinterpret_cast<u32x4*>(p));
}
__device__ __forceinline__ Chunk load_stream(const void* p) {
  return __builtin_bit_cast(Chunk, __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p)));
}
// The same 16 bytes at any address that an element may have: global accesses need no alignment beyond their
// element's (the loads and stores stay single instructions; a row of an odd length is as wide as an even one).
typedef u32x4 __attribute__((aligned(2))) u32x4_any;
__device__ __forceinline__ Chunk load_any(const void* p) {
  return __builtin_bit_cast(Chunk, static_cast<u32x4>(*reinterpret_cast<const u32x4_any*>(p)));
}
__device__ __forceinline__ void store_any(void* p, const Chunk& c) {
  *reinterpret_cast<u32x4_any*>(p) = __builtin_bit_cast(u32x4, c);
}
__device__ __forceinline__ void store_stream_any(void* p, const Chunk& c) {
  __builtin_nontemporal_store(__builtin_bit_cast(u32x4, c), reinterpret_cast<u32x4_any*>(p));
}
template <bool STREAM>
__device__ __forceinline__ Chunk load_chunk_as(const void* p) {
  if constexpr (STREAM) return load_stream(p);
  else return load_chunk(p);
}

}  // namespace mote
