// The largest of the lanes' unsigned words, in every lane (wave_max of common.hpp for whole numbers).
#pragma once

#include <type_traits>

#include "common.hpp"

namespace mote {

__device__ __forceinline__ uint32_t wave_umax(uint32_t x) {
  u32x2 a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  x = max(a[0], a[1]);
  a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = max(a[0], a[1]);
  auto step = [&](auto ctrl) { x = max(x, uint32_t(__builtin_amdgcn_mov_dpp(int(x), decltype(ctrl)::value, 0xF, 0xF, false))); };
  step(std::integral_constant<int, kDppRor8>{});
  step(std::integral_constant<int, kDppNext4>{});
  step(std::integral_constant<int, kDppXor2>{});
  step(std::integral_constant<int, kDppXor1>{});
  return x;
}

}  // namespace mote
