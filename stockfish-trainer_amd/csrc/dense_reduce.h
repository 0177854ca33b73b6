// Reductions over groups of 2 .. 64 neighbouring lanes, in registers: the exchanges are
// register moves (DPP, permlane swaps), not LDS traffic.
#pragma once

#include "common.h"

namespace sft {
namespace dense {

// x of the lane across distance M.  Distances 4 and 8 are mirrors within 8 and 16
// lanes, which serve a reduction whose smaller distances are done.
template <int M>
__device__ __forceinline__ void exchange(uint32_t x, uint32_t &a, uint32_t &b) {
#ifdef __HIP_DEVICE_COMPILE__
  if constexpr (M <= 8) {
    constexpr int ctrl = M == 1 ? 0xB1 : M == 2 ? 0x4E : M == 4 ? 0x141 : 0x140;
    a = x;
    b = __builtin_amdgcn_update_dpp(0, x, ctrl, 0xf, 0xf, true);
  } else if constexpr (M == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    a = r[0];
    b = r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    a = r[0];
    b = r[1];
  }
#endif
}
// op over groups of G lanes from distance FROM on: every lane gets the group's result.
template <int G, int FROM = 1, typename T, typename Op>
__device__ __forceinline__ T group_reduce(T x, Op op) {
  if constexpr (FROM < G) {
    uint32_t a = 0, b = 0;
    exchange<FROM>(__builtin_bit_cast(uint32_t, x), a, b);
    return group_reduce<G, FROM * 2>(op(__builtin_bit_cast(T, a), __builtin_bit_cast(T, b)), op);
  } else {
    return x;
  }
}
template <int G>
__device__ __forceinline__ float group_max(float x) {
  return group_reduce<G>(x, [](float a, float b) { return fmaxf(a, b); });
}
template <int G, typename T>
__device__ __forceinline__ T group_sum(T x) {
  return group_reduce<G>(x, [](T a, T b) { return a + b; });
}

}  // namespace dense
}  // namespace sft
