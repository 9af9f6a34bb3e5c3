// Reductions and lane exchanges inside groups of 16 lanes and whole waves, for the row-wise operators.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace gg {

// The value of another lane of the same 16: exchanges by DPP, which need neither LDS nor a wait.  The four steps below
// pair lanes as a butterfly does, once the steps before them made the lanes of a half equal: every lane ends with the
// same bits, also of a float sum.  (Every source lane is there; with the 0 for one that is not, the compiler makes the exchange part of the
// instruction that uses it.)
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
enum : int { kDppXor1 = 0xb1, kDppXor2 = 0x4e, kDppHalfMirror = 0x141, kDppMirror = 0x140 };

// All lanes of a group of G (4, 8, 16, 32 or 64) get op over the group.
template <int G, typename T, typename Op>
__device__ __forceinline__ T group_reduce(T v, Op op) {
  static_assert(sizeof(T) == 4 && (G == 4 || G == 8 || G == 16 || G == 32 || G == 64), "");
  auto step = [&](auto other) { v = op(v, __builtin_bit_cast(T, other)); };
  step(dpp<kDppXor1>(__builtin_bit_cast(uint32_t, v)));
  step(dpp<kDppXor2>(__builtin_bit_cast(uint32_t, v)));
  if constexpr (G >= 8) step(dpp<kDppHalfMirror>(__builtin_bit_cast(uint32_t, v)));
  if constexpr (G >= 16) step(dpp<kDppMirror>(__builtin_bit_cast(uint32_t, v)));
  if constexpr (G >= 32) v = op(v, __shfl_xor(v, 16));
  if constexpr (G == 64) v = op(v, __shfl_xor(v, 32));
  return v;
}

template <int G>
__device__ __forceinline__ float group_sum(float v) {
  return group_reduce<G>(v, [](float a, float b) { return a + b; });
}
template <int G>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
  return group_reduce<G>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
template <int G>
__device__ __forceinline__ uint32_t group_min(uint32_t v) {
  return group_reduce<G>(v, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
}

// Inclusive prefix sum over the 64 lanes of a wave.
__device__ __forceinline__ int wave_prefix(int v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int distance = 1; distance < 64; distance <<= 1) {
    const int o = __shfl_up(v, distance);
    if (lane >= distance) v += o;
  }
  return v;
}

}  // namespace gg
