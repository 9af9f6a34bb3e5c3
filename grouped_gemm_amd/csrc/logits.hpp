// Router logits of three element types, a token's in 4, 16 or 64 lanes, and the functions of them: what the router and its losses share.
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "gmm_kernel.hpp"
#include "operators.hpp"

namespace gg {

template <int DT>
struct Logit;
template <>
struct Logit<kF32> {
  using T = uint32_t;
  static __device__ __forceinline__ float widen(T v) { return __builtin_bit_cast(float, v); }
  static __device__ __forceinline__ T narrow(float v) { return __builtin_bit_cast(uint32_t, v); }
};
template <>
struct Logit<kBF16> {
  using T = uint16_t;
  static __device__ __forceinline__ float widen(T v) { return __builtin_bit_cast(float, (uint32_t)v << 16); }
  static __device__ __forceinline__ T narrow(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
};
template <>
struct Logit<kF16> {
  using T = uint16_t;
  static __device__ __forceinline__ float widen(T v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ __forceinline__ T narrow(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
};

// VPL neighbouring elements on any boundary (rows of any length): CDNA takes wide accesses on any boundary of an element.
template <typename T, int VPL>
struct __attribute__((packed, aligned(sizeof(T)))) Row {
  T v[VPL];
};

// The exponential by the hardware's power of two, off by 2^-24 |x| and a unit in the last place: for the scores of all experts, whose
// sums and gradients that does not show in.  The chosen weights are computed with the full functions.
__device__ __forceinline__ float quick_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }
__device__ __forceinline__ float quick_sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + quick_exp(-x)); }
__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + expf(-x)); }
// sigmoid(x) / exp(min(top, 0)), for x up to top: of a token all of whose sigmoids are too small for a float, what is left of them to compare.
__device__ __forceinline__ float scaled_sigmoid(float x, float top) {
  return (x >= 0.0f ? 1.0f : expf(x - fminf(top, 0.0f))) / (1.0f + expf(-fabsf(x)));
}

// The VPL logits of one lane, from `column` of its token on; columns past the last read as -inf.
template <int DT, int VPL>
__device__ __forceinline__ Row<typename Logit<DT>::T, VPL> load_logits(const void* logits, int64_t token, int experts, int column) {
  using T = typename Logit<DT>::T;
  const T* from = static_cast<const T*>(logits) + token * experts + column;
  Row<T, VPL> r;
  if (column + VPL <= experts) {
    r = *reinterpret_cast<const Row<T, VPL>*>(from);
  } else {
#pragma unroll
    for (int v = 0; v < VPL; ++v) r.v[v] = column + v < experts ? from[v] : Logit<DT>::narrow(-INFINITY);
  }
  return r;
}

}  // namespace gg
