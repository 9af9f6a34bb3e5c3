// Launches of the operators around the grouped GEMM that the C ABI (gmm_api.hip) is built on: the router
// (route_kernels.hip), the gated expert layer for a few tokens (few_tokens_kernels.hip), low-rank adapters
// (adapter_kernels.hip).  Arguments are checked by the caller.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace gg {

constexpr int kF32 = 4;   // element type of logits besides kBF16 and kF16

constexpr int64_t kRouteMaxExperts = 1024;
constexpr int64_t kRouteMaxTopK = 32;

struct RouteArgs {
  const void* logits;   // (tokens, experts), element type dt
  int dt;
  int64_t tokens;
  int32_t experts, top_k;
  bool sigmoid, normalize;
  float* weights;          // (tokens, top_k)
  int32_t* chosen;         // (tokens, top_k)
  int64_t* batch_sizes;    // (experts)
  int32_t* row_index;      // (tokens * top_k)
  int32_t* order;          // (tokens * top_k)
  float* mass;             // (experts) or null
  void* scratch;           // route_scratch_bytes, any contents
};
uint64_t route_scratch_bytes(int64_t tokens, int64_t experts, int64_t top_k);
hipError_t route(const RouteArgs& args, hipStream_t stream);

struct RouteBackwardArgs {
  const void* logits;
  int dt;
  int64_t tokens;
  int32_t experts, top_k;
  bool sigmoid, normalize;
  const int32_t* chosen;       // as route wrote it
  const float* weights_grad;   // (tokens, top_k) or null
  const float* mass_grad;      // (experts) or null
  void* logits_grad;           // (tokens, experts), element type dt
};
hipError_t route_backward(const RouteBackwardArgs& args, hipStream_t stream);

}  // namespace gg
