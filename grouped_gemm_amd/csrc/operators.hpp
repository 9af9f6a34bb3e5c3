// Launches of the operators around the grouped GEMM that the C ABI (operators_api.hip) is built on: the router
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

constexpr int64_t kFewMaxTokens = 64;
constexpr int64_t kFewMaxExperts = 1024;
constexpr int64_t kFewMaxSlots = kFewMaxTokens * kRouteMaxTopK;

struct FewTokensArgs {
  const void* x;           // (tokens, hidden), element type dt (kBF16, kF16)
  const void* w13;         // (experts, hidden, 2 * ffn), or (experts, 2 * ffn, hidden) with trans_b
  const void* w2;          // (experts, ffn, hidden), or (experts, hidden, ffn) with trans_b
  const int32_t* chosen;   // (tokens, top_k)
  const float* weights;    // (tokens, top_k)
  void* out;               // (tokens, hidden)
  void* scratch;           // few_tokens_scratch_bytes, 256-byte aligned, any contents
  int dt;
  bool trans_b;
  int32_t tokens, experts, top_k, hidden, ffn;
};
// Whether 32 bits hold the offsets and thread counts of such a call.
bool few_tokens_fits(int64_t tokens, int64_t experts, int64_t top_k, int64_t hidden, int64_t ffn, bool trans_b);
uint64_t few_tokens_scratch_bytes(int64_t tokens, int64_t experts, int64_t top_k, int64_t hidden, int64_t ffn, bool trans_b);
hipError_t few_tokens(const FewTokensArgs& args, hipStream_t stream);

constexpr int64_t kAdapterMaxRank = 256;

struct AdapterArgs {
  const void* x;             // (rows, hidden_in), element type dt (kBF16, kF16)
  const void* a;             // (num, rank, hidden_in)
  const void* b;             // (num, hidden_out, rank)
  const int32_t* adapters;   // (rows)
  const float* scales;       // (num) or null: 1
  const void* base;          // (rows, hidden_out) or null: 0
  void* out;                 // (rows, hidden_out), may be base
  void* scratch;             // adapters_scratch_bytes, 16-byte aligned, any contents
  int dt;
  int64_t rows;
  int32_t num, rank, hidden_in, hidden_out;
};
// Whether 32 bits hold the thread counts of such a call.
bool adapters_fit(int64_t rows, int64_t num, int64_t rank, int64_t hidden_in, int64_t hidden_out);
uint64_t adapters_scratch_bytes(int64_t rows, int64_t num, int64_t rank, int64_t hidden_in, int64_t hidden_out);
hipError_t adapters(const AdapterArgs& args, hipStream_t stream);

}  // namespace gg
