// Launches of the operators around the grouped GEMM that the C ABI (operators_api.hip) is built on: the router
// (route_kernels.hip), its balance loss (balance_kernels.hip), the gated expert layer for a few tokens (few_tokens_kernels.hip), low-rank adapters
// (adapter_kernels.hip), rows in 8-bit integers (int8_row_kernels.hip).  Arguments are checked by the caller.
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

struct BalanceArgs {
  const void* logits;        // (tokens, experts), element type dt
  int dt;
  bool sigmoid;
  int64_t tokens;
  int32_t experts, top_k, sequences;
  const int32_t* chosen;     // (tokens, top_k)
  const int32_t* offsets;    // (sequences + 1), or null: one sequence of all tokens
  const uint8_t* mask;       // (tokens), 0: not counted; or null
  float *balance, *z;        // one number each
  int32_t* counts;           // (sequences, experts)
  float* share;              // (sequences, experts): counts * experts / (top_k * tokens of the sequence), for the gradient
  float* inverse;            // one number: 1 / counted tokens, for the gradient
  void* scratch;             // balance_scratch_bytes, 4-byte aligned, any contents
};
uint64_t balance_scratch_bytes(int64_t tokens, int64_t experts, int64_t sequences);
hipError_t balance(const BalanceArgs& args, hipStream_t stream);

struct BalanceBackwardArgs {
  const void* logits;
  int dt;
  bool sigmoid;
  int64_t tokens;
  int32_t experts, sequences;
  const int32_t* offsets;
  const uint8_t* mask;
  const float *share, *inverse;          // as balance wrote them
  const float *balance_grad, *z_grad;    // one number each, or null
  void* logits_grad;                     // (tokens, experts), element type dt
};
hipError_t balance_backward(const BalanceBackwardArgs& args, hipStream_t stream);

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

struct QuantizeArgs {
  const void* x;              // rows x_stride elements apart, element type dt (kBF16, kF16, kF32): cols of them, or gate | up
  int dt;
  bool gated;                 // silu(gate) * up of 2 * cols elements
  int64_t rows, cols, x_stride;
  const int32_t* row_index;   // (rows): the row of x that is meant, or null: rows in place
  int64_t x_rows;
  int8_t* q;                  // (rows, cols)
  float* scales;              // (rows)
};
hipError_t quantize(const QuantizeArgs& args, hipStream_t stream);

// One launch of the product of 8-bit integers for few rows and for any sizes (int8_product_kernels.hip): at most kMaxGroups groups.
struct Int8Args {
  const int8_t* a;            // (tokens, hidden_in)
  const float* a_scales;      // (tokens)
  const int8_t* b;            // (all groups, hidden_out, hidden_in)
  const float* b_scales;      // (all groups, hidden_out)
  void* c;                    // (tokens, hidden_out)
  bool to_f16;                // c in f16, otherwise in bf16
  const int64_t* sizes_dev;   // sizes of all groups, or null: HostSizes
  int32_t* status;            // as in GmmParams
  int64_t tokens, row_base;   // row_base: rows before first_group's (host-resident sizes)
  int32_t first_group, num_groups, hidden_in, hidden_out;
  int32_t* arrivals;          // set by int8_rows
  int32_t* parts;
};
struct HostSizes;
// Whether 32 bits count the tasks of such a call.
bool int8_rows_fit(int64_t tokens, int64_t num_groups, int64_t hidden_in, int64_t hidden_out);
// Whether it can make use of a workspace: kWsCounterBytes of zeros, left as they are found, and partial sums.
bool int8_rows_in_pieces(int64_t tokens, int64_t num_groups, int64_t hidden_in, int64_t hidden_out);
hipError_t int8_rows(Int8Args args, const HostSizes& hs, void* workspace, uint64_t workspace_bytes, hipStream_t stream);

}  // namespace gg
