// Entry points of the operators around the grouped GEMM (include/grouped_gemm_hip.h): argument checks and launches.  No allocation,
// no sync.
#include "../../include/grouped_gemm_hip.h"

#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdio>

#include "operators.hpp"

namespace gg {
int set_error(int code, const char* message);   // gmm_api.hip
int prepare_device();
}  // namespace gg

namespace {

int fail(int code, const char* fmt, ...) {
  char message[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(message, sizeof(message), fmt, ap);
  va_end(ap);
  return gg::set_error(code, message);
}

#define GG_HIP(call)                                                                     \
  do {                                                                                   \
    hipError_t err__ = (call);                                                           \
    if (err__ != hipSuccess)                                                             \
      return fail(GG_EHIP, "%s failed: %s", #call, hipGetErrorString(err__));            \
  } while (0)

}  // namespace

extern "C" {

static int check_route(const void* logits, int dtype, int64_t tokens, int64_t experts, int64_t top_k, int score) {
  if (dtype != GG_DTYPE_BF16 && dtype != GG_DTYPE_F16 && dtype != GG_DTYPE_F32)
    return fail(GG_EINVAL, "dtype must be GG_DTYPE_BF16, GG_DTYPE_F16 or GG_DTYPE_F32");
  if (tokens < 0 || experts < 1 || top_k < 1) return fail(GG_EINVAL, "tokens must not be negative, experts and top_k at least 1");
  if (top_k > experts) return fail(GG_EINVAL, "top_k must not be more than experts");
  if (experts > GG_ROUTE_MAX_EXPERTS || top_k > GG_ROUTE_MAX_TOP_K)
    return fail(GG_ELIMIT, "at most %d experts, top_k at most %d", GG_ROUTE_MAX_EXPERTS, GG_ROUTE_MAX_TOP_K);
  if (tokens >= (int64_t(1) << 31) / top_k) return fail(GG_ELIMIT, "tokens * top_k must be below 2^31");
  if (score != GG_SCORE_SOFTMAX && score != GG_SCORE_SIGMOID) return fail(GG_EINVAL, "score must be one of GG_SCORE_*");
  if (tokens > 0 && logits == nullptr) return fail(GG_EINVAL, "logits is null");
  return GG_OK;
}

uint64_t gg_route_scratch_bytes(int64_t tokens, int64_t experts, int64_t top_k) {
  if (tokens < 0 || experts < 1 || top_k < 1 || experts > GG_ROUTE_MAX_EXPERTS || top_k > GG_ROUTE_MAX_TOP_K ||
      tokens >= (int64_t(1) << 31) / top_k)
    return 0;
  return gg::route_scratch_bytes(tokens, experts, top_k);
}

int gg_route(const void* logits, int dtype, int64_t tokens, int64_t experts, int64_t top_k, int score, int normalize,
             float* weights, int32_t* chosen, int64_t* batch_sizes, int32_t* row_index, int32_t* order, float* mass,
             void* scratch, void* stream) {
  const int rc = check_route(logits, dtype, tokens, experts, top_k, score);
  if (rc != GG_OK) return rc;
  if (batch_sizes == nullptr || (tokens > 0 && (weights == nullptr || chosen == nullptr || row_index == nullptr || order == nullptr)))
    return fail(GG_EINVAL, "weights, chosen, batch_sizes, row_index or order is null");
  if (scratch == nullptr && gg::route_scratch_bytes(tokens, experts, top_k) > 0) return fail(GG_EINVAL, "scratch is null");
  const int init = gg::prepare_device();
  if (init != GG_OK) return init;
  const gg::RouteArgs a = {logits, dtype, tokens, (int32_t)experts, (int32_t)top_k, score == GG_SCORE_SIGMOID, normalize != 0,
                           weights, chosen, batch_sizes, row_index, order, mass, scratch};
  GG_HIP(gg::route(a, static_cast<hipStream_t>(stream)));
  return GG_OK;
}

int gg_route_backward(const void* logits, int dtype, int64_t tokens, int64_t experts, int64_t top_k, int score, int normalize,
                      const int32_t* chosen, const float* weights_grad, const float* mass_grad, void* logits_grad, void* stream) {
  const int rc = check_route(logits, dtype, tokens, experts, top_k, score);
  if (rc != GG_OK) return rc;
  if (tokens == 0) return GG_OK;
  if (chosen == nullptr || logits_grad == nullptr) return fail(GG_EINVAL, "chosen or logits_grad is null");
  const int init = gg::prepare_device();
  if (init != GG_OK) return init;
  const gg::RouteBackwardArgs a = {logits, dtype, tokens, (int32_t)experts, (int32_t)top_k, score == GG_SCORE_SIGMOID,
                                   normalize != 0, chosen, weights_grad, mass_grad, logits_grad};
  GG_HIP(gg::route_backward(a, static_cast<hipStream_t>(stream)));
  return GG_OK;
}

static int check_few_tokens(int dtype, int64_t tokens, int64_t experts, int64_t top_k, int64_t hidden, int64_t ffn, int trans_b) {
  if (dtype != GG_DTYPE_BF16 && dtype != GG_DTYPE_F16) return fail(GG_EINVAL, "dtype must be GG_DTYPE_BF16 or GG_DTYPE_F16");
  if (tokens < 0 || experts < 1 || top_k < 1 || hidden < 1 || ffn < 1)
    return fail(GG_EINVAL, "tokens must not be negative, experts, top_k and hidden sizes at least 1");
  if (tokens > GG_FEW_TOKENS_MAX || experts > GG_ROUTE_MAX_EXPERTS || top_k > GG_ROUTE_MAX_TOP_K)
    return fail(GG_ELIMIT, "at most %d tokens, %d experts, top_k at most %d", GG_FEW_TOKENS_MAX, GG_ROUTE_MAX_EXPERTS, GG_ROUTE_MAX_TOP_K);
  if (hidden >= (1 << 22) || ffn >= (1 << 22)) return fail(GG_ELIMIT, "hidden sizes must be below 2^22");
  if (!gg::few_tokens_fits(tokens, experts, top_k, hidden, ffn, trans_b != 0))
    return fail(GG_ELIMIT, "experts times hidden sizes are too large for one launch");
  return GG_OK;
}

uint64_t gg_moe_few_tokens_scratch_bytes(int64_t tokens, int64_t experts, int64_t top_k, int64_t hidden, int64_t ffn, int trans_b) {
  if (check_few_tokens(GG_DTYPE_BF16, tokens, experts, top_k, hidden, ffn, trans_b) != GG_OK) return 0;
  return gg::few_tokens_scratch_bytes(tokens, experts, top_k, hidden, ffn, trans_b != 0);
}

int gg_moe_few_tokens(const void* x, const void* w13, const void* w2, const int32_t* chosen, const float* weights, void* out,
                      int dtype, int64_t tokens, int64_t experts, int64_t top_k, int64_t hidden, int64_t ffn, int trans_b,
                      void* scratch, void* stream) {
  const int rc = check_few_tokens(dtype, tokens, experts, top_k, hidden, ffn, trans_b);
  if (rc != GG_OK) return rc;
  if (tokens == 0) return GG_OK;
  if (x == nullptr || w13 == nullptr || w2 == nullptr || chosen == nullptr || weights == nullptr || out == nullptr || scratch == nullptr)
    return fail(GG_EINVAL, "x, w13, w2, chosen, weights, out or scratch is null");
  if (reinterpret_cast<uintptr_t>(scratch) & 255) return fail(GG_ELIMIT, "scratch must be on a 256-byte boundary");
  const int init = gg::prepare_device();
  if (init != GG_OK) return init;
  const gg::FewTokensArgs a = {x, w13, w2, chosen, weights, out, scratch, dtype, trans_b != 0, (int32_t)tokens, (int32_t)experts,
                               (int32_t)top_k, (int32_t)hidden, (int32_t)ffn};
  GG_HIP(gg::few_tokens(a, static_cast<hipStream_t>(stream)));
  return GG_OK;
}

static int check_lora(int dtype, int64_t rows, int64_t num, int64_t rank, int64_t hidden_in, int64_t hidden_out) {
  if (dtype != GG_DTYPE_BF16 && dtype != GG_DTYPE_F16) return fail(GG_EINVAL, "dtype must be GG_DTYPE_BF16 or GG_DTYPE_F16");
  if (rows < 0 || num < 1 || rank < 1 || hidden_in < 1 || hidden_out < 1)
    return fail(GG_EINVAL, "rows must not be negative, adapters, rank and hidden sizes at least 1");
  if (rank > GG_LORA_MAX_RANK) return fail(GG_ELIMIT, "rank must be at most %d", GG_LORA_MAX_RANK);
  if (rows >= (int64_t(1) << 31) || num >= (int64_t(1) << 31)) return fail(GG_ELIMIT, "rows and adapters must be below 2^31");
  if (hidden_in >= (1 << 22) || hidden_out >= (1 << 22)) return fail(GG_ELIMIT, "hidden sizes must be below 2^22");
  if (rows > 0 && !gg::adapters_fit(rows, num, rank, hidden_in, hidden_out)) return fail(GG_ELIMIT, "rows times hidden sizes are too large for one launch");
  return GG_OK;
}

uint64_t gg_lora_scratch_bytes(int64_t rows, int64_t num, int64_t rank, int64_t hidden_in, int64_t hidden_out) {
  if (check_lora(GG_DTYPE_BF16, rows, num, rank, hidden_in, hidden_out) != GG_OK || rows == 0) return 0;
  return gg::adapters_scratch_bytes(rows, num, rank, hidden_in, hidden_out);
}

int gg_lora(const void* x, const void* a, const void* b, const int32_t* adapters, const float* scales, const void* base, void* out,
            int dtype, int64_t rows, int64_t num, int64_t rank, int64_t hidden_in, int64_t hidden_out, void* scratch, void* stream) {
  const int rc = check_lora(dtype, rows, num, rank, hidden_in, hidden_out);
  if (rc != GG_OK) return rc;
  if (rows == 0) return GG_OK;
  if (x == nullptr || a == nullptr || b == nullptr || adapters == nullptr || out == nullptr || scratch == nullptr)
    return fail(GG_EINVAL, "x, a, b, adapters, out or scratch is null");
  if (reinterpret_cast<uintptr_t>(scratch) & 15) return fail(GG_ELIMIT, "scratch must be on a 16-byte boundary");
  const int init = gg::prepare_device();
  if (init != GG_OK) return init;
  const gg::AdapterArgs args = {x, a, b, adapters, scales, base, out, scratch, dtype, rows, (int32_t)num, (int32_t)rank,
                                (int32_t)hidden_in, (int32_t)hidden_out};
  GG_HIP(gg::adapters(args, static_cast<hipStream_t>(stream)));
  return GG_OK;
}

}  // extern "C"
