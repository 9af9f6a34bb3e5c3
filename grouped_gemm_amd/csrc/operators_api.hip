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

static int check_balance(const void* logits, int dtype, int64_t tokens, int64_t experts, int64_t top_k, int score, const int32_t* offsets,
                         int64_t sequences) {
  const int rc = check_route(logits, dtype, tokens, experts, top_k, score);
  if (rc != GG_OK) return rc;
  if (sequences < 0 || (offsets == nullptr && sequences != 1)) return fail(GG_EINVAL, "sequences must not be negative, and 1 without offsets");
  if (sequences >= (int64_t(1) << 31) - 1) return fail(GG_ELIMIT, "sequences must be below 2^31 - 1");
  return GG_OK;
}

uint64_t gg_balance_scratch_bytes(int64_t tokens, int64_t experts, int64_t top_k, int64_t sequences) {
  if (tokens < 0 || experts < 1 || top_k < 1 || experts > GG_ROUTE_MAX_EXPERTS || top_k > GG_ROUTE_MAX_TOP_K || sequences < 0 ||
      tokens >= (int64_t(1) << 31) / top_k || sequences >= (int64_t(1) << 31) - 1)
    return 0;
  return gg::balance_scratch_bytes(tokens, experts, sequences);
}

int gg_balance(const void* logits, int dtype, int64_t tokens, int64_t experts, int64_t top_k, int score, const int32_t* chosen,
               const int32_t* offsets, int64_t sequences, const uint8_t* mask, float* balance, float* z, int32_t* counts, float* share,
               float* inverse, void* scratch, void* stream) {
  const int rc = check_balance(logits, dtype, tokens, experts, top_k, score, offsets, sequences);
  if (rc != GG_OK) return rc;
  if (tokens > 0 && chosen == nullptr) return fail(GG_EINVAL, "chosen is null");
  if (balance == nullptr || z == nullptr || inverse == nullptr || scratch == nullptr || (sequences > 0 && (counts == nullptr || share == nullptr)))
    return fail(GG_EINVAL, "balance, z, counts, share, inverse or scratch is null");
  const int init = gg::prepare_device();
  if (init != GG_OK) return init;
  const gg::BalanceArgs a = {logits, dtype, score == GG_SCORE_SIGMOID, tokens, (int32_t)experts, (int32_t)top_k, (int32_t)sequences, chosen,
                             offsets, mask, balance, z, counts, share, inverse, scratch};
  GG_HIP(gg::balance(a, static_cast<hipStream_t>(stream)));
  return GG_OK;
}

int gg_balance_backward(const void* logits, int dtype, int64_t tokens, int64_t experts, int score, const int32_t* offsets,
                        int64_t sequences, const uint8_t* mask, const float* share, const float* inverse, const float* balance_grad,
                        const float* z_grad, void* logits_grad, void* stream) {
  const int rc = check_balance(logits, dtype, tokens, experts, 1, score, offsets, sequences);
  if (rc != GG_OK) return rc;
  if (tokens == 0) return GG_OK;
  if (logits_grad == nullptr || inverse == nullptr || (sequences > 0 && share == nullptr)) return fail(GG_EINVAL, "logits_grad, share or inverse is null");
  const int init = gg::prepare_device();
  if (init != GG_OK) return init;
  const gg::BalanceBackwardArgs a = {logits, dtype, score == GG_SCORE_SIGMOID, tokens, (int32_t)experts, (int32_t)sequences, offsets, mask,
                                     share, inverse, balance_grad, z_grad, logits_grad};
  GG_HIP(gg::balance_backward(a, static_cast<hipStream_t>(stream)));
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

static int check_quantize(const void* x, int dtype, int64_t rows, int64_t cols, int64_t stride, int64_t least, int8_t* q, float* scales) {
  if (dtype != GG_DTYPE_BF16 && dtype != GG_DTYPE_F16 && dtype != GG_DTYPE_F32)
    return fail(GG_EINVAL, "dtype must be GG_DTYPE_BF16, GG_DTYPE_F16 or GG_DTYPE_F32");
  if (rows < 0 || cols < 1) return fail(GG_EINVAL, "rows must not be negative, cols at least 1");
  if (cols >= (1 << 22)) return fail(GG_ELIMIT, "cols must be below 2^22");
  if (rows >= (int64_t(1) << 40)) return fail(GG_ELIMIT, "rows must be below 2^40");
  if (rows > 1 && stride < least) return fail(GG_EINVAL, "rows overlap: they are closer together than they are long");
  if (stride >= (int64_t(1) << 40)) return fail(GG_ELIMIT, "rows are too far apart");
  if (rows > 0 && (q == nullptr || scales == nullptr)) return fail(GG_EINVAL, "q or scales is null");
  return GG_OK;
}

static int run_quantize(const gg::QuantizeArgs& a, void* stream) {
  const int init = gg::prepare_device();
  if (init != GG_OK) return init;
  GG_HIP(gg::quantize(a, static_cast<hipStream_t>(stream)));
  return GG_OK;
}

int gg_quantize_rows(const void* x, int dtype, int64_t rows, int64_t cols, int64_t x_stride, const int32_t* row_index, int64_t x_rows,
                     int8_t* q, float* scales, void* stream) {
  const int rc = check_quantize(x, dtype, rows, cols, x_stride, cols, q, scales);
  if (rc != GG_OK) return rc;
  if (x_rows < 0 || (row_index == nullptr && x_rows < rows)) return fail(GG_EINVAL, "x_rows must not be negative, nor without a row index below rows");
  if (rows == 0) return GG_OK;
  if (x == nullptr && x_rows > 0) return fail(GG_EINVAL, "x is null");
  return run_quantize({x, dtype, false, rows, cols, x_stride, row_index, x_rows, q, scales}, stream);
}

int gg_swiglu_quantize(const void* gate_up, int dtype, int64_t rows, int64_t cols, int64_t stride, int8_t* q, float* scales, void* stream) {
  const int rc = check_quantize(gate_up, dtype, rows, cols, stride, 2 * cols, q, scales);
  if (rc != GG_OK) return rc;
  if (rows == 0) return GG_OK;
  if (gate_up == nullptr) return fail(GG_EINVAL, "gate_up is null");
  return run_quantize({gate_up, dtype, true, rows, cols, stride, nullptr, rows, q, scales}, stream);
}

}  // extern "C"
