// PyTorch-ROCm binding of the operators around the grouped GEMM: checks of the tensors, outputs and scratch from
// torch's allocator, one call into the C ABI on torch's current stream.
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/extension.h>

#include <tuple>

#include "../../include/grouped_gemm_hip.h"

namespace grouped_gemm {

// torch_binding.cpp
torch::Tensor AttachCallWorkspace(gg_gmm_args* g, uint64_t bytes, const torch::Device& device, void* stream);
int32_t* CallSizeStatusWord();

namespace {

void* CurrentStream(const torch::Device& device) {
  return static_cast<void*>(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(device.index()).stream());
}

torch::Tensor Scratch(uint64_t bytes, const torch::Tensor& like) {
  if (bytes == 0) return torch::Tensor();
  return torch::empty({(int64_t)bytes}, like.options().dtype(torch::kUInt8).requires_grad(false));
}

void* Pointer(const torch::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// Kernels see values only: a tangent that came in would be dropped without a word (in any mode of gradients, which forward mode does not heed).
void RefuseTangents(std::initializer_list<const torch::Tensor*> tensors, const char* name) {
  for (const torch::Tensor* t : tensors)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), "grouped_gemm: ", name, " has no forward-mode derivative");
}

// torch hands a leaf's gradient over on the stream where a graph of the leaf was first made, as long as one lives.  From a captured backward pass to the
// default stream, which a capture cannot wait for, that ends the process: an error here, before torch gets there.
void RefuseLivingGraph(const torch::Tensor& leaf, const char* name) {
  if (!leaf.is_leaf()) return;
  const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(leaf);
  if (accumulator == nullptr) return;
  const auto made_on = accumulator->stream();
  if (!made_on.has_value() || made_on->id() != 0) return;   // (0: the default one)
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(static_cast<hipStream_t>(CurrentStream(leaf.device())), &status) != hipSuccess) {
    (void)hipGetLastError();
    return;
  }
  TORCH_CHECK(status == hipStreamCaptureStatusNone, "grouped_gemm: a captured backward pass of ", name,
              " cannot reach a leaf of which a graph made outside the capture still lives: free what that graph returned first");
}

// ------------------------------------------------------------------ router

int LogitsType(torch::ScalarType t) {
  return t == torch::kFloat32 ? GG_DTYPE_F32 : (t == torch::kFloat16 ? GG_DTYPE_F16 : GG_DTYPE_BF16);
}

int Score(const std::string& score) {
  TORCH_CHECK(score == "softmax" || score == "sigmoid", "grouped_gemm: score must be 'softmax' or 'sigmoid'");
  return score == "softmax" ? GG_SCORE_SOFTMAX : GG_SCORE_SIGMOID;
}

void CheckLogits(const torch::Tensor& logits, int64_t top_k) {
  TORCH_CHECK(logits.dim() == 2, "grouped_gemm: logits must be 2-d (tokens, experts)");
  TORCH_CHECK(logits.scalar_type() == torch::kFloat32 || logits.scalar_type() == torch::kBFloat16 ||
                  logits.scalar_type() == torch::kFloat16,
              "grouped_gemm: logits must be float32, bfloat16 or float16");
  TORCH_CHECK(logits.is_contiguous(), "grouped_gemm: logits must be contiguous");
  TORCH_CHECK(top_k >= 1 && top_k <= logits.size(1), "grouped_gemm: top_k must be between 1 and the number of experts");
  TORCH_CHECK(logits.size(1) <= GG_ROUTE_MAX_EXPERTS && top_k <= GG_ROUTE_MAX_TOP_K, "grouped_gemm: at most ",
              GG_ROUTE_MAX_EXPERTS, " experts and a top_k of at most ", GG_ROUTE_MAX_TOP_K);
  TORCH_CHECK(logits.is_cuda(), "grouped_gemm: logits must be a GPU tensor");
}

// weights, chosen, batch_sizes, row_index, order, mass (undefined where it is not wanted)
torch::autograd::variable_list RunRoute(const torch::Tensor& logits, int64_t top_k, int score, bool normalize, bool with_mass) {
  c10::hip::HIPGuardMasqueradingAsCUDA guard(logits.device());
  const int64_t tokens = logits.size(0), experts = logits.size(1);
  const auto f32 = logits.options().dtype(torch::kFloat32).requires_grad(false);
  const auto i32 = f32.dtype(torch::kInt32);
  torch::Tensor weights = torch::empty({tokens, top_k}, f32), chosen = torch::empty({tokens, top_k}, i32);
  torch::Tensor batch_sizes = torch::empty({experts}, f32.dtype(torch::kInt64));
  torch::Tensor row_index = torch::empty({tokens * top_k}, i32), order = torch::empty({tokens * top_k}, i32);
  torch::Tensor mass = with_mass ? torch::empty({experts}, f32) : torch::Tensor();
  const torch::Tensor scratch = Scratch(gg_route_scratch_bytes(tokens, experts, top_k), weights);
  const int rc = gg_route(logits.data_ptr(), LogitsType(logits.scalar_type()), tokens, experts, top_k, score, normalize,
                          weights.data_ptr<float>(), chosen.data_ptr<int32_t>(), batch_sizes.data_ptr<int64_t>(),
                          row_index.data_ptr<int32_t>(), order.data_ptr<int32_t>(), static_cast<float*>(Pointer(mass)),
                          Pointer(scratch), CurrentStream(logits.device()));
  TORCH_CHECK(rc == GG_OK, "grouped_gemm: ", gg_last_error());
  return {weights, chosen, batch_sizes, row_index, order, mass};
}

torch::Tensor RunRouteBackward(const torch::Tensor& logits, const torch::Tensor& chosen, torch::Tensor weights_grad, torch::Tensor mass_grad,
                               int score, bool normalize) {
  c10::hip::HIPGuardMasqueradingAsCUDA guard(logits.device());
  if (weights_grad.defined()) weights_grad = weights_grad.contiguous();
  if (mass_grad.defined()) mass_grad = mass_grad.contiguous();
  torch::Tensor out = torch::empty(logits.sizes(), logits.options().requires_grad(false));
  const int rc = gg_route_backward(logits.data_ptr(), LogitsType(logits.scalar_type()), logits.size(0), logits.size(1), chosen.size(1), score,
                                   normalize, chosen.data_ptr<int32_t>(), static_cast<const float*>(Pointer(weights_grad)),
                                   static_cast<const float*>(Pointer(mass_grad)), out.data_ptr(), CurrentStream(logits.device()));
  TORCH_CHECK(rc == GG_OK, "grouped_gemm: ", gg_last_error());
  return out;
}

// The gradient where a graph of it is wanted (create_graph): a second derivative through it is an error, not a silent zero.
class RouteGradientNode : public torch::autograd::Function<RouteGradientNode> {
 public:
  static torch::Tensor forward(torch::autograd::AutogradContext*, const torch::Tensor& logits, const torch::Tensor& chosen,
                               const c10::optional<torch::Tensor>& weights_grad, const c10::optional<torch::Tensor>& mass_grad, int64_t score,
                               bool normalize) {
    return RunRouteBackward(logits, chosen, weights_grad.value_or(torch::Tensor()), mass_grad.value_or(torch::Tensor()), (int)score, normalize);
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext*, torch::autograd::variable_list) {
    TORCH_CHECK(false, "grouped_gemm: route has no second derivative");
  }
};

class RouteNode : public torch::autograd::Function<RouteNode> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const torch::Tensor& logits, int64_t top_k,
                                                int64_t score, bool normalize, bool with_mass) {
    auto out = RunRoute(logits, top_k, (int)score, normalize, with_mass);
    ctx->save_for_backward({logits, out[1]});
    ctx->saved_data["score"] = score;
    ctx->saved_data["normalize"] = normalize;
    ctx->mark_non_differentiable({out[1], out[2], out[3], out[4]});
    ctx->set_materialize_grads(false);
    if (!with_mass) out.pop_back();
    return out;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const torch::Tensor &logits = saved[0], &chosen = saved[1];
    const torch::Tensor weights_grad = grads[0], mass_grad = grads.size() > 5 ? grads[5] : torch::Tensor(), none;
    if (!weights_grad.defined() && !mass_grad.defined()) return {none, none, none, none, none};
    RefuseTangents({&weights_grad, &mass_grad}, "the gradient of route");
    RefuseLivingGraph(logits, "route");
    const int64_t score = ctx->saved_data["score"].toInt();
    const bool normalize = ctx->saved_data["normalize"].toBool();
    torch::Tensor out;
    if (torch::GradMode::is_enabled()) {
      const auto given = [](const torch::Tensor& t) { return t.defined() ? c10::optional<torch::Tensor>(t) : c10::nullopt; };
      out = RouteGradientNode::apply(logits, chosen, given(weights_grad), given(mass_grad), score, normalize);
    } else {
      out = RunRouteBackward(logits, chosen, weights_grad, mass_grad, (int)score, normalize);
    }
    return {out, none, none, none, none};
  }
};

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor, c10::optional<torch::Tensor>> Route(
    const torch::Tensor& logits, int64_t top_k, const std::string& score, bool normalize, bool with_mass) {
  const int which = Score(score);
  CheckLogits(logits, top_k);
  RefuseTangents({&logits}, "route");
  torch::autograd::variable_list out;
  if (torch::GradMode::is_enabled() && logits.requires_grad()) {
    out = RouteNode::apply(logits, top_k, (int64_t)which, normalize, with_mass);
  } else {
    out = RunRoute(logits, top_k, which, normalize, with_mass);
  }
  c10::optional<torch::Tensor> mass;
  if (with_mass) mass = out[5];
  return {out[0], out[1], out[2], out[3], out[4], mass};
}

// ------------------------------------------------------------------ balance loss

struct BalanceInputs {
  torch::Tensor logits, offsets, mask;   // the last two undefined: one sequence, every token counts
  int score;
  int64_t sequences() const { return offsets.defined() ? offsets.size(0) - 1 : 1; }
  const int32_t* offsets_data() const { return static_cast<const int32_t*>(Pointer(offsets)); }
  const uint8_t* mask_data() const { return static_cast<const uint8_t*>(Pointer(mask)); }
};

// balance, z, counts, and what the gradient takes besides the inputs: (sequences, experts) shares, and behind them the inverse of the tokens' number
torch::autograd::variable_list RunBalance(const BalanceInputs& in, const torch::Tensor& chosen) {
  const torch::Tensor& logits = in.logits;
  c10::hip::HIPGuardMasqueradingAsCUDA guard(logits.device());
  const int64_t tokens = logits.size(0), experts = logits.size(1);
  const auto f32 = logits.options().dtype(torch::kFloat32).requires_grad(false);
  const int64_t shares = in.sequences() * experts;
  torch::Tensor balance = torch::empty({}, f32), z = torch::empty({}, f32), kept = torch::empty({shares + 1}, f32);
  torch::Tensor counts = torch::empty({in.sequences(), experts}, f32.dtype(torch::kInt32));
  const torch::Tensor scratch = Scratch(gg_balance_scratch_bytes(tokens, experts, chosen.size(1), in.sequences()), balance);
  const int rc = gg_balance(logits.data_ptr(), LogitsType(logits.scalar_type()), tokens, experts, chosen.size(1), in.score,
                            chosen.data_ptr<int32_t>(), in.offsets_data(), in.sequences(), in.mask_data(), balance.data_ptr<float>(),
                            z.data_ptr<float>(), counts.data_ptr<int32_t>(), kept.data_ptr<float>(), kept.data_ptr<float>() + shares, Pointer(scratch),
                            CurrentStream(logits.device()));
  TORCH_CHECK(rc == GG_OK, "grouped_gemm: ", gg_last_error());
  return {balance, z, counts, kept};
}

torch::Tensor RunBalanceBackward(const BalanceInputs& in, const torch::Tensor& kept, torch::Tensor balance_grad, torch::Tensor z_grad) {
  const torch::Tensor& logits = in.logits;
  c10::hip::HIPGuardMasqueradingAsCUDA guard(logits.device());
  torch::Tensor out = torch::empty(logits.sizes(), logits.options().requires_grad(false));
  const int rc = gg_balance_backward(logits.data_ptr(), LogitsType(logits.scalar_type()), logits.size(0), logits.size(1), in.score, in.offsets_data(),
                                     in.sequences(), in.mask_data(), kept.data_ptr<float>(), kept.data_ptr<float>() + in.sequences() * logits.size(1),
                                     static_cast<const float*>(Pointer(balance_grad)), static_cast<const float*>(Pointer(z_grad)), out.data_ptr(),
                                     CurrentStream(logits.device()));
  TORCH_CHECK(rc == GG_OK, "grouped_gemm: ", gg_last_error());
  return out;
}

c10::optional<torch::Tensor> Given(const torch::Tensor& t) { return t.defined() ? c10::optional<torch::Tensor>(t) : c10::nullopt; }

// (as RouteGradientNode)
class BalanceGradientNode : public torch::autograd::Function<BalanceGradientNode> {
 public:
  static torch::Tensor forward(torch::autograd::AutogradContext*, const torch::Tensor& logits, const torch::Tensor& kept,
                               const c10::optional<torch::Tensor>& offsets, const c10::optional<torch::Tensor>& mask,
                               const c10::optional<torch::Tensor>& balance_grad, const c10::optional<torch::Tensor>& z_grad, int64_t score) {
    const torch::Tensor none;
    return RunBalanceBackward({logits, offsets.value_or(none), mask.value_or(none), (int)score}, kept, balance_grad.value_or(none),
                              z_grad.value_or(none));
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext*, torch::autograd::variable_list) {
    TORCH_CHECK(false, "grouped_gemm: balance_loss has no second derivative");
  }
};

class BalanceNode : public torch::autograd::Function<BalanceNode> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const torch::Tensor& logits, const torch::Tensor& chosen,
                                                const c10::optional<torch::Tensor>& offsets, const c10::optional<torch::Tensor>& mask, int64_t score) {
    const BalanceInputs in = {logits, offsets.value_or(torch::Tensor()), mask.value_or(torch::Tensor()), (int)score};
    auto out = RunBalance(in, chosen);
    ctx->save_for_backward({logits, in.offsets, in.mask, out[3]});
    ctx->saved_data["score"] = score;
    ctx->mark_non_differentiable({out[2]});
    ctx->set_materialize_grads(false);
    out.resize(3);
    return out;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const torch::Tensor &balance_grad = grads[0], &z_grad = grads[1], none;
    if (!balance_grad.defined() && !z_grad.defined()) return {none, none, none, none, none};
    RefuseTangents({&balance_grad, &z_grad}, "the gradient of balance_loss");
    RefuseLivingGraph(saved[0], "balance_loss");
    const BalanceInputs in = {saved[0], saved[1], saved[2], (int)ctx->saved_data["score"].toInt()};
    torch::Tensor out;
    if (torch::GradMode::is_enabled()) {
      out = BalanceGradientNode::apply(in.logits, saved[3], Given(in.offsets), Given(in.mask), Given(balance_grad), Given(z_grad), (int64_t)in.score);
    } else {
      out = RunBalanceBackward(in, saved[3], balance_grad, z_grad);
    }
    return {out, none, none, none, none};
  }
};

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> BalanceLoss(const torch::Tensor& logits, const torch::Tensor& experts,
                                                                    const c10::optional<torch::Tensor>& offsets,
                                                                    const c10::optional<torch::Tensor>& mask, const std::string& score) {
  const int which = Score(score);
  TORCH_CHECK(experts.dim() == 2 && experts.scalar_type() == torch::kInt32, "grouped_gemm: experts must be int32 (tokens, top_k)");
  TORCH_CHECK(logits.dim() != 2 || experts.size(0) == logits.size(0), "grouped_gemm: experts must be int32 (tokens, top_k), a row to each of logits");
  TORCH_CHECK(experts.is_contiguous(), "grouped_gemm: experts must be contiguous");
  CheckLogits(logits, experts.size(1));
  TORCH_CHECK(experts.device() == logits.device(), "grouped_gemm: logits and experts must be on the same GPU");
  if (offsets.has_value())
    TORCH_CHECK(offsets->dim() == 1 && offsets->size(0) >= 1 && offsets->scalar_type() == torch::kInt32 && offsets->is_contiguous() &&
                    offsets->device() == logits.device(),
                "grouped_gemm: offsets must be int32 (sequences + 1), contiguous and on the logits' GPU");
  if (mask.has_value())
    TORCH_CHECK(mask->dim() == 1 && mask->size(0) == logits.size(0) && mask->scalar_type() == torch::kBool && mask->is_contiguous() &&
                    mask->device() == logits.device(),
                "grouped_gemm: mask must be bool (tokens), contiguous and on the logits' GPU");
  RefuseTangents({&logits}, "balance_loss");
  torch::autograd::variable_list out;
  if (torch::GradMode::is_enabled() && logits.requires_grad()) {
    out = BalanceNode::apply(logits, experts, offsets, mask, (int64_t)which);
  } else {
    out = RunBalance({logits, offsets.value_or(torch::Tensor()), mask.value_or(torch::Tensor()), which}, experts);
  }
  return {out[0], out[1], out[2]};
}

// ------------------------------------------------------------------ gated expert layer for a few tokens

bool IsTwoByte(const torch::Tensor& t) { return t.scalar_type() == torch::kBFloat16 || t.scalar_type() == torch::kFloat16; }

// Operators for serving have no gradient: a graph that asks for one is an error, not a silent zero.
void RefuseGradients(std::initializer_list<const torch::Tensor*> tensors, const char* name, const char* instead) {
  RefuseTangents(tensors, name);
  if (!torch::GradMode::is_enabled()) return;
  for (const torch::Tensor* t : tensors)
    TORCH_CHECK(!t->defined() || !t->requires_grad(), "grouped_gemm: ", name, " has no gradient (", instead, ")");
}

torch::Tensor MoeFewTokens(const torch::Tensor& x, const torch::Tensor& w13, const torch::Tensor& w2, const torch::Tensor& experts,
                           const torch::Tensor& weights, bool trans_b) {
  TORCH_CHECK(x.dim() == 2, "grouped_gemm: x must be 2-d (tokens, hidden)");
  TORCH_CHECK(IsTwoByte(x), "grouped_gemm: x must be bfloat16 or float16");
  TORCH_CHECK(w13.dim() == 3 && w2.dim() == 3, "grouped_gemm: w13 and w2 must be 3-d");
  TORCH_CHECK(w13.scalar_type() == x.scalar_type() && w2.scalar_type() == x.scalar_type(),
              "grouped_gemm: w13 and w2 must have the element type of x");
  const int64_t tokens = x.size(0), hidden = x.size(1), num = w13.size(0), both = w13.size(trans_b ? 1 : 2);
  TORCH_CHECK(w13.size(trans_b ? 2 : 1) == hidden, "grouped_gemm: contraction dimensions of x and w13 differ");
  TORCH_CHECK(both % 2 == 0, "grouped_gemm: w13 must hold gate | up, an even number of columns");
  TORCH_CHECK(w2.size(0) == num && w2.size(trans_b ? 2 : 1) == both / 2 && w2.size(trans_b ? 1 : 2) == hidden,
              "grouped_gemm: w2 must take gate's columns back to the columns of x, for as many experts as w13");
  TORCH_CHECK(experts.dim() == 2 && experts.size(0) == tokens && experts.scalar_type() == torch::kInt32,
              "grouped_gemm: experts must be int32 (tokens, top_k)");
  TORCH_CHECK(weights.sizes() == experts.sizes() && weights.scalar_type() == torch::kFloat32,
              "grouped_gemm: weights must be float32, of the shape of experts");
  TORCH_CHECK(tokens <= GG_FEW_TOKENS_MAX, "grouped_gemm: at most ", GG_FEW_TOKENS_MAX,
              " tokens (more belong in gmm_swiglu and gmm_scatter with the indices of route)");
  for (const torch::Tensor* t : {&x, &w13, &w2, &experts, &weights})
    TORCH_CHECK(t->is_contiguous(), "grouped_gemm: x, w13, w2, experts and weights must be contiguous");
  for (const torch::Tensor* t : {&x, &w13, &w2, &experts, &weights})
    TORCH_CHECK(t->is_cuda() && t->device() == x.device(), "grouped_gemm: x, w13, w2, experts and weights must be on the same GPU");
  RefuseGradients({&x, &w13, &w2, &weights}, "moe_few_tokens", "train through gmm_swiglu and gmm_scatter");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  torch::Tensor out = torch::empty({tokens, hidden}, x.options().requires_grad(false));
  if (tokens == 0) return out;
  const torch::Tensor scratch =
      Scratch(gg_moe_few_tokens_scratch_bytes(tokens, num, experts.size(1), hidden, both / 2, trans_b), out);
  const int rc = gg_moe_few_tokens(x.data_ptr(), w13.data_ptr(), w2.data_ptr(), experts.data_ptr<int32_t>(),
                                   weights.data_ptr<float>(), out.data_ptr(), x.scalar_type() == torch::kFloat16 ? GG_DTYPE_F16 : GG_DTYPE_BF16,
                                   tokens, num, experts.size(1), hidden, both / 2, trans_b, Pointer(scratch), CurrentStream(x.device()));
  TORCH_CHECK(rc == GG_OK, "grouped_gemm: ", gg_last_error());
  return out;
}

// ------------------------------------------------------------------ low-rank adapters

bool Overlap(const torch::Tensor& t, const torch::Tensor& u) {
  const auto begin = [](const torch::Tensor& v) { return reinterpret_cast<uintptr_t>(v.data_ptr()); };
  return begin(t) < begin(u) + u.nbytes() && begin(u) < begin(t) + t.nbytes();
}

torch::Tensor Lora(const torch::Tensor& x, const torch::Tensor& a, const torch::Tensor& b, const torch::Tensor& adapters,
                   const c10::optional<torch::Tensor>& base, const c10::optional<torch::Tensor>& scales,
                   const c10::optional<torch::Tensor>& c) {
  TORCH_CHECK(x.dim() == 2, "grouped_gemm: x must be 2-d (rows, hidden_in)");
  TORCH_CHECK(IsTwoByte(x), "grouped_gemm: x must be bfloat16 or float16");
  TORCH_CHECK(a.dim() == 3 && b.dim() == 3, "grouped_gemm: a and b must be 3-d");
  TORCH_CHECK(a.scalar_type() == x.scalar_type() && b.scalar_type() == x.scalar_type(),
              "grouped_gemm: a and b must have the element type of x");
  const int64_t rows = x.size(0), num = a.size(0), rank = a.size(1), hidden_in = x.size(1), hidden_out = b.size(1);
  TORCH_CHECK(a.size(2) == hidden_in, "grouped_gemm: a must be (adapters, rank, hidden_in)");
  TORCH_CHECK(b.size(0) == num && b.size(2) == rank, "grouped_gemm: b must be (adapters, hidden_out, rank)");
  TORCH_CHECK(rank <= GG_LORA_MAX_RANK, "grouped_gemm: a rank of at most ", GG_LORA_MAX_RANK);
  TORCH_CHECK(adapters.dim() == 1 && adapters.size(0) == rows && adapters.scalar_type() == torch::kInt32,
              "grouped_gemm: adapters must be int32, one number per row of x");
  if (scales.has_value())
    TORCH_CHECK(scales->dim() == 1 && scales->size(0) == num && scales->scalar_type() == torch::kFloat32,
                "grouped_gemm: scales must be float32, one per adapter");
  torch::Tensor none;
  const torch::Tensor &from = base.has_value() ? *base : none, &scale = scales.has_value() ? *scales : none, &to = c.has_value() ? *c : none;
  for (const torch::Tensor* t : {&from, &to})
    TORCH_CHECK(!t->defined() || (t->dim() == 2 && t->size(0) == rows && t->size(1) == hidden_out && t->scalar_type() == x.scalar_type()),
                "grouped_gemm: base and c must be (rows, hidden_out), of the element type of x");
  for (const torch::Tensor* t : {&x, &a, &b, &adapters, &from, &scale, &to})
    TORCH_CHECK(!t->defined() || t->is_contiguous(), "grouped_gemm: x, a, b, adapters, base, scales and c must be contiguous");
  for (const torch::Tensor* t : {&x, &a, &b, &adapters, &from, &scale, &to})
    TORCH_CHECK(!t->defined() || (t->is_cuda() && t->device() == x.device()),
                "grouped_gemm: x, a, b, adapters, base, scales and c must be on the same GPU");
  RefuseGradients({&x, &a, &b, &from, &scale, &to}, "lora", "train adapters through gmm, on rows sorted by adapter");
  if (to.defined()) {
    for (const torch::Tensor* t : {&x, &a, &b, &adapters, &scale})
      TORCH_CHECK(!t->defined() || !Overlap(*t, to), "grouped_gemm: c must not overlap x, a, b, adapters or scales");
    TORCH_CHECK(!from.defined() || from.data_ptr() == to.data_ptr() || !Overlap(from, to), "grouped_gemm: c must be base or not overlap it");
  }
  c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  torch::Tensor out = to.defined() ? to : torch::empty({rows, hidden_out}, x.options().requires_grad(false));
  if (rows == 0) return out;
  const torch::Tensor scratch = Scratch(gg_lora_scratch_bytes(rows, num, rank, hidden_in, hidden_out), out);
  const int rc = gg_lora(x.data_ptr(), a.data_ptr(), b.data_ptr(), adapters.data_ptr<int32_t>(), static_cast<const float*>(Pointer(scale)),
                         Pointer(from), out.data_ptr(), x.scalar_type() == torch::kFloat16 ? GG_DTYPE_F16 : GG_DTYPE_BF16, rows, num, rank,
                         hidden_in, hidden_out, Pointer(scratch), CurrentStream(x.device()));
  TORCH_CHECK(rc == GG_OK, "grouped_gemm: ", gg_last_error());
  if (to.defined() && !to.is_inference()) to.unsafeGetTensorImpl()->bump_version();   // (a write that a graph which saved c has to notice)
  return out;
}

// ------------------------------------------------------------------ 8-bit integers

void CheckQuantized(const torch::Tensor& x, const char* what) {
  TORCH_CHECK(x.scalar_type() == torch::kFloat32 || x.scalar_type() == torch::kBFloat16 || x.scalar_type() == torch::kFloat16, "grouped_gemm: ", what,
              " must be float32, bfloat16 or float16");
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, "grouped_gemm: ", what, " must have rows of at least one element");
  // (rows may lie further apart than they are long)
  TORCH_CHECK(x.is_contiguous() || (x.dim() == 2 && x.stride(1) == 1 && (x.size(0) <= 1 || x.stride(0) >= x.size(1))), "grouped_gemm: ", what,
              " must be contiguous, or 2-d with contiguous rows that do not overlap");
  TORCH_CHECK(x.is_cuda(), "grouped_gemm: ", what, " must be a GPU tensor");
}

int64_t RowStride(const torch::Tensor& x) { return !x.is_contiguous() ? x.stride(0) : x.size(-1); }

std::tuple<torch::Tensor, torch::Tensor> QuantizeRows(const torch::Tensor& x, const c10::optional<torch::Tensor>& row_index) {
  CheckQuantized(x, "x");
  if (row_index.has_value()) {
    TORCH_CHECK(x.dim() == 2, "grouped_gemm: with row_index, x must be 2-d");
    TORCH_CHECK(row_index->dim() == 1 && row_index->scalar_type() == torch::kInt32 && row_index->is_contiguous() && row_index->device() == x.device(),
                "grouped_gemm: row_index must be a contiguous 1-d int32 tensor on x's GPU");
  }
  RefuseGradients({&x}, "quantize_rows", "round to 8 bits what is served, not what is trained");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  const int64_t cols = x.size(-1), x_rows = x.numel() / cols, rows = row_index.has_value() ? row_index->size(0) : x_rows;
  std::vector<int64_t> shape = x.sizes().vec(), of_scales(shape.begin(), shape.end() - 1);
  if (row_index.has_value()) shape = {rows, cols}, of_scales = {rows};
  const auto options = x.options().requires_grad(false);
  torch::Tensor q = torch::empty(shape, options.dtype(torch::kInt8)), scales = torch::empty(of_scales, options.dtype(torch::kFloat32));
  const int rc = gg_quantize_rows(x.data_ptr(), LogitsType(x.scalar_type()), rows, cols, RowStride(x),
                                  row_index.has_value() ? row_index->data_ptr<int32_t>() : nullptr, x_rows, q.data_ptr<int8_t>(),
                                  scales.data_ptr<float>(), CurrentStream(x.device()));
  TORCH_CHECK(rc == GG_OK, "grouped_gemm: ", gg_last_error());
  return {q, scales};
}

std::tuple<torch::Tensor, torch::Tensor> SwigluQuantize(const torch::Tensor& gate_up) {
  CheckQuantized(gate_up, "gate_up");
  TORCH_CHECK(gate_up.size(-1) % 2 == 0, "grouped_gemm: gate_up must hold gate | up, an even number of columns");
  RefuseGradients({&gate_up}, "swiglu_quantize", "round to 8 bits what is served, not what is trained");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(gate_up.device());
  const int64_t cols = gate_up.size(-1) / 2, rows = gate_up.numel() / (2 * cols);
  std::vector<int64_t> shape = gate_up.sizes().vec(), of_scales(shape.begin(), shape.end() - 1);
  shape.back() = cols;
  const auto options = gate_up.options().requires_grad(false);
  torch::Tensor q = torch::empty(shape, options.dtype(torch::kInt8)), scales = torch::empty(of_scales, options.dtype(torch::kFloat32));
  const int rc = gg_swiglu_quantize(gate_up.data_ptr(), LogitsType(gate_up.scalar_type()), rows, cols, RowStride(gate_up), q.data_ptr<int8_t>(),
                                    scales.data_ptr<float>(), CurrentStream(gate_up.device()));
  TORCH_CHECK(rc == GG_OK, "grouped_gemm: ", gg_last_error());
  return {q, scales};
}

constexpr int64_t kInt8PadRows = 128;   // average rows to a group

torch::Tensor GmmInt8(const torch::Tensor& a, const torch::Tensor& a_scales, const torch::Tensor& b, const torch::Tensor& b_scales,
                      const torch::Tensor& batch_sizes, bool to_f16, const c10::optional<torch::Tensor>& c) {
  TORCH_CHECK(a.dim() == 2 && a.scalar_type() == torch::kInt8, "grouped_gemm: a must be int8 (tokens, hidden_in)");
  TORCH_CHECK(b.dim() == 3 && b.scalar_type() == torch::kInt8, "grouped_gemm: b must be int8 (experts, hidden_out, hidden_in)");
  const int64_t tokens = a.size(0), hidden_in = a.size(1), experts = b.size(0), hidden_out = b.size(1);
  TORCH_CHECK(b.size(2) == hidden_in, "grouped_gemm: contraction dimensions of a and b differ");
  TORCH_CHECK(a_scales.dim() == 1 && a_scales.size(0) == tokens && a_scales.scalar_type() == torch::kFloat32,
              "grouped_gemm: a_scales must be float32, one per row of a");
  TORCH_CHECK(b_scales.dim() == 2 && b_scales.size(0) == experts && b_scales.size(1) == hidden_out && b_scales.scalar_type() == torch::kFloat32,
              "grouped_gemm: b_scales must be float32 (experts, hidden_out)");
  TORCH_CHECK(batch_sizes.dim() == 1 && batch_sizes.size(0) == experts && batch_sizes.scalar_type() == torch::kInt64,
              "grouped_gemm: batch_sizes must be int64, one per expert");
  TORCH_CHECK(batch_sizes.is_cpu() || batch_sizes.is_contiguous(), "grouped_gemm: batch_sizes must be contiguous");
  const torch::Tensor none, &to = c.has_value() ? *c : none;
  const auto type = to_f16 ? torch::kFloat16 : torch::kBFloat16;
  if (to.defined())
    TORCH_CHECK(to.dim() == 2 && to.size(0) == tokens && to.size(1) == hidden_out && to.scalar_type() == type,
                "grouped_gemm: c must be (tokens, hidden_out), of the type asked for");
  for (const torch::Tensor* t : {&a, &a_scales, &b, &b_scales, &to})
    TORCH_CHECK(!t->defined() || t->is_contiguous(), "grouped_gemm: a, a_scales, b, b_scales and c must be contiguous");
  for (const torch::Tensor* t : {&a, &a_scales, &b, &b_scales, &to})
    TORCH_CHECK(!t->defined() || (t->is_cuda() && t->device() == a.device()), "grouped_gemm: a, a_scales, b, b_scales and c must be on the same GPU");
  TORCH_CHECK(batch_sizes.is_cpu() || batch_sizes.device() == a.device(), "grouped_gemm: batch_sizes must be on the host or on a's GPU");
  RefuseGradients({&a_scales, &b_scales, &to}, "gmm_int8", "train through gmm");
  if (to.defined())
    for (const torch::Tensor* t : {&a, &a_scales, &b, &b_scales, &batch_sizes})
      TORCH_CHECK(!Overlap(*t, to), "grouped_gemm: c must not overlap a, b, their scales or batch_sizes");
  const torch::Tensor sizes = batch_sizes.is_cpu() ? batch_sizes.contiguous() : batch_sizes;
  c10::hip::HIPGuardMasqueradingAsCUDA guard(a.device());
  torch::Tensor out = to.defined() ? to : torch::empty({tokens, hidden_out}, a.options().dtype(type));
  TORCH_CHECK(gg_init() == GG_OK, "grouped_gemm: ", gg_last_error());
  torch::Tensor lhs = a, rhs = b;
  int64_t depth = hidden_in;
  // Rows that do not begin on boundaries of 16 bytes are read by the kernel for few rows, at a third of the streaming kernel's rate; with this many
  // of them it pays to lay them out again, with zeros behind.  us, padded / as they are, by rows to a group: 8 groups,
  // 2047 -> 1023: 64 27 / 19, 128 27 / 29, 256 31 / 48, 1024 53 / 117; 8, 4095 -> 4097: 96 95 / 97, 128 93 / 123, 1024 223 / 686; 64, 2047 -> 1407: 64 127 /
  // 117, 128 143 / 179; 32, 4095 -> 2047: 96 209 / 181, 128 214 / 241; 8, 1021 -> 1021: 128 23 / 19, 256 24 / 30.
  const bool aligned = hidden_in % 16 == 0 && ((reinterpret_cast<uintptr_t>(a.data_ptr()) | reinterpret_cast<uintptr_t>(b.data_ptr())) & 15) == 0;
  const int64_t padded = (hidden_in + 15) / 16 * 16;
  if (!aligned && experts > 0 && tokens >= kInt8PadRows * experts && hidden_in > 0 && hidden_out > 0 && padded <= GG_INT8_MAX_DEPTH) {
    depth = padded;
    lhs = torch::empty({tokens, depth}, a.options());
    rhs = torch::empty({experts, hidden_out, depth}, a.options());
    int rc = gg_pad_rows(a.data_ptr(), lhs.data_ptr(), 1, tokens, hidden_in, tokens, depth, 1, CurrentStream(a.device()));
    if (rc == GG_OK) rc = gg_pad_rows(b.data_ptr(), rhs.data_ptr(), 1, experts * hidden_out, hidden_in, experts * hidden_out, depth, 1, CurrentStream(a.device()));
    TORCH_CHECK(rc == GG_OK, "grouped_gemm: ", gg_last_error());
  }
  gg_gmm_args g = {};
  g.struct_bytes = sizeof(g);
  g.dtype = to_f16 ? GG_DTYPE_F16 : GG_DTYPE_BF16;
  g.a = lhs.data_ptr();
  g.b = rhs.data_ptr();
  g.c = out.data_ptr();
  g.batch_sizes = sizes.data_ptr<int64_t>();
  g.batch_sizes_on_device = sizes.is_cuda() ? 1 : 0;
  g.trans_b = 1;
  g.num_groups = experts;
  g.tokens = tokens;
  g.hidden_in = depth;
  g.hidden_out = hidden_out;
  g.stream = CurrentStream(a.device());
  if (sizes.is_cuda()) g.size_status = CallSizeStatusWord();
  const torch::Tensor workspace = AttachCallWorkspace(&g, gg_gmm_int8_workspace_bytes(&g), a.device(), g.stream);
  const int rc = gg_gmm_int8(&g, a_scales.data_ptr<float>(), b_scales.data_ptr<float>());
  TORCH_CHECK(rc == GG_OK, "grouped_gemm: ", gg_last_error());
  if (to.defined() && !to.is_inference()) to.unsafeGetTensorImpl()->bump_version();   // (as in Lora)
  return out;
}

}  // namespace

void RegisterOperators(pybind11::module_& m) {
  m.def("route", &Route, "weights, chosen experts, batch_sizes, row_index, order and mass of router logits.");
  m.def("balance_loss", &BalanceLoss, "Balance loss and z-loss of router logits, and the experts' counts.");
  m.def("quantize_rows", &QuantizeRows, "Rows as 8-bit integers, and their scales.");
  m.def("swiglu_quantize", &SwigluQuantize, "silu(gate) * up as 8-bit integers, and their scales.");
  m.def("gmm_int8", &GmmInt8, "Grouped GEMM of 8-bit integers with scales per row and column.");
  m.def("moe_few_tokens", &MoeFewTokens, "A gated expert layer for a few tokens.");
  m.attr("moe_few_tokens_max") = GG_FEW_TOKENS_MAX;
  m.def("lora", &Lora, "base + scale * (x @ a^T) @ b^T, with the adapter of each row.");
  m.attr("lora_max_rank") = GG_LORA_MAX_RANK;
  m.attr("route_max_experts") = GG_ROUTE_MAX_EXPERTS;
  m.attr("route_max_top_k") = GG_ROUTE_MAX_TOP_K;
}

}  // namespace grouped_gemm
