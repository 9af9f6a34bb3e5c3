// PyTorch-ROCm binding of the operators around the grouped GEMM: checks of the tensors, outputs and scratch from
// torch's allocator, one call into the C ABI on torch's current stream.
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/extension.h>

#include <tuple>

#include "../../include/grouped_gemm_hip.h"

namespace grouped_gemm {

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

}  // namespace

void RegisterOperators(pybind11::module_& m) {
  m.def("route", &Route, "weights, chosen experts, batch_sizes, row_index, order and mass of router logits.");
  m.def("moe_few_tokens", &MoeFewTokens, "A gated expert layer for a few tokens.");
  m.attr("moe_few_tokens_max") = GG_FEW_TOKENS_MAX;
  m.def("lora", &Lora, "base + scale * (x @ a^T) @ b^T, with the adapter of each row.");
  m.attr("lora_max_rank") = GG_LORA_MAX_RANK;
  m.attr("route_max_experts") = GG_ROUTE_MAX_EXPERTS;
  m.attr("route_max_top_k") = GG_ROUTE_MAX_TOP_K;
}

}  // namespace grouped_gemm
