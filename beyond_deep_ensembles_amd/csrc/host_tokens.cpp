// Autograd nodes of the token-model operators in C++ (part of lib/_bde_host.so, beside those of host_autograd.cpp): the argument
// checks, allocations and C-ABI calls of lookup.py's and distill.py's Python path, which remains the fallback when the helper is
// not built (same kernels, same results).  No arithmetic lives in this file.
#include <torch/extension.h>
#include <c10/hip/HIPStream.h>
#include <c10/core/DeviceGuard.h>

#include <mutex>

#include "../../include/bde_hip.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void* current_stream(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// the capture a stream takes part in (0: none): one number per capture of the process
uint64_t capture_of(void* stream) { hipStreamCaptureStatus s = hipStreamCaptureStatusNone; unsigned long long id = 0; return hipStreamGetCaptureInfo(static_cast<hipStream_t>(stream), &s, &id) == hipSuccess && s != hipStreamCaptureStatusNone ? id + 1 : 0; }

// the kernels produce plain tensors: a second differentiation through a node would silently see constants
void check_once_differentiable(const variable_list& grad_outputs) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && grad_outputs[0].defined() && grad_outputs[0].requires_grad()),
              "the token-model operators are differentiable once (no double backward)");
}
at::Tensor opt(const c10::optional<at::Tensor>& t) { return t.has_value() ? *t : at::Tensor(); }

// A refused argument raises the package's own error class, as the Python path does.  (Called under the interpreter's lock only.)
template <typename... Args>
[[noreturn]] void refuse(const Args&... args) {
  const std::string text = c10::str(args...);
  py::object cls = py::module_::import("beyond_deep_ensembles_amd.ops").attr("BdeKernelError");
  PyErr_SetString(cls.ptr(), text.c_str());
  throw py::error_already_set();
}
int type_code(at::ScalarType t) { return t == at::kFloat ? BDE_F32 : t == at::kBFloat16 ? BDE_BF16 : t == at::kHalf ? BDE_F16 : -1; }
void need_device(const at::Tensor& t, const char* name) {
  const bool there = t.is_cuda() && t.layout() == at::kStrided;
  if (!there)
    refuse(name, ": expected a CUDA (HIP) tensor, got device ", t.device().str(), "; beyond_deep_ensembles_amd has no CPU path");
}
void same_device(const at::Tensor& ref, const at::Tensor& t, const char* name) {
  if (t.defined() && t.device() != ref.device()) refuse(name, ": on ", t.device().str(), ", the other operands are on ", ref.device().str());
}
void need_index_type(const at::Tensor& t, const char* name) {
  if (t.scalar_type() != at::kLong && t.scalar_type() != at::kInt) refuse(name, ": expected int64 / int32, got ", t.scalar_type());
}
// rows that may lie apart, their elements not
at::Tensor row_major(const at::Tensor& t) {
  return (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1)) ? t : t.contiguous();
}
int64_t row_step(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
void* data(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* fdata(const at::Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

struct EmbeddingNode : public torch::autograd::Function<EmbeddingNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& weight, const c10::optional<at::Tensor>& rho_, const at::Tensor& tokens,
                            const c10::optional<at::Tensor>& eps_, int64_t out_type, int64_t noise, int64_t seed, int64_t stream_id,
                            double scale, int64_t padding) {
    const at::Tensor rho = opt(rho_), eps = opt(eps_);
    c10::DeviceGuard guard(weight.device());
    const at::Tensor w = row_major(weight.detach()), t = tokens.contiguous();
    at::Tensor r;
    if (rho.defined()) r = row_major(rho.detach());
    const int64_t n = t.numel(), v = w.size(0), d = w.size(1);
    std::vector<int64_t> shape = tokens.sizes().vec();
    shape.push_back(d);
    at::Tensor out = at::empty(shape, w.options().dtype(static_cast<at::ScalarType>(out_type)));
    const int rc = bde_embedding_fwd(data(w), type_code(w.scalar_type()), row_step(w), fdata(r), r.defined() ? row_step(r) : 0, data(t),
                                     t.scalar_type() == at::kLong, fdata(eps), eps.defined() ? row_step(eps) : 0, static_cast<int>(noise),
                                     static_cast<uint64_t>(seed), static_cast<uint64_t>(stream_id), static_cast<float>(scale), padding,
                                     data(out), type_code(out.scalar_type()), n, v, d, current_stream(w));
    if (rc != 0) refuse("bde_embedding_fwd failed with code ", rc, rc == -1 ? " (invalid argument)" : " (hipError)");
    ctx->save_for_backward({t, rho, eps});
    ctx->saved_data["i"] = std::vector<int64_t>{v, d, static_cast<int64_t>(w.scalar_type()), noise, seed, stream_id, padding};
    ctx->saved_data["scale"] = scale;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grad_outputs) {
    check_once_differentiable(grad_outputs);
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &t = saved[0], &rho = saved[1];
    at::Tensor eps = saved[2];
    const std::vector<int64_t> i = ctx->saved_data["i"].toIntVector();
    const int64_t n = t.numel(), v = i[0], d = i[1];
    const auto type = static_cast<at::ScalarType>(i[2]);
    int64_t noise = i[3];
    c10::DeviceGuard guard(t.device());
    at::Tensor g = grad_outputs[0].reshape({n, d});
    if (d > 1 && g.stride(1) != 1) g = g.contiguous();      // (rows may coincide: a broadcast gradient is read as it is)
    at::Tensor gw = at::empty({v, d}, g.options().dtype(type)), gr, r;
    if (rho.defined() && ctx->needs_input_grad(1)) {
      r = row_major(rho.detach());
      gr = at::empty({v, d}, g.options().dtype(at::kFloat));
    } else {                                                // the mean's gradient is the plain lookup's
      noise = 0;
      eps = at::Tensor();
    }
    const size_t bytes = bde_embedding_bwd_ws_bytes(n, d, static_cast<int>(noise));
    TORCH_CHECK(bytes > 0, "embedding: unsupported size N=", n, ", D=", d);
    at::Tensor ws = at::empty({static_cast<int64_t>(bytes)}, g.options().dtype(at::kByte));
    const int rc = bde_embedding_bwd(data(g), type_code(g.scalar_type()), n > 1 ? g.stride(0) : d, data(t), t.scalar_type() == at::kLong, fdata(r),
                                     r.defined() ? row_step(r) : 0, fdata(eps), eps.defined() ? row_step(eps) : 0,
                                     static_cast<int>(noise), static_cast<uint64_t>(i[4]), static_cast<uint64_t>(i[5]),
                                     static_cast<float>(ctx->saved_data["scale"].toDouble()), i[6], data(gw), type_code(type), fdata(gr), n, v, d,
                                     data(ws), bytes, current_stream(t));
    TORCH_CHECK(rc == 0, "bde_embedding_bwd failed with code ", rc);
    if (!ctx->needs_input_grad(0)) gw = at::Tensor();
    return {gw, gr, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

at::Tensor embedding(const at::Tensor& tokens, const at::Tensor& weight, const c10::optional<at::Tensor>& rho_,
                     const c10::optional<at::Tensor>& eps_, int64_t noise, int64_t seed, int64_t stream_id, double scale,
                     const c10::optional<int64_t>& padding_, const c10::optional<at::ScalarType>& out_) {
  need_index_type(tokens, "tokens");
  if (weight.dim() != 2 || type_code(weight.scalar_type()) < 0)
    refuse("weight: expected a float32 / bfloat16 / float16 [V, D] tensor, got ", weight.scalar_type(), " ", weight.sizes());
  need_device(weight, "weight");
  need_device(tokens, "tokens");
  same_device(weight, tokens, "tokens");
  const at::ScalarType out = out_.value_or(weight.scalar_type());
  if (type_code(out) < 0 || (weight.scalar_type() != at::kFloat && out != weight.scalar_type()))
    refuse("out_dtype: a ", weight.scalar_type(), " weight does not give ", out);
  const int64_t v = weight.size(0), d = weight.size(1), n = tokens.numel();
  if (n > BDE_EMBEDDING_MAX_TOKENS || v < 1 || v > BDE_EMBEDDING_MAX_ROWS || d < 1 || d > BDE_EMBEDDING_MAX_DIM)
    refuse("embedding: unsupported size N=", n, ", V=", v, ", D=", d);
  int64_t padding = -1;
  if (padding_.has_value()) {
    padding = *padding_;
    if (padding < -v || padding >= v) refuse("padding_idx ", padding, " is outside the table of ", v, " rows");
    if (padding < 0) padding += v;
  }
  at::Tensor rho = opt(rho_), eps = opt(eps_);
  if (rho.defined()) {
    if (weight.scalar_type() != at::kFloat || rho.scalar_type() != at::kFloat || rho.sizes() != weight.sizes() || rho.device() != weight.device())
      refuse("gaussian_embedding: mean and rho must be float32 tensors of one shape and device");
    if (eps.defined()) {
      std::vector<int64_t> want = noise == 2 ? std::vector<int64_t>{v} : tokens.sizes().vec();
      want.push_back(d);
      if (eps.sizes() != at::IntArrayRef(want) || eps.scalar_type() != at::kFloat || eps.device() != weight.device())
        refuse("eps: expected a float32 tensor of shape ", at::IntArrayRef(want), " on ", weight.device().str(), ", got ", eps.scalar_type(), " ", eps.sizes(),
               " on ", eps.device().str());
      if (eps.requires_grad()) refuse("eps: the noise is a constant of this operator (no gradient); detach it");
      eps = row_major(eps.reshape({noise == 2 ? v : n, d}));
    }
  }
  return EmbeddingNode::apply(weight, rho.defined() ? c10::make_optional(rho) : c10::nullopt, tokens,
                              eps.defined() ? c10::make_optional(eps) : c10::nullopt, static_cast<int64_t>(out), noise, seed, stream_id, scale, padding);
}

// [..., V] -> [N, V], rows possibly apart
at::Tensor logit_rows(const at::Tensor& logits) {
  if (logits.dim() < 1 || logits.size(-1) < 1 || type_code(logits.scalar_type()) < 0)
    refuse("logits: expected a float32 / bfloat16 / float16 [..., V] tensor, got ", logits.scalar_type(), " ", logits.sizes());
  need_device(logits, "logits");
  const int64_t v = logits.size(-1);
  return row_major(logits.dim() == 2 ? logits : logits.reshape({logits.numel() / v, v}));
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> topk_logits(const at::Tensor& logits, int64_t k, double temperature) {
  const at::Tensor z = logit_rows(logits.detach());
  const int64_t n = z.size(0), v = z.size(1);
  int max_v = 0, max_k = 0;
  bde_topk_limits(&max_v, &max_k);
  if (k < 1 || k > v || k > max_k || v > max_v || n > INT32_MAX)
    refuse("topk_logits: 1 <= k <= min(V, ", max_k, "), V <= ", max_v, " and fewer than 2^31 rows supported, got k=", k, ", V=", v, ", ", n, " rows");
  c10::DeviceGuard guard(z.device());
  std::vector<int64_t> shape = logits.sizes().vec();
  shape.back() = k;
  at::Tensor values = at::empty(shape, z.options()), indices = at::empty(shape, z.options().dtype(at::kLong));
  shape.pop_back();
  at::Tensor rest = at::empty(shape, z.options().dtype(at::kFloat));
  const int rc = bde_topk_logits(data(z), type_code(z.scalar_type()), row_step(z), static_cast<float>(temperature), static_cast<int>(n),
                                 static_cast<int>(v), static_cast<int>(k), data(values), indices.data_ptr<int64_t>(), fdata(rest), current_stream(z));
  if (rc != 0) refuse("bde_topk_logits failed with code ", rc, rc == -1 ? " (invalid argument)" : " (hipError)");
  return {values, indices, rest};
}

// Under sum / mean the forward writes the gradient for d objective / d loss = 1 in the pass that computes the loss; the backward
// returns that buffer after a launch that leaves it alone where the value IS 1 and recomputes it from the logits where it is not.
// Later backward passes of a retained graph, and one that is not part of the very capture its forward was part of (captured
// alone, or into another graph: replayed without that forward), use a buffer of their own.
struct DistillNode : public torch::autograd::Function<DistillNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& values, const at::Tensor& indices,
                            const c10::optional<at::Tensor>& rest_, const c10::optional<at::Tensor>& weight_, int64_t reduction, double scale,
                            double temperature, bool differentiated) {
    const at::Tensor rest = opt(rest_), weight = opt(weight_);
    c10::DeviceGuard guard(logits.device());
    const at::Tensor z = logit_rows(logits.detach());
    const int64_t n = z.size(0), v = z.size(1), k = values.size(1);
    const auto f32 = z.options().dtype(at::kFloat);
    at::Tensor rows = at::empty(reduction == 0 ? at::IntArrayRef(logits.sizes().data(), logits.dim() - 1) : at::IntArrayRef(n), f32), loss, inv, grad;
    if (reduction != 0) {
      loss = at::empty({}, f32);
      if (differentiated) grad = at::empty({n, v}, z.options());
    }
    if (reduction == 2 && weight.defined()) inv = at::empty({}, f32);
    void* const stream = current_stream(z);
    const int rc = bde_distill_fwd(data(z), type_code(z.scalar_type()), row_step(z), data(values), type_code(values.scalar_type()), data(indices),
                                   indices.scalar_type() == at::kLong, fdata(rest), fdata(weight), static_cast<int>(reduction),
                                   static_cast<float>(scale), static_cast<float>(temperature), static_cast<int>(n), static_cast<int>(v),
                                   static_cast<int>(k), fdata(rows), fdata(loss), data(grad), fdata(inv), stream);
    if (rc != 0) refuse("bde_distill_fwd failed with code ", rc, rc == -1 ? " (invalid argument)" : " (hipError)");
    ctx->save_for_backward({logits, values, indices, rest, weight, inv});
    ctx->saved_data["i"] = std::vector<int64_t>{reduction, static_cast<int64_t>(capture_of(stream))};
    ctx->saved_data["f"] = std::vector<double>{scale, temperature};
    if (grad.defined()) ctx->saved_data["unit"] = grad;
    return reduction == 0 ? rows : loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grad_outputs) {
    check_once_differentiable(grad_outputs);
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &logits = saved[0], &values = saved[1], &indices = saved[2], &rest = saved[3], &weight = saved[4], &inv = saved[5];
    const std::vector<int64_t> i = ctx->saved_data["i"].toIntVector();
    const std::vector<double> f = ctx->saved_data["f"].toDoubleVector();
    c10::DeviceGuard guard(logits.device());
    const int64_t v = logits.size(-1), n = logits.numel() / v;
    const at::Tensor z = row_major(logits.detach().reshape({n, v}));
    void* const stream = current_stream(z);
    at::Tensor grad;
    {
      static std::mutex taking;                            // two backward passes of one retained graph, from two threads
      std::lock_guard<std::mutex> lock(taking);
      auto it = ctx->saved_data.find("unit");
      if (it != ctx->saved_data.end()) {
        grad = it->second.toTensor();
        ctx->saved_data.erase(it);
      }
    }
    const bool ready = grad.defined() && i[1] == static_cast<int64_t>(capture_of(stream));
    if (!ready) grad = at::empty({n, v}, z.options());
    const at::Tensor up = grad_outputs[0].contiguous();
    const int rc = bde_distill_bwd(data(z), type_code(z.scalar_type()), row_step(z), data(values), type_code(values.scalar_type()), data(indices),
                                   indices.scalar_type() == at::kLong, fdata(rest), fdata(weight), fdata(inv), i[0] == 2,
                                   static_cast<float>(f[0]), static_cast<float>(f[1]), fdata(up), i[0] == 0 ? 1 : 0, ready ? 1 : 0,
                                   static_cast<int>(n), static_cast<int>(v), static_cast<int>(values.size(1)), data(grad), stream);
    TORCH_CHECK(rc == 0, "bde_distill_bwd failed with code ", rc);
    return {grad.view(logits.sizes()), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

at::Tensor distillation_loss(const at::Tensor& logits, const at::Tensor& values, const at::Tensor& indices, const c10::optional<at::Tensor>& rest_,
                             const c10::optional<at::Tensor>& weight_, int64_t reduction, double scale, double temperature) {
  if (logits.dim() < 1 || logits.size(-1) < 1 || type_code(logits.scalar_type()) < 0)
    refuse("logits: expected a float32 / bfloat16 / float16 [..., V] tensor, got ", logits.scalar_type(), " ", logits.sizes());
  need_device(logits, "logits");
  const at::IntArrayRef lead(logits.sizes().data(), logits.dim() - 1);
  const int64_t v = logits.size(-1), n = logits.numel() / v;
  if (values.dim() != logits.dim() || values.sizes().slice(0, lead.size()) != lead || indices.sizes() != values.sizes())
    refuse("distillation_loss: values and indices of shape ", lead, " + [K] expected, got ", values.sizes(), " and ", indices.sizes());
  const int64_t k = values.size(-1);
  int max_v = 0, max_k = 0;
  bde_distill_limits(&max_v, &max_k);
  if (k < 1 || k > max_k || v > max_v || n > INT32_MAX)
    refuse("distillation_loss: 1 <= K <= ", max_k, ", 1 <= V <= ", max_v, " and fewer than 2^31 rows supported, got K=", k, ", V=", v, ", ", n, " rows");
  if (type_code(values.scalar_type()) < 0) refuse("values: expected float32 / bfloat16 / float16, got ", values.scalar_type());
  need_index_type(indices, "indices");
  same_device(logits, values, "values");
  same_device(logits, indices, "indices");
  const at::Tensor rest = opt(rest_), weight = opt(weight_);
  auto per_row = [&](const at::Tensor& t, const char* name) -> c10::optional<at::Tensor> {
    if (!t.defined()) return c10::nullopt;
    if (t.sizes() != lead) refuse(name, ": expected shape ", lead, ", got ", t.sizes());
    if (t.scalar_type() != at::kFloat) refuse(name, ": expected float32, got ", t.scalar_type());
    same_device(logits, t, name);
    if (t.requires_grad()) refuse(name, ": the teacher's side and the weights are constants of this loss (no gradient); detach them");
    return t.reshape({n}).contiguous();
  };
  if (values.requires_grad()) refuse("values: the teacher's side and the weights are constants of this loss (no gradient); detach them");
  return DistillNode::apply(logits, values.reshape({n, k}).contiguous(), indices.reshape({n, k}).contiguous(), per_row(rest, "rest"),
                            per_row(weight, "weight"), reduction, scale, temperature, at::GradMode::is_enabled() && logits.requires_grad());
}

}  // namespace

void bind_token_nodes(py::module_& m) {
  m.def("embedding", &embedding, "scaled / Gaussian embedding lookup (lookup.py)", py::arg("tokens"), py::arg("weight"), py::arg("rho"), py::arg("eps"),
        py::arg("noise"), py::arg("seed"), py::arg("stream_id"), py::arg("scale"), py::arg("padding_idx"), py::arg("out_dtype"));
  m.def("topk_logits", &topk_logits, "(values, indices, rest) of a teacher's logits (distill.py)", py::arg("logits"), py::arg("k"), py::arg("temperature"));
  m.def("distillation_loss", &distillation_loss, "loss over a teacher's top logits (distill.py)", py::arg("logits"), py::arg("values"),
        py::arg("indices"), py::arg("rest"), py::arg("weight"), py::arg("reduction"), py::arg("scale"), py::arg("temperature"));
}
