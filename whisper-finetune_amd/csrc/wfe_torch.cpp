// wfe_torch.cpp -- the decoder's vocabulary operators as differentiable torch functions: a Python module
// (wfe_amd._decoder) over the C ABI.  Host code only.  It is C++ because the calls are short: as a Python
// torch.autograd.Function a training step of 16 x 48 tokens spent 92 us on the embedding and its gradient, of which
// the kernels are 33; from here it takes 54 (the backward pass of a Python function runs Python on autograd's own thread).
//
// Nothing here links to libwfe_hip.so: wfe_amd._lib loads that and hands over its entry points (bind).
#include <ATen/autocast_mode.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/AutogradState.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <cstring>
#include <string>

#include "../../include/wfe.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Abi {
  decltype(&wfe_last_error) last_error;
  decltype(&wfe_linear_ce_state_bytes) ce_state;
  decltype(&wfe_linear_ce_workspace_bytes) ce_workspace;
  decltype(&wfe_linear_ce_forward) ce_forward;
  decltype(&wfe_linear_ce_backward) ce_backward;
  decltype(&wfe_embedding) embedding;
  decltype(&wfe_embedding_workspace_bytes) embedding_workspace;
  decltype(&wfe_embedding_backward) embedding_backward;
} entry;

PyObject* wfe_error = nullptr;                 // wfe_amd._lib.WfeError
struct WfeFailure : std::runtime_error {
  using std::runtime_error::runtime_error;
};

[[noreturn]] void refuse(const std::string& text) { throw pybind11::value_error(text); }

void check(int64_t rc) {
  if (rc >= 0) return;
  const char* text = entry.last_error(nullptr);
  const std::string message = std::string("wfe: ") + (text ? text : "");
  if (rc == WFE_ERR_ARG || rc == WFE_ERR_SAMPLING) refuse(message);
  throw WfeFailure(message);
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return WFE_F32;
    case at::kHalf: return WFE_F16;
    case at::kBFloat16: return WFE_BF16;
    default: return -1;
  }
}
at::ScalarType type_of(int32_t code) { return code == WFE_F32 ? at::kFloat : code == WFE_F16 ? at::kHalf : at::kBFloat16; }
std::string name_of(at::ScalarType t) {        // as Python has it
  switch (t) {
    case at::kDouble: return "float64";
    case at::kFloat: return "float32";
    case at::kHalf: return "float16";
    case at::kBFloat16: return "bfloat16";
    case at::kLong: return "int64";
    case at::kInt: return "int32";
    case at::kShort: return "int16";
    case at::kChar: return "int8";
    case at::kByte: return "uint8";
    case at::kBool: return "bool";
    default: return c10::toString(t);
  }
}
std::string shape_of(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}

constexpr int64_t kMaxTokens = 1 << 24, kMaxVocab = 1 << 24, kMaxDim = 16384, kMaxLogits = (int64_t)1 << 37;

void check_matrix(const char* name, const Tensor& weight, const char* index_name, const Tensor& index) {
  const std::string who = std::string(name) + ": ";
  if (weight.dim() != 2) refuse(who + "weight must be (vocab, dim), got " + shape_of(weight));
  if (dtype_code(weight.scalar_type()) < 0)
    refuse(who + "weight is " + name_of(weight.scalar_type()) + "; float32, float16 or bfloat16 is needed");
  if (weight.size(0) < 1 || weight.size(0) > kMaxVocab || weight.size(1) < 1 || weight.size(1) > kMaxDim)
    refuse(who + "weight of " + shape_of(weight) + " outside 1.." + std::to_string(kMaxVocab) + " x 1.." +
           std::to_string(kMaxDim));
  if (index.scalar_type() != at::kLong && index.scalar_type() != at::kInt)
    refuse(who + index_name + " are " + name_of(index.scalar_type()) + "; int32 or int64 is needed");
  if (index.numel() > kMaxTokens)
    refuse(who + std::to_string(index.numel()) + " tokens are more than " + std::to_string(kMaxTokens));
  if (index.device() != weight.device())
    refuse(who + index_name + " are on " + index.device().str() + ", weight on " + weight.device().str());
}

// What differentiates or batches a call behind autograd's back would get the values alone: forward-mode tangents, which are
// not tied to requires_grad, and the function transforms' wrappers.  -> its name, or null
const char* unknown_mode(const Tensor& t) {
  constexpr c10::DispatchKeySet wrapped({c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::FuncTorchBatched});
  if (t.key_set().has_any(wrapped)) return "a function transform (torch.func)";
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t.unsafeGetTensorImpl()->_fw_grad(0, t).defined())
    return "forward-mode differentiation";
  return nullptr;
}

void check_modes(const char* name, std::initializer_list<Tensor> inputs) {
  for (const Tensor& t : inputs)
    if (const char* mode = unknown_mode(t)) {
      PyErr_SetString(PyExc_NotImplementedError, (std::string(name) + ": " + mode + " is not supported").c_str());
      throw pybind11::error_already_set();
    }
}

// The same in a backward pass, which runs on autograd's own threads
void check_upstream(const char* name, const Tensor& grad) {
  if (const char* mode = unknown_mode(grad))
    throw std::runtime_error(std::string(name) + ": " + mode + " of the gradient is not supported");
}

void check_device(const char* name, const Tensor& weight) {
  if (!weight.is_cuda())
    throw WfeFailure(std::string(name) + ": tensors are on " + weight.device().str() +
                     "; an MI355X is needed, there is no CPU path");
}

c10::hip::HIPStream stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()); }
void* raw(const c10::hip::HIPStream& s) { return reinterpret_cast<void*>(s.stream()); }

Tensor bytes(int64_t n, const Tensor& like) {
  check(n);
  return at::empty({n}, like.options().dtype(at::kByte));
}
void* pointer(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// t in memory as it reads: a lazily negated view (torch keeps such for the imaginary part of a conjugate) holds the opposite
Tensor as_read(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }
Tensor dense(const Tensor& t) { return as_read(t).contiguous(); }
// the same with its last dimension contiguous
Tensor dense_rows(const Tensor& t) { return t.size(-1) == 1 || t.stride(-1) == 1 ? as_read(t) : dense(t); }

// A saved tensor as it was when it was saved, strides apart: hooks on saved tensors may bring back another one.
void check_saved(const char* name, const Tensor& t, at::IntArrayRef sizes, at::ScalarType type, const c10::Device& device) {
  if (!t.defined() || t.layout() != at::kStrided || t.sizes() != sizes || t.scalar_type() != type || t.device() != device)
    throw std::runtime_error(std::string(name) + ": a tensor saved for the backward pass came back with another shape, type "
                             "or device (from hooks on saved tensors)");
}

// Refuses to record a call on parameters that a graph of an earlier call on the default stream, still alive, holds on to.
// Autograd keeps one accumulation node per parameter while any graph refers to it, on the stream it was made on; a captured
// backward pass would make that stream wait for the capture.  Another stream is drawn into the capture and joined again at
// the pass's end (warming up on a side stream is how a capture is prepared); the default stream cannot be, which ends the
// process.
void check_capture(const char* name, std::initializer_list<Tensor> inputs) {
  for (const Tensor& t : inputs) {
    if (!t.requires_grad() || !t.is_leaf()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
    if (!node) continue;
    const auto made_on = node->stream();
    if (!made_on || made_on->id() != c10::hip::getDefaultHIPStream(t.device().index()).id()) continue;
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(static_cast<hipStream_t>(raw(stream_of(t))), &status) != hipSuccess) {
      (void)hipGetLastError();
      continue;
    }
    if (status == hipStreamCaptureStatusNone) continue;
    throw std::runtime_error(std::string(name) + ": captured while the autograd graph of an earlier call on the default stream "
                             "with the same parameter is alive; drop that call's results (or detach them) before capturing");
  }
}

// Gradients that come from kernels cannot be differentiated again
variable_list once(const char* name, variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;           // create_graph was not asked for
  for (Tensor& g : grads)
    if (g.defined()) g = g.detach().set_requires_grad(true);
  return torch::autograd::DelayedError(std::string(name) + " can be differentiated once only", (int64_t)grads.size())
      .apply(std::move(grads));
}

template <class D> std::string packed(const D& d) { return std::string(reinterpret_cast<const char*>(&d), sizeof d); }
template <class D> D unpacked(const std::string& s) {
  D d;
  std::memcpy(&d, s.data(), sizeof d);
  return d;
}

// ---- cross entropy -----------------------------------------------------------------------------------------
constexpr const char* kCe = "linear_cross_entropy";

struct CeCall {
  wfe_linear_ce desc{};
  Tensor weight, loss, state;
};

CeCall ce_forward(Tensor hidden, const Tensor& weight, const Tensor& labels_, int64_t ignore_index, int64_t reduction,
                  bool keep) {
  CeCall c;
  c.weight = dense_rows(weight);
  hidden = dense_rows(hidden);
  // the leading dimensions merged, from the last one on: at most two strides, else a copy
  int64_t size[2] = {1, 1}, stride[2] = {hidden.size(-1), 0};
  int levels = 0;
  for (int64_t i = hidden.dim() - 2; i >= 0; --i) {
    if (hidden.size(i) == 1) continue;
    if (levels > 0 && hidden.stride(i) == size[levels - 1] * stride[levels - 1]) {
      size[levels - 1] *= hidden.size(i);
    } else if (levels == 2) {
      hidden = hidden.contiguous();
      levels = 1;
      size[0] = hidden.numel() / hidden.size(-1);
      stride[0] = hidden.size(-1);
      break;
    } else {
      size[levels] = hidden.size(i);
      stride[levels++] = hidden.stride(i);
    }
  }
  const Tensor labels = dense(labels_);
  wfe_linear_ce& d = c.desc;
  d.device = weight.device().index();
  d.dtype = d.grad_hidden_dtype = d.grad_weight_dtype = dtype_code(weight.scalar_type());
  d.rows = labels.numel();
  d.inner = size[0] > 0 ? size[0] : 1;
  d.inner_stride = stride[0];
  d.outer_stride = levels == 2 ? stride[1] : 0;
  d.weight_stride = c.weight.stride(0);
  d.vocab = (int32_t)weight.size(0);
  d.dim = (int32_t)weight.size(1);
  d.label_bits = labels.scalar_type() == at::kLong ? 64 : 32;
  d.reduction = (int32_t)reduction;
  d.ignore_index = ignore_index;
  c.loss = at::empty(reduction == WFE_REDUCE_NONE ? labels.sizes() : at::IntArrayRef{},
                     weight.options().dtype(at::kFloat).requires_grad(false));
  const int64_t state = entry.ce_state(&d), workspace = entry.ce_workspace(&d, c.weight.data_ptr(), 0, 0);
  check(state);
  check(workspace);
  const int64_t at = (state + 255) / 256 * 256;            // without a backward pass: one buffer for both
  c.state = bytes(keep ? state : at + workspace, c.weight);
  const Tensor scratch = keep ? bytes(workspace, c.weight) : Tensor();
  check(entry.ce_forward(&d, hidden.data_ptr(), c.weight.data_ptr(), labels.data_ptr(), c.loss.data_ptr<float>(),
                       c.state.data_ptr(), keep ? scratch.data_ptr() : static_cast<char*>(c.state.data_ptr()) + at,
                       workspace, raw(stream_of(c.weight))));
  return c;
}

struct LinearCrossEntropy : torch::autograd::Function<LinearCrossEntropy> {
  static Tensor forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const Tensor& labels,
                        int64_t dtype, int64_t ignore_index, int64_t reduction) {
    const auto type = static_cast<at::ScalarType>(dtype);
    CeCall c = ce_forward(hidden.to(type), weight.to(type), labels, ignore_index, reduction, true);
    // a gradient in float32 is written as such; any other type is the products' own, cast where the input's differs
    if (hidden.scalar_type() == at::kFloat) c.desc.grad_hidden_dtype = WFE_F32;
    if (weight.scalar_type() == at::kFloat) c.desc.grad_weight_dtype = WFE_F32;
    ctx->save_for_backward({c.weight, c.state});
    ctx->saved_data["desc"] = packed(c.desc);
    ctx->saved_data["shape"] = hidden.sizes();
    ctx->saved_data["types"] = std::vector<int64_t>{(int64_t)hidden.scalar_type(), (int64_t)weight.scalar_type()};
    return c.loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list result(6);
    if (!grads[0].defined()) return result;
    check_upstream(kCe, grads[0]);
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      const auto saved = ctx->get_saved_variables();
      auto d = unpacked<wfe_linear_ce>(ctx->saved_data["desc"].toStringRef());
      const auto types = ctx->saved_data["types"].toIntVector();
      check_saved(kCe, saved[0], {d.vocab, d.dim}, type_of(d.dtype), grads[0].device());
      check_saved(kCe, saved[1], {entry.ce_state(&d)}, at::kByte, grads[0].device());
      const Tensor weight = dense_rows(saved[0]), state = dense(saved[1]);
      d.weight_stride = weight.stride(0);
      const Tensor upstream = dense(grads[0].to(at::kFloat));
      Tensor grad_hidden, grad_weight;
      const auto kind = [&](int32_t code) { return code == WFE_F32 ? at::kFloat : weight.scalar_type(); };
      if (ctx->needs_input_grad(0))
        grad_hidden = at::empty(ctx->saved_data["shape"].toIntVector(), weight.options().dtype(kind(d.grad_hidden_dtype)));
      if (ctx->needs_input_grad(1))
        grad_weight = at::empty(weight.sizes(), weight.options().dtype(kind(d.grad_weight_dtype)));
      const int64_t need = entry.ce_workspace(&d, weight.data_ptr(), 1,
                                            (grad_hidden.defined() ? WFE_GRAD_HIDDEN : 0) |
                                                (grad_weight.defined() ? WFE_GRAD_WEIGHT : 0));
      const Tensor workspace = bytes(need, weight);
      check(entry.ce_backward(&d, weight.data_ptr(), state.data_ptr(), upstream.data_ptr<float>(), pointer(grad_hidden),
                            pointer(grad_weight), workspace.data_ptr(), need, raw(stream_of(weight))));
      if (grad_hidden.defined()) result[0] = grad_hidden.to(static_cast<at::ScalarType>(types[0]));
      if (grad_weight.defined()) result[1] = grad_weight.to(static_cast<at::ScalarType>(types[1]));
    }
    return once(kCe, std::move(result));
  }
};

Tensor linear_cross_entropy(const Tensor& hidden, const Tensor& weight, const Tensor& labels, int64_t ignore_index,
                            int64_t reduction) {
  check_modes(kCe, {hidden, weight, labels});
  check_matrix(kCe, weight, "labels", labels);
  const std::string who = std::string(kCe) + ": ";
  if (hidden.dim() < 1 || hidden.size(-1) != weight.size(1) || hidden.sizes().slice(0, hidden.dim() - 1) != labels.sizes())
    refuse(who + "hidden " + shape_of(hidden) + " does not fit labels " + shape_of(labels) + " and weight " +
           shape_of(weight));
  if (labels.numel() * weight.size(0) > kMaxLogits)
    refuse(who + std::to_string(labels.numel()) + " tokens by a vocabulary of " + std::to_string(weight.size(0)) +
           " are more than 2^37 logits");
  if (hidden.device() != weight.device())
    refuse(who + "hidden is on " + hidden.device().str() + ", weight on " + weight.device().str());
  check_device(kCe, weight);
  at::ScalarType type = weight.scalar_type();
  if (at::autocast::is_autocast_enabled(at::kCUDA)) {
    type = at::autocast::get_autocast_dtype(at::kCUDA);
    if (dtype_code(hidden.scalar_type()) < 0 || dtype_code(type) < 0)
      refuse(who + name_of(hidden.scalar_type()) + " under autocast to " + name_of(type));
  } else if (hidden.scalar_type() != type) {
    refuse(who + "hidden is " + name_of(hidden.scalar_type()) + ", weight " + name_of(type) +
           "; outside autocast they must agree");
  }
  if (at::GradMode::is_enabled() && (hidden.requires_grad() || weight.requires_grad())) {
    check_capture(kCe, {hidden, weight});
    return LinearCrossEntropy::apply(hidden, weight, labels, (int64_t)type, ignore_index, reduction);
  }
  const at::AutoDispatchBelowADInplaceOrView below;
  return ce_forward(hidden.to(type), weight.to(type), labels, ignore_index, reduction, false).loss;
}

// ---- embedding ---------------------------------------------------------------------------------------------
constexpr const char* kEmbed = "token_embedding";

struct EmbedCall {
  wfe_embedding_desc desc{};
  Tensor ids, out;
};

EmbedCall embed_forward(const Tensor& ids, const Tensor& weight_, double scale, int64_t padding_idx) {
  EmbedCall c;
  const Tensor weight = dense_rows(weight_);
  c.ids = dense(ids);
  wfe_embedding_desc& d = c.desc;
  d.device = weight.device().index();
  d.dtype = d.grad_weight_dtype = dtype_code(weight.scalar_type());
  d.rows = ids.numel();
  d.weight_stride = weight.stride(0);
  d.vocab = (int32_t)weight.size(0);
  d.dim = (int32_t)weight.size(1);
  d.id_bits = ids.scalar_type() == at::kLong ? 64 : 32;
  d.padding_idx = padding_idx;
  d.scale = (float)scale;
  std::vector<int64_t> shape = ids.sizes().vec();
  shape.push_back(d.dim);
  c.out = at::empty(shape, weight.options().requires_grad(false));
  check(entry.embedding(&d, c.ids.data_ptr(), weight.data_ptr(), c.out.data_ptr(), raw(stream_of(weight))));
  return c;
}

struct TokenEmbedding : torch::autograd::Function<TokenEmbedding> {
  static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& weight, double scale,
                        int64_t padding_idx) {
    EmbedCall c = embed_forward(ids, weight, scale, padding_idx);
    ctx->save_for_backward({c.ids});
    ctx->saved_data["desc"] = packed(c.desc);
    return c.out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list result(4);
    if (!grads[0].defined()) return result;
    check_upstream(kEmbed, grads[0]);
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      const Tensor saved = ctx->get_saved_variables()[0];
      auto d = unpacked<wfe_embedding_desc>(ctx->saved_data["desc"].toStringRef());
      check_saved(kEmbed, saved, grads[0].sizes().slice(0, grads[0].dim() - 1), d.id_bits == 64 ? at::kLong : at::kInt,
                  grads[0].device());
      const Tensor ids = dense(saved);
      Tensor rows = dense_rows(grads[0]);
      if (!rows.is_contiguous()) rows = rows.reshape({-1, d.dim});     // a view where the leading dimensions allow one
      d.grad_stride = rows.is_contiguous() ? d.dim : rows.stride(0);
      const Tensor grad_weight = at::empty({d.vocab, d.dim}, rows.options());
      const int64_t need = entry.embedding_workspace(&d);
      const Tensor workspace = bytes(need, rows);
      check(entry.embedding_backward(&d, ids.data_ptr(), rows.data_ptr(), grad_weight.data_ptr(), workspace.data_ptr(),
                                   need, raw(stream_of(rows))));
      result[1] = grad_weight;
    }
    return once(kEmbed, std::move(result));
  }
};

Tensor token_embedding(const Tensor& ids, const Tensor& weight, double scale, std::optional<int64_t> padding_idx) {
  check_modes(kEmbed, {ids, weight});
  check_matrix(kEmbed, weight, "ids", ids);
  int64_t padding = -1;
  if (padding_idx) {
    if (*padding_idx < -weight.size(0) || *padding_idx >= weight.size(0))
      refuse(std::string(kEmbed) + ": padding_idx " + std::to_string(*padding_idx) + " outside a vocabulary of " +
             std::to_string(weight.size(0)));
    padding = *padding_idx < 0 ? *padding_idx + weight.size(0) : *padding_idx;
  }
  check_device(kEmbed, weight);
  if (at::GradMode::is_enabled() && weight.requires_grad()) {
    check_capture(kEmbed, {weight});
    return TokenEmbedding::apply(ids, weight, scale, padding);
  }
  const at::AutoDispatchBelowADInplaceOrView below;
  return embed_forward(ids, weight, scale, padding).out;
}

template <class F> void take(F& f, uintptr_t address) { f = reinterpret_cast<F>(address); }

}  // namespace

PYBIND11_MODULE(_decoder, m) {
  pybind11::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const WfeFailure& e) {
      PyErr_SetString(wfe_error ? wfe_error : PyExc_RuntimeError, e.what());
    }
  });
  m.def("bind", [](const std::vector<uintptr_t>& a, pybind11::object error) {
    if (a.size() != 8) refuse("bind: 8 entry points are needed");
    take(entry.last_error, a[0]);
    take(entry.ce_state, a[1]);
    take(entry.ce_workspace, a[2]);
    take(entry.ce_forward, a[3]);
    take(entry.ce_backward, a[4]);
    take(entry.embedding, a[5]);
    take(entry.embedding_workspace, a[6]);
    take(entry.embedding_backward, a[7]);
    wfe_error = error.release().ptr();
  });
  m.def("linear_cross_entropy", &linear_cross_entropy);
  m.def("token_embedding", &token_embedding);
}
