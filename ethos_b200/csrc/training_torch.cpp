// torch binding of the training operators: argument checks, memory and
// autograd around the C ABI of include/ethos_b200.h.
//
// These operators are short (tens of microseconds), and torch runs a backward
// in a worker thread.  With the nodes in Python a lookup and its gradient took
// 85 us of host time: 26 us forward and 22 us backward (17 and 17 on a warm
// core), the rest the engine's.  Nodes in C++ need neither the interpreter nor
// its lock in that thread: 55 us, of which the engine's round trip is 30 to 36.  ethos_b200/ops.py holds the same calls without
// autograd.
#include <torch/extension.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <dlfcn.h>

#include <limits>
#include <stdexcept>
#include <string>

#include "ethos_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The library that ethos_b200._lib has loaded (its path is the user's to
// choose, so nothing is linked).
struct Library {
  decltype(&::ethos_balance_backward) ethos_balance_backward;
  decltype(&::ethos_balance_forward) ethos_balance_forward;
  decltype(&::ethos_balance_scratch_size) ethos_balance_scratch_size;
  decltype(&::ethos_embedding_backward) ethos_embedding_backward;
  decltype(&::ethos_embedding_backward_workspace_size) ethos_embedding_backward_workspace_size;
  decltype(&::ethos_embedding_forward) ethos_embedding_forward;
  decltype(&::ethos_status_string) ethos_status_string;
  decltype(&::ethos_xent_backward) ethos_xent_backward;
  decltype(&::ethos_xent_backward_workspace_size) ethos_xent_backward_workspace_size;
  decltype(&::ethos_xent_forward) ethos_xent_forward;
  decltype(&::ethos_xent_forward_backward) ethos_xent_forward_backward;
  decltype(&::ethos_xent_forward_backward_workspace_size) ethos_xent_forward_backward_workspace_size;
  decltype(&::ethos_xent_forward_workspace_size) ethos_xent_forward_workspace_size;
  decltype(&::ethos_xent_save_size) ethos_xent_save_size;
  decltype(&::ethos_xent_scale) ethos_xent_scale;
} L;

void load(const std::string& path) {
  void* so = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
  TORCH_CHECK(so != nullptr, dlerror());
  auto find = [so](auto& f, const char* name) {
    f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(dlsym(so, name));
    TORCH_CHECK(f != nullptr, name, " is not in the library");
  };
  find(L.ethos_balance_backward, "ethos_balance_backward");
  find(L.ethos_balance_forward, "ethos_balance_forward");
  find(L.ethos_balance_scratch_size, "ethos_balance_scratch_size");
  find(L.ethos_embedding_backward, "ethos_embedding_backward");
  find(L.ethos_embedding_backward_workspace_size, "ethos_embedding_backward_workspace_size");
  find(L.ethos_embedding_forward, "ethos_embedding_forward");
  find(L.ethos_status_string, "ethos_status_string");
  find(L.ethos_xent_backward, "ethos_xent_backward");
  find(L.ethos_xent_backward_workspace_size, "ethos_xent_backward_workspace_size");
  find(L.ethos_xent_forward, "ethos_xent_forward");
  find(L.ethos_xent_forward_backward, "ethos_xent_forward_backward");
  find(L.ethos_xent_forward_backward_workspace_size, "ethos_xent_forward_backward_workspace_size");
  find(L.ethos_xent_forward_workspace_size, "ethos_xent_forward_workspace_size");
  find(L.ethos_xent_save_size, "ethos_xent_save_size");
  find(L.ethos_xent_scale, "ethos_xent_scale");
}

// A status of the library: ethos_b200._lib.EthosError in a forward call, its
// text in a RuntimeError where the autograd engine carries it.
struct StatusError : std::runtime_error {
  int status;
  const char* call;
  StatusError(int s, const char* c) : std::runtime_error(std::string(c) + ": " + L.ethos_status_string(s)), status(s), call(c) {}
};
void check(int status, const char* call) {
  if (status != ETHOS_OK) throw StatusError(status, call);
}

// The device's error word (ops.device_error_word), registered before its first
// use.
int* g_err[64];
int* error_word(const Tensor& t) { return g_err[t.get_device()]; }
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

void need_cuda(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor: the ETHOS B200 layer has no CPU path");
}
void need_on(const Tensor& ref, const Tensor& t, const char* name) {
  need_cuda(t, name);
  TORCH_CHECK_VALUE(t.get_device() == ref.get_device(), name, " is on ", t.device(), ", not on ", ref.device());
}
int dtype_code(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16, name, ": fp32 or bf16, not ",
                    t.scalar_type());
  return t.scalar_type() == at::kBFloat16 ? ETHOS_BF16 : ETHOS_F32;
}
int ids_i64(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, name, ": int32 or int64, not ",
                    t.scalar_type());
  return t.scalar_type() == at::kLong;
}
Tensor bytes(size_t n, const Tensor& like) {
  return at::empty({static_cast<int64_t>(n)}, like.options().dtype(at::kByte));
}
Tensor fp32(at::IntArrayRef sizes, const Tensor& like) { return at::empty(sizes, like.options().dtype(at::kFloat)); }

// The gradients are not built of differentiable parts: better an error than
// a second derivative that lacks a term.
void once(const char* name) {
  TORCH_CHECK(!at::GradMode::is_enabled(), name, ": its gradient cannot be differentiated (create_graph=True)");
}

// Rows with unit column stride and a pitch of at least their width.
Tensor as_rows(const Tensor& t) {
  return t.stride(1) == 1 && t.stride(0) >= t.size(1) ? t : t.contiguous();
}
// (a single row may carry any stride)
int64_t pitch(const Tensor& t) { return std::max(t.stride(0), t.size(1)); }

// -------------------------------------------------------------- embedding --
struct Embedding : torch::autograd::Function<Embedding> {
  static Tensor forward(AutogradContext* ctx, const Tensor& ids_, const Tensor& weight, double scale, int64_t padding) {
    need_cuda(weight, "weight");
    need_on(weight, ids_, "ids");
    TORCH_CHECK_VALUE(weight.dim() == 2, "weight: [vocab, dim]");
    const int code = dtype_code(weight, "weight"), i64 = ids_i64(ids_, "ids");
    const int64_t V = weight.size(0), d = weight.size(1);
    const c10::cuda::CUDAGuard guard(weight.device());
    const Tensor ids = ids_.contiguous();
    const Tensor w = as_rows(weight);
    std::vector<int64_t> shape = ids.sizes().vec();
    shape.push_back(d);
    Tensor out = at::empty(shape, weight.options());
    check(L.ethos_embedding_forward(ids.const_data_ptr(), i64, w.const_data_ptr(), pitch(w), code, ids.numel(), V, d,
                                  static_cast<float>(scale), out.mutable_data_ptr(), error_word(w), stream_of(w)),
          "ethos_embedding_forward");
    ctx->save_for_backward({ids});
    ctx->saved_data["p"] = std::vector<int64_t>{V, d, padding};
    ctx->saved_data["scale"] = scale;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    once("embedding");
    const Tensor ids = ctx->get_saved_variables()[0];
    const std::vector<int64_t> p = ctx->saved_data["p"].toIntVector();
    const Tensor dy = grads[0].contiguous();
    const c10::cuda::CUDAGuard guard(dy.device());
    const int64_t T = ids.numel(), V = p[0], d = p[1];
    Tensor dw = at::empty({V, d}, dy.options());
    const size_t need = L.ethos_embedding_backward_workspace_size(T, V, d);
    Tensor ws = bytes(need, dy);
    check(L.ethos_embedding_backward(ids.const_data_ptr(), ids_i64(ids, "ids"), dy.const_data_ptr(), dtype_code(dy, "dy"),
                                   T, V, d, p[2], static_cast<float>(ctx->saved_data["scale"].toDouble()),
                                   dw.mutable_data_ptr(), ws.mutable_data_ptr(), need, error_word(dy), stream_of(dy)),
          "ethos_embedding_backward");
    return {Tensor(), dw, Tensor(), Tensor()};
  }
};

// ---------------------------------------------------------------- balance --
struct Balance : torch::autograd::Function<Balance> {
  static variable_list forward(AutogradContext* ctx, const Tensor& weights_, const Tensor& ids_, int64_t experts,
                               const std::optional<Tensor>& mask_) {
    need_cuda(weights_, "weights");
    need_on(weights_, ids_, "ids");
    const int code = dtype_code(weights_, "weights"), i64 = ids_i64(ids_, "ids");
    TORCH_CHECK_VALUE(weights_.dim() == 3 && ids_.sizes() == weights_.sizes(),
                      "weights and ids: [tokens, heads, k], of one shape");
    const int64_t T = weights_.size(0), H = weights_.size(1), k = weights_.size(2);
    const c10::cuda::CUDAGuard guard(weights_.device());
    Tensor mask;
    if (mask_) {
      need_on(weights_, *mask_, "mask");
      TORCH_CHECK_VALUE(mask_->scalar_type() == at::kBool && mask_->dim() == 1 && mask_->size(0) == T,
                        "mask: bool [tokens]");
      mask = mask_->contiguous();
    }
    const Tensor w = weights_.contiguous(), ids = ids_.contiguous();
    const size_t need = L.ethos_balance_scratch_size(T, H, k);
    Tensor counts = at::empty({experts}, w.options().dtype(at::kInt));
    Tensor loss = fp32({}, w);
    Tensor scratch = bytes(need, w);
    check(L.ethos_balance_forward(ids.const_data_ptr(), i64, w.const_data_ptr(), code,
                                mask.defined() ? static_cast<const uint8_t*>(mask.const_data_ptr()) : nullptr, T, H, k,
                                experts, static_cast<int32_t*>(counts.mutable_data_ptr()),
                                static_cast<float*>(loss.mutable_data_ptr()), scratch.mutable_data_ptr(), need,
                                error_word(w), stream_of(w)),
          "ethos_balance_forward");
    ctx->save_for_backward({scratch});
    ctx->saved_data["p"] = std::vector<int64_t>{T, H, k, experts, code};
    ctx->mark_non_differentiable({counts});
    ctx->set_materialize_grads(false);  // no zeros for the counts
    return {loss, counts};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    once("balance_loss");
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const Tensor scratch = ctx->get_saved_variables()[0];
    const std::vector<int64_t> p = ctx->saved_data["p"].toIntVector();
    const c10::cuda::CUDAGuard guard(scratch.device());
    const Tensor grad = grads[0].to(at::kFloat);
    Tensor dw = at::empty({p[0], p[1], p[2]}, scratch.options().dtype(p[4] == ETHOS_BF16 ? at::kBFloat16 : at::kFloat));
    check(L.ethos_balance_backward(static_cast<int>(p[4]), p[0], p[1], p[2], p[3], scratch.const_data_ptr(),
                                 static_cast<size_t>(scratch.numel()), static_cast<const float*>(grad.const_data_ptr()),
                                 dw.mutable_data_ptr(), stream_of(scratch)),
          "ethos_balance_backward");
    return {dw, Tensor(), Tensor(), Tensor()};
  }
};

// ---------------------------------------------------------- cross entropy --
// What the products read in place: rows of 16-byte pieces (other widths go
// through packed copies in the workspace).
Tensor as_table(const Tensor& t) {
  const Tensor w = as_rows(t);
  if (w.scalar_type() == at::kBFloat16 && w.size(1) % 8 == 0 &&
      (reinterpret_cast<uintptr_t>(w.const_data_ptr()) % 16 != 0 || pitch(w) % 8 != 0))
    return w.clone(at::MemoryFormat::Contiguous);
  return w;
}

struct CrossEntropy : torch::autograd::Function<CrossEntropy> {
  // what: bit 0 d_hidden, bit 1 d_weight, bit 2 keep the exponentials if that way is open
  static Tensor forward(AutogradContext* ctx, const Tensor& hidden_, const Tensor& weight_, const Tensor& labels_,
                        int64_t ignore_index, int64_t reduction, int64_t what) {
    const Tensor h = as_rows(hidden_), w = as_table(weight_), y = labels_.contiguous();
    const c10::cuda::CUDAGuard guard(h.device());
    const int64_t T = h.size(0), d = h.size(1), V = w.size(0);
    const int code = dtype_code(h, "hidden"), i64 = ids_i64(y, "labels"), red = static_cast<int>(reduction);
    Tensor loss = red == ETHOS_XENT_NONE ? fp32({T}, h) : fp32({}, h);
    Tensor save, dh, dw;
    if (T == 0) {  // as torch: nothing, 0, and the mean of nothing
      if (red != ETHOS_XENT_NONE) loss.fill_(red == ETHOS_XENT_SUM ? 0.0 : std::numeric_limits<double>::quiet_NaN());
    } else {
      const size_t save_bytes = L.ethos_xent_save_size(T, V, d, code);
      save = bytes(save_bytes, h);
      const size_t keep_bytes = (what & 4) && (what & 3) && red != ETHOS_XENT_NONE
                                    ? L.ethos_xent_forward_backward_workspace_size(T, V, d, code)
                                    : 0;
      if (keep_bytes > 0) {
        if (what & 1) dh = at::empty({T, d}, h.options());
        if (what & 2) dw = at::empty({V, d}, w.options());
        Tensor ws = bytes(keep_bytes, h);
        check(L.ethos_xent_forward_backward(
                  h.const_data_ptr(), pitch(h), w.const_data_ptr(), pitch(w), code, y.const_data_ptr(), i64,
                  ignore_index, red, T, V, d, static_cast<float*>(loss.mutable_data_ptr()), save.mutable_data_ptr(),
                  save_bytes, (what & 1) ? dh.mutable_data_ptr() : nullptr,
                  (what & 2) ? dw.mutable_data_ptr() : nullptr, ws.mutable_data_ptr(), keep_bytes, error_word(h),
                  stream_of(h)),
              "ethos_xent_forward_backward");
      } else {
        const size_t n = L.ethos_xent_forward_workspace_size(T, V, d, code);
        Tensor ws = bytes(n, h);
        check(L.ethos_xent_forward(h.const_data_ptr(), pitch(h), w.const_data_ptr(), pitch(w), code, y.const_data_ptr(),
                                 i64, ignore_index, red, T, V, d, static_cast<float*>(loss.mutable_data_ptr()),
                                 save.mutable_data_ptr(), save_bytes, ws.mutable_data_ptr(), n, error_word(h),
                                 stream_of(h)),
              "ethos_xent_forward");
      }
    }
    if (what & 3) {
      ctx->save_for_backward({hidden_, weight_, save});
      ctx->saved_data["p"] = std::vector<int64_t>{reduction};
      // the gradients of a loss whose own gradient is 1, until the first backward
      if (dh.defined()) ctx->saved_data["dh"] = dh;
      if (dw.defined()) ctx->saved_data["dw"] = dw;
    }
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    once("linear_cross_entropy");
    const variable_list s = ctx->get_saved_variables();
    const std::vector<int64_t> p = ctx->saved_data["p"].toIntVector();
    const bool need_h = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    const Tensor &hidden = s[0], &weight = s[1], &save = s[2];
    const c10::cuda::CUDAGuard guard(hidden.device());
    const Tensor grad = grads[0].to(at::kFloat).contiguous();
    const int code = dtype_code(hidden, "hidden"), red = static_cast<int>(p[0]);
    Tensor dh, dw;
    auto take = [&](const char* name, bool need) {
      const auto it = ctx->saved_data.find(name);
      if (it == ctx->saved_data.end()) return Tensor();
      const Tensor t = it->second.toTensor();
      ctx->saved_data.erase(it);
      return need ? t : Tensor();
    };
    const bool kept = ctx->saved_data.count("dh") + ctx->saved_data.count("dw") > 0;
    dh = take("dh", need_h);
    dw = take("dw", need_w);
    if (kept) {
      check(L.ethos_xent_scale(static_cast<const float*>(grad.const_data_ptr()),
                             dh.defined() ? dh.mutable_data_ptr() : nullptr, dh.defined() ? dh.numel() : 0,
                             dw.defined() ? dw.mutable_data_ptr() : nullptr, dw.defined() ? dw.numel() : 0, code,
                             stream_of(hidden)),
            "ethos_xent_scale");
      return {dh, dw, Tensor(), Tensor(), Tensor(), Tensor()};
    }
    // also a second pass through the graph: the first one's results belong to its caller
    const Tensor h = as_rows(hidden), w = as_table(weight);
    const int64_t T = h.size(0), d = h.size(1), V = w.size(0);
    if (need_h) dh = at::empty({T, d}, h.options());
    if (need_w) dw = at::empty({V, d}, w.options());
    if (T == 0) {
      if (need_w) dw.zero_();
    } else {
      const size_t n = L.ethos_xent_backward_workspace_size(T, V, d, code);
      Tensor ws = bytes(n, h);
      check(L.ethos_xent_backward(h.const_data_ptr(), pitch(h), w.const_data_ptr(), pitch(w), code, red, T, V, d,
                                static_cast<const float*>(grad.const_data_ptr()), save.const_data_ptr(),
                                static_cast<size_t>(save.numel()), need_h ? dh.mutable_data_ptr() : nullptr,
                                need_w ? dw.mutable_data_ptr() : nullptr, ws.mutable_data_ptr(), n, error_word(h),
                                stream_of(h)),
            "ethos_xent_backward");
    }
    return {dh, dw, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor cross_entropy(const Tensor& hidden, const Tensor& weight, const Tensor& labels, int64_t ignore_index,
                     int64_t reduction, bool keep) {
  need_cuda(hidden, "hidden");
  need_on(hidden, weight, "weight");
  need_on(hidden, labels, "labels");
  dtype_code(hidden, "hidden");
  ids_i64(labels, "labels");
  TORCH_CHECK_VALUE(hidden.dim() >= 1 && weight.dim() == 2 && hidden.size(-1) == weight.size(1),
                    "hidden [T, d] and weight [V, d]: got ", hidden.sizes(), " and ", weight.sizes());
  TORCH_CHECK_VALUE(weight.scalar_type() == hidden.scalar_type(), "hidden is ", hidden.scalar_type(), ", weight ",
                    weight.scalar_type());
  TORCH_CHECK_VALUE(labels.sizes() == hidden.sizes().slice(0, hidden.dim() - 1), "labels ", labels.sizes(),
                    " do not belong to hidden ", hidden.sizes());
  const Tensor flat = hidden.dim() == 2 ? hidden : hidden.reshape({-1, hidden.size(-1)});
  const bool grad = at::GradMode::is_enabled();
  const int64_t what = (grad && hidden.requires_grad() ? 1 : 0) | (grad && weight.requires_grad() ? 2 : 0) | (keep ? 4 : 0);
  const Tensor loss = CrossEntropy::apply(flat, weight, labels.dim() == 1 ? labels : labels.reshape({-1}), ignore_index,
                                          reduction, what);
  return reduction == ETHOS_XENT_NONE && labels.dim() != 1 ? loss.view(labels.sizes()) : loss;
}

// f() without the interpreter's lock.
template <class F>
auto call(F f) {
  try {
    const py::gil_scoped_release off;
    return f();
  } catch (const StatusError& e) {
    const py::object cls = py::module_::import("ethos_b200._lib").attr("EthosError");
    PyErr_SetObject(cls.ptr(), cls(e.status, e.call).ptr());
    throw py::error_already_set();
  }
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("load", torch::wrap_pybind_function(load));
  m.def("set_error_word", torch::wrap_pybind_function([](int64_t device, int64_t ptr) {
          TORCH_CHECK(device >= 0 && device < 64, "device ", device);
          g_err[device] = reinterpret_cast<int*>(ptr);
        }));
  m.def("embedding", torch::wrap_pybind_function(
                         [](const Tensor& ids, const Tensor& weight, double scale, int64_t padding) {
                           return call([&] { return Embedding::apply(ids, weight, scale, padding); });
                         }));
  m.def("balance_loss",
        torch::wrap_pybind_function(
            [](const Tensor& weights, const Tensor& ids, int64_t experts, const std::optional<Tensor>& mask) {
              return call([&] {
                const variable_list r = Balance::apply(weights, ids, experts, mask);
                return std::make_tuple(r[0], r[1]);
              });
            }));
  m.def("cross_entropy", torch::wrap_pybind_function([](const Tensor& hidden, const Tensor& weight,
                                                        const Tensor& labels, int64_t ignore_index, int64_t reduction,
                                                        bool keep) {
          return call([&] { return cross_entropy(hidden, weight, labels, ignore_index, reduction, keep); });
        }));
}
