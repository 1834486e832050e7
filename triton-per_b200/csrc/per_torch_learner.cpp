// Python binding of the learner's operators for torch tensors: layer norm as
// an autograd node, the global gradient norm and its clipping. Checks the
// tensors, allocates outputs and workspaces with ATen on the current stream
// (one workspace per call, so calls on different streams and captured graphs
// share none) and calls the C ABI. No kernels here.
#include <torch/extension.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <algorithm>
#include <mutex>
#include <optional>
#include <string>
#include <utility>
#include <vector>

#include "per_b200.h"

namespace py = pybind11;

namespace {

using at::Tensor;

std::string error_text(const char* what, int rc) {
  std::string s = std::string("per_b200: ") + what + " failed: " + per_error_string(rc);
  if (rc == PER_ERR_CUDA) s += ", cudaError " + std::to_string(per_last_cuda_error());
  return s;
}

// Raises per_b200._lib.PerError (the GIL is held).
void check(const char* what, int rc) {
  if (rc == PER_OK) return;
  py::object cls = py::module_::import("per_b200._lib").attr("PerError");
  PyErr_SetObject(cls.ptr(), cls(what, rc).ptr());
  throw py::error_already_set();
}

int32_t code_of(at::ScalarType t) {
  return t == at::kFloat ? PER_F32 : t == at::kBFloat16 ? PER_BF16 : t == at::kHalf ? PER_F16 : -1;
}

void* stream_of(const Tensor& t) {
  return c10::cuda::getCurrentCUDAStream(t.get_device()).stream();
}

// A new tensor on the current stream, without the dispatcher's detour (about
// 1 us of host time less than at::empty, of which a training step makes six).
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, c10::Device device) {
  return Tensor(at::detail::empty_cuda(sizes, type, device, std::nullopt));
}

// A tracer records what the dispatcher sees, and these calls pass beneath it:
// their results would go into the trace as constants. Refused while one is at
// work: torch.jit.trace (and ONNX export by it), make_fx, fake tensors,
// functionalization, torch.export. Other dispatch modes (counters, selective
// recomputation) change no result by not seeing the call.
bool being_traced() {
  using Modes = c10::impl::TorchDispatchModeTLS;
  using Key = c10::impl::TorchDispatchModeKey;
  using D = c10::DispatchKey;
  constexpr c10::DispatchKeySet tracers({D::Tracer, D::PreDispatch}), modes(D::Python);
  const c10::DispatchKeySet tls = c10::impl::tls_local_dispatch_key_set().included_;
  if (C10_LIKELY(!tls.has_any(tracers | modes))) return false;
  return tls.has_any(tracers) ||
         (Modes::get_mode(Key::PROXY) || Modes::get_mode(Key::FAKE) || Modes::get_mode(Key::FUNCTIONAL));
}

void refuse_tracing(const char* what) {
  if (being_traced())
    throw std::runtime_error(std::string("per_b200.") + what +
                             " cannot be traced or exported (its result would be recorded as a "
                             "constant); use torch's own operator in what is traced");
}

// Tensors of vmap, torch.func and functionalization have no memory of their own.
void refuse_wrapped(const Tensor& t, const char* what) {
  using D = c10::DispatchKey;
  constexpr c10::DispatchKeySet wrappers(
      {D::FuncTorchBatched, D::BatchedNestedTensor, D::FuncTorchGradWrapper, D::Functionalize});
  if (C10_UNLIKELY(t.key_set().has_any(wrappers)))
    throw std::runtime_error(std::string("per_b200.") + what +
                             " takes plain tensors only (it cannot be used under vmap, torch.func "
                             "transforms or functionalization)");
}

// ------------------------------------------------------------- layer norm

// `t` as rows of `dim` values: the elements between the starts of two rows,
// or -1 where its strides are no such rows (then it has to be copied).
// `norm_dims`: trailing dimensions that make up a row. Stride 0 (one row for
// all, as an expanded gradient has) only if `broadcast`.
int64_t row_stride(const Tensor& t, int64_t norm_dims, int64_t dim, bool broadcast) {
  const auto sizes = t.sizes();
  const auto strides = t.strides();
  const int64_t lead = t.dim() - norm_dims;
  int64_t want = 1;
  for (int64_t d = t.dim() - 1; d >= lead; --d) {
    if (sizes[d] != 1 && strides[d] != want) return -1;
    want *= sizes[d];
  }
  int64_t stride = -1;
  for (int64_t d = lead - 1; d >= 0; --d) {
    if (sizes[d] == 1) continue;
    if (stride < 0) {
      stride = strides[d];
      want = stride * sizes[d];
    } else {
      if (strides[d] != want) return -1;
      want *= sizes[d];
    }
  }
  if (stride < 0) return dim;  // at most one row
  if (stride == 0) return broadcast ? 0 : -1;
  return stride < dim ? -1 : stride;
}

// `t` itself or a contiguous copy, and its row stride
std::pair<Tensor, int64_t> rows_of(const Tensor& t, int64_t norm_dims, int64_t dim,
                                   bool broadcast = false) {
  const int64_t s = row_stride(t, norm_dims, dim, broadcast);
  if (s >= 0) return {t, s};
  return {t.contiguous(), dim};
}

// The values in memory: a lazily negated view (the imaginary part of a
// conjugated tensor) holds them with the other sign.
Tensor plain(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }

void* ptr_or_null(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

struct Shape {
  int64_t norm_dims = 0, dim = 1, rows = 1;
};

struct LayerNormBackward : public torch::autograd::Node {
  torch::autograd::SavedVariable x, weight;
  Tensor stats;
  bool has_weight = false, has_bias = false;
  at::ScalarType param_type = at::kFloat;
  Shape shape;

  std::string name() const override { return "PerLayerNormBackward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    x.reset_data();
    weight.reset_data();
    stats.reset();
  }

  torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    torch::autograd::variable_list out(3);
    if (grads.empty() || !grads[0].defined()) return out;
    TORCH_CHECK(!being_traced(), "per_b200.layer_norm: its backward pass cannot be traced");
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "per_b200.layer_norm: its gradient is not differentiable again "
                "(backward with create_graph=True)");
    const Tensor xv = plain(x.unpack());
    const Tensor wv = has_weight ? plain(weight.unpack()).contiguous() : Tensor();
    const bool want_x = task_should_compute_output(0);
    const bool want_w = has_weight && task_should_compute_output(1);
    const bool want_b = has_bias && task_should_compute_output(2);
    c10::cuda::CUDAGuard guard(xv.device());
    TORCH_CHECK(grads[0].device() == xv.device() && grads[0].scalar_type() == xv.scalar_type(),
                "per_b200.layer_norm: the gradient must have the input's type and device");
    const auto [xr, xs] = rows_of(xv, shape.norm_dims, shape.dim);
    const auto [dy, ds] = rows_of(plain(grads[0]), shape.norm_dims, shape.dim, true);
    if (want_x) out[0] = fresh(xv.sizes(), xv.scalar_type(), xv.device());
    const auto norm_sizes = xv.sizes().slice(xv.dim() - shape.norm_dims);
    if (want_w) out[1] = fresh(norm_sizes, param_type, xv.device());
    if (want_b) out[2] = fresh(norm_sizes, param_type, xv.device());
    if (shape.dim == 0) return out;
    const per_norm_t n{shape.rows, shape.dim, code_of(xv.scalar_type()), code_of(param_type), 0.f};
    int64_t bytes = 0;
    Tensor ws;
    if (shape.rows > 0) {
      bytes = per_layer_norm_backward_workspace(&n);
      ws = fresh({bytes}, at::kByte, xv.device());
    }
    const int rc = per_layer_norm_backward(
        &n, dy.data_ptr(), ds, xr.data_ptr(), xs, ptr_or_null(wv), stats.data_ptr<float>(),
        ptr_or_null(out[0]), shape.dim, ptr_or_null(out[1]),
        ptr_or_null(out[2]), ptr_or_null(ws), bytes, stream_of(xv));
    TORCH_CHECK(rc == PER_OK, error_text("per_layer_norm_backward", rc));
    return out;
  }
};

// A leaf whose gradient accumulator lives on, from an eager pass, on the
// default stream cannot take part in a captured backward pass: the engine
// would wait on the default stream within the capture, which ends the
// process. Refused here, while nothing of it has been captured.
void check_capture(const Tensor& t, const char* name) {
  if (!t.defined() || !t.requires_grad() || !t.is_leaf()) return;
  const auto acc = torch::autograd::impl::try_get_grad_accumulator(t);
  if (!acc) return;
  const auto s = acc->stream();
  if (s && s->id() == c10::cuda::getDefaultCUDAStream(t.get_device()).id())
    throw std::runtime_error(
        std::string("per_b200.layer_norm: ") + name + " is still part of an eager graph made on "
        "the default stream; drop that graph's outputs (del loss) before capturing, or make it on "
        "a side stream");
}

Tensor layer_norm(const Tensor& x, const std::vector<int64_t>& normalized_shape,
                  const std::optional<Tensor>& weight, const std::optional<Tensor>& bias,
                  double eps) {
  refuse_tracing("layer_norm");
  if (!x.is_cuda())
    throw std::runtime_error("per_b200.layer_norm runs on CUDA devices only (no CPU fallback)");
  if (x.layout() != at::kStrided) throw py::type_error("layer_norm: input must be strided");
  if (code_of(x.scalar_type()) < 0)
    throw py::type_error("layer_norm: input must be float32, bfloat16 or float16");
  Shape s;
  s.norm_dims = (int64_t)normalized_shape.size();
  if (s.norm_dims < 1 || s.norm_dims > x.dim())
    throw py::value_error("layer_norm: normalized_shape must name at least one trailing dimension "
                          "of the input");
  const int64_t lead = x.dim() - s.norm_dims;
  for (int64_t d = 0; d < s.norm_dims; ++d) {
    if (x.size(lead + d) != normalized_shape[d])
      throw py::value_error("layer_norm: the input's trailing dimensions differ from "
                            "normalized_shape");
    s.dim *= normalized_shape[d];
  }
  for (int64_t d = 0; d < lead; ++d) s.rows *= x.size(d);
  if (!(eps >= 0)) throw py::value_error("layer_norm: eps must not be negative");
  Tensor w = weight ? *weight : Tensor(), b = bias ? *bias : Tensor();
  for (const Tensor* t : {&x, static_cast<const Tensor*>(&w), static_cast<const Tensor*>(&b)}) {
    if (!t->defined()) continue;
    refuse_wrapped(*t, "layer_norm");
    if (t->_fw_grad(0).defined())
      throw std::runtime_error("per_b200.layer_norm has no forward-mode derivative");
  }
  at::ScalarType param_type = at::kFloat;
  for (const Tensor* p : {&w, &b}) {
    if (!p->defined()) continue;
    if (p->sizes() != at::IntArrayRef(normalized_shape))
      throw py::value_error("layer_norm: weight and bias must have the shape normalized_shape");
    if (p->device() != x.device())
      throw py::value_error("layer_norm: weight and bias must be on the input's device");
    if (p->scalar_type() != at::kFloat && p->scalar_type() != x.scalar_type())
      throw py::type_error("layer_norm: weight and bias must be float32 or of the input's type");
    param_type = p->scalar_type();
  }
  if (w.defined() && b.defined() && w.scalar_type() != b.scalar_type())
    throw py::type_error("layer_norm: weight and bias must have one type");

  c10::cuda::CUDAGuard guard(x.device());
  const bool grad = at::GradMode::is_enabled() &&
                    (x.requires_grad() || (w.defined() && w.requires_grad()) ||
                     (b.defined() && b.requires_grad()));
  const auto stream = c10::cuda::getCurrentCUDAStream(x.get_device());
  if (grad) {
    cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(stream.stream(), &cs) == cudaSuccess &&
        cs != cudaStreamCaptureStatusNone) {
      check_capture(x, "the input");
      check_capture(w, "weight");
      check_capture(b, "bias");
    }
  }
  Tensor y, xr, stats;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    int64_t xs = 0;
    std::tie(xr, xs) = rows_of(plain(x), s.norm_dims, s.dim);
    y = fresh(x.sizes(), x.scalar_type(), x.device());
    if (grad) stats = fresh({s.rows, 4}, at::kFloat, x.device());
    if (s.rows > 0 && s.dim > 0) {
      const Tensor wc = w.defined() ? plain(w).contiguous() : w;
      const Tensor bc = b.defined() ? plain(b).contiguous() : b;
      const per_norm_t n{s.rows, s.dim, code_of(x.scalar_type()), code_of(param_type), (float)eps};
      check("per_layer_norm",
            per_layer_norm(&n, xr.data_ptr(), xs, ptr_or_null(wc), ptr_or_null(bc), y.data_ptr(),
                           s.dim, grad ? stats.data_ptr<float>() : nullptr, stream.stream()));
    }
  }
  if (grad) {
    auto node = std::shared_ptr<LayerNormBackward>(new LayerNormBackward(),
                                                   torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, w, b));
    node->x = torch::autograd::SavedVariable(x, false);
    if (w.defined()) node->weight = torch::autograd::SavedVariable(w, false);
    node->stats = stats;
    node->has_weight = w.defined();
    node->has_bias = b.defined();
    node->param_type = param_type;
    node->shape = s;
    const auto nr = node->add_input_metadata(y);
    torch::autograd::impl::set_gradient_edge(y, {node, nr});
  }
  return y;
}

// ------------------------------------------------------- gradient norms

// The list as the C ABI takes it; checks type, device and memory layout.
// `writes`: also that no two tensors share memory.
struct List {
  // borrowed: the caller's list holds them (or the parameters whose gradients
  // they are), and the GIL is held until the call's work is enqueued
  std::vector<at::TensorImpl*> impl;
  std::vector<per_tensor_t> t;
  c10::Device device{c10::kCPU};

  void add(const Tensor& g, const char* what) {
    if (!g.is_cuda())
      throw std::runtime_error(std::string("per_b200.") + what +
                               " runs on CUDA devices only (no CPU fallback)");
    if (g.layout() != at::kStrided)
      throw py::type_error(std::string(what) + ": gradients must be strided (dense) tensors");
    refuse_wrapped(g, what);
    const int32_t code = code_of(g.scalar_type());
    if (code < 0)
      throw py::type_error(std::string(what) + ": gradients must be float32, bfloat16 or float16");
    if (t.empty())
      device = g.device();
    else if (g.device() != device)
      throw py::value_error(std::string(what) + ": gradients must be on one device");
    if (!g.is_non_overlapping_and_dense())
      throw py::value_error(std::string(what) +
                            ": gradients must fill their memory without gaps or overlaps");
    impl.push_back(g.unsafeGetTensorImpl());
    const int64_t n = g.numel();
    t.push_back(per_tensor_t{n ? g.data_ptr() : nullptr, n, code, 0});
  }

  void check_disjoint(const char* what) const {
    std::vector<std::pair<uintptr_t, uintptr_t>> r;
    r.reserve(t.size());
    bool sorted = true;
    for (const auto& e : t) {
      if (!e.count) continue;
      const uintptr_t a = (uintptr_t)e.data;
      if (!r.empty() && a < r.back().first) sorted = false;
      r.emplace_back(a, a + (uintptr_t)e.count * (e.dtype == PER_F32 ? 4 : 2));
    }
    if (!sorted) std::sort(r.begin(), r.end());
    for (size_t i = 1; i < r.size(); ++i)
      if (r[i].first < r[i - 1].second)
        throw py::value_error(std::string(what) + ": two gradients share memory (is a parameter "
                                                  "listed twice?)");
  }

  void* stream() const { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }
  // the tensors have been written to
  void written() const {
    for (at::TensorImpl* g : impl)
      if (!g->is_inference()) g->bump_version();
  }
};

List list_of(const py::list& tensors, bool take_grads, const char* what) {
  refuse_tracing(what);
  List l;
  l.impl.reserve(tensors.size());
  l.t.reserve(tensors.size());
  for (const py::handle& h : tensors) {
    if (!THPVariable_Check(h.ptr())) throw py::type_error(std::string(what) + ": expected tensors");
    const Tensor& v = THPVariable_Unpack(h.ptr());
    if (!take_grads) {
      l.add(v, what);
    } else if (v.grad().defined()) {
      l.add(v.grad(), what);
    }
  }
  return l;
}

std::pair<Tensor, Tensor> norm_and_workspace(const List& l, int64_t* bytes) {
  *bytes = per_grad_norm_workspace((int64_t)l.t.size());
  return {fresh({}, at::kFloat, l.device), fresh({*bytes}, at::kByte, l.device)};
}

// grad_norm(tensors, kind) -> float32 scalar on the device; None for an empty list
py::object grad_norm(const py::list& tensors, bool take_grads, int kind) {
  const List l = list_of(tensors, take_grads, "grad_norm");
  if (l.t.empty()) return py::none();
  c10::cuda::CUDAGuard guard(l.device);
  int64_t bytes = 0;
  auto [norm, ws] = norm_and_workspace(l, &bytes);
  check("per_grad_norm", per_grad_norm(l.t.data(), (int64_t)l.t.size(), kind,
                                       norm.data_ptr<float>(), ws.data_ptr(), bytes, l.stream()));
  return py::cast(norm);
}

py::object clip_grad_norm(const py::list& params, int kind, double max_norm) {
  const List l = list_of(params, true, "clip_grad_norm_");
  if (l.t.empty()) return py::none();
  l.check_disjoint("clip_grad_norm_");
  c10::cuda::CUDAGuard guard(l.device);
  int64_t bytes = 0;
  auto [norm, ws] = norm_and_workspace(l, &bytes);
  check("per_clip_grad_norm",
        per_clip_grad_norm(l.t.data(), (int64_t)l.t.size(), kind, (float)max_norm,
                           norm.data_ptr<float>(), ws.data_ptr(), bytes, l.stream()));
  l.written();
  return py::cast(norm);
}

void clip_grads_with_norm(const py::list& params, double max_norm, const Tensor& norm) {
  const List l = list_of(params, true, "clip_grads_with_norm_");
  if (l.t.empty()) return;
  l.check_disjoint("clip_grads_with_norm_");
  refuse_wrapped(norm, "clip_grads_with_norm_");
  if (norm.device() != l.device || norm.scalar_type() != at::kFloat || norm.numel() != 1)
    throw py::value_error("clip_grads_with_norm_: total_norm must be one float32 value on the "
                          "gradients' device");
  for (const auto& e : l.t)
    if (e.count && (uintptr_t)norm.data_ptr() >= (uintptr_t)e.data &&
        (uintptr_t)norm.data_ptr() < (uintptr_t)e.data + (uintptr_t)e.count * (e.dtype == PER_F32 ? 4 : 2))
      throw py::value_error("clip_grads_with_norm_: total_norm must not be part of a gradient");
  c10::cuda::CUDAGuard guard(l.device);
  const Tensor value = plain(norm);
  check("per_scale_grads", per_scale_grads(l.t.data(), (int64_t)l.t.size(), (float)max_norm,
                                           value.data_ptr<float>(), l.stream()));
  l.written();
}

}  // namespace

void per_register_learner(py::module_& m) {
  m.def("layer_norm", &layer_norm);
  m.def("grad_norm", &grad_norm);
  m.def("clip_grad_norm", &clip_grad_norm);
  m.def("clip_grads_with_norm", &clip_grads_with_norm);
}
