// torch binding of the training-step operators (include/purin_ops.h): autograd nodes, outputs
// and workspaces in C++.  A training step calls these operators many times with little work
// in each; the nodes' host time in Python (16 us forward, 25 us backward) was most of such a
// call.  Arguments are checked by the Python modules that call this one.
#include <c10/core/InferenceMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime.h>
#include <nvtx3/nvToolsExt.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <atomic>
#include <mutex>
#include <optional>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include "../../include/purin_ops.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::Variable;
using torch::autograd::variable_list;

int32_t code_of(at::ScalarType type) {
  switch (type) {
    case at::kDouble: return PURIN_OPS_FLOAT64;
    case at::kFloat: return PURIN_OPS_FLOAT32;
    case at::kBFloat16: return PURIN_OPS_BFLOAT16;
    case at::kHalf: return PURIN_OPS_FLOAT16;
    default: TORCH_CHECK(false, "unsupported element type ", type);
  }
}

// ---- calls ---------------------------------------------------------------------------

struct Launch {
  const char* name;
  cudaEvent_t start, end;
};
std::atomic<bool> g_recording{false};
std::mutex g_launches_mutex;
std::vector<Launch> g_launches;

void check(int32_t status, const char* name) {
  TORCH_CHECK(status == PURIN_OK, name, " failed (status ", status, "): ", purin_cp_last_error());
}

// Two events around one call, recorded on its stream.
struct Recording {
  Launch launch;
  bool on;
  cudaStream_t stream;
  Recording(const char* name, int device, cudaStream_t s) : launch{name, nullptr, nullptr}, on(false), stream(s) {
    if (!g_recording.load(std::memory_order_relaxed)) return;
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    // A captured call runs at each replay: it has no time of its own.
    on = cudaStreamIsCapturing(s, &capture) == cudaSuccess;
    if (!on) cudaGetLastError();
    on = on && capture == cudaStreamCaptureStatusNone;
    if (!on) return;
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));  // the events are the stream's device's
    on = cudaEventCreate(&launch.start) == cudaSuccess && cudaEventCreate(&launch.end) == cudaSuccess &&
         cudaEventRecord(launch.start, s) == cudaSuccess;
    if (!on) cudaGetLastError();  // not the call's error
  }
  void end() {
    if (!on || cudaEventRecord(launch.end, stream) != cudaSuccess) return;
    std::lock_guard<std::mutex> lock(g_launches_mutex);
    g_launches.push_back(launch);
    launch = {};
  }
  ~Recording() {
    if (launch.start) cudaEventDestroy(launch.start);
    if (launch.end) cudaEventDestroy(launch.end);
  }
};

// Runs one entry point on the device's current stream in an NVTX range, between two events
// while launches are recorded.
template <typename F>
void call(const char* name, int device, F&& f) {
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device).stream();
  Recording recording(name, device, stream);
  nvtxRangePushA(name);
  const int32_t status = f(static_cast<void*>(stream));
  nvtxRangePop();
  recording.end();
  check(status, name);
}

void record_launches(bool on) { g_recording.store(on); }

// (name, milliseconds) of the calls recorded since the last time, oldest first; waits for them.
std::vector<std::pair<std::string, float>> recorded_launches() {
  std::vector<Launch> launches;
  {
    std::lock_guard<std::mutex> lock(g_launches_mutex);
    launches.swap(g_launches);
  }
  std::vector<std::pair<std::string, float>> out;
  for (const Launch& l : launches) {
    float ms = 0.f;
    if (cudaEventSynchronize(l.end) != cudaSuccess || cudaEventElapsedTime(&ms, l.start, l.end) != cudaSuccess)
      cudaGetLastError();
    cudaEventDestroy(l.start);
    cudaEventDestroy(l.end);
    out.emplace_back(l.name, ms);
  }
  return out;
}

Tensor workspace(size_t bytes, const Tensor& like) {
  if (bytes == 0) return Tensor();
  return at::empty({int64_t(bytes)}, like.options().dtype(at::kByte));
}
void* pointer(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
size_t bytes_of(const Tensor& t) { return t.defined() ? size_t(t.numel()) : 0; }

// The same rows with adjacent elements, and the stride between them.
std::pair<Tensor, int64_t> rows_of(const Tensor& t) {
  if (t.is_contiguous()) return {t, t.size(1)};
  const Tensor rows = t.size(1) > 1 && t.stride(1) != 1 ? t.contiguous() : t;
  return {rows, rows.size(0) <= 1 ? rows.size(1) : rows.stride(0)};
}

// A tracer sees the outputs' allocation and not what is written to them by pointer: the traced
// function would return memory that nobody wrote.
void refuse_tracing(const char* what) {
  using c10::impl::TorchDispatchModeTLS;
  const bool traced = torch::jit::tracer::isTracing() ||
                      c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch) ||
                      (TorchDispatchModeTLS::any_modes_set() &&
                       TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value());
  TORCH_CHECK(!traced, what, " cannot be traced");
}

// The operators have no forward-mode derivative; outputs made without one would lose it.
void refuse_tangent(const char* what, const Tensor& t) {
  TORCH_CHECK(!t._fw_grad(0).defined(), what, " has no forward-mode derivative");
}

bool needs_gradient(std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t->requires_grad()) return true;
  return false;
}

// The same values, with a node that raises when it is differentiated.
variable_list raising(variable_list values, const char* message) {
  variable_list defined;
  for (const Variable& v : values)
    if (v.defined()) defined.push_back(v.detach().requires_grad_());
  if (defined.empty()) return values;
  auto node = std::make_shared<torch::autograd::DelayedError>(message, int64_t(defined.size()));
  at::AutoGradMode enabled(true);
  variable_list wrapped = (*node)(std::move(defined));
  size_t at = 0;
  for (Variable& v : values)
    if (v.defined()) v = wrapped[at++];
  return values;
}

// The gradients of a node that is differentiable once, which create_graph may ask for.
variable_list once(variable_list grads, bool graph) {
  return graph ? raising(std::move(grads), "this operator's gradient is not differentiable") : grads;
}

// ---- embedding -----------------------------------------------------------------------

PurinEmbeddingArgs embedding_args(const Tensor& like, const Tensor& ids, int64_t vocab, int64_t dim,
                                  double scale, int64_t padding) {
  PurinEmbeddingArgs a = {};
  a.device = like.get_device();
  a.dtype = code_of(like.scalar_type());
  a.ids_64bit = ids.scalar_type() == at::kLong;
  a.tokens = ids.numel();
  a.vocab = vocab;
  a.dim = dim;
  a.scale = scale;
  a.padding = padding;
  a.ids = ids.data_ptr();
  return a;
}

Tensor lookup(const Tensor& table, const Tensor& ids, double scale, int64_t padding) {
  const auto [rows, stride] = rows_of(table);
  Tensor out = at::empty({ids.numel(), table.size(1)}, table.options());
  PurinEmbeddingArgs a = embedding_args(table, ids, table.size(0), table.size(1), scale, padding);
  a.table = rows.data_ptr();
  a.table_stride = stride;
  a.out = out.data_ptr();
  call("purin_embedding_forward", a.device, [&](void* s) { return purin_embedding_forward(&a, s); });
  return out;
}

struct Embedding : Function<Embedding> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& ids, double scale,
                        int64_t padding) {
    ctx->save_for_backward({ids});
    ctx->saved_data["shape"] = std::make_tuple(table.size(0), table.size(1), scale, padding);
    return lookup(table, ids, scale, padding);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool graph = at::GradMode::is_enabled();
    torch::NoGradGuard no_grad;
    refuse_tracing("token_embedding");
    refuse_tangent("token_embedding", grads[0]);
    const Tensor ids = ctx->get_saved_variables()[0];
    const auto shape = ctx->saved_data["shape"].toTuple();
    const int64_t vocab = shape->elements()[0].toInt(), dim = shape->elements()[1].toInt();
    const auto [grad, stride] = rows_of(grads[0]);
    Tensor out = at::empty({vocab, dim}, grad.options());
    PurinEmbeddingArgs a = embedding_args(grad, ids, vocab, dim, shape->elements()[2].toDouble(),
                                          shape->elements()[3].toInt());
    a.grad_out = grad.data_ptr();
    a.grad_out_stride = stride;
    a.grad_table = out.data_ptr();
    size_t bytes = 0;
    check(purin_embedding_backward_workspace_size(&a, &bytes), "purin_embedding_backward");
    const Tensor ws = workspace(bytes, grad);
    call("purin_embedding_backward", a.device,
         [&](void* s) { return purin_embedding_backward(&a, pointer(ws), bytes_of(ws), s); });
    return once({out, Tensor(), Tensor(), Tensor()}, graph);
  }
};

Tensor embedding(const Tensor& table, const Tensor& ids, double scale, int64_t padding) {
  refuse_tracing("token_embedding");
  refuse_tangent("token_embedding", table);
  const Tensor flat = ids.dim() == 1 && ids.is_contiguous() ? ids : ids.reshape({-1}).contiguous();
  const Tensor out = needs_gradient({&table}) ? Embedding::apply(table, flat, scale, padding)
                                              : lookup(table, flat, scale, padding);
  if (ids.dim() == 1) return out;
  std::vector<int64_t> shape(ids.sizes().begin(), ids.sizes().end());
  shape.push_back(table.size(1));
  return out.view(shape);
}

// ---- routing -------------------------------------------------------------------------

std::tuple<Tensor, Tensor, Tensor> route(const Tensor& given, int64_t num_experts) {
  refuse_tracing("route_to_experts");
  const Tensor experts = given.contiguous();
  const auto options = experts.options().dtype(at::kInt);
  Tensor offsets = at::empty({num_experts + 1}, options);
  Tensor position = at::empty(experts.sizes(), options);
  Tensor source = at::empty({experts.numel()}, options);
  PurinRouteArgs a = {};
  a.device = experts.get_device();
  a.experts_64bit = experts.scalar_type() == at::kLong;
  a.tokens = experts.size(0);
  a.slots = experts.size(1);
  a.num_experts = num_experts;
  a.experts = experts.data_ptr();
  a.offsets = offsets.data_ptr<int32_t>();
  a.position = position.data_ptr<int32_t>();
  a.source = source.data_ptr<int32_t>();
  size_t bytes = 0;
  check(purin_route_workspace_size(&a, &bytes), "purin_route");
  const Tensor ws = workspace(bytes, experts);
  call("purin_route", a.device, [&](void* s) { return purin_route(&a, pointer(ws), bytes_of(ws), s); });
  return {offsets, position, source};
}

// A routing that a kernel may read, whole and on x's device.  `source` may be undefined.
void check_routing(const std::string& what, const Tensor& x, const Tensor& offsets, const Tensor& position,
                   const std::optional<Tensor>& source) {
  TORCH_CHECK_VALUE(position.dim() == 2 && position.size(1) >= 1 && offsets.dim() == 1 && offsets.size(0) >= 2, what,
                    ": the routing's position must have shape (tokens, slots) and offsets (experts + 1,), got ",
                    position.sizes(), " and ", offsets.sizes());
  TORCH_CHECK_TYPE(position.scalar_type() == at::kInt && offsets.scalar_type() == at::kInt, what,
                   ": the routing's position and offsets must be int32, got ", position.scalar_type(), " and ",
                   offsets.scalar_type());
  TORCH_CHECK_VALUE(position.is_contiguous() && offsets.is_contiguous(), what,
                    ": the routing's position and offsets must be contiguous, as route_to_experts makes them");
  // Positions name rows of the whole routing: of a part of it, rows that are not there.
  TORCH_CHECK_VALUE(!source || source->numel() == position.numel(), what, ": the routing has ", source->numel(),
                    " slots but ", position.numel(), " positions");
  TORCH_CHECK(x.is_cuda(), what, " runs on CUDA devices only; got a tensor on ", x.device());
  TORCH_CHECK_VALUE(position.device() == x.device() && offsets.device() == x.device(), what, ": tensors are on ",
                    x.device(), ", ", position.device(), " and ", offsets.device());
}

PurinRouteRowsArgs rows_args(const Tensor& rows, const Tensor& offsets, const Tensor& position) {
  PurinRouteRowsArgs a = {};
  a.device = rows.get_device();
  a.dtype = code_of(rows.scalar_type());
  a.weights_dtype = PURIN_OPS_FLOAT32;
  a.tokens = position.size(0);
  a.slots = position.size(1);
  a.num_experts = offsets.size(0) - 1;
  a.dim = rows.size(1);
  a.offsets = offsets.data_ptr<int32_t>();
  a.position = position.data_ptr<int32_t>();
  return a;
}

Tensor spread(const Tensor& x, const Tensor& offsets, const Tensor& position) {
  const auto [rows, stride] = rows_of(x);
  Tensor out = at::empty({position.numel(), x.size(1)}, x.options());
  PurinRouteRowsArgs a = rows_args(x, offsets, position);
  a.token_rows = rows.data_ptr();
  a.token_stride = stride;
  a.sorted_out = out.data_ptr();
  call("purin_route_spread", a.device, [&](void* s) { return purin_route_spread(&a, s); });
  return out;
}

Tensor gather(const Tensor& sorted, const Tensor& weights, const Tensor& offsets, const Tensor& position) {
  const auto [rows, stride] = rows_of(sorted);
  Tensor out = at::empty({position.size(0), sorted.size(1)}, sorted.options());
  PurinRouteRowsArgs a = rows_args(sorted, offsets, position);
  a.sorted_rows = rows.data_ptr();
  a.sorted_stride = stride;
  if (weights.defined()) {
    a.weights = weights.data_ptr();
    a.weights_dtype = code_of(weights.scalar_type());
  }
  a.token_out = out.data_ptr();
  call("purin_route_gather", a.device, [&](void* s) { return purin_route_gather(&a, s); });
  return out;
}

struct Dispatch : Function<Dispatch> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& offsets, const Tensor& position) {
    ctx->save_for_backward({offsets, position});
    return spread(x, offsets, position);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool graph = at::GradMode::is_enabled();
    torch::NoGradGuard no_grad;
    refuse_tracing("dispatch_to_experts");
    refuse_tangent("dispatch_to_experts", grads[0]);
    const variable_list saved = ctx->get_saved_variables();
    return once({gather(grads[0], Tensor(), saved[0], saved[1]), Tensor(), Tensor()}, graph);
  }
};

struct Combine : Function<Combine> {
  static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& weights,
                        const Tensor& offsets, const Tensor& position) {
    ctx->save_for_backward({rows, weights, offsets, position});
    return gather(rows, weights, offsets, position);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool graph = at::GradMode::is_enabled();
    torch::NoGradGuard no_grad;
    refuse_tracing("combine_from_experts");
    refuse_tangent("combine_from_experts", grads[0]);
    const variable_list saved = ctx->get_saved_variables();
    const auto [grad, grad_stride] = rows_of(grads[0]);
    const auto [rows, rows_stride] = rows_of(saved[0]);
    const Tensor& weights = saved[1];
    PurinRouteRowsArgs a = rows_args(grad, saved[2], saved[3]);
    a.token_rows = grad.data_ptr();
    a.token_stride = grad_stride;
    a.sorted_rows = rows.data_ptr();
    a.sorted_stride = rows_stride;
    a.weights = weights.data_ptr();
    a.weights_dtype = code_of(weights.scalar_type());
    Tensor grad_rows, grad_weights;
    if (ctx->needs_input_grad(0)) grad_rows = at::empty(rows.sizes(), rows.options());
    if (ctx->needs_input_grad(1)) grad_weights = at::empty(weights.sizes(), weights.options());
    a.sorted_out = pointer(grad_rows);
    a.grad_weights = pointer(grad_weights);
    call("purin_route_combine_backward", a.device,
         [&](void* s) { return purin_route_combine_backward(&a, s); });
    return once({grad_rows, grad_weights, Tensor(), Tensor()}, graph);
  }
};

Tensor dispatch(const Tensor& x, const Tensor& offsets, const Tensor& position) {
  refuse_tracing("dispatch_to_experts");
  refuse_tangent("dispatch_to_experts", x);
  return needs_gradient({&x}) ? Dispatch::apply(x, offsets, position) : spread(x, offsets, position);
}
Tensor combine(const Tensor& rows, const Tensor& given, const Tensor& offsets, const Tensor& position) {
  refuse_tracing("combine_from_experts");
  refuse_tangent("combine_from_experts", rows);
  refuse_tangent("combine_from_experts", given);
  const Tensor weights = given.contiguous();
  return needs_gradient({&rows, &weights}) ? Combine::apply(rows, weights, offsets, position)
                                           : gather(rows, weights, offsets, position);
}

// ---- linear cross entropy ------------------------------------------------------------

enum Reduction : int64_t { kNone = 0, kSum = 1, kMean = 2 };

// The arguments; `kept` holds each row's softmax data, then the mean's divisor.
PurinLossArgs loss_args(const Tensor& hidden, int64_t hidden_stride, const Tensor& weight,
                        int64_t weight_stride, const Tensor& targets, int64_t ignore, const Tensor& kept) {
  PurinLossArgs a = {};
  a.device = hidden.get_device();
  a.dtype = code_of(hidden.scalar_type());
  a.targets_64bit = targets.scalar_type() == at::kLong;
  a.tokens = hidden.size(0);
  a.vocab = weight.size(0);
  a.dim = hidden.size(1);
  a.ignore = ignore;
  a.hidden = hidden.data_ptr();
  a.hidden_stride = hidden_stride;
  a.weight = weight.data_ptr();
  a.weight_stride = weight_stride;
  a.targets = targets.data_ptr();
  a.softmax = kept.data_ptr<float>();
  return a;
}

std::pair<Tensor, Tensor> loss_forward(const Tensor& hidden, const Tensor& weight, const Tensor& targets,
                                       int64_t ignore, int64_t reduction) {
  const auto [h, h_stride] = rows_of(hidden);
  const auto [w, w_stride] = rows_of(weight);
  const auto options = hidden.options().dtype(at::kFloat);
  const int64_t tokens = hidden.size(0);
  Tensor kept = at::empty({2 * tokens + 1}, options);
  Tensor each = at::empty({tokens}, options);
  Tensor loss = reduction == kNone ? each : at::empty({}, options);
  PurinLossArgs a = loss_args(h, h_stride, w, w_stride, targets, ignore, kept);
  a.loss = each.data_ptr<float>();
  if (reduction == kSum) a.sum = loss.data_ptr<float>();
  if (reduction == kMean) {
    a.mean = loss.data_ptr<float>();
    a.count = kept.data_ptr<float>() + 2 * tokens;
  }
  size_t bytes = 0;
  check(purin_loss_workspace_size(&a, 0, &bytes), "purin_loss_forward");
  const Tensor ws = workspace(bytes, hidden);
  call("purin_loss_forward", a.device,
       [&](void* s) { return purin_loss_forward(&a, pointer(ws), bytes_of(ws), s); });
  return {loss, kept};
}

struct LinearCrossEntropy : Function<LinearCrossEntropy> {
  static Tensor forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight,
                        const Tensor& targets, int64_t ignore, int64_t reduction) {
    const auto [loss, kept] = loss_forward(hidden, weight, targets, ignore, reduction);
    ctx->save_for_backward({hidden, weight, targets, kept});
    ctx->saved_data["call"] = std::make_tuple(ignore, reduction);
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool graph = at::GradMode::is_enabled();
    torch::NoGradGuard no_grad;
    refuse_tracing("linear_cross_entropy");
    refuse_tangent("linear_cross_entropy", grads[0]);
    const variable_list saved = ctx->get_saved_variables();
    const auto options = ctx->saved_data["call"].toTuple();
    const int64_t ignore = options->elements()[0].toInt(), reduction = options->elements()[1].toInt();
    const auto [h, h_stride] = rows_of(saved[0]);
    const auto [w, w_stride] = rows_of(saved[1]);
    const Tensor grad = grads[0].contiguous();
    PurinLossArgs a = loss_args(h, h_stride, w, w_stride, saved[2], ignore, saved[3]);
    a.grad_loss = grad.data_ptr<float>();
    a.grad_stride = reduction == kNone ? 1 : 0;
    a.divisor = reduction == kMean ? saved[3].data_ptr<float>() + 2 * h.size(0) : nullptr;
    Tensor grad_hidden, grad_weight;
    if (ctx->needs_input_grad(0)) grad_hidden = at::empty(h.sizes(), h.options());
    if (ctx->needs_input_grad(1)) grad_weight = at::empty(w.sizes(), w.options());
    a.grad_hidden = pointer(grad_hidden);
    a.grad_weight = pointer(grad_weight);
    size_t bytes = 0;
    check(purin_loss_workspace_size(&a, 1, &bytes), "purin_loss_backward");
    const Tensor ws = workspace(bytes, h);
    call("purin_loss_backward", a.device,
         [&](void* s) { return purin_loss_backward(&a, pointer(ws), bytes_of(ws), s); });
    return once({grad_hidden, grad_weight, Tensor(), Tensor(), Tensor()}, graph);
  }
};

Tensor linear_cross_entropy(const Tensor& hidden, const Tensor& weight, const Tensor& given,
                            int64_t ignore, int64_t reduction) {
  refuse_tracing("linear_cross_entropy");
  refuse_tangent("linear_cross_entropy", hidden);
  refuse_tangent("linear_cross_entropy", weight);
  const Tensor targets = given.contiguous();
  if (needs_gradient({&hidden, &weight}))
    return LinearCrossEntropy::apply(hidden, weight, targets, ignore, reduction);
  return loss_forward(hidden, weight, targets, ignore, reduction).first;
}

// ---- gradients -----------------------------------------------------------------------

// Every tensor's elements fill a range of memory, outs[i] in tensors[i]'s order.
Tensor gradients(const std::vector<Tensor>& tensors, const std::vector<Tensor>& outs, bool clip,
                 double max_norm, double eps) {
  const char* what = clip ? "clip_gradients" : "gradient_norm";
  refuse_tracing(what);
  const bool forward_mode = torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr;
  std::vector<PurinGradient> list(tensors.size());
  bool wide = false, graph = false;
  for (size_t i = 0; i < tensors.size(); ++i) {
    if (forward_mode) refuse_tangent(what, tensors[i]);
    if (clip) {
      if (forward_mode) refuse_tangent(what, outs[i]);
      // Counting the change below would raise, behind a launch that has written.
      TORCH_CHECK(!outs[i].is_inference() || c10::InferenceMode::is_enabled(), what,
                  ": a tensor of inference mode is not written outside it");
    }
    list[i] = {tensors[i].data_ptr(), outs[i].data_ptr(), tensors[i].numel(),
               code_of(tensors[i].scalar_type()), 0};
    wide |= list[i].dtype == PURIN_OPS_FLOAT64;
    graph |= tensors[i].requires_grad();
  }
  Tensor norm = at::empty({}, tensors[0].options().dtype(wide ? at::kDouble : at::kFloat));
  PurinGradientsArgs a = {};
  a.device = norm.get_device();
  a.norm_dtype = wide ? PURIN_OPS_FLOAT64 : PURIN_OPS_FLOAT32;
  a.tensors = int64_t(list.size());
  a.list = list.data();
  a.clip = clip;
  a.max_norm = max_norm;
  a.eps = eps;
  a.norm = norm.data_ptr();
  size_t bytes = 0;
  check(purin_gradients_workspace_size(&a, &bytes), "purin_gradients");
  const Tensor ws = workspace(bytes, norm);
  call("purin_gradients", a.device, [&](void* s) { return purin_gradients(&a, pointer(ws), bytes_of(ws), s); });
  if (clip)  // autograd learns of what was written in place
    for (const Tensor& o : outs) o.unsafeGetTensorImpl()->bump_version();
  else if (graph && at::GradMode::is_enabled())
    return raising({norm}, "gradient_norm is not differentiable")[0];
  return norm;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("embedding", &embedding);
  m.def("route", &route);
  m.def("check_routing", &check_routing);
  m.def("dispatch", &dispatch);
  m.def("combine", &combine);
  m.def("linear_cross_entropy", &linear_cross_entropy);
  m.def("gradients", &gradients);
  m.def("record_launches", &record_launches, "Record every native call from here on, or stop.");
  m.def("recorded_launches", &recorded_launches,
        "(name, milliseconds) of the calls recorded since the last time; waits for them.");
}
