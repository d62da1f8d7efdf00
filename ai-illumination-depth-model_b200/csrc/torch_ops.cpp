// The token operators and the AdamW step as calls on torch tensors: argument
// checks, result allocation (on the current stream of the tensors' device) and
// the C entry point, in one native call. A small call's kernel takes a few
// microseconds; checking and allocating from the interpreter took three times
// as long.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>

#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "illumina.h"

namespace py = pybind11;

namespace {

typedef std::optional<at::Tensor> MaybeTensor;

// Becomes illumina.IlluminaError(status, message).
struct Refused {
  int status;
  std::string message;
};

[[noreturn]] void refuse(std::string message) { throw Refused{ILLUMINA_INVALID_ARG, std::move(message)}; }
inline void need(bool ok, const char *message) {
  if (!ok) refuse(message);
}
inline void need(bool ok, const char *name, const char *message) {
  if (!ok) refuse(std::string(name) + " " + message);
}
inline void check(illumina_status status) {
  if (status != ILLUMINA_OK) throw Refused{status, illumina_last_error()};
}

// Makes the device of `x` current; `stream` is its current stream.
struct On {
  c10::cuda::OptionalCUDAGuard guard;
  cudaStream_t stream;
  explicit On(const at::Tensor &x) {
    guard.set_device(x.device());
    stream = c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
  }
};

// The calls record nothing for autograd: a tensor whose gradient or tangent
// would be lost is refused.
inline void no_gradient(const at::Tensor &x) {
  need(!(c10::GradMode::is_enabled() && x.requires_grad()),
       "a tensor requires a gradient, which these calls do not record: detach it, or call under torch.no_grad()");
  need(!x._fw_grad(0).defined(), "a tensor carries a tangent, which these calls do not pass on");
}
inline void no_gradient(const MaybeTensor &x) {
  if (x.has_value()) no_gradient(*x);
}
template <typename... X>
void no_gradients(const X &...x) {
  (no_gradient(x), ...);
}

// A view whose negation is still to be done (z.conj().imag) has other values in
// memory than it stands for.
inline void as_stored(const char *name, const at::Tensor &x) {
  need(!x.is_neg(), name, "is a view with a lazy negation: call resolve_neg() on it");
}

// A storage tensor: on a CUDA device, float32 or bfloat16, contiguous in its
// last dimension; returns its precision.
int storage(const char *name, const at::Tensor &x, int dims = -1) {
  need(x.is_cuda(), name, "must be a CUDA tensor");
  as_stored(name, x);
  if (dims >= 0 && x.dim() != dims) refuse(std::string(name) + " must have " + std::to_string(dims) + " dimensions");
  need(x.dim() > 0 && (x.size(-1) <= 1 || x.stride(-1) == 1), name, "must be contiguous in its last dimension");
  const auto t = x.scalar_type();
  if (t == at::kFloat) return ILLUMINA_PRECISION_F32;
  need(t == at::kBFloat16, name, "must be float32 or bfloat16");
  return ILLUMINA_PRECISION_BF16;
}
void storage_like(const char *name, const at::Tensor &x, const at::Tensor &like, int dims = -1) {
  storage(name, x, dims);
  need(x.scalar_type() == like.scalar_type() && x.device() == like.device(), name, "must have the type and device of the others");
}

// A contiguous vector of n values; nullptr for none.
template <typename T>
T *vector_of(const char *name, const MaybeTensor &x, int64_t n, const at::Tensor &like, at::ScalarType type) {
  if (!x.has_value()) return nullptr;
  if (!(x->scalar_type() == type && x->device() == like.device() && x->numel() == n && x->is_contiguous()))
    refuse(std::string(name) + " must be " + std::to_string(n) + " contiguous " +
           (type == at::kInt ? "int32" : type == at::kDouble ? "float64" : "float32") + " values on the device of the others");
  as_stored(name, *x);
  return static_cast<T *>(x->data_ptr());
}
float *floats(const char *name, const MaybeTensor &x, int64_t n, const at::Tensor &like) {
  return vector_of<float>(name, x, n, like, at::kFloat);
}

// The leading dimensions as evenly spaced rows.
struct Rows {
  int64_t rows = 1, width, stride;
  Rows(const char *name, const at::Tensor &x) : width(x.size(-1)), stride(x.size(-1)) {
    bool seen = false;
    for (int64_t d = x.dim() - 2; d >= 0; d--) {
      const int64_t n = x.size(d);
      if (n != 1) {
        if (!seen) stride = x.stride(d);
        need(rows == 0 || !seen || x.stride(d) == stride * rows, name, "must have evenly spaced rows (reshape it to two dimensions)");
        seen = true;
      }
      rows *= n;
    }
  }
};

// Bytes from the first element of x to the end of its last.
int64_t span_of(const at::Tensor &x) {
  int64_t n = 1;
  for (int64_t d = 0; d < x.dim(); d++) n += (x.size(d) - 1) * x.stride(d);
  return n * (int64_t)x.element_size();
}

// An output that the caller gives: no element may lie under another, which is
// sure where every dimension steps over all those with smaller strides.
void writable(const char *name, const at::Tensor &x, const at::Tensor &like) {
  storage_like(name, x, like);
  need(x.sizes() == like.sizes(), name, "must have the shape of its input");
  if (x.numel() == 0) return;
  for (int64_t d = 0; d < x.dim(); d++) {
    if (x.size(d) <= 1) continue;
    int64_t below = 1;
    for (int64_t e = 0; e < x.dim(); e++)
      if (x.size(e) > 1 && e != d && (x.stride(e) < x.stride(d) || (x.stride(e) == x.stride(d) && e < d)))
        below += (x.size(e) - 1) * x.stride(e);
    need(x.stride(d) >= below, name, "must not be broadcast or lie under itself");
  }
}

// Whether x repeats with a pitch of `pitch` bytes: every stride is a multiple
// of it, or belongs to the `width` bytes that x takes of each.
bool repeats(const at::Tensor &x, int64_t pitch, int64_t &width) {
  width = (int64_t)x.element_size();
  for (int64_t d = 0; d < x.dim(); d++) {
    if (x.size(d) <= 1) continue;
    const int64_t step = x.stride(d) * (int64_t)x.element_size();
    if (step < pitch) width += (x.size(d) - 1) * step;
    else if (step % pitch) return false;
  }
  return width <= pitch;
}

// Whether no byte belongs to both: their ranges of addresses are apart, or they
// take different parts of one pitch (the heads of a packed projection, columns
// of the same rows).
bool separate(const at::Tensor &x, const at::Tensor &y) {
  if (x.numel() == 0 || y.numel() == 0) return true;
  const uintptr_t a = reinterpret_cast<uintptr_t>(x.const_data_ptr()), b = reinterpret_cast<uintptr_t>(y.const_data_ptr());
  if (a + span_of(x) <= b || b + span_of(y) <= a) return true;
  for (const at::Tensor *t : {&x, &y})
    for (int64_t d = 0; d < t->dim(); d++) {
      const int64_t pitch = t->stride(d) * (int64_t)t->element_size();
      int64_t wx, wy;
      if (t->size(d) <= 1 || pitch <= 0 || !repeats(x, pitch, wx) || !repeats(y, pitch, wy)) continue;
      const int64_t at = (int64_t)((b % pitch + pitch - a % pitch) % pitch);  // y's part, from the start of x's
      if (at >= wx && at + wy <= pitch) return true;
    }
  return false;
}

// An output may be the input whose place it takes, element for element, but
// must not share memory with it, or with another input, in any other way.
void apart(const char *name, const at::Tensor &out, const at::Tensor &in, bool in_place) {
  if (in_place && out.const_data_ptr() == in.const_data_ptr() && out.sizes() == in.sizes()) {
    bool same = true;
    for (int64_t d = 0; d < out.dim(); d++) same = same && (out.size(d) <= 1 || out.stride(d) == in.stride(d));
    if (same) return;
  }
  need(separate(out, in), name, "must not overlap an input");
}

// x was written in place: autograd finds it changed if it had saved it.
void written(const at::Tensor &x) {
  if (!x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
}
void written(const MaybeTensor &x) {
  if (x.has_value()) written(*x);
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> layer_norm(const at::Tensor &x, const MaybeTensor &weight,
                                                          const MaybeTensor &bias, double eps, const MaybeTensor &out) {
  no_gradients(x, weight, bias, out);
  const int precision = storage("x", x);
  const Rows r("x", x);
  need(r.width > 0, "x must not have a width of zero");
  need(r.width < (1 << 28), "x must be narrower than 2^28");
  const float *w = floats("weight", weight, r.width, x), *b = floats("bias", bias, r.width, x);
  On on(x);
  at::Tensor y;
  int64_t y_stride = r.width;
  if (out.has_value()) {
    y = *out;
    writable("out", y, x);
    apart("out", y, x, true);
    if (weight.has_value()) apart("out", y, *weight, false);
    if (bias.has_value()) apart("out", y, *bias, false);
    y_stride = Rows("out", y).stride;
  } else {
    y = at::empty(x.sizes(), x.options());
  }
  const auto f32 = x.options().dtype(at::kFloat);
  at::Tensor mean = at::empty({r.rows}, f32), rstd = at::empty({r.rows}, f32);
  check(illumina_op_layer_norm(precision, x.data_ptr(), r.stride, r.rows, (int)r.width, w, b, (float)eps, y.data_ptr(),
                               y_stride, mean.data_ptr<float>(), rstd.data_ptr<float>(), on.stream));
  written(out);
  return {std::move(y), std::move(mean), std::move(rstd)};
}

std::tuple<at::Tensor, MaybeTensor, MaybeTensor> layer_norm_backward(const at::Tensor &dy, const at::Tensor &x,
                                                                     const MaybeTensor &mean, const MaybeTensor &rstd,
                                                                     const MaybeTensor &weight, bool need_weight) {
  no_gradients(dy, x, mean, rstd, weight);
  const int precision = storage("x", x);
  storage_like("dy", dy, x);
  need(dy.sizes() == x.sizes(), "dy must have the shape of x");
  const Rows r("x", x), g("dy", dy);
  need(r.width > 0, "x must not have a width of zero");
  need(r.width < (1 << 28), "x must be narrower than 2^28");
  const float *w = floats("weight", weight, r.width, x);
  need(mean.has_value() && rstd.has_value(), "mean and rstd of the forward pass are needed");
  const float *m = floats("mean", mean, r.rows, x), *s = floats("rstd", rstd, r.rows, x);
  On on(x);
  at::Tensor dx = at::empty(x.sizes(), x.options());
  MaybeTensor dw, db;
  at::Tensor workspace;
  size_t size = 0;
  if (need_weight) {
    check(illumina_op_layer_norm_workspace(r.rows, (int)r.width, &size));
    const auto f32 = x.options().dtype(at::kFloat);
    dw = at::empty({r.width}, f32), db = at::empty({r.width}, f32);
    workspace = at::empty({(int64_t)size}, x.options().dtype(at::kByte));
  }
  check(illumina_op_layer_norm_backward(precision, dy.data_ptr(), g.stride, x.data_ptr(), r.stride, r.rows, (int)r.width,
                                        w, m, s, dx.data_ptr(), r.width, need_weight ? dw->data_ptr<float>() : nullptr,
                                        need_weight ? db->data_ptr<float>() : nullptr,
                                        need_weight ? workspace.data_ptr() : nullptr, size, on.stream));
  return {std::move(dx), std::move(dw), std::move(db)};
}

std::tuple<at::Tensor, MaybeTensor> rotary(const at::Tensor &q, const MaybeTensor &k, const at::Tensor &positions,
                                           const at::Tensor &turns, const at::Tensor &axis, int64_t axes, int64_t head_dim,
                                           bool interleaved, bool inverse, const MaybeTensor &out_q,
                                           const MaybeTensor &out_k) {
  no_gradients(q, k, positions, turns, out_q, out_k);
  illumina_rotary_args a{};
  a.precision = storage("q", q, 4);
  const int64_t b = q.size(0), t = q.size(1), d = q.size(3);
  if (d != head_dim) refuse("q must have the plan's " + std::to_string(head_dim) + " elements a head");
  const int64_t pairs = turns.numel();
  need(pairs <= d / 2, "the plan must have at most headDim / 2 pairs");
  a.turns = vector_of<double>("the plan's turns", turns, pairs, q, at::kDouble);
  a.axis = vector_of<int>("the plan's axis", axis, pairs, q, at::kInt);
  const bool fractional = positions.scalar_type() == at::kFloat;
  need(positions.device() == q.device() && (fractional || positions.scalar_type() == at::kInt),
       "positions must be int32 or float32 on the device of q");
  as_stored("positions", positions);
  const int64_t pd = positions.dim();
  need((pd == 2 || pd == 3) && positions.size(0) == axes && positions.size(-1) == t && (pd == 2 || positions.size(1) == b),
       "positions must be [axes, tokens] or [axes, batch, tokens]");
  if (k.has_value()) {
    storage_like("k", *k, q, 4);
    need(k->size(0) == b && k->size(1) == t && k->size(3) == d, "k must have the batch, tokens and head size of q");
  }
  On on(q);
  a.batch = b, a.tokens = t, a.head_dim = (int)d, a.pairs = (int)pairs, a.axes = (int)axes;
  a.interleaved = interleaved, a.inverse = inverse;
  auto fill = [&](illumina_rotary_tensor &slot, const at::Tensor &x, const MaybeTensor &out, const char *name) {
    at::Tensor y;
    if (out.has_value()) {
      y = *out;
      writable(name, y, x);
      apart(name, y, x, true);
      for (const at::Tensor *t : {&positions, &turns, &axis}) apart(name, y, *t, false);
    } else {
      y = at::empty(x.sizes(), x.options());
    }
    slot.x = x.data_ptr(), slot.y = y.data_ptr(), slot.heads = (int)x.size(2);
    for (int i = 0; i < 3; i++) slot.x_stride[i] = x.stride(i), slot.y_stride[i] = y.stride(i);
    return y;
  };
  at::Tensor yq = fill(a.first, q, out_q, "outQ");
  MaybeTensor yk;
  if (k.has_value()) {
    yk = fill(a.second, *k, out_k, "outK");
    if (out_q.has_value()) apart("outQ", yq, *k, false);
    if (out_k.has_value()) apart("outK", *yk, q, false);
    if (out_q.has_value() && out_k.has_value()) apart("outQ", yq, *yk, false);
  }
  a.positions = positions.data_ptr(), a.positions_float = fractional;
  a.position_stride[0] = positions.stride(0), a.position_stride[1] = pd == 3 ? positions.stride(1) : 0;
  a.position_stride[2] = positions.stride(-1);
  check(illumina_op_rotary(&a, on.stream));
  written(out_q), written(out_k);
  return {std::move(yq), std::move(yk)};
}

void set(illumina_attention_tensor &slot, const at::Tensor &x) {
  slot.data = x.data_ptr();
  for (int i = 0; i < 3; i++) slot.stride[i] = x.stride(i);
}

illumina_attention_args attention_args(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v,
                                       std::optional<double> scale, int64_t causal_block, const MaybeTensor &q_lens,
                                       const MaybeTensor &k_lens) {
  illumina_attention_args a{};
  a.precision = storage("q", q, 4);
  storage_like("k", k, q, 4);
  storage_like("v", v, q, 4);
  const int64_t b = q.size(0), tq = q.size(1), h = q.size(2), d = q.size(3), tk = k.size(1), hk = k.size(2);
  need(k.sizes() == v.sizes() && k.size(0) == b && k.size(3) == d, "k and v must have q's batch and head size, and one shape");
  need(hk > 0 && h % hk == 0, "q's heads must be a multiple of the key heads");
  need(d >= 1 && d <= 128, "head sizes from 1 to 128 are supported");
  constexpr int64_t most = 1 << 28;
  need(b <= most && h <= most && tq <= most && tk <= most, "attention: size beyond 2^28");
  need(causal_block >= 0 && causal_block < (1ll << 31), "causalBlock must be a token count, 0 for none");
  a.batch = (int)b, a.heads = (int)h, a.kv_heads = (int)hk, a.head_dim = (int)d;
  a.q_tokens = (int)tq, a.k_tokens = (int)tk, a.causal_block = (int)causal_block;
  a.scale = scale.has_value() ? (float)*scale : (float)(1.0 / std::sqrt((double)d));
  a.q_lens = vector_of<int>("qLens", q_lens, b, q, at::kInt), a.k_lens = vector_of<int>("kLens", k_lens, b, q, at::kInt);
  set(a.q, q), set(a.k, k), set(a.v, v);
  return a;
}

at::Tensor attention_workspace(illumina_attention_args &a, int backward, const at::Tensor &like) {
  size_t size = 0;
  check(illumina_op_attention_workspace(&a, backward, &size));
  if (!size) return {};
  at::Tensor w = at::empty({(int64_t)size}, like.options().dtype(at::kByte));
  a.workspace = w.data_ptr(), a.workspace_bytes = size;
  return w;
}

std::tuple<at::Tensor, at::Tensor> attention(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v,
                                             std::optional<double> scale, int64_t causal_block, const MaybeTensor &q_lens,
                                             const MaybeTensor &k_lens) {
  no_gradients(q, k, v);
  illumina_attention_args a = attention_args(q, k, v, scale, causal_block, q_lens, k_lens);
  On on(q);
  at::Tensor out = at::empty(q.sizes(), q.options());
  at::Tensor lse = at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat));
  set(a.out, out);
  a.lse = lse.data_ptr<float>();
  const at::Tensor workspace = attention_workspace(a, 0, q);
  check(illumina_op_attention(&a, on.stream));
  return {std::move(out), std::move(lse)};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> attention_backward(const at::Tensor &dout, const at::Tensor &q,
                                                                  const at::Tensor &k, const at::Tensor &v,
                                                                  const at::Tensor &out, const MaybeTensor &lse,
                                                                  std::optional<double> scale, int64_t causal_block,
                                                                  const MaybeTensor &q_lens, const MaybeTensor &k_lens) {
  no_gradients(dout, q, k, v, out, lse);
  illumina_attention_args a = attention_args(q, k, v, scale, causal_block, q_lens, k_lens);
  storage_like("dOut", dout, q, 4);
  storage_like("out", out, q, 4);
  need(dout.sizes() == q.sizes() && out.sizes() == q.sizes(), "dOut and out must have the shape of q");
  need(lse.has_value(), "lse of the forward pass is needed");
  a.lse = floats("lse", lse, q.size(0) * q.size(1) * q.size(2), q);
  On on(q);
  at::Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()),
             dv = at::empty(v.sizes(), v.options());
  set(a.dout, dout), set(a.out, out), set(a.dq, dq), set(a.dk, dk), set(a.dv, dv);
  const at::Tensor workspace = attention_workspace(a, 1, q);
  check(illumina_op_attention_backward(&a, on.stream));
  return {std::move(dq), std::move(dk), std::move(dv)};
}

// What a step of an optimiser checks its gradients against, and the tensors
// whose places the optimiser was created with.
struct Stepper {
  illumina_adamw *handle;
  std::vector<at::Tensor> params, moments;
  std::vector<int64_t> counts;
  std::vector<const void *> pointers, places;
  c10::Device device;
  bool bf16;
  Stepper(uintptr_t h, std::vector<at::Tensor> p, std::vector<at::Tensor> m, int64_t index, bool b)
      : handle((illumina_adamw *)h), params(std::move(p)), moments(std::move(m)),
        device(c10::kCUDA, (c10::DeviceIndex)index), bf16(b) {
    for (const at::Tensor &x : params) counts.push_back(x.numel()), places.push_back(x.data_ptr());
    for (const at::Tensor &x : moments) places.push_back(x.data_ptr());
    pointers.resize(counts.size());
  }

  // A tensor that was given other memory (p.data = ..., a module moved to another type or device) no longer lies
  // where the optimiser writes.
  void stay() const {
    for (size_t i = 0; i < params.size(); i++)
      if (params[i].const_data_ptr() != places[i] || params[i].numel() != counts[i])
        refuse("adamw: parameter " + std::to_string(i) + " has moved since the optimizer was created");
    for (size_t i = 0; i < moments.size(); i++)
      need(moments[i].const_data_ptr() == places[params.size() + i], "adamw: the moments have moved since the optimizer was created");
  }

  void step(const py::sequence &grads, const py::object &lr, double beta1, double beta2, double eps, double decay) {
    illumina_adamw_hyper h{};
    if (THPVariable_Check(lr.ptr())) {
      const at::Tensor &t = THPVariable_Unpack(lr.ptr());
      need(t.scalar_type() == at::kFloat && t.device() == device && t.numel() == 1,
           "lr must be a number or one float32 value on the device of the others");
      as_stored("adamw: lr", t);
      h.lr_device = t.data_ptr<float>();
    } else {
      h.lr = lr.cast<double>();
    }
    need(py::len(grads) == counts.size(), "adamw: one gradient for each parameter is needed");
    const auto type = bf16 ? at::kBFloat16 : at::kFloat;
    // a list or tuple holds its items; one that may make them as they are asked for is kept as a list until the launch
    py::object held = grads;
    if (!PyList_CheckExact(grads.ptr()) && !PyTuple_CheckExact(grads.ptr())) {
      py::list made;
      for (size_t i = 0; i < counts.size(); i++) made.append(grads[i]);
      held = std::move(made);
    }
    stay();  // after the last call into the interpreter
    PyObject *const *items = PySequence_Fast_ITEMS(held.ptr());
    for (size_t i = 0; i < counts.size(); i++) {
      const at::Tensor *g = THPVariable_Check(items[i]) ? &THPVariable_Unpack(items[i]) : nullptr;
      if (!g || g->scalar_type() != type || g->device() != device || g->numel() != counts[i] || !g->is_contiguous())
        refuse("adamw: gradient " + std::to_string(i) + " must be " + std::to_string(counts[i]) + " contiguous " +
               (bf16 ? "bfloat16" : "float32") + " values on " + device.str());
      as_stored("adamw: a gradient", *g);
      pointers[i] = g->const_data_ptr();
    }
    h.beta1 = beta1, h.beta2 = beta2, h.eps = eps, h.weight_decay = decay;
    check(illumina_adamw_step(handle, pointers.data(), &h, c10::cuda::getCurrentCUDAStream(device.index()).stream()));
    for (const at::Tensor &x : params) written(x);
  }
};

}  // namespace

PYBIND11_MODULE(_torch_ops, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const Refused &e) {
      const py::object cls = py::module_::import("illumina._lib").attr("IlluminaError");
      PyErr_SetObject(cls.ptr(), cls(e.status, e.message).ptr());
    }
  });
  m.def("layer_norm", &layer_norm);
  m.def("layer_norm_backward", &layer_norm_backward);
  m.def("rotary", &rotary);
  m.def("attention", &attention);
  m.def("attention_backward", &attention_backward);
  py::class_<Stepper>(m, "Stepper")
      .def(py::init<uintptr_t, std::vector<at::Tensor>, std::vector<at::Tensor>, int64_t, bool>())
      .def("stay", &Stepper::stay)
      .def("step", &Stepper::step);
}
