// The decoder operators on torch tensors without Python's per-attribute costs (about 0.1 us each, and
// some sixty of them in a call): a call whose tensors are as the kernels take them is checked, given its
// output and workspace, and launched here.  Every function returns None where it does not take the call
// as it is -- other layouts, empty tensors, what needs a gradient, and everything that is refused: the
// Python functions then do what is left, and raise the errors.  The package runs without this module: they then do all, and
// refuse captured rotations of leaves, whose living graphs only the module sees.
#define PY_SSIZE_T_CLEAN
#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <utility>

#include "../../include/biops.h"

namespace {

int type_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return BIOPS_F32;
    case at::kHalf: return BIOPS_F16;
    case at::kBFloat16: return BIOPS_BF16;
    default: return -1;
  }
}
bool is_index(const at::Tensor& t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong; }
int is_long(const at::Tensor& t) { return t.scalar_type() == at::kLong ? 1 : 0; }
bool unit_last(const at::Tensor& t) { return t.stride(-1) == 1; }

bool needs_grad(const at::Tensor& t) { return c10::GradMode::is_enabled() && t.requires_grad(); }
// A plain tensor with elements on the current device that needs no gradient here (`grad`: or does) and has no tangent.
const at::Tensor* take(PyObject* o, c10::DeviceIndex device, bool grad = false) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.layout() != at::kStrided || t.get_device() != device || t.numel() == 0 || t.is_neg() ||
      t._fw_grad(0).defined())
    return nullptr;
  return !grad && needs_grad(t) ? nullptr : &t;
}
bool number(PyObject* o, int64_t* v) {
  if (!PyLong_CheckExact(o)) return false;
  int over = 0;
  *v = PyLong_AsLongLongAndOverflow(o, &over);
  return over == 0;
}
// A float, or None for 1 / sqrt(d).
bool scale_of(PyObject* o, int64_t d, float* v) {
  if (o == Py_None) {
    *v = (float)(1.0 / std::sqrt((double)d));
    return true;
  }
  if (!PyFloat_CheckExact(o)) return false;
  *v = (float)PyFloat_AS_DOUBLE(o);
  return std::isfinite(*v);
}
void* stream_on(c10::DeviceIndex device) { return (void*)c10::hip::getCurrentHIPStream(device).stream(); }
char* ptr(const at::Tensor& t) { return static_cast<char*>(t.data_ptr()); }

#define TAKE(name, object)                              \
  const at::Tensor* name##_ = take(object, device);     \
  if (!name##_) Py_RETURN_NONE;                         \
  const at::Tensor& name = *name##_

// The GIL is released around the library's calls (a gradient's runs without it from the start).
struct WithoutGil {
  PyThreadState* held = PyGILState_Check() ? PyEval_SaveThread() : nullptr;
  ~WithoutGil() {
    if (held) PyEval_RestoreThread(held);
  }
};
#define LAUNCH(rc, call) \
  int rc;                \
  {                      \
    WithoutGil without;  \
    rc = (call);         \
  }

struct Rotation {
  const double* turns;
  const uint8_t* axis;
  int64_t pairs;
  int neighbours;
};

// Rotated copies of [tokens, heads, dim] or [batch, tokens, heads, dim] tensors (either may be undefined); any strides, and
// lazily negated (a gradient comes as the engine has it).
std::pair<at::Tensor, at::Tensor> rotated(const at::Tensor& query, const at::Tensor& key, const at::Tensor& p, const Rotation& r, bool inverse) {
  auto unit = [](const at::Tensor& x) {
    const at::Tensor t = x.defined() ? x.resolve_neg() : x;
    return !t.defined() || unit_last(t) ? t : t.contiguous();
  };
  auto like = [](const at::Tensor& t) {
    if (!t.defined()) return t;
    at::Tensor y = at::empty_like(t);
    return unit_last(y) ? y : at::empty(t.sizes(), t.options());
  };
  const at::Tensor q = unit(query), k = unit(key);
  at::Tensor oq = like(q), ok = like(k);
  const at::Tensor& some = q.defined() ? q : k;
  const bool four = some.dim() == 4;
  auto at_ = [](const at::Tensor& t) { return t.defined() ? ptr(t) : nullptr; };
  auto st = [](const at::Tensor& t, int i) { return t.defined() ? t.stride(i) : (int64_t)0; };
  auto sb = [four, st](const at::Tensor& t) { return four ? st(t, 0) : (int64_t)0; };
  const int pos = p.scalar_type() == at::kLong ? 0 : p.scalar_type() == at::kInt ? 1 : 2;
  LAUNCH(rc, biops_rotary(type_code(some.scalar_type()), four ? some.size(0) : 1, some.size(-3), q.defined() ? q.size(-2) : 0,
                          k.defined() ? k.size(-2) : 0, some.size(-1), at_(q), sb(q), st(q, -3), st(q, -2), at_(oq), sb(oq),
                          st(oq, -3), st(oq, -2), at_(k), sb(k), st(k, -3), st(k, -2), at_(ok), sb(ok), st(ok, -3),
                          st(ok, -2), ptr(p), pos, p.stride(0), four ? p.stride(1) : 0, p.stride(-1), r.pairs, r.turns,
                          r.axis, r.neighbours, inverse ? 1 : 0, stream_on(some.get_device())))
  TORCH_CHECK(rc == BIOPS_OK, "biops_rotary failed (", rc, "): ", biops_last_error());
  return {oq, ok};
}

// The rotation with its gradient, the inverse rotation (and so on).  The frequencies are copied: the graph may
// outlive the table that they came from.  A call without keys has no `key` (not an undefined one).
struct RotaryFunction : torch::autograd::Function<RotaryFunction> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q,
                                                const std::optional<at::Tensor>& key, const at::Tensor& p,
                                                const at::Tensor& turns, const at::Tensor& axis, bool neighbours,
                                                bool inverse) {
    const at::Tensor k = key.value_or(at::Tensor());
    ctx->save_for_backward({p});
    ctx->saved_data["turns"] = turns;
    ctx->saved_data["axis"] = axis;
    ctx->saved_data["neighbours"] = neighbours;
    ctx->saved_data["inverse"] = inverse;
    ctx->saved_data["both"] = k.defined();
    ctx->set_materialize_grads(false);
    const Rotation r{turns.const_data_ptr<double>(), axis.const_data_ptr<uint8_t>(), turns.numel(), neighbours ? 1 : 0};
    auto y = rotated(q, k, p, r, inverse);
    torch::autograd::variable_list out{y.first};
    if (k.defined()) out.push_back(y.second);
    // what comes of a tensor without a gradient has none
    if (!q.requires_grad()) ctx->mark_non_differentiable({y.first});
    else if (k.defined() && !k.requires_grad()) ctx->mark_non_differentiable({y.second});
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
    const at::Tensor p = ctx->get_saved_variables()[0], turns = ctx->saved_data["turns"].toTensor(),
                     axis = ctx->saved_data["axis"].toTensor();
    const bool neighbours = ctx->saved_data["neighbours"].toBool(), inverse = ctx->saved_data["inverse"].toBool();
    torch::autograd::variable_list out(7);  // one for each argument of forward
    const at::Tensor first = ctx->needs_input_grad(0) ? g[0] : at::Tensor();
    const at::Tensor second = ctx->saved_data["both"].toBool() && ctx->needs_input_grad(1) ? g[1] : at::Tensor();
    if (!first.defined() && !second.defined()) return out;
    if (c10::GradMode::is_enabled()) {  // create_graph
      const bool alone = !first.defined();  // (the first tensor of a call is a defined one)
      const std::optional<at::Tensor> other = alone || !second.defined() ? std::nullopt : std::optional<at::Tensor>(second);
      auto y = RotaryFunction::apply(alone ? second : first, other, p, turns, axis, neighbours, !inverse);
      out[alone ? 1 : 0] = y[0];
      if (y.size() > 1) out[1] = y[1];
    } else {
      const Rotation r{turns.const_data_ptr<double>(), axis.const_data_ptr<uint8_t>(), turns.numel(), neighbours ? 1 : 0};
      auto y = rotated(first, second, p, r, !inverse);
      out[0] = y.first;
      out[1] = y.second;
    }
    return out;
  }
};

// Whether a gradient that is captured into a graph here would run into one outside of it: an older graph of the leaf that
// is still held keeps the leaf's accumulation node on another stream, and the engine would make that stream wait
// for the capturing one in the middle of a backward pass, where no error leads back to the caller.
bool held_elsewhere(const at::Tensor& t, c10::DeviceIndex device) {
  if (!t.requires_grad() || !t.is_leaf()) return false;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
  if (!node) return false;
  const auto stream = node->stream();
  return stream && *stream != c10::hip::getCurrentHIPStream(device).unwrap();
}
bool capturing(c10::DeviceIndex device) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  return hipStreamIsCapturing((hipStream_t)stream_on(device), &status) == hipSuccess && status != hipStreamCaptureStatusNone;
}

// held(tensors...) -> whether one of them is such a leaf, for the rotations that the Python function launches
PyObject* held(PyObject*, PyObject* const* args, Py_ssize_t n) {
  for (Py_ssize_t i = 0; i < n; ++i)
    if (THPVariable_Check(args[i]) && held_elsewhere(THPVariable_Unpack(args[i]), c10::hip::current_device())) Py_RETURN_TRUE;
  Py_RETURN_FALSE;
}

// rotary(query, key or None, positions, axes, pairs, turns, axis, neighbours) -> query or (query, key)
PyObject* rotary(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 8) Py_RETURN_NONE;
  const auto device = c10::hip::current_device();
  const bool both = args[1] != Py_None;
  const at::Tensor* q_ = take(args[0], device, true);
  const at::Tensor* k_ = both ? take(args[1], device, true) : nullptr;
  if (!q_ || (both && !k_)) Py_RETURN_NONE;
  TAKE(p, args[2]);
  const at::Tensor& q = *q_;
  const at::Tensor k = both ? *k_ : at::Tensor();
  if (c10::GradMode::is_enabled() && capturing(device) && (held_elsewhere(q, device) || (both && held_elsewhere(k, device)))) {
    PyErr_SetString(PyExc_RuntimeError, "multi_axis_rotary: a graph of this leaf from outside of the capture is still alive; "
                                        "delete its outputs (or capture on the stream that they were made on)");
    return nullptr;
  }
  int64_t axes, pairs, turns, axis, neighbours;
  if (!number(args[3], &axes) || !number(args[4], &pairs) || !number(args[5], &turns) || !number(args[6], &axis) ||
      !number(args[7], &neighbours))
    Py_RETURN_NONE;
  const int64_t nd = q.dim();
  if ((nd != 3 && nd != 4) || type_code(q.scalar_type()) < 0 || 2 * pairs > q.size(-1)) Py_RETURN_NONE;
  const int lead = (int)nd - 2;
  const bool known = p.scalar_type() == at::kLong || p.scalar_type() == at::kInt || p.scalar_type() == at::kFloat;
  if (!known || p.dim() != lead + 1 || p.size(0) != axes) Py_RETURN_NONE;
  for (int i = 0; i < lead; ++i)
    if (p.size(i + 1) != q.size(i)) Py_RETURN_NONE;
  if (both) {
    if (k.dim() != nd || k.scalar_type() != q.scalar_type() || k.size(-1) != q.size(-1)) Py_RETURN_NONE;
    for (int i = 0; i < lead; ++i)
      if (k.size(i) != q.size(i)) Py_RETURN_NONE;
  }
  const Rotation r{reinterpret_cast<const double*>(turns), reinterpret_cast<const uint8_t*>(axis), pairs, (int)neighbours};
  std::pair<at::Tensor, at::Tensor> out;
  if (needs_grad(q) || (both && needs_grad(k))) {
    at::Tensor t = at::empty({pairs}, at::kDouble), a = at::empty({pairs}, at::kByte);
    std::copy_n(r.turns, pairs, t.data_ptr<double>());
    std::copy_n(r.axis, pairs, a.data_ptr<uint8_t>());
    const std::optional<at::Tensor> key = both ? std::optional<at::Tensor>(k) : std::nullopt;
    auto y = RotaryFunction::apply(q, key, p, t, a, neighbours != 0, false);
    out.first = y[0];
    if (both) out.second = y[1];
  } else {
    out = rotated(q, k, p, r, false);
  }
  if (!both) return THPVariable_Wrap(std::move(out.first));
  PyObject* pair = PyTuple_New(2);
  if (!pair) return nullptr;
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(out.first)));
  PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(out.second)));
  return pair;
}

bool caches(const at::Tensor& kc, const at::Tensor& vc) {
  if (kc.dim() != 4 || vc.dim() != 4 || kc.scalar_type() != vc.scalar_type() || !unit_last(kc) || !unit_last(vc)) return false;
  for (int i = 0; i < 3; ++i)
    if (kc.size(i) != vc.size(i)) return false;
  return true;
}

// paged_write(key, value, key_cache, value_cache, slots, flag) -> True
PyObject* paged_write(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 6) Py_RETURN_NONE;
  const auto device = c10::hip::current_device();
  TAKE(k, args[0]);
  TAKE(v, args[1]);
  TAKE(kc, args[2]);
  TAKE(vc, args[3]);
  TAKE(slots, args[4]);
  int64_t flag;
  const int code = type_code(k.scalar_type());
  if (!number(args[5], &flag) || code < 0 || !caches(kc, vc) || k.scalar_type() != kc.scalar_type() ||
      v.scalar_type() != kc.scalar_type())
    Py_RETURN_NONE;
  // (caches that overlap themselves or one another are refused in Python)
  if (!kc.is_non_overlapping_and_dense() || !vc.is_non_overlapping_and_dense()) Py_RETURN_NONE;
  const int64_t gap = vc.storage_offset() - kc.storage_offset();
  if (kc.is_alias_of(vc) && gap < kc.numel() && -gap < vc.numel()) Py_RETURN_NONE;
  if (k.dim() != 3 || v.dim() != 3 || !unit_last(k) || !unit_last(v) || k.size(0) != v.size(0) || k.size(1) != kc.size(2) ||
      v.size(1) != kc.size(2) || k.size(2) != kc.size(3) || v.size(2) != vc.size(3))
    Py_RETURN_NONE;
  if (slots.dim() != 1 || !is_index(slots) || slots.size(0) != k.size(0)) Py_RETURN_NONE;
  LAUNCH(rc, biops_paged_write(code, k.size(0), k.size(1), k.size(2), v.size(2), ptr(k), k.stride(0), k.stride(1), ptr(v),
                               v.stride(0), v.stride(1), ptr(kc), kc.stride(0), kc.stride(1), kc.stride(2), ptr(vc),
                               vc.stride(0), vc.stride(1), vc.stride(2), kc.size(0), kc.size(1), ptr(slots),
                               is_long(slots), slots.stride(0), reinterpret_cast<int*>(flag), stream_on(device)))
  if (rc != BIOPS_OK) Py_RETURN_NONE;
  for (const at::Tensor* c : {&kc, &vc})  // autograd has to know of the change, as of any other in place
    if (!c->is_inference()) c->unsafeGetTensorImpl()->bump_version();
  Py_RETURN_TRUE;
}

// paged_attention(query, key_cache, value_cache, table, lengths, scale or None, window or 0, sinks, max_length or -1,
//                 flag) -> output
PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 10) Py_RETURN_NONE;
  const auto device = c10::hip::current_device();
  TAKE(q, args[0]);
  TAKE(kc, args[1]);
  TAKE(vc, args[2]);
  TAKE(table, args[3]);
  TAKE(lengths, args[4]);
  int64_t window, sinks, bound, flag;
  float scale;
  const int code = type_code(q.scalar_type());
  if (code < 0 || q.dim() != 3 || !unit_last(q) || !caches(kc, vc) || q.scalar_type() != kc.scalar_type()) Py_RETURN_NONE;
  const int64_t batch = q.size(0), hq = q.size(1), hkv = kc.size(2), d = q.size(2), dv = vc.size(3);
  if (!scale_of(args[5], d, &scale) || !number(args[6], &window) || !number(args[7], &sinks) || !number(args[8], &bound) ||
      !number(args[9], &flag) || window < 0 || sinks < 0)
    Py_RETURN_NONE;
  if (d != kc.size(3) || hq % hkv != 0 || table.dim() != 2 || table.size(0) != batch || !is_index(table) ||
      lengths.dim() != 1 || lengths.size(0) != batch || !is_index(lengths))
    Py_RETURN_NONE;
  const int64_t page = kc.size(1), width = table.size(1);
  const int64_t need = biops_paged_attention_workspace_size(batch, hq, dv, width, page, bound, window, sinks);
  if (need < 0) Py_RETURN_NONE;
  at::Tensor out = at::empty({batch, hq, dv}, q.options());
  at::Tensor ws;
  if (need > 0) ws = at::empty({need}, q.options().dtype(at::kByte));
  LAUNCH(rc, biops_paged_attention(code, batch, hq, hkv, d, dv, ptr(q), q.stride(0), q.stride(1), ptr(kc), kc.stride(0),
                                   kc.stride(1), kc.stride(2), ptr(vc), vc.stride(0), vc.stride(1), vc.stride(2),
                                   kc.size(0), page, ptr(table), is_long(table), table.stride(0), table.stride(1), width,
                                   ptr(lengths), is_long(lengths), lengths.stride(0), bound, window, sinks, scale, ptr(out),
                                   reinterpret_cast<int*>(flag), need > 0 ? ptr(ws) : nullptr, need, stream_on(device)))
  if (rc != BIOPS_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
}

// window_attention(query, key, value, window, sinks, scale or None, enable_gqa) -> output   [batch, heads, tokens, dim]
PyObject* window_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 7) Py_RETURN_NONE;
  const auto device = c10::hip::current_device();
  TAKE(q, args[0]);
  TAKE(k, args[1]);
  TAKE(v, args[2]);
  int64_t window, sinks;
  float scale;
  const int code = type_code(q.scalar_type());
  if (code < 0 || q.dim() != 4 || k.dim() != 4 || v.dim() != 4 || k.scalar_type() != q.scalar_type() ||
      v.scalar_type() != q.scalar_type() || !unit_last(q) || !unit_last(k) || !unit_last(v))
    Py_RETURN_NONE;
  const int64_t batch = q.size(0), hq = q.size(1), lq = q.size(2), d = q.size(3), hkv = k.size(1), lk = k.size(2);
  const int64_t dv = v.size(3);
  if (!number(args[3], &window) || !number(args[4], &sinks) || !scale_of(args[5], d, &scale) || window < 1 || sinks < 0)
    Py_RETURN_NONE;
  if (k.size(0) != batch || v.size(0) != batch || v.size(1) != hkv || v.size(2) != lk || k.size(3) != d || hq % hkv != 0 ||
      (hq != hkv && args[6] != Py_True))
    Py_RETURN_NONE;
  // tokens before heads in memory where the queries have them so
  at::Tensor out = q.stride(1) < q.stride(2) ? at::empty({batch, lq, hq, dv}, q.options()).transpose(1, 2)
                                             : at::empty({batch, hq, lq, dv}, q.options());
  const int64_t need = biops_window_attention_workspace_size(batch, hq, lq, lk, dv, window, sinks);
  if (need < 0) Py_RETURN_NONE;
  at::Tensor ws;
  if (need > 0) ws = at::empty({need}, q.options().dtype(at::kByte));
  LAUNCH(rc, biops_window_attention(code, batch, hq, hkv, lq, lk, d, dv, ptr(q), q.stride(0), q.stride(2), q.stride(1),
                                    ptr(k), k.stride(0), k.stride(2), k.stride(1), ptr(v), v.stride(0), v.stride(2),
                                    v.stride(1), ptr(out), out.stride(0), out.stride(2), out.stride(1), nullptr, 0, 0,
                                    nullptr, 0, 0, window, sinks, scale, nullptr, need > 0 ? ptr(ws) : nullptr, need,
                                    stream_on(device)))
  if (rc != BIOPS_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
}

// window_packed(query, key, value, cu_q, cu_kv, window, sinks, scale or None, flag) -> output   [1, tokens, heads, dim]
PyObject* window_packed(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 9) Py_RETURN_NONE;
  const auto device = c10::hip::current_device();
  TAKE(q, args[0]);
  TAKE(k, args[1]);
  TAKE(v, args[2]);
  TAKE(cu_q, args[3]);
  TAKE(cu_k, args[4]);
  int64_t window, sinks, flag;
  float scale;
  const int code = type_code(q.scalar_type());
  if (code < 0 || q.dim() != 4 || k.dim() != 4 || v.dim() != 4 || k.scalar_type() != q.scalar_type() ||
      v.scalar_type() != q.scalar_type() || !unit_last(q) || !unit_last(k) || !unit_last(v))
    Py_RETURN_NONE;
  const int64_t lq = q.size(1), hq = q.size(2), d = q.size(3), lk = k.size(1), hkv = k.size(2), dv = v.size(3);
  if (!number(args[5], &window) || !number(args[6], &sinks) || !scale_of(args[7], d, &scale) || !number(args[8], &flag) ||
      window < 1 || sinks < 0)
    Py_RETURN_NONE;
  if (q.size(0) != 1 || k.size(0) != 1 || v.size(0) != 1 || v.size(1) != lk || v.size(2) != hkv || k.size(3) != d ||
      hq % hkv != 0 || cu_q.dim() != 1 || cu_k.dim() != 1 || cu_q.size(0) != cu_k.size(0) || !is_index(cu_q) || !is_index(cu_k))
    Py_RETURN_NONE;
  at::Tensor out = at::empty({1, lq, hq, dv}, q.options());
  LAUNCH(rc, biops_window_attention(code, cu_q.size(0) - 1, hq, hkv, lq, lk, d, dv, ptr(q), 0, q.stride(1), q.stride(2),
                                    ptr(k), 0, k.stride(1), k.stride(2), ptr(v), 0, v.stride(1), v.stride(2), ptr(out), 0,
                                    out.stride(1), out.stride(2), ptr(cu_q), is_long(cu_q), cu_q.stride(0), ptr(cu_k),
                                    is_long(cu_k), cu_k.stride(0), window, sinks, scale, reinterpret_cast<int*>(flag),
                                    nullptr, 0, stream_on(device)))
  if (rc != BIOPS_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
}

// C++ exceptions (out of memory) end here: the Python function then meets the same condition and raises it.
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  try {
    if (at::tracer::impl::is_dispatch_enabled()) Py_RETURN_NONE;  // (refused in Python)
    return F(self, args, n);
  } catch (...) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<F>));
}

PyMethodDef methods[] = {
    {"held", fast<held>(), METH_FASTCALL, "whether a graph of a leaf is alive on another stream, or None"},
    {"rotary", fast<rotary>(), METH_FASTCALL, "biops_rotary on tensors, or None"},
    {"paged_write", fast<paged_write>(), METH_FASTCALL, "biops_paged_write on tensors, or None"},
    {"paged_attention", fast<paged_attention>(), METH_FASTCALL, "biops_paged_attention on tensors, or None"},
    {"window_attention", fast<window_attention>(), METH_FASTCALL, "biops_window_attention on dense tensors, or None"},
    {"window_packed", fast<window_packed>(), METH_FASTCALL, "biops_window_attention on packed tensors, or None"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_biops_tensor", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__biops_tensor(void) { return PyModule_Create(&module); }
