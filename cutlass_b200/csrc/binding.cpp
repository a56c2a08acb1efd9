// Python calls of the operators whose kernels take a few microseconds, without the interpreter's share of the work: a call
// through ctypes with its checks in Python takes 10 to 15 microseconds of host time, which such kernels do not hide.
//
// Every function here either makes the whole call (checks, outputs, launch on torch's current stream) and returns its
// results, or returns None without having done anything: for whatever is not the plain case -- wrong types and shapes, other
// devices than the current one, tensors that want a gradient -- the caller goes on in Python, which says what is wrong or does
// it step by step.  The library's C entry points are handed over by address (bind), so that there is one copy of the library.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/autograd/python_variable.h>

#include <exception>
#include <initializer_list>

#include "../../include/bsgemm.h"

namespace {

struct {
  decltype(&bsg_int8_linear_run) int8_linear_run;
  decltype(&bsg_int8_scratch_rows) int8_scratch_rows;
  decltype(&bsg_act_forward) act_forward;
  decltype(&bsg_act_backward) act_backward;
  decltype(&bsg_route_forward) route_forward;
  decltype(&bsg_route_backward) route_backward;
  decltype(&bsg_route_scratch_size) route_scratch_size;
  decltype(&bsg_last_error_string) last_error_string;
} g;
// Objects of the Python side: what is called with the status code of a call that failed; activation name -> code; device -> status
// words; the named tuples that the operators return.
struct {
  PyObject *raise, *activations, *workspaces, *checkpoint, *routing;
} g_py;

constexpr int64_t kMaxExperts = 1024, kMaxTopK = 32;

int kind_of(at::ScalarType t, bool with_f32) {
  if (t == at::kBFloat16) return BSG_OUT_BF16;
  if (t == at::kHalf) return BSG_OUT_F16;
  return with_f32 && t == at::kFloat ? BSG_OUT_F32 : -1;
}

// The tensor of an argument that is a plain torch.Tensor (or Parameter) on CUDA device `device`; null otherwise.
const at::Tensor* tensor(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.defined() && t.layout() == at::kStrided && t.is_cuda() && !t.is_neg() ? &t : nullptr;
}
const at::Tensor* array(PyObject* o, at::ScalarType type, at::IntArrayRef shape, int device) {
  const at::Tensor* t = tensor(o);
  return t && t->scalar_type() == type && t->get_device() == device && t->sizes() == shape && t->is_contiguous() ? t : nullptr;
}
struct Matrix {
  const at::Tensor* t;
  int kind, device;
  int64_t rows, cols, pitch;
};
bool matrix(PyObject* o, bool with_f32, Matrix* m) {
  m->t = tensor(o);
  if (!m->t || m->t->dim() != 2) return false;
  m->kind = kind_of(m->t->scalar_type(), with_f32);
  m->device = m->t->get_device();
  m->rows = m->t->size(0);
  m->cols = m->t->size(1);
  m->pitch = m->rows > 1 ? m->t->stride(0) : m->cols;
  return m->kind >= 0 && m->device == c10::cuda::current_device() && m->cols >= 1 && (m->cols == 1 || m->t->stride(1) == 1) && m->pitch >= m->cols;
}
bool has_tangent(const at::Tensor* t) { return t && c10::AutogradState::get_tls_state().get_fw_grad_mode() && t->_fw_grad(0).defined(); }
bool wants_gradient(const at::Tensor* t) { return t && ((t->requires_grad() && at::GradMode::is_enabled()) || has_tangent(t)); }

at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, const at::Tensor& like) { return at::Tensor(at::detail::empty_cuda(shape, type, like.device(), std::nullopt)); }

// Part of a buffer as a tensor of its own (contiguous, `offset` in elements of `type`); not a view for autograd.
at::Tensor part(const at::Tensor& buffer, at::ScalarType type, int64_t offset, at::IntArrayRef shape) {
  auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(buffer.storage()), buffer.key_set(), c10::scalarTypeToTypeMeta(type));
  impl->set_storage_offset(offset);
  impl->set_sizes_contiguous(shape);
  return at::Tensor(std::move(impl));
}

void* current_stream(int device) { return c10::cuda::getCurrentCUDAStream(device).stream(); }

PyObject* failed(int32_t code) { return PyObject_CallFunction(g_py.raise, "i", int(code)); }      // raises

// A tuple of the (named) tuple type `type`; takes the items over.
PyObject* tuple_of(PyObject* type, std::initializer_list<PyObject*> items) {
  PyTypeObject* t = reinterpret_cast<PyTypeObject*>(type);
  PyObject* made = t->tp_alloc(t, Py_ssize_t(items.size()));
  bool whole = made != nullptr;
  Py_ssize_t i = 0;
  for (PyObject* o : items) {
    whole = whole && o;
    if (made) PyTuple_SET_ITEM(made, i++, o); else Py_XDECREF(o);
  }
  if (!whole) Py_CLEAR(made);
  return made;
}
// Activation code of a name; -1 where there is none.
int32_t activation_of(PyObject* name) {
  PyObject* code = PyUnicode_Check(name) ? PyDict_GetItem(g_py.activations, name) : nullptr;
  return code ? int32_t(PyLong_AsLong(code)) : -1;
}

// The interpreter's lock is given up while memory is allocated and kernels are launched: both may wait, for the device or for a full
// queue, and other Python threads go on.  (The arguments are the caller's and stay alive.)
class Unlocked {
 public:
  Unlocked() : state_(PyEval_SaveThread()) {}
  ~Unlocked() { PyEval_RestoreThread(state_); }
  Unlocked(const Unlocked&) = delete;
  Unlocked& operator=(const Unlocked&) = delete;

 private:
  PyThreadState* state_;
};

template <class F>
PyObject* guarded(F body) {
  try {
    return body();
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(PyExc_MemoryError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// int8_linear(x, weight, weight_scale, bias, activation, offsets, rows, out_dtype) -> y
PyObject* int8_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Matrix x;
    if (n != 8 || !matrix(a[0], false, &x)) Py_RETURN_NONE;
    const int dev = x.device;
    const bool grouped = a[5] != Py_None;
    PyObject* device_key = PyLong_FromLong(dev);
    PyObject* words = device_key ? PyDict_GetItem(g_py.workspaces, device_key) : nullptr;      // borrowed
    Py_XDECREF(device_key);
    const at::Tensor *w = tensor(a[1]), *status = words ? tensor(words) : nullptr;
    if (!w || !status || w->scalar_type() != at::kChar || w->get_device() != dev || w->dim() != (grouped ? 3 : 2)) Py_RETURN_NONE;
    const int64_t K = x.cols, N = w->size(-2), groups = grouped ? w->size(0) : 1, whole = (K + 15) & ~int64_t(15);
    const int64_t pitch = K <= 128 ? whole : (K + 127) & ~int64_t(127);      // of the scratch
    const int64_t ldw = N > 1 ? w->stride(-2) : whole, group_stride = groups > 1 ? w->stride(0) : 0;
    if (w->size(-1) != K || N < 1 || groups < 1 || groups > BSG_MAX_GROUPS || (K > 1 && w->stride(-1) != 1) || ldw < K || ((ldw | group_stride) & 15) != 0 || (groups > 1 && group_stride < K) || K > 131071 ||
        (reinterpret_cast<uintptr_t>(w->const_data_ptr()) & 15) != 0)
      Py_RETURN_NONE;
    const auto per_channel = w->sizes().slice(0, grouped ? 2 : 1);
    const at::Tensor* ws = array(a[2], at::kFloat, per_channel, dev);
    const at::Tensor* bias = a[3] == Py_None ? nullptr : array(a[3], at::kFloat, per_channel, dev);
    const at::Tensor* offsets = grouped ? array(a[5], at::kInt, w->sizes().slice(0, 1), dev) : nullptr;
    const at::Tensor* rows = a[6] == Py_None ? nullptr : tensor(a[6]);
    if (!ws || (a[3] != Py_None && !bias) || (grouped && !offsets)) Py_RETURN_NONE;
    if (a[6] != Py_None && (!grouped || !rows || rows->scalar_type() != at::kInt || rows->dim() != 1 || rows->get_device() != dev || !rows->is_contiguous())) Py_RETURN_NONE;
    if (wants_gradient(x.t) || wants_gradient(ws) || wants_gradient(bias)) Py_RETURN_NONE;
    at::ScalarType out_type = x.t->scalar_type();
    if (a[7] != Py_None) {
      if (!THPDtype_Check(a[7])) Py_RETURN_NONE;
      out_type = reinterpret_cast<THPDtype*>(a[7])->scalar_type;
    }
    const int out_kind = kind_of(out_type, true);
    const int32_t act = activation_of(a[4]);
    const int64_t R = rows ? rows->size(0) : x.rows;
    if (out_kind < 0 || act < 0 || R == 0) Py_RETURN_NONE;
    bsg_int8_args c{};
    c.in_kind = x.kind; c.out_kind = out_kind; c.num_groups = int32_t(groups); c.activation = act;
    c.rows = R; c.tokens = x.rows; c.N = N; c.K = K;
    c.X = x.t->const_data_ptr(); c.ldx = x.pitch; c.index = rows ? rows->const_data_ptr<int32_t>() : nullptr; c.ldq = pitch;
    c.W = w->const_data_ptr(); c.ldw = ldw; c.group_stride_w = group_stride; c.w_scale = ws->const_data_ptr<float>();
    c.bias = bias ? bias->const_data_ptr<float>() : nullptr; c.offsets = offsets ? offsets->const_data_ptr<int32_t>() : nullptr;
    c.ldd = N;
    at::Tensor scratch, y;
    void* const status_words = status->mutable_data_ptr();
    int32_t code;
    {
      Unlocked unlocked;
      if (grouped || R > 4 || (R <= 2 ? R : 4) * whole > 65536) {      // else the tokens are quantised inside the product's kernel
        int64_t held = R;
        if (rows) g.int8_scratch_rows(&c, &held);
        scratch = empty({held * (pitch + 4)}, at::kChar, *x.t);        // 8-bit tokens, then their scales
        c.Q = scratch.mutable_data_ptr();
        c.q_scale = reinterpret_cast<float*>(static_cast<char*>(c.Q) + held * pitch);
      }
      y = empty({R, N}, out_type, *x.t);
      c.D = y.mutable_data_ptr();
      code = g.int8_linear_run(&c, status_words, 16, current_stream(dev));
    }
    return code ? failed(code) : THPVariable_Wrap(std::move(y));
  });
}

// act_forward(x, activation, gated) -> (h, ActivationCheckpoint)
PyObject* act_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Matrix x;
    if (n != 3 || !matrix(a[0], false, &x) || wants_gradient(x.t)) Py_RETURN_NONE;
    const int32_t act = activation_of(a[1]);
    const bool gated = a[2] == Py_True;
    if (act < 0 || (!gated && a[2] != Py_False) || (gated && x.cols % 2 != 0)) Py_RETURN_NONE;
    const int64_t parts = gated ? 2 : 1, T = x.rows, F = x.cols / parts, split = T * parts * ((F + 15) & ~int64_t(15));
    at::Tensor data, h;
    bsg_act_args c{};
    c.type = x.kind; c.activation = act; c.gated = gated; c.rows = T; c.width = F;
    c.in = x.t->const_data_ptr(); c.ld_in = x.pitch; c.ld_out = F;
    int32_t code;
    {
      Unlocked unlocked;
      data = empty({split + 4 * T * parts * ((F + 127) / 128)}, at::kChar, *x.t);
      h = empty({T, F}, x.t->scalar_type(), *x.t);
      c.out = h.mutable_data_ptr();
      c.kept = data.mutable_data_ptr(); c.kept_scale = reinterpret_cast<float*>(static_cast<char*>(c.kept) + split);
      code = g.act_forward(&c, current_stream(x.device));
    }
    if (code) return failed(code);
    PyObject* dtype = reinterpret_cast<PyObject*>(torch::getTHPDtype(x.t->scalar_type()));
    Py_INCREF(a[1]);
    Py_INCREF(a[2]);
    Py_INCREF(dtype);
    PyObject* kept = tuple_of(g_py.checkpoint, {THPVariable_Wrap(std::move(data)), a[1], a[2], PyLong_FromLongLong(T), PyLong_FromLongLong(F), dtype});
    return kept ? tuple_of(reinterpret_cast<PyObject*>(&PyTuple_Type), {THPVariable_Wrap(std::move(h)), kept}) : nullptr;
  });
}

// act_backward(grad, kept) -> dx
PyObject* act_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Matrix d;
    if (n != 2 || !matrix(a[0], false, &d) || wants_gradient(d.t) || reinterpret_cast<PyObject*>(Py_TYPE(a[1])) != g_py.checkpoint || PyTuple_GET_SIZE(a[1]) != 6) Py_RETURN_NONE;
    PyObject* const* kept = &PyTuple_GET_ITEM(a[1], 0);      // data, activation, gated, rows, width, dtype
    const int32_t act = activation_of(kept[1]);
    const bool gated = kept[2] == Py_True;
    if (act < 0 || !PyLong_Check(kept[3]) || !PyLong_Check(kept[4]) || !THPDtype_Check(kept[5])) Py_RETURN_NONE;
    const int64_t T = d.rows, F = d.cols, parts = gated ? 2 : 1, split = T * parts * ((F + 15) & ~int64_t(15));
    if (PyLong_AsLongLong(kept[3]) != T || PyLong_AsLongLong(kept[4]) != F || reinterpret_cast<THPDtype*>(kept[5])->scalar_type != d.t->scalar_type()) {
      PyErr_Clear();
      Py_RETURN_NONE;
    }
    const at::Tensor* data = array(kept[0], at::kChar, {split + 4 * T * parts * ((F + 127) / 128)}, d.device);
    if (!data) Py_RETURN_NONE;
    at::Tensor dx;
    bsg_act_args c{};
    c.type = d.kind; c.activation = act; c.gated = gated; c.rows = T; c.width = F;
    c.in = d.t->const_data_ptr(); c.ld_in = d.pitch; c.ld_out = parts * F;
    c.kept = const_cast<void*>(data->const_data_ptr());
    c.kept_scale = reinterpret_cast<float*>(static_cast<char*>(c.kept) + split);
    int32_t code;
    {
      Unlocked unlocked;
      dx = empty({T, parts * F}, d.t->scalar_type(), *d.t);
      c.out = dx.mutable_data_ptr();
      code = g.act_backward(&c, current_stream(d.device));
    }
    return code ? failed(code) : THPVariable_Wrap(std::move(dx));
  });
}

bool routable(const Matrix& l, int64_t k) { return l.cols <= kMaxExperts && k >= 1 && k <= kMaxTopK && k <= l.cols && l.rows * k <= 0x7FFFFFFFll; }

// route_forward(logits, top_k, token_mask, normalize) -> Routing
PyObject* route_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Matrix l;
    if (n != 4 || !matrix(a[0], true, &l) || !PyLong_CheckExact(a[1]) || (a[3] != Py_True && a[3] != Py_False) || wants_gradient(l.t)) Py_RETURN_NONE;
    const int64_t T = l.rows, E = l.cols, k = PyLong_AsLongLong(a[1]);
    if (k < 1 || !routable(l, k)) { PyErr_Clear(); Py_RETURN_NONE; }
    const at::Tensor* mask = a[2] == Py_None ? nullptr : array(a[2], at::kBool, {T}, l.device);
    if (a[2] != Py_None && !mask) Py_RETURN_NONE;
    const int64_t slots = T * k;
    // one allocation: softmax (2 T), experts, rows, positions, weights (slots each), counts, offsets (E each), live, loss
    int64_t at_ = 0;
    auto take = [&](int64_t count) { const int64_t o = at_; at_ += count; return o; };
    const int64_t soft = take(2 * T), experts = take(slots), rows = take(slots), positions = take(slots), weights = take(slots), counts = take(E), offsets = take(E),
                  live = take(1), loss = take(1);
    bsg_route_args c{};
    c.type = l.kind; c.experts = int32_t(E); c.k = int32_t(k); c.normalize = a[3] == Py_True; c.tokens = T;
    c.logits = l.t->const_data_ptr(); c.ld = l.pitch; c.mask = mask ? static_cast<const uint8_t*>(mask->const_data_ptr()) : nullptr;
    size_t bytes = 0;
    if (g.route_scratch_size(&c, &bytes) != BSG_OK) Py_RETURN_NONE;
    at::Tensor all, scratch;
    int32_t code;
    {
      Unlocked unlocked;
      all = empty({at_}, at::kInt, *l.t);
      int32_t* p = static_cast<int32_t*>(all.mutable_data_ptr());
      c.chosen = p + experts; c.weights = reinterpret_cast<float*>(p + weights); c.counts = p + counts; c.live = p + live;
      c.softmax = reinterpret_cast<float*>(p + soft); c.offsets = p + offsets; c.rows = p + rows; c.positions = p + positions;
      c.loss = reinterpret_cast<float*>(p + loss);
      if (bytes) scratch = empty({int64_t(bytes)}, at::kByte, *l.t);
      code = g.route_forward(&c, bytes ? scratch.mutable_data_ptr() : nullptr, bytes, current_stream(l.device));
    }
    if (code) return failed(code);
    auto ints = [&](int64_t o, at::IntArrayRef s) { return THPVariable_Wrap(part(all, at::kInt, o, s)); };
    auto reals = [&](int64_t o, at::IntArrayRef s) { return THPVariable_Wrap(part(all, at::kFloat, o, s)); };
    Py_INCREF(a[3]);
    return tuple_of(g_py.routing, {ints(experts, {T, k}), reals(weights, {T, k}), ints(counts, {E}), ints(offsets, {E}), ints(rows, {slots}),
                                   ints(positions, {T, k}), reals(loss, {}), ints(live, {1}), ints(soft, {2 * T}), a[3]});
  });
}

// route_backward(logits, routing, grad_weights, grad_loss) -> grad_logits
PyObject* route_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Matrix l;
    if (n != 4 || !matrix(a[0], true, &l) || reinterpret_cast<PyObject*>(Py_TYPE(a[1])) != g_py.routing || PyTuple_GET_SIZE(a[1]) != 10) Py_RETURN_NONE;
    // experts, weights, counts, offsets, rows, positions, balance_loss, num_tokens, softmax, normalize
    PyObject* const* r = &PyTuple_GET_ITEM(a[1], 0);
    const at::Tensor* experts = tensor(r[0]);
    if (!experts || experts->dim() != 2) Py_RETURN_NONE;
    const int64_t T = l.rows, E = l.cols, k = experts->size(1);
    if (!routable(l, k)) Py_RETURN_NONE;
    experts = array(r[0], at::kInt, {T, k}, l.device);
    const at::Tensor *weights = array(r[1], at::kFloat, {T, k}, l.device), *counts = array(r[2], at::kInt, {E}, l.device), *live = array(r[7], at::kInt, {1}, l.device),
                     *soft = array(r[8], at::kInt, {2 * T}, l.device);
    const at::Tensor* gw = a[2] == Py_None ? nullptr : array(a[2], at::kFloat, {T, k}, l.device);
    const at::Tensor* gl = a[3] == Py_None ? nullptr : tensor(a[3]);
    if (!experts || !weights || !counts || !live || !soft || (a[2] != Py_None && !gw)) Py_RETURN_NONE;
    if (has_tangent(l.t) || has_tangent(weights) || has_tangent(gw) || has_tangent(gl)) Py_RETURN_NONE;
    if (a[3] != Py_None && (!gl || gl->scalar_type() != at::kFloat || gl->numel() != 1 || gl->get_device() != l.device)) Py_RETURN_NONE;
    at::Tensor d;
    bsg_route_args c{};
    c.type = l.kind; c.experts = int32_t(E); c.k = int32_t(k); c.normalize = r[9] == Py_True; c.tokens = T;
    c.logits = l.t->const_data_ptr(); c.ld = l.pitch;
    c.chosen = const_cast<int32_t*>(experts->const_data_ptr<int32_t>()); c.weights = const_cast<float*>(weights->const_data_ptr<float>());
    c.counts = const_cast<int32_t*>(counts->const_data_ptr<int32_t>()); c.live = const_cast<int32_t*>(live->const_data_ptr<int32_t>());
    c.softmax = reinterpret_cast<float*>(const_cast<int32_t*>(soft->const_data_ptr<int32_t>()));
    c.grad_weights = gw ? gw->const_data_ptr<float>() : nullptr; c.grad_loss = gl ? gl->const_data_ptr<float>() : nullptr;
    c.ld_grad = E;
    int32_t code;
    {
      Unlocked unlocked;
      d = empty({T, E}, l.t->scalar_type(), *l.t);
      c.grad_logits = d.mutable_data_ptr();
      code = g.route_backward(&c, current_stream(l.device));
    }
    return code ? failed(code) : THPVariable_Wrap(std::move(d));
  });
}

// bind(raise, activations, workspaces, checkpoint, routing, address, ...): the objects of `g_py`, then the entry points in the
// order of `g`.
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  PyObject** objects = reinterpret_cast<PyObject**>(&g_py);
  void** slots = reinterpret_cast<void**>(&g);
  constexpr Py_ssize_t kObjects = Py_ssize_t(sizeof(g_py) / sizeof(PyObject*)), kSlots = Py_ssize_t(sizeof(g) / sizeof(void*));
  if (n != kObjects + kSlots || !PyDict_Check(a[1]) || !PyDict_Check(a[2]) || !PyType_Check(a[3]) || !PyType_Check(a[4])) {
    PyErr_Format(PyExc_TypeError, "bind takes a function, two dicts, two tuple types and %zd addresses", kSlots);
    return nullptr;
  }
  for (Py_ssize_t i = 0; i < kSlots; ++i) {
    slots[i] = PyLong_AsVoidPtr(a[kObjects + i]);
    if (PyErr_Occurred()) return nullptr;
  }
  for (Py_ssize_t i = 0; i < kObjects; ++i) {
    Py_INCREF(a[i]);
    objects[i] = a[i];
  }
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(bind)), METH_FASTCALL, nullptr},
    {"int8_linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(int8_linear)), METH_FASTCALL, nullptr},
    {"act_forward", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(act_forward)), METH_FASTCALL, nullptr},
    {"act_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(act_backward)), METH_FASTCALL, nullptr},
    {"route_forward", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(route_forward)), METH_FASTCALL, nullptr},
    {"route_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(route_backward)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

#ifndef BSG_BINDING_FOR
#error "BSG_BINDING_FOR names the Python and the torch that this is compiled for"
#endif
PyMODINIT_FUNC PyInit__binding() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "made_for", BSG_BINDING_FOR) != 0) Py_CLEAR(m);
  return m;
}
