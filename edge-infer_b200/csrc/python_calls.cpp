// The operators for long contexts as Python calls them: takes torch tensors apart (device, type, shape, strides, address) and
// calls the C ABI. Through ctypes that took some ten microseconds a call, as long as the smaller kernels run.
//
// Every function returns the ei_status of its call; a tensor of another device, type or rank raises ValueError, which a C
// entry, that only sees pointers, could not tell. Nothing of torch is linked: tensors are asked by their Python methods.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include "../../include/edge_infer_b200.h"

namespace {

PyObject *name_get_device, *name_dtype, *name_data_ptr, *name_shape, *name_stride, *name_numel, *name_element_size;
PyObject *type_bf16, *type_f32, *type_i32;  // torch's, given by configure()

// Owned reference that is dropped on every way out.
struct Held {
  PyObject* object;
  explicit Held(PyObject* o) : object(o) {}
  ~Held() { Py_XDECREF(object); }
  Held(const Held&) = delete;
  Held& operator=(const Held&) = delete;
  explicit operator bool() const { return object != nullptr; }
};

bool as_size(PyObject* o, size_t* out) {
  *out = PyLong_AsSize_t(o);
  return !(*out == size_t(-1) && PyErr_Occurred());
}

bool on_device(PyObject* t, const ei_context* ctx) {
  Held device(PyObject_CallMethodNoArgs(t, name_get_device));
  if (!device) return false;
  const long found = PyLong_AsLong(device.object);
  if (found == -1 && PyErr_Occurred()) return false;
  if (found == ctx->device) return true;
  if (found < 0) PyErr_Format(PyExc_ValueError, "a tensor is on cpu, the execution context on cuda:%d", int(ctx->device));
  else PyErr_Format(PyExc_ValueError, "a tensor is on cuda:%ld, the execution context on cuda:%d", found, int(ctx->device));
  return false;
}

bool address(PyObject* t, void** out) {
  Held pointer(PyObject_CallMethodNoArgs(t, name_data_ptr));
  if (!pointer) return false;
  *out = PyLong_AsVoidPtr(pointer.object);
  return !(*out == nullptr && PyErr_Occurred());
}

bool sizes(PyObject* tuple, int rank, size_t* out) {
  if (!PyTuple_Check(tuple) || PyTuple_GET_SIZE(tuple) != rank) {
    PyErr_Format(PyExc_ValueError, "expected a tensor with %d axes, not %zd", rank, PyTuple_Check(tuple) ? PyTuple_GET_SIZE(tuple) : -1);
    return false;
  }
  for (int i = 0; i < rank; ++i)
    if (!as_size(PyTuple_GET_ITEM(tuple, i), out + i)) return false;
  return true;
}

template <typename View>
bool view(PyObject* t, const ei_context* ctx, PyObject* type, View* out) {
  constexpr int rank = int(sizeof(out->shape) / sizeof(out->shape[0]));
  if (!on_device(t, ctx)) return false;
  Held found(PyObject_GetAttr(t, name_dtype));
  if (!found) return false;
  if (found.object != type) {
    PyErr_Format(PyExc_ValueError, "expected a %S tensor, not %S", type, found.object);
    return false;
  }
  Held shape(PyObject_GetAttr(t, name_shape));
  if (!shape || !sizes(shape.object, rank, out->shape)) return false;
  Held stride(PyObject_CallMethodNoArgs(t, name_stride));
  if (!stride || !sizes(stride.object, rank, out->stride)) return false;
  return address(t, &out->data);
}

// `count` packed int32 values on the device, or None.
bool values(PyObject* t, const ei_context* ctx, size_t count, const char* name, int32_t** out) {
  *out = nullptr;
  if (t == Py_None) return true;
  ei_view1 v;
  if (!view(t, ctx, type_i32, &v)) return false;
  if (v.shape[0] != count || (count > 1 && v.stride[0] != 1)) {
    PyErr_Format(PyExc_ValueError, "%s must hold %zu packed values", name, count);
    return false;
  }
  *out = static_cast<int32_t*>(v.data);
  return true;
}

bool scratch_of(PyObject* t, const ei_context* ctx, void** data, size_t* bytes) {
  *data = nullptr;
  *bytes = 0;
  if (t == Py_None) return true;
  if (!on_device(t, ctx)) return false;
  Held count(PyObject_CallMethodNoArgs(t, name_numel)), each(PyObject_CallMethodNoArgs(t, name_element_size));
  size_t n = 0, size = 0;
  if (!count || !each || !as_size(count.object, &n) || !as_size(each.object, &size)) return false;
  *bytes = n * size;
  return address(t, data);
}

// The context is given by its address (a ctypes structure); the arguments behind it are counted here.
bool begin(PyObject* const* args, Py_ssize_t given, Py_ssize_t wanted, const ei_context** ctx) {
  if (given != wanted) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, not %zd", wanted, given);
    return false;
  }
  if (!type_bf16) {
    PyErr_SetString(PyExc_RuntimeError, "configure() has not been called");
    return false;
  }
  *ctx = static_cast<const ei_context*>(PyLong_AsVoidPtr(args[0]));
  if (!*ctx && !PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "execution context is null");
  return *ctx != nullptr;
}

// The C call runs without the interpreter's lock, as calls through ctypes do: a launch waits while the device's queue is full, and
// what empties the queue may need the interpreter. The caller holds the tensors and the context meanwhile.
template <typename Call>
PyObject* status_of(Call call) {
  PyThreadState* const thread = PyEval_SaveThread();
  const ei_status status = call();
  PyEval_RestoreThread(thread);
  return PyLong_FromLong(status);
}

PyObject* configure(PyObject*, PyObject* const* args, Py_ssize_t given) {
  if (given != 3) return PyErr_Format(PyExc_TypeError, "expected 3 types");
  PyObject** const types[3] = {&type_bf16, &type_f32, &type_i32};
  for (int i = 0; i < 3; ++i) {
    Py_INCREF(args[i]);
    Py_XSETREF(*types[i], args[i]);
  }
  Py_RETURN_NONE;
}

// (ctx, q, k, table, q_out, k_out, positions, offset, q_weight, k_weight, epsilon, interleaved)
PyObject* qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t given) {
  const ei_context* ctx;
  ei_view3 q, k, q_out, k_out;
  ei_view2 table;
  ei_view1 q_weight{}, k_weight{};
  int32_t* positions;
  size_t offset;
  if (!begin(a, given, 12, &ctx) || !view(a[1], ctx, type_bf16, &q) || !view(a[2], ctx, type_bf16, &k) || !view(a[3], ctx, type_f32, &table) ||
      !view(a[4], ctx, type_bf16, &q_out) || !view(a[5], ctx, type_bf16, &k_out) || !values(a[6], ctx, q.shape[0], "positions", &positions) ||
      !as_size(a[7], &offset) || (a[8] != Py_None && !view(a[8], ctx, type_bf16, &q_weight)) ||
      (a[9] != Py_None && !view(a[9], ctx, type_bf16, &k_weight)))
    return nullptr;
  const double epsilon = PyFloat_AsDouble(a[10]);
  const int interleaved = PyObject_IsTrue(a[11]);
  if (PyErr_Occurred()) return nullptr;
  return status_of([&] {
    return ei_qk_norm_rope_bf16(ctx, q, k, table, positions, offset, q_weight, k_weight, float(epsilon), interleaved, q_out, k_out);
  });
}

// (ctx, q, k, v, output, window, sinks, lengths, length)
PyObject* attention_window(PyObject*, PyObject* const* a, Py_ssize_t given) {
  const ei_context* ctx;
  ei_view3 q, out;
  ei_view4 k, v;
  int32_t* lengths;
  size_t window, sinks, length;
  if (!begin(a, given, 9, &ctx) || !view(a[1], ctx, type_bf16, &q) || !view(a[2], ctx, type_bf16, &k) || !view(a[3], ctx, type_bf16, &v) ||
      !view(a[4], ctx, type_bf16, &out) || !as_size(a[5], &window) || !as_size(a[6], &sinks) ||
      !values(a[7], ctx, k.shape[0], "lengths", &lengths) || !as_size(a[8], &length))
    return nullptr;
  return status_of([&] { return ei_attention_window_bf16(ctx, q, k, v, out, lengths, length, window, sinks); });
}

// (ctx, q, prefix_k, prefix_v, k, v, output, scratch, lengths, length)
PyObject* attention_shared_prefix(PyObject*, PyObject* const* a, Py_ssize_t given) {
  const ei_context* ctx;
  ei_view3 q, prefix_k, prefix_v, out;
  ei_view4 k, v;
  int32_t* lengths;
  void* scratch;
  size_t scratch_bytes, length;
  if (!begin(a, given, 10, &ctx) || !view(a[1], ctx, type_bf16, &q) || !view(a[2], ctx, type_bf16, &prefix_k) ||
      !view(a[3], ctx, type_bf16, &prefix_v) || !view(a[4], ctx, type_bf16, &k) || !view(a[5], ctx, type_bf16, &v) ||
      !view(a[6], ctx, type_bf16, &out) || !scratch_of(a[7], ctx, &scratch, &scratch_bytes) ||
      !values(a[8], ctx, k.shape[0], "lengths", &lengths) || !as_size(a[9], &length))
    return nullptr;
  return status_of([&] {
    return ei_attention_shared_prefix_bf16(ctx, q, prefix_k, prefix_v, k, v, out, lengths, length, scratch, scratch_bytes);
  });
}

// (ctx, q, k, v, output, scores, scores_out, scratch, lengths, length)
PyObject* attention_accumulate(PyObject*, PyObject* const* a, Py_ssize_t given) {
  const ei_context* ctx;
  ei_view3 q, out, scores{}, scores_out;
  ei_view4 k, v;
  int32_t* lengths;
  void* scratch;
  size_t scratch_bytes, length;
  if (!begin(a, given, 10, &ctx) || !view(a[1], ctx, type_bf16, &q) || !view(a[2], ctx, type_bf16, &k) || !view(a[3], ctx, type_bf16, &v) ||
      !view(a[4], ctx, type_bf16, &out) || (a[5] != Py_None && !view(a[5], ctx, type_f32, &scores)) ||
      !view(a[6], ctx, type_f32, &scores_out) || !scratch_of(a[7], ctx, &scratch, &scratch_bytes) ||
      !values(a[8], ctx, k.shape[0], "lengths", &lengths) || !as_size(a[9], &length))
    return nullptr;
  return status_of([&] {
    return ei_attention_accumulate_bf16(ctx, q, k, v, out, lengths, length, scores, scores_out, scratch, scratch_bytes);
  });
}

// (ctx, k, v, scores, k_out, v_out, scores_out, kept, lengths_out, sinks, recent, lengths, length)
PyObject* evict_kv(PyObject*, PyObject* const* a, Py_ssize_t given) {
  const ei_context* ctx;
  ei_view4 k, v, k_out, v_out;
  ei_view3 scores, scores_out, kept;
  int32_t *lengths, *lengths_out;
  size_t sinks, recent, length;
  if (!begin(a, given, 13, &ctx) || !view(a[1], ctx, type_bf16, &k) || !view(a[2], ctx, type_bf16, &v) || !view(a[3], ctx, type_f32, &scores) ||
      !view(a[4], ctx, type_bf16, &k_out) || !view(a[5], ctx, type_bf16, &v_out) || !view(a[6], ctx, type_f32, &scores_out) ||
      !view(a[7], ctx, type_i32, &kept) || !values(a[8], ctx, k.shape[0], "lengths_out", &lengths_out) || !as_size(a[9], &sinks) ||
      !as_size(a[10], &recent) || !values(a[11], ctx, k.shape[0], "lengths", &lengths) || !as_size(a[12], &length))
    return nullptr;
  return status_of([&] {
    return ei_evict_kv_bf16(ctx, k, v, scores, lengths, length, sinks, recent, k_out, v_out, scores_out, kept, lengths_out);
  });
}

#define CALL(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {CALL(configure),            CALL(qk_norm_rope), CALL(attention_window), CALL(attention_shared_prefix),
                         CALL(attention_accumulate), CALL(evict_kv),     {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", "Operator calls on torch tensors over the C ABI.", -1, methods,
                      nullptr,               nullptr,  nullptr,                                            nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() {
  struct {
    PyObject** to;
    const char* text;
  } const names[] = {{&name_get_device, "get_device"}, {&name_dtype, "dtype"}, {&name_data_ptr, "data_ptr"},       {&name_shape, "shape"},
                     {&name_stride, "stride"},         {&name_numel, "numel"}, {&name_element_size, "element_size"}};
  for (const auto& name : names)
    if (!(*name.to = PyUnicode_InternFromString(name.text))) return nullptr;
  return PyModule_Create(&module);
}
