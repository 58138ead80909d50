// attention.cpp -- torch tensors to the window-cache entry points of the C ABI
// (include/streaming_b200.h): the checks of streaming_transformer_b200/attention.py
// and the descriptors the C calls take, as a CPython extension module.
//
// It is compiled because the calls are short: reading ten tensors' types,
// shapes, strides and addresses through Python objects took 10 to 15 us where
// the kernels of a small call take 3 to 6.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <sstream>
#include <string>

#include "streaming_b200.h"

namespace {

PyObject* g_error = nullptr;  // StreamError(code, message)

// A refusal on its way out: the status and its message.
struct Refusal {
  int code;
  std::string message;
};
[[noreturn]] void refuse(const std::string& message, int code = ST_ERR_INVALID) { throw Refusal{code, message}; }
void check(int code) {
  if (code != ST_OK) refuse(st_cache_error(), code);
}

std::string shape_text(c10::IntArrayRef s) {
  std::ostringstream o;
  o << '(';
  for (size_t i = 0; i < s.size(); ++i) o << (i ? ", " : "") << s[i];
  o << (s.size() == 1 ? ",)" : ")");
  return o.str();
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(std::string(name) + ": expected a tensor");
  return THPVariable_Unpack(o);
}
const at::Tensor* optional_tensor(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }

const char* type_name(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kHalf: return "torch.float16";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kDouble: return "torch.float64";
    case at::kLong: return "torch.int64";
    case at::kInt: return "torch.int32";
    case at::kByte: return "torch.uint8";
    default: return c10::toString(t);
  }
}

int mode_of(at::ScalarType t) {
  return t == at::kFloat ? ST_MODE_FP32 : t == at::kHalf ? ST_MODE_FP16 : t == at::kBFloat16 ? ST_MODE_BF16 : -1;
}
int row_mode(const at::Tensor& t, const char* name) {
  const int mode = mode_of(t.scalar_type());
  if (mode < 0) refuse(std::string(name) + ": " + type_name(t.scalar_type()) + " is no row type");
  return mode;
}

// Refuses tensors whose derivative a call would drop: every floating-point one that it reads or writes is named here,
// before any other check. Forward-mode tangents (there is one level, 0) count with gradients off as well.
void no_gradient(std::initializer_list<const at::Tensor*> tensors) {
  const c10::AutogradState& state = c10::AutogradState::get_tls_state();
  for (const at::Tensor* t : tensors) {
    if (!t) continue;
    if (state.get_grad_mode() && t->requires_grad())
      refuse("there is no backward pass: detach the inputs or call under torch.no_grad()");
    if (state.get_fw_grad_mode() && t->_fw_grad(0).defined()) refuse("there is no forward-mode derivative: detach the inputs");
  }
}

// Counts a write, so that a backward pass which saved the old values of one of these raises, as for torch's own.
void written(std::initializer_list<const at::Tensor*> tensors) {
  for (const at::Tensor* t : tensors)
    if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

void placed(const at::Tensor& t, const char* name, c10::Device device, at::ScalarType type) {
  if (t.device() != device || t.scalar_type() != type) {
    std::ostringstream o;
    o << name << ": expected " << type_name(type) << " on " << device << ", got " << type_name(t.scalar_type()) << " on " << t.device();
    refuse(o.str());
  }
}

// [rows, heads, head_dim] with contiguous columns, any row and head strides.
st_rows rows_of(const at::Tensor& t, const char* name, c10::Device device, at::ScalarType type, int64_t rows,
                int64_t heads, int64_t head_dim) {
  placed(t, name, device, type);
  const auto z = t.sizes();
  if (z.size() != 3 || z[0] != rows || z[1] != heads || z[2] != head_dim)
    refuse(std::string(name) + ": expected shape " + shape_text({rows, heads, head_dim}) + ", got " + shape_text(z));
  const auto s = t.strides();
  if (s[2] != 1 && head_dim > 1) refuse(std::string(name) + ": columns must be contiguous");
  return {t.data_ptr(), rows > 1 ? s[0] : heads * head_dim, heads > 1 ? s[1] : head_dim};
}

// The address of a contiguous one-dimensional tensor of `count` values.
const void* values_of(const at::Tensor& t, const char* name, c10::Device device, at::ScalarType type, int64_t count) {
  placed(t, name, device, type);
  if (t.dim() != 1 || t.size(0) != count || (count > 1 && t.stride(0) != 1))
    refuse(std::string(name) + ": expected " + std::to_string(count) + " contiguous values, got shape " + shape_text(t.sizes()));
  return t.data_ptr();
}

st_cache cache_of(const at::Tensor& keys, const at::Tensor& values, const at::Tensor* key_scales,
                  const at::Tensor* value_scales, int64_t sinks) {
  if (sinks < 0 || sinks > INT32_MAX) refuse("sinks: " + std::to_string(sinks) + " is out of range");
  if (!keys.is_cuda()) refuse("keys: expected a CUDA tensor, got " + keys.device().str());
  const bool four = keys.scalar_type() == at::kByte;
  const int mode = mode_of(keys.scalar_type());
  if (!four && mode < 0) refuse(std::string("keys: ") + type_name(keys.scalar_type()) + " is no cache type");
  const auto z = keys.sizes();
  if (z.size() != 4 || z[0] < 1 || z[1] < 1 || z[3] < 1 || z[3] > 4096)
    refuse("keys: expected [streams, heads, slots, columns], got " + shape_text(z));
  const int64_t streams = z[0], heads = z[1], slots = z[2], columns = z[3];
  if (streams > 65535 || heads > 65535) refuse("cache streams and heads are 1 to 65535");
  if (slots > (1 << 30)) refuse("a cache has at most 2^30 slots");
  const auto s = keys.strides();
  if (values.sizes() != z || values.scalar_type() != keys.scalar_type() || values.device() != keys.device() ||
      (keys.numel() && values.strides() != s))
    refuse("values must have the keys' shape, strides, type and device");
  if ((columns > 1 && s[3] != 1) || (slots > 1 && s[2] != columns)) refuse("the slots of a cache head must be contiguous");
  if ((streams > 1 && s[0] % columns) || (heads > 1 && s[1] % columns)) refuse("cache strides must be whole rows");
  // a stride along a dimension of one element is never used
  const int64_t stream_stride = streams > 1 ? s[0] / columns : heads * slots, head_stride = heads > 1 ? s[1] / columns : slots;
  if (four != (key_scales != nullptr) || four != (value_scales != nullptr))
    refuse("a 4-bit cache has scales, any other has none");
  const int64_t head_dim = four ? columns * 2 : columns, groups = head_dim / ST_CACHE_GROUP;
  if (four) {
    const at::Tensor* sides[2] = {key_scales, value_scales};
    for (int i = 0; i < 2; ++i) {
      const at::Tensor& t = *sides[i];
      const std::string name = i ? "value_scales" : "key_scales";
      const auto y = t.sizes();
      if (t.scalar_type() != at::kBFloat16 || t.device() != keys.device() || y.size() != 5 || y[0] != streams ||
          y[1] != heads || y[2] != slots || y[3] != groups || y[4] != 2)
        refuse(name + ": expected bfloat16 " + shape_text({streams, heads, slots, groups, 2}) + " on " + keys.device().str());
      const auto x = t.strides();
      if (t.numel() && (x[4] != 1 || (groups > 1 && x[3] != 2) || (slots > 1 && x[2] != 2 * groups) ||
                        (streams > 1 && x[0] != stream_stride * 2 * groups) ||
                        (heads > 1 && x[1] != head_stride * 2 * groups)))
        refuse(name + ": strides must be those of the rows");
    }
  }
  st_cache c{};
  c.device = keys.device().index();
  c.type = four ? ST_CACHE_INT4 : mode;
  c.streams = (int)streams;
  c.heads = (int)heads;
  c.head_dim = (int)head_dim;
  c.sinks = (int)sinks;
  c.window = (int)(slots - sinks < 0 ? 0 : slots - sinks);
  c.stream_stride = stream_stride;
  c.head_stride = head_stride;
  c.keys = keys.data_ptr();
  c.values = values.data_ptr();
  c.key_scales = four ? key_scales->data_ptr() : nullptr;
  c.value_scales = four ? value_scales->data_ptr() : nullptr;
  return c;
}

int heads_of(const at::Tensor& q, const char* what) {
  if (q.dim() != 3) refuse(std::string("q: expected ") + what + ", got " + shape_text(q.sizes()));
  if (q.size(1) > 65535) refuse("query heads are 1 to 65535");
  return (int)q.size(1);
}

at::Tensor fresh(std::initializer_list<int64_t> shape, at::ScalarType type, c10::Device device) {
  return at::empty(c10::IntArrayRef(shape), at::TensorOptions().dtype(type).device(device));
}
void* stream_of(c10::Device device) { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }

double number(PyObject* o, const char* name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(std::string(name) + ": expected a number");
  }
  return v;
}
// An integer of any type that is one (numpy's among them); one past 64 bits becomes the nearest that fits.
int64_t integer(PyObject* o, const char* name) {
  PyObject* index = PyNumber_Index(o);
  if (!index) {
    PyErr_Clear();
    refuse(std::string(name) + ": expected an integer");
  }
  int over = 0;
  const long long v = PyLong_AsLongLongAndOverflow(index, &over);
  Py_DECREF(index);
  return over > 0 ? INT64_MAX : over < 0 ? INT64_MIN : v;
}

// q, k, v, keys, values, positions, frequencies, sinks, starts, q_gain, k_gain, epsilon, key_scales, value_scales,
// rotated_keys, out
PyObject* do_append(PyObject* const* o) {
  const at::Tensor &q = tensor(o[0], "q"), &k = tensor(o[1], "k"), &v = tensor(o[2], "v"), &keys = tensor(o[3], "keys"),
                   &values = tensor(o[4], "values"), &positions = tensor(o[5], "positions"),
                   &frequencies = tensor(o[6], "frequencies");
  const at::Tensor *starts = optional_tensor(o[8], "starts"), *q_gain = optional_tensor(o[9], "q_gain"),
                   *k_gain = optional_tensor(o[10], "k_gain"), *key_scales = optional_tensor(o[12], "key_scales"),
                   *value_scales = optional_tensor(o[13], "value_scales"), *given = optional_tensor(o[15], "out");
  no_gradient({&q, &k, &v, &keys, &values, &frequencies, q_gain, k_gain, key_scales, value_scales, given});
  const st_cache c = cache_of(keys, values, key_scales, value_scales, integer(o[7], "sinks"));
  const c10::Device device = keys.device();
  const at::ScalarType type = q.scalar_type();
  st_append a{};
  a.mode = row_mode(q, "q");
  a.heads = heads_of(q, "[rows, heads, head_dim]");
  const int64_t rows = a.rows = q.size(0);
  a.q = rows_of(q, "q", device, type, rows, a.heads, c.head_dim);
  a.k = rows_of(k, "k", device, type, rows, c.heads, c.head_dim);
  a.v = rows_of(v, "v", device, type, rows, c.heads, c.head_dim);
  at::Tensor out = given ? *given : fresh({rows, a.heads, c.head_dim}, type, device), turned;
  a.q_out = rows_of(out, "out", device, type, rows, a.heads, c.head_dim);
  const int both = PyObject_IsTrue(o[14]);
  if (both < 0) {
    PyErr_Clear();
    refuse("rotated_keys: expected True or False");
  }
  if (both) {
    turned = fresh({rows, c.heads, c.head_dim}, type, device);
    a.k_out = rows_of(turned, "k", device, type, rows, c.heads, c.head_dim);
  }
  if (q_gain) a.q_gain = static_cast<const float*>(values_of(*q_gain, "q_gain", device, at::kFloat, c.head_dim));
  if (k_gain) a.k_gain = static_cast<const float*>(values_of(*k_gain, "k_gain", device, at::kFloat, c.head_dim));
  a.epsilon = (float)number(o[11], "epsilon");
  if (frequencies.dim() != 1 || frequencies.size(0) > ST_CACHE_MAX_HEAD_DIM)
    refuse("frequencies: expected one dimension; rotary is 0 to head_dim / 2");
  a.rotary = (int)frequencies.size(0);
  a.frequencies = static_cast<const double*>(values_of(frequencies, "frequencies", device, at::kDouble, a.rotary));
  a.positions = static_cast<const int64_t*>(values_of(positions, "positions", device, at::kLong, c.streams));
  if (starts) a.starts = static_cast<const int32_t*>(values_of(*starts, "starts", device, at::kInt, c.streams + 1));
  check(st_cache_append(&c, &a, stream_of(device)));
  written({&keys, &values, key_scales, value_scales, given});
  PyObject* first = THPVariable_Wrap(std::move(out));
  if (!both || !first) return first;
  PyObject* second = THPVariable_Wrap(std::move(turned));
  PyObject* pair = second ? PyTuple_Pack(2, first, second) : nullptr;
  Py_DECREF(first);
  Py_XDECREF(second);
  return pair;
}

// q, keys, values, positions, key_scales, value_scales, scale, out
PyObject* do_attend(PyObject* const* o) {
  const at::Tensor &q = tensor(o[0], "q"), &keys = tensor(o[1], "keys"), &values = tensor(o[2], "values"),
                   &positions = tensor(o[3], "positions");
  const at::Tensor *key_scales = optional_tensor(o[4], "key_scales"), *value_scales = optional_tensor(o[5], "value_scales"),
                   *given = optional_tensor(o[7], "out");
  no_gradient({&q, &keys, &values, key_scales, value_scales, given});
  const st_cache c = cache_of(keys, values, key_scales, value_scales, 0);
  const c10::Device device = keys.device();
  const at::ScalarType type = q.scalar_type();
  st_attend a{};
  a.mode = row_mode(q, "q");
  a.heads = heads_of(q, "[streams, heads, head_dim]");
  a.scale = o[6] == Py_None ? (float)(1.0 / std::sqrt((double)c.head_dim)) : (float)number(o[6], "scale");
  a.q = rows_of(q, "q", device, type, c.streams, a.heads, c.head_dim);
  at::Tensor out = given ? *given : fresh({c.streams, a.heads, c.head_dim}, type, device), work;
  a.out = rows_of(out, "out", device, type, c.streams, a.heads, c.head_dim);
  a.positions = static_cast<const int64_t*>(values_of(positions, "positions", device, at::kLong, c.streams));
  check(st_cache_attention_workspace(&c, a.heads, &a.workspace_bytes));
  if (a.workspace_bytes) {
    // from torch's stream-ordered allocator: calls on other streams, and captured graphs, get their own
    work = fresh({(int64_t)a.workspace_bytes}, at::kByte, device);
    a.workspace = work.data_ptr();
  }
  check(st_cache_attention(&c, &a, stream_of(device)));
  written({given});
  return THPVariable_Wrap(std::move(out));
}

// keys, values, key_scales, value_scales, a tensor of the wanted type
PyObject* do_unpack(PyObject* const* o) {
  const at::Tensor &keys = tensor(o[0], "keys"), &values = tensor(o[1], "values");
  const at::Tensor *key_scales = optional_tensor(o[2], "key_scales"), *value_scales = optional_tensor(o[3], "value_scales");
  no_gradient({key_scales, value_scales});
  const st_cache c = cache_of(keys, values, key_scales, value_scales, 0);
  const at::ScalarType type = tensor(o[4], "dtype").scalar_type();
  const int mode = row_mode(THPVariable_Unpack(o[4]), "dtype");
  const int64_t slots = keys.size(2);
  at::Tensor outs[2];
  for (at::Tensor& t : outs) t = fresh({c.streams, c.heads, slots, c.head_dim}, type, keys.device());
  check(st_cache_unpack(&c, mode, outs[0].data_ptr(), outs[1].data_ptr(), stream_of(keys.device())));
  PyObject *first = THPVariable_Wrap(std::move(outs[0])), *second = first ? THPVariable_Wrap(std::move(outs[1])) : nullptr;
  PyObject* pair = second ? PyTuple_Pack(2, first, second) : nullptr;
  Py_XDECREF(first);
  Py_XDECREF(second);
  return pair;
}

// q, k, v, window, sinks, starts, scale, out
PyObject* do_window(PyObject* const* o) {
  const at::Tensor &q = tensor(o[0], "q"), &k = tensor(o[1], "k"), &v = tensor(o[2], "v");
  const at::Tensor *starts = optional_tensor(o[5], "starts"), *given = optional_tensor(o[7], "out");
  no_gradient({&q, &k, &v, given});
  if (!q.is_cuda()) refuse("q: expected a CUDA tensor, got " + q.device().str());
  const c10::Device device = q.device();
  const at::ScalarType type = q.scalar_type();
  st_window a{};
  a.device = device.index();
  a.mode = row_mode(q, "q");
  a.heads = heads_of(q, "[rows, heads, head_dim]");
  if (k.dim() != 3 || k.size(1) > 65535) refuse("k: expected [rows, key heads, head_dim]");
  const int64_t window = integer(o[3], "window"), sinks = integer(o[4], "sinks"), rows = a.rows = q.size(0), dim = q.size(2);
  if (window < 1 || sinks < 0) refuse("window is at least 1 and sinks at least 0");
  // no sequence is longer than the largest int: a wider window sees as much
  a.window = (int)std::min<int64_t>(window, INT32_MAX);
  a.sinks = (int)std::min<int64_t>(sinks, INT32_MAX);
  a.kv_heads = (int)k.size(1);
  if (dim < 1 || dim > ST_CACHE_MAX_HEAD_DIM) refuse("head_dim is a multiple of 8 up to 256");
  a.head_dim = (int)dim;
  a.scale = o[6] == Py_None ? (float)(1.0 / std::sqrt((double)dim)) : (float)number(o[6], "scale");
  a.q = rows_of(q, "q", device, type, rows, a.heads, dim);
  a.k = rows_of(k, "k", device, type, rows, a.kv_heads, dim);
  a.v = rows_of(v, "v", device, type, rows, a.kv_heads, dim);
  at::Tensor out = given ? *given : fresh({rows, a.heads, dim}, type, device);
  a.out = rows_of(out, "out", device, type, rows, a.heads, dim);
  a.sequences = 1;
  if (starts) {
    if (starts->dim() != 1 || starts->size(0) < 1 || starts->size(0) > INT32_MAX) refuse("starts: expected [sequences + 1]");
    a.sequences = (int)(starts->size(0) - 1);
    a.starts = static_cast<const int32_t*>(values_of(*starts, "starts", device, at::kInt, a.sequences + 1));
  }
  check(st_window_attention(&a, stream_of(device)));
  written({given});
  return THPVariable_Wrap(std::move(out));
}

// Runs `f` on exactly N arguments; no C++ exception leaves it.
template <int N, PyObject* (*F)(PyObject* const*)>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", N, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Refusal& r) {
    PyObject* e = PyObject_CallFunction(g_error, "is", r.code, r.message.c_str());
    if (e) {
      PyErr_SetObject(g_error, e);
      Py_DECREF(e);
    }
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "unknown error");
  }
  return nullptr;
}

PyObject* set_error(PyObject*, PyObject* type) {
  Py_INCREF(type);
  Py_XDECREF(g_error);
  g_error = type;
  Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&entry<16, do_append>)), METH_FASTCALL, nullptr},
    {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&entry<8, do_attend>)), METH_FASTCALL, nullptr},
    {"unpack", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&entry<5, do_unpack>)), METH_FASTCALL, nullptr},
    {"window", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&entry<8, do_window>)), METH_FASTCALL, nullptr},
    {"set_error", set_error, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "attention_binding", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_attention_binding() { return PyModule_Create(&g_module); }
