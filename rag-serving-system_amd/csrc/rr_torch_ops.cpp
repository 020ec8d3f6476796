// rr_torch_ops.cpp — the torch side of rag_service_amd.ops: checks of tensors, results and scratch memory from torch's
// allocator, the current stream, and one call of the C-ABI (include/rag_retrieval.h) for each operator. A CPython module of its
// own (rag_service_amd/_torch_ops.so), so that librag_retrieval.so stays free of torch; the C-ABI functions are looked up in
// the library that rag_service_amd._lib has loaded (bind()). In C++ because a call of a few microseconds of GPU work is
// otherwise mostly the host's: block_norm of one row 11.6 us through Python checks and ctypes, of which the launch is 3.5.
//
// Errors: ValueError / TypeError for arguments (as Python raises them), the C-ABI's negative code as an int otherwise, which
// ops.py turns into HipRetrievalError.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <dlfcn.h>

#include <stdexcept>
#include <string>

#include "rag_retrieval.h"

namespace {

using at::ScalarType;
using at::Tensor;

decltype(&rr_quantize_rows) p_quantize_rows;
decltype(&rr_linear_i8) p_linear_i8;
decltype(&rr_linear_i8_workspace) p_linear_i8_workspace;
decltype(&rr_block_norm) p_block_norm;
decltype(&rr_cross_attention) p_cross_attention;
decltype(&rr_cross_attention_workspace) p_cross_attention_workspace;

struct BadValue : std::runtime_error {
  using std::runtime_error::runtime_error;
};
struct BadType : std::runtime_error {
  using std::runtime_error::runtime_error;
};
struct Refused {   // the C-ABI's code
  int64_t code;
};

std::string shape_of(const Tensor& t) {
  std::string s = "(";
  for (int64_t d : t.sizes()) s += std::to_string(d) + ", ";
  return s.size() > 1 ? s.substr(0, s.size() - 2) + ")" : "()";
}
std::string strides_of(const Tensor& t) {
  std::string s = "(";
  for (int64_t d : t.strides()) s += std::to_string(d) + ", ";
  return s.size() > 1 ? s.substr(0, s.size() - 2) + ")" : "()";
}

int code_of(ScalarType t) {
  return t == ScalarType::Float ? RR_TYPE_F32 : t == ScalarType::BFloat16 ? RR_TYPE_BF16 : t == ScalarType::Half ? RR_TYPE_F16
         : t == ScalarType::Char ? RR_TYPE_I8 : -1;
}
bool is_float(ScalarType t) { return t == ScalarType::Float || t == ScalarType::BFloat16 || t == ScalarType::Half; }

const Tensor* tensor(const char* name, PyObject* o) {
  if (!THPVariable_Check(o)) throw BadType(std::string(name) + " must be a torch tensor, not " + Py_TYPE(o)->tp_name);
  const Tensor& t = THPVariable_Unpack(o);
  if (t.requires_grad() && c10::GradMode::is_enabled())
    throw BadValue(std::string(name) + " requires a gradient; these operators are for inference (torch.no_grad())");
  // What the operators would pass by without a word: a tangent, and values that a view's bit says are negated (or zeros).
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined())
    throw BadValue(std::string(name) + " has a forward-mode tangent; these operators are for inference (unpack_dual(...).primal)");
  if (t.is_neg() || t._is_zerotensor())
    throw BadValue(std::string(name) + " is a negated view or has no values of its own; resolve_neg() or clone() it first");
  return &t;
}
void on_gpu(const char* name, const Tensor& t) {
  if (!t.is_cuda() || t.layout() != c10::kStrided)
    throw BadValue(std::string(name) + " is on " + t.device().str() + "; these operators run on the GPU only (dense tensors)");
}
// a floating-point tensor on a GPU
const Tensor* floating(const char* name, PyObject* o) {
  const Tensor* t = tensor(name, o);
  if (!is_float(t->scalar_type()))
    throw BadValue(std::string(name) + " has type " + c10::toString(t->scalar_type()) + "; expected float32, bfloat16 or float16");
  on_gpu(name, *t);
  return t;
}
// a tensor of this type on this device
const Tensor* like(const char* name, PyObject* o, ScalarType type, c10::Device device) {
  const Tensor* t = tensor(name, o);
  if (t->scalar_type() != type)
    throw BadValue(std::string(name) + " has type " + c10::toString(t->scalar_type()) + "; expected " + c10::toString(type));
  on_gpu(name, *t);
  if (t->device() != device) throw BadValue(std::string(name) + " is on " + t->device().str() + "; expected " + device.str());
  return t;
}
void shaped(const char* name, const Tensor& t, at::IntArrayRef want) {
  if (t.sizes() == want) return;
  std::string w = "(";
  for (int64_t d : want) w += std::to_string(d) + ", ";
  throw BadValue(std::string(name) + " has shape " + shape_of(t) + "; expected " + (want.empty() ? "()" : w.substr(0, w.size() - 2) + ")"));
}

// a tensor (..., cols) as evenly spaced rows, without a copy
struct Rows {
  void* p = nullptr;
  int64_t rows = 0, cols = 0, ld = 0;
};
Rows rows_of(const char* name, const Tensor& t) {
  if (t.dim() < 1 || t.size(-1) < 1) throw BadValue(std::string(name) + " has shape " + shape_of(t) + "; expected (..., columns)");
  Rows r{t.data_ptr(), t.numel() / t.size(-1), t.size(-1), t.size(-1)};
  if (t.is_contiguous() || r.rows == 0) return r;
  if (r.cols > 1 && t.stride(-1) != 1)
    throw BadValue(std::string(name) + ": the last dimension must be contiguous (strides " + strides_of(t) + ")");
  // the innermost of the other dimensions that has more than one entry sets the spacing; those outside must continue it
  int64_t expect = -1;
  for (int64_t d = t.dim() - 2; d >= 0; --d) {
    if (t.size(d) == 1) continue;
    if (expect < 0) {
      r.ld = t.stride(d);
      expect = r.ld * t.size(d);
    } else {
      if (t.stride(d) != expect)
        throw BadValue(std::string(name) + ": rows of shape " + shape_of(t) + ", strides " + strides_of(t) + " are not evenly spaced");
      expect *= t.size(d);
    }
  }
  if (r.rows > 1 && r.ld < r.cols) throw BadValue(std::string(name) + ": rows overlap (strides " + strides_of(t) + ")");
  return r;
}

// a vector of n values, made contiguous into `hold` if it is not; null for None
const void* vector_of(const char* name, PyObject* o, ScalarType type, c10::Device device, int64_t n, Tensor& hold) {
  if (o == Py_None) return nullptr;
  const Tensor* t = like(name, o, type, device);
  shaped(name, *t, {n});
  if (t->is_contiguous()) return t->data_ptr();
  hold = t->contiguous();
  return hold.data_ptr();
}

int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
int32_t as_int32(const char* name, int64_t v) {
  if (v < INT32_MIN || v > INT32_MAX) throw BadValue(std::string(name) + " of " + std::to_string(v) + " is out of range");
  return (int32_t)v;
}

at::TensorOptions options(ScalarType type, c10::Device device) { return at::TensorOptions().dtype(type).device(device); }
Tensor scratch(int64_t bytes, c10::Device device) {
  if (bytes < 0) throw Refused{bytes};
  return bytes ? at::empty({bytes}, options(ScalarType::Byte, device)) : Tensor();
}
void* stream_of(c10::Device device) { return c10::hip::getCurrentHIPStream(device.index()).stream(); }
void check(int rc) {
  if (rc != RR_OK) throw Refused{rc};
}

PyObject* wrap(Tensor t) { return t.defined() ? THPVariable_Wrap(std::move(t)) : Py_NewRef(Py_None); }
template <class... T>
PyObject* tuple_of(T... t) {
  PyObject* items[] = {wrap(std::move(t))...};
  PyObject* r = PyTuple_New(sizeof...(T));
  for (size_t i = 0; i < sizeof...(T); ++i) PyTuple_SET_ITEM(r, i, items[i]);
  return r;
}

template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments expected, got %zd", N, n);
    return nullptr;
  }
  if (!p_cross_attention_workspace) {
    PyErr_SetString(PyExc_RuntimeError, "bind() has not been called");
    return nullptr;
  }
  if (torch::jit::tracer::isTracing() ||
      c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value()) {
    PyErr_SetString(PyExc_ValueError, "these operators cannot be traced: a trace would keep their results as constants");
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Refused& e) {
    return PyLong_FromLongLong(e.code);
  } catch (const BadValue& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const BadType& e) {
    PyErr_SetString(PyExc_TypeError, e.what());
  } catch (python_error& e) {
    e.restore();
  } catch (const c10::Error& e) {   // (out of memory among them)
    torch::translate_exception_to_python(std::current_exception());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// (x)
PyObject* quantize_rows(PyObject* const* args) {
  const Tensor& x = *floating("x", args[0]);
  const Rows r = rows_of("x", x);
  const int32_t cols = as_int32("x: a row", r.cols);
  const auto dev = x.device();
  Tensor q = at::empty(x.sizes(), options(ScalarType::Char, dev));
  Tensor s = at::empty(x.sizes().slice(0, x.dim() - 1), options(ScalarType::Float, dev));
  check(p_quantize_rows(dev.index(), stream_of(dev), code_of(x.scalar_type()), r.p, r.ld, r.rows, cols,
                        (int8_t*)q.data_ptr(), r.cols, (float*)s.data_ptr()));
  return tuple_of(q, s);
}

// (x, w, w_scale, x_scale, bias, act, out_dtype)
PyObject* linear_int8(PyObject* const* args) {
  const bool eight = args[3] != Py_None;
  const Tensor& x = eight ? *tensor("x", args[0]) : *floating("x", args[0]);
  const auto dev = x.device();
  if (eight) like("x", args[0], ScalarType::Char, dev);
  ScalarType out_type = eight ? ScalarType::Float : x.scalar_type();
  if (args[6] != Py_None) {
    if (!THPDtype_Check(args[6])) throw BadType("out_dtype must be a torch dtype");
    out_type = reinterpret_cast<THPDtype*>(args[6])->scalar_type;
    if (!is_float(out_type)) throw BadValue("out_dtype must be float32, bfloat16 or float16");
  }
  const Rows xr = rows_of("x", x);
  const Tensor& w = *like("w", args[1], ScalarType::Char, dev);
  if (w.dim() != 2 || w.size(1) != xr.cols)
    throw BadValue("w has shape " + shape_of(w) + "; expected (n, " + std::to_string(xr.cols) + ")");
  const Rows wr = rows_of("w", w);
  Tensor hold[3];
  if (args[2] == Py_None) throw BadType("w_scale must be a torch tensor, not NoneType");
  const void* w_scale = vector_of("w_scale", args[2], ScalarType::Float, dev, wr.rows, hold[0]);
  const void* bias = vector_of("bias", args[4], ScalarType::Float, dev, wr.rows, hold[1]);
  const void* x_scale = nullptr;
  int type = code_of(x.scalar_type());
  if (eight) {
    const Tensor& s = *like("x_scale", args[3], ScalarType::Float, dev);
    shaped("x_scale", s, x.sizes().slice(0, x.dim() - 1));
    hold[2] = s.contiguous();
    x_scale = hold[2].data_ptr();
  }
  const int32_t n = as_int32("w: rows", wr.rows), k = as_int32("x: a row", xr.cols);
  const int64_t need = p_linear_i8_workspace(type, xr.rows, n, k);
  Tensor ws = scratch(need, dev);
  auto sizes = x.sizes().vec();
  sizes.back() = n;
  Tensor out = at::empty(sizes, options(out_type, dev));
  // (no rows: nothing is read, and an empty tensor has no address; the scale's absence would say another type)
  if (xr.rows)
    check(p_linear_i8(dev.index(), stream_of(dev), type, xr.p, xr.ld, (const float*)x_scale, (const int8_t*)wr.p, wr.ld,
                      (const float*)w_scale, (const float*)bias, (int)integer(args[5]), code_of(out_type), out.data_ptr(), n,
                      xr.rows, n, k, ws.defined() ? ws.data_ptr() : nullptr, need));
  return wrap(out);
}

// (y, residual, residual_scale, gate, rows_per_gate, post_norm, post_weight, post_bias, next_norm, next_weight, next_bias, eps,
//  stream, normed, rows8)
PyObject* block_norm(PyObject* const* args) {
  const Tensor& y = *floating("y", args[0]);
  const auto dev = y.device();
  const auto type = y.scalar_type();
  const Rows yr = rows_of("y", y);
  const int32_t cols = as_int32("y: a row", yr.cols);
  Rows xr, gr;
  if (args[1] != Py_None) {
    const Tensor& x = *like("residual", args[1], type, dev);
    shaped("residual", x, y.sizes());
    xr = rows_of("residual", x);
  }
  int64_t per = integer(args[4]);
  if (args[3] != Py_None) {
    const Tensor& g = *like("gate", args[3], type, dev);
    if (g.dim() < 1 || g.dim() > 2 || g.size(-1) != yr.cols)
      throw BadValue("gate has shape " + shape_of(g) + "; expected (" + std::to_string(yr.cols) + ",) or (gate_rows, " +
                     std::to_string(yr.cols) + ")");
    gr = rows_of("gate", g);
    if (gr.rows == 0 && yr.rows) throw BadValue("gate has no rows");   // (and no address, which would say that there is no gate)
    if (g.dim() == 1) per = yr.rows > 1 ? yr.rows : 1;
  }
  Tensor hold[4];
  const void* pw = vector_of("post_weight", args[6], type, dev, yr.cols, hold[0]);
  const void* pb = vector_of("post_bias", args[7], type, dev, yr.cols, hold[1]);
  const void* nw = vector_of("next_weight", args[9], type, dev, yr.cols, hold[2]);
  const void* nb = vector_of("next_bias", args[10], type, dev, yr.cols, hold[3]);
  const bool want_h = args[12] == Py_True, want_o = args[13] == Py_True, want_q = args[14] == Py_True;
  Tensor h, o, q, s;
  if (want_h) h = at::empty(y.sizes(), options(type, dev));
  if (want_o) o = at::empty(y.sizes(), options(type, dev));
  if (want_q) {
    q = at::empty(y.sizes(), options(ScalarType::Char, dev));
    s = at::empty(y.sizes().slice(0, y.dim() - 1), options(ScalarType::Float, dev));
  }
  auto at_ = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
  if (yr.rows)
    check(p_block_norm(dev.index(), stream_of(dev), code_of(type), yr.rows, cols, yr.p, yr.ld, xr.p, xr.ld,
                       (float)number(args[2]), gr.p, gr.ld, gr.rows, per, (int)integer(args[5]), pw, pb,
                       (int)integer(args[8]), nw, nb, (float)number(args[11]), at_(h), cols, at_(o), cols,
                       (int8_t*)at_(q), cols, (float*)at_(s)));
  return tuple_of(h, o, q, s);
}

// (q, k, v, scale, key_lengths, key_mask, q_offsets, k_offsets, max_q, max_k)
PyObject* cross_attention(PyObject* const* args) {
  const Tensor& q = *floating("q", args[0]);
  const auto dev = q.device();
  const auto type = q.scalar_type();
  const Tensor& k = *like("k", args[1], type, dev);
  const Tensor& v = *like("v", args[2], type, dev);
  const bool q_dense = args[6] == Py_None, k_dense = args[7] == Py_None;
  if (q.dim() != (q_dense ? 4 : 3))
    throw BadValue("q has shape " + shape_of(q) + "; expected (batch, queries, heads, d), or (rows, heads, d) with q_offsets");
  if (k.dim() != (k_dense ? 4 : 3))
    throw BadValue("k has shape " + shape_of(k) + "; expected (batch, keys, kv_heads, d), or (rows, kv_heads, d) with k_offsets");
  if (v.sizes() != k.sizes()) throw BadValue("v has shape " + shape_of(v) + ", k " + shape_of(k));
  const int64_t heads = q.size(-2), d = q.size(-1), kv_heads = k.size(-2);
  if (k.size(-1) != d) throw BadValue("q has head size " + std::to_string(d) + ", k " + std::to_string(k.size(-1)));
  const std::pair<const char*, const Tensor*> all[] = {{"q", &q}, {"k", &k}, {"v", &v}};
  for (const auto& [name, t] : all)
    if (t->size(-1) > 1 && t->stride(-1) != 1)
      throw BadValue(std::string(name) + ": the last dimension must be contiguous (strides " + strides_of(*t) + ")");
  const int32_t* offsets[2] = {nullptr, nullptr};
  int64_t batches[2] = {q_dense ? q.size(0) : 0, k_dense ? k.size(0) : 0};
  int64_t longest[2] = {q_dense ? q.size(1) : 0, k_dense ? k.size(1) : 0};
  for (int i = 0; i < 2; ++i) {
    PyObject* o = args[6 + i];
    if (o == Py_None) continue;
    const char* name = i ? "k_offsets" : "q_offsets";
    const Tensor& t = *like(name, o, ScalarType::Int, dev);
    if (t.dim() != 1 || t.size(0) < 1 || !t.is_contiguous())
      throw BadValue(std::string(name) + " must be a contiguous vector of batch + 1 row numbers");
    if (args[8 + i] == Py_None || (longest[i] = integer(args[8 + i])) < 0)
      throw BadValue(std::string(name) + " goes with max_q / max_k, the longest sequence");
    offsets[i] = t.data_ptr<int32_t>();
    batches[i] = t.size(0) - 1;
  }
  if (batches[0] != batches[1]) throw BadValue("queries and keys have different batch sizes");
  const int64_t batch = batches[0];
  Tensor hold[2];
  const void* lengths = vector_of("key_lengths", args[4], ScalarType::Int, dev, batch, hold[0]);
  const uint8_t* mask = nullptr;
  int64_t mask_stride = 0;
  if (args[5] != Py_None) {
    if (!k_dense) throw BadValue("key_mask goes with dense keys");
    const Tensor* m = tensor("key_mask", args[5]);
    if (m->scalar_type() != ScalarType::Bool) m = like("key_mask", args[5], ScalarType::Byte, dev);
    else m = like("key_mask", args[5], ScalarType::Bool, dev);
    shaped("key_mask", *m, {batch, longest[1]});
    if ((longest[1] > 1 && m->stride(1) != 1) || (batch > 1 && m->stride(0) < longest[1])) {
      hold[1] = m->contiguous();
      m = &hold[1];
    }
    mask = static_cast<const uint8_t*>(m->data_ptr());
    mask_stride = batch > 1 ? m->stride(0) : longest[1];
  }
  const double scale = args[3] == Py_None ? 1.0 / std::sqrt((double)d) : number(args[3]);
  const int code = code_of(type);
  const int32_t b32 = as_int32("batch", batch), h32 = as_int32("heads", heads), kv32 = as_int32("kv_heads", kv_heads),
                d32 = as_int32("head size", d), mq = as_int32("max_q", longest[0]), mk = as_int32("max_k", longest[1]);
  const int64_t need = p_cross_attention_workspace(code, b32, h32, kv32, d32, mq, mk);
  Tensor ws = scratch(need, dev);
  Tensor out = at::empty(q.sizes(), options(type, dev));
  auto s = [](const Tensor& t, bool dense, int i) { return dense ? t.stride(i) : i ? t.stride(i - 1) : 0; };
  check(p_cross_attention(dev.index(), stream_of(dev), code, q.data_ptr(), s(q, q_dense, 0), s(q, q_dense, 1),
                          s(q, q_dense, 2), k.data_ptr(), s(k, k_dense, 0), s(k, k_dense, 1), s(k, k_dense, 2),
                          v.data_ptr(), s(v, k_dense, 0), s(v, k_dense, 1), s(v, k_dense, 2), out.data_ptr(),
                          s(out, q_dense, 0), s(out, q_dense, 1), s(out, q_dense, 2), b32, h32, kv32, d32, mq, mk,
                          q_dense ? 0 : q.size(0), k_dense ? 0 : k.size(0), offsets[0], offsets[1],
                          (const int32_t*)lengths, mask, mask_stride, (float)scale,
                          ws.defined() ? ws.data_ptr() : nullptr, need));
  return wrap(out);
}

// bind(path): looks the C-ABI up in the library at `path`, which is loaded already
PyObject* bind(PyObject*, PyObject* path) {
  const char* at = PyUnicode_AsUTF8(path);
  if (!at) return nullptr;
  void* lib = dlopen(at, RTLD_NOW | RTLD_NOLOAD);
  if (!lib) return PyErr_Format(PyExc_RuntimeError, "%s is not loaded", at);
  auto find = [&](auto& f, const char* name) {
    f = reinterpret_cast<std::decay_t<decltype(f)>>(dlsym(lib, name));
    if (!f) PyErr_Format(PyExc_RuntimeError, "%s has no %s", at, name);
    return f != nullptr;
  };
  if (!find(p_quantize_rows, "rr_quantize_rows") || !find(p_linear_i8, "rr_linear_i8") ||
      !find(p_linear_i8_workspace, "rr_linear_i8_workspace") || !find(p_block_norm, "rr_block_norm") ||
      !find(p_cross_attention, "rr_cross_attention") ||
      !find(p_cross_attention_workspace, "rr_cross_attention_workspace"))
    return nullptr;
  Py_RETURN_NONE;
}

#define FAST(f, n) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<f, n>)), METH_FASTCALL
PyMethodDef methods[] = {
    {"quantize_rows", FAST(quantize_rows, 1), nullptr},     {"linear_int8", FAST(linear_int8, 7), nullptr},
    {"block_norm", FAST(block_norm, 15), nullptr},          {"cross_attention", FAST(cross_attention, 10), nullptr},
    {"bind", bind, METH_O, nullptr},                        {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_ops", "torch side of rag_service_amd.ops", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_ops(void) { return PyModule_Create(&module); }
