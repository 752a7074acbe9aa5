// torch_binding.cpp -- the layer operators' host side for torch tensors: checks the
// arguments, allocates the outputs on the current stream and calls the C ABI.
//
// The operators' kernels take 3 to 20 us on a decode step's sizes, about as long as a
// Python wrapper spends on checks, allocations and ctypes (norm of one token: 16 us,
// of which the launch is 5); here that is done in C++ (see fused.py for the Python
// side).  Functions return (status, tensors...); a refused argument raises
// ValueError or TypeError.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>
#include <string>

#include "../../include/qgemm.h"

namespace {

struct Refusal {
  PyObject* type;
  std::string what;
};
[[noreturn]] void refuse_value(const std::string& s) { throw Refusal{PyExc_ValueError, s}; }
[[noreturn]] void refuse_type(const std::string& s) { throw Refusal{PyExc_TypeError, s}; }

const at::Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) refuse_type(std::string(what) + " must be a tensor");
  return THPVariable_Unpack(o);
}
const at::Tensor* optional_tensor(PyObject* o, const char* what) {
  return o == Py_None ? nullptr : &tensor(o, what);
}
int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse_type("expected an integer");
  }
  return v;
}
// A layout as the C ABI's int (which of them an operator takes is the ABI's to say).
int layout_code(PyObject* o) {
  const int64_t v = integer(o);
  if (v != static_cast<int>(v)) refuse_value("unknown layout " + std::to_string(v));
  return static_cast<int>(v);
}
double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse_type("expected a number");
  }
  return v;
}
bool flag(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) {
    PyErr_Clear();
    refuse_type("expected a truth value");
  }
  return v == 1;
}

int dtype_code(const at::Tensor& t, const char* what) {
  if (t.scalar_type() == at::kFloat) return QG_DTYPE_F32;
  if (t.scalar_type() == at::kBFloat16) return QG_DTYPE_BF16;
  refuse_type(std::string(what) + ": unsupported dtype; use float32 or bfloat16");
}

c10::Device cuda_matrix(const at::Tensor& t, const char* what) {
  if (t.dim() != 2 || !t.is_cuda())
    refuse_value(std::string(what) + " must be a 2-D CUDA tensor");
  return t.device();
}

// Checks a matrix and returns its row stride (arbitrary in torch for a single row).
int64_t matrix(const at::Tensor& t, const char* what, int64_t rows, int64_t cols, c10::Device dev) {
  if (t.dim() != 2 || t.size(0) != rows || t.size(1) != cols)
    refuse_value(std::string(what) + " must be " + std::to_string(rows) + " x " +
                 std::to_string(cols));
  if (t.device() != dev || (t.stride(1) != 1 && cols > 1))
    refuse_value(std::string(what) + " must be on " + dev.str() + " with unit column stride");
  return rows > 1 ? t.stride(0) : cols;
}
void same_type(const at::Tensor& t, const char* what, const at::Tensor& as) {
  if (t.scalar_type() != as.scalar_type())
    refuse_type(std::string(what) + " must have the dtype of the matrix that it goes with");
}
void vec(const at::Tensor& t, const char* what, int64_t n, c10::Device dev) {
  if (t.dim() != 1 || t.size(0) != n || t.device() != dev || (n > 1 && t.stride(0) != 1))
    refuse_value(std::string(what) + " must be a contiguous vector of " + std::to_string(n) +
                 " values on " + dev.str());
}

int64_t scale_bytes(int64_t rows, int64_t k, int sv, int layout) {
  return layout == QG_LAYOUT_REF_LINEAR ? rows * (k / sv) : qg_scale_bytes(rows, k, sv);
}

// A quantised operand's buffers against its shape.  format: qg_format.
c10::Device held(const at::Tensor& q, const at::Tensor& sf, int64_t rows, int64_t k, int layout,
                 int format, const char* what) {
  int64_t values = 0;
  // 2^48 values: no device holds them, and nothing below can wrap round.
  if (__builtin_mul_overflow(rows, k, &values) || values > int64_t{1} << 48)
    refuse_value(std::string(what) + ": buffers are smaller than the shape needs");
  if (format != QG_FORMAT_MXFP8) values /= 2;
  const int sv = format == QG_FORMAT_NVFP4 ? 16 : 32;
  if (rows < 0 || k < 0 || q.numel() < values || sf.numel() < scale_bytes(rows, k, sv, layout))
    refuse_value(std::string(what) + ": buffers are smaller than the shape needs");
  if (!q.is_contiguous() || !sf.is_contiguous())
    refuse_value(std::string(what) + ": buffers must be contiguous");
  if (q.scalar_type() != at::kByte || sf.scalar_type() != at::kByte)
    refuse_type(std::string(what) + ": buffers must be uint8");
  if (!q.is_cuda() || sf.device() != q.device())
    refuse_value(std::string(what) + ": buffers must be on one CUDA device");
  return q.device();
}

at::Tensor empty(at::IntArrayRef size, at::ScalarType type, c10::Device dev) {
  return at::Tensor(at::detail::empty_cuda(size, type, dev, std::nullopt));
}

// The device of the call made current, and its current stream.
struct Here {
  c10::cuda::OptionalCUDAGuard guard;
  qg_stream_t stream;
  explicit Here(c10::Device dev) {
    if (dev.index() != c10::cuda::current_device()) guard.set_device(dev);
    stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  }
};

void* ptr(const at::Tensor& t) { return t.data_ptr(); }
void* ptr(const at::Tensor* t) { return t ? t->data_ptr() : nullptr; }

// (status, tensors...); an undefined tensor becomes None.
template <typename... T>
PyObject* result(int rc, T&&... t) {
  PyObject* r = PyTuple_New(1 + sizeof...(T));
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, PyLong_FromLong(rc));
  Py_ssize_t i = 1;
  auto put = [&](at::Tensor&& x) {
    if (x.defined()) {
      PyTuple_SET_ITEM(r, i++, THPVariable_Wrap(std::move(x)));
    } else {
      Py_INCREF(Py_None);
      PyTuple_SET_ITEM(r, i++, Py_None);
    }
  };
  (put(std::forward<T>(t)), ...);
  return r;
}

template <typename F>
PyObject* guarded(Py_ssize_t got, Py_ssize_t want, F&& body) {
  if (got != want) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  HANDLE_TH_ERRORS  // torch's exceptions as torch's Python errors (OutOfMemoryError)
  try {
    return body();
  } catch (const Refusal& r) {
    PyErr_SetString(r.type, r.what.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// x, weight, residual | None, eps, layout, h | None -> status, q, sf, h | None, rstd
PyObject* rmsnorm_mxfp8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 6, [&] {
    const at::Tensor& x = tensor(a[0], "x");
    const at::Tensor& w = tensor(a[1], "weight");
    const at::Tensor* res = optional_tensor(a[2], "residual");
    const float eps = static_cast<float>(real(a[3]));
    const int layout = layout_code(a[4]);
    const at::Tensor* h_in = optional_tensor(a[5], "h");
    const c10::Device dev = cuda_matrix(x, "x");
    const int64_t rows = x.size(0), k = x.size(1);
    const int code = dtype_code(x, "x"), w_code = dtype_code(w, "weight");
    const int64_t ldx = matrix(x, "x", rows, k, dev);
    vec(w, "weight", k, dev);
    int64_t ldr = 0, ldh = 0;
    if (res) {
      same_type(*res, "residual", x);
      ldr = matrix(*res, "residual", rows, k, dev);
    }
    if (h_in) {
      same_type(*h_in, "h", x);
      ldh = matrix(*h_in, "h", rows, k, dev);
    }
    Here here(dev);
    at::Tensor q = empty({rows * k}, at::kByte, dev);
    at::Tensor sf = empty({scale_bytes(rows, k, 32, layout)}, at::kByte, dev);
    at::Tensor rstd = empty({rows}, at::kFloat, dev), h;
    if (!h_in && res) {
      h = empty({rows, k}, x.scalar_type(), dev);
      ldh = k;
    }
    const int rc = qg_rmsnorm_mxfp8(ptr(x), code, ldx, ptr(res), ldr, ptr(w), w_code, eps, rows, k,
                                    layout, ptr(q), ptr(sf), h.defined() ? ptr(h) : ptr(h_in), ldh,
                                    static_cast<float*>(ptr(rstd)), here.stream);
    return result(rc, std::move(q), std::move(sf), std::move(h), std::move(rstd));
  });
}

// dy, h, rstd, weight, dres | None, want dweight -> status, dx, dweight | None
PyObject* rmsnorm_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 6, [&] {
    const at::Tensor& dy = tensor(a[0], "dy");
    const at::Tensor& h = tensor(a[1], "h");
    const at::Tensor& rstd = tensor(a[2], "rstd");
    const at::Tensor& w = tensor(a[3], "weight");
    const at::Tensor* dres = optional_tensor(a[4], "dres");
    const c10::Device dev = cuda_matrix(h, "h");
    const int64_t rows = h.size(0), k = h.size(1);
    const int code = dtype_code(h, "h"), w_code = dtype_code(w, "weight");
    const int64_t ldh = matrix(h, "h", rows, k, dev), lddy = matrix(dy, "dy", rows, k, dev);
    same_type(dy, "dy", h);
    vec(rstd, "rstd", rows, dev);
    vec(w, "weight", k, dev);
    if (rstd.scalar_type() != at::kFloat) refuse_type("rstd must be float32");
    int64_t ldr = 0;
    if (dres) {
      same_type(*dres, "dres", h);
      ldr = matrix(*dres, "dres", rows, k, dev);
    }
    Here here(dev);
    at::Tensor dx = empty({rows, k}, h.scalar_type(), dev), dw, ws;
    int64_t need = 0;
    if (flag(a[5])) {
      dw = empty({k}, at::kFloat, dev);
      need = static_cast<int64_t>(qg_rmsnorm_backward_workspace_bytes(rows, k));
      if (need) ws = empty({need}, at::kByte, dev);
    }
    const int rc = qg_rmsnorm_backward(
        ptr(dy), lddy, ptr(h), ldh, code, static_cast<float*>(ptr(rstd)), ptr(w), w_code, ptr(dres),
        ldr, rows, k, ptr(dx), k, dw.defined() ? static_cast<float*>(ptr(dw)) : nullptr,
        ws.defined() ? ptr(ws) : nullptr, static_cast<size_t>(need), here.stream);
    return result(rc, std::move(dx), std::move(dw));
  });
}

// format, a (q, sf, ts | None, rows), b (the same), k, sf_layout, bias | None, act,
// residual | None, out dtype, out | None, out_layout, checkpoint, ckpt_layout,
// status | None -> status, out, out_sf | None, ckpt q | None, ckpt sf | None
PyObject* gemm_fused(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 20, [&] {
    const int format = static_cast<int>(integer(a[0]));
    const at::Tensor& aq = tensor(a[1], "a");
    const at::Tensor& asf = tensor(a[2], "a");
    const at::Tensor* ats = optional_tensor(a[3], "a");
    const int64_t m = integer(a[4]);
    const at::Tensor& bq = tensor(a[5], "b");
    const at::Tensor& bsf = tensor(a[6], "b");
    const at::Tensor* bts = optional_tensor(a[7], "b");
    const int64_t nn = integer(a[8]), k = integer(a[9]);
    const int sf_layout = layout_code(a[10]);
    const at::Tensor* bias = optional_tensor(a[11], "bias");
    const int act = static_cast<int>(integer(a[12]));
    const at::Tensor* res = optional_tensor(a[13], "residual");
    const int out_dtype = static_cast<int>(integer(a[14]));
    const at::Tensor* out_in = optional_tensor(a[15], "out");
    const int out_layout = layout_code(a[16]);
    const bool ckpt = flag(a[17]);
    const int ckpt_layout = layout_code(a[18]);
    const at::Tensor* status = optional_tensor(a[19], "status");
    const c10::Device dev = held(aq, asf, m, k, sf_layout, format, "a");
    if (held(bq, bsf, nn, k, sf_layout, format, "b") != dev)
      refuse_value("operands must be on one device");
    for (const at::Tensor* ts : {ats, bts})
      if (format == QG_FORMAT_NVFP4 && ts &&
          (ts->device() != dev || ts->scalar_type() != at::kFloat || ts->numel() < 1))
        refuse_value("tensor scales must be float32 on " + dev.str());
    const int64_t cols = act == QG_ACT_SWIGLU ? nn / 2 : nn;
    qg_epilogue e{};
    e.act = act;
    if (bias) {
      vec(*bias, "bias", nn, dev);
      e.bias = ptr(bias);
      e.bias_dtype = dtype_code(*bias, "bias");
    }
    if (res) {
      e.ldr = matrix(*res, "residual", m, cols, dev);
      e.residual = ptr(res);
      e.residual_dtype = dtype_code(*res, "residual");
    }
    if (status &&
        (status->device() != dev || status->numel() < 1 || status->element_size() != 4))
      refuse_value("status must be a 32-bit word on " + dev.str());
    Here here(dev);
    at::Tensor out, out_sf, zq, zsf;
    e.out_dtype = out_dtype;
    if (out_in) {
      e.ldc = matrix(*out_in, "out", m, cols, dev);
      e.out_dtype = dtype_code(*out_in, "out");
      e.out = ptr(out_in);
    } else if (out_dtype == QG_DTYPE_MXFP8) {
      out = empty({m * cols}, at::kByte, dev);
      out_sf = empty({scale_bytes(m, cols, 32, out_layout)}, at::kByte, dev);
      e.out = ptr(out);
      e.out_sf = ptr(out_sf);
      e.out_layout = out_layout;
    } else {
      out = empty({m, cols}, out_dtype == QG_DTYPE_BF16 ? at::kBFloat16 : at::kFloat, dev);
      e.out = ptr(out);
      e.ldc = cols;
    }
    if (ckpt) {
      zq = empty({m * nn}, at::kByte, dev);
      zsf = empty({scale_bytes(m, nn, 32, ckpt_layout)}, at::kByte, dev);
      e.ckpt_q = ptr(zq);
      e.ckpt_sf = ptr(zsf);
      e.ckpt_layout = ckpt_layout;
    }
    const int rc = qg_gemm_fused(format, ptr(aq), ptr(asf), static_cast<float*>(ptr(ats)), ptr(bq),
                                 ptr(bsf), static_cast<float*>(ptr(bts)), m, nn, k, sf_layout, &e,
                                 static_cast<uint32_t*>(ptr(status)), here.stream);
    return result(rc, std::move(out), std::move(out_sf), std::move(zq), std::move(zsf));
  });
}

// dout, z (q, sf, or both None), z rows, z columns, z_layout, act, layout, want dbias
// -> status, dz q, dz sf, dzt q, dzt sf, dbias | None
PyObject* act_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 9, [&] {
    const at::Tensor& d = tensor(a[0], "dout");
    const bool z = a[1] != Py_None || a[2] != Py_None;
    const at::Tensor* zq = z ? &tensor(a[1], "checkpoint") : nullptr;
    const at::Tensor* zsf = z ? &tensor(a[2], "checkpoint") : nullptr;
    const int z_layout = layout_code(a[5]);
    const int act = static_cast<int>(integer(a[6])), layout = layout_code(a[7]);
    const c10::Device dev = cuda_matrix(d, "dout");
    const int64_t m = d.size(0), cols = d.size(1), nn = act == QG_ACT_SWIGLU ? 2 * cols : cols;
    const int code = dtype_code(d, "dout");
    if (z && (integer(a[3]) != m || integer(a[4]) != nn ||
               held(*zq, *zsf, m, nn, z_layout, QG_FORMAT_MXFP8, "checkpoint") != dev))
      refuse_value("checkpoint must be " + std::to_string(m) + " x " + std::to_string(nn) +
                   " on the device of dout");
    const int64_t ldd = matrix(d, "dout", m, cols, dev);
    Here here(dev);
    const int64_t mt = (m + 31) / 32 * 32;
    at::Tensor dz = empty({m * nn}, at::kByte, dev), dzt = empty({nn * mt}, at::kByte, dev);
    at::Tensor dz_sf = empty({scale_bytes(m, nn, 32, layout)}, at::kByte, dev);
    at::Tensor dzt_sf = empty({scale_bytes(nn, mt, 32, layout)}, at::kByte, dev);
    at::Tensor db, ws;
    int64_t need = 0;
    if (flag(a[8])) {
      db = empty({nn}, at::kFloat, dev);
      need = static_cast<int64_t>(qg_act_backward_workspace_bytes(m, nn));
      if (need) ws = empty({need}, at::kByte, dev);
    }
    const int rc = qg_act_backward_mxfp8(
        ptr(d), code, ldd, ptr(zq), ptr(zsf), z_layout, act, m, nn, ptr(dz), ptr(dz_sf), ptr(dzt),
        ptr(dzt_sf), layout, db.defined() ? static_cast<float*>(ptr(db)) : nullptr,
        ws.defined() ? ptr(ws) : nullptr, static_cast<size_t>(need), here.stream);
    return result(rc, std::move(dz), std::move(dz_sf), std::move(dzt), std::move(dzt_sf),
                  std::move(db));
  });
}

// q, sf, rows, k, layout, out layout -> status, tq, tsf
PyObject* transpose_mxfp8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 6, [&] {
    const at::Tensor& q = tensor(a[0], "a");
    const at::Tensor& sf = tensor(a[1], "a");
    const int64_t rows = integer(a[2]), k = integer(a[3]);
    const int layout = layout_code(a[4]), to = layout_code(a[5]);
    const c10::Device dev = held(q, sf, rows, k, layout, QG_FORMAT_MXFP8, "a");
    Here here(dev);
    const int64_t rt = (rows + 31) / 32 * 32;
    at::Tensor tq = empty({k * rt}, at::kByte, dev);
    at::Tensor tsf = empty({scale_bytes(k, rt, 32, to)}, at::kByte, dev);
    const int rc = qg_transpose_mxfp8(ptr(q), ptr(sf), layout, rows, k, ptr(tq), ptr(tsf), to,
                                      here.stream);
    return result(rc, std::move(tq), std::move(tsf));
  });
}

#define QG_METHOD(f) \
  {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {QG_METHOD(rmsnorm_mxfp8), QG_METHOD(rmsnorm_backward),
                         QG_METHOD(gemm_fused), QG_METHOD(act_backward),
                         QG_METHOD(transpose_mxfp8), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() { return PyModule_Create(&module); }
