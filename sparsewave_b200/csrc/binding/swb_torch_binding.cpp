// The device-tensor operator calls of the Python layer, natively: reads the operands of torch tensors, keeps parsed
// option text, takes torch's current stream and calls the C ABI.
//
// A small operator is bound by what the host does per call.  The same steps through Python attribute calls and ctypes
// (five operands x four attributes, option parsing, a stream object) took 11 us a call against 2.8 us of GPU time for
// a 4096 x 4096 SpMV.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>
#include <unordered_map>
#include <vector>

#include "../../../include/sparsewave_b200.h"

namespace {

PyObject *g_error = nullptr;         // SparseWaveError(status, message)
PyTypeObject *g_options = nullptr;   // ctypes SwbOptions

struct Failed {};  // a Python exception is set

[[noreturn]] void raise_status(int status, const char *message) {
  PyObject *e = PyObject_CallFunction(g_error, "is", status, message ? message : "");
  if (e) {
    PyErr_SetObject(g_error, e);
    Py_DECREF(e);
  }
  throw Failed();
}

[[noreturn]] void raise_type(const char *name, const char *what) {
  PyErr_Format(PyExc_TypeError, "%s %s", name, what);
  throw Failed();
}

// Parsed option texts.  The GIL guards the table; a program uses a handful of texts, and the table starts over at 256.
const swb_options &parsed(const char *text, Py_ssize_t length) {
  static std::unordered_map<std::string, swb_options> table;
  std::string key(text, (size_t)length);
  auto it = table.find(key);
  if (it != table.end()) return it->second;
  swb_options o;
  swb_options_default(&o);
  const int st = swb_options_parse(nullptr, &o, key.c_str());
  if (st != SWB_OK) raise_status(st, swb_last_error(nullptr));
  if (table.size() >= 256) table.clear();
  return table.emplace(std::move(key), o).first->second;
}

// A copy: the caller's block may change and the table may move while the GIL is released.
swb_options options_of(PyObject *obj) {
  if (PyUnicode_Check(obj)) {
    Py_ssize_t n = 0;
    const char *s = PyUnicode_AsUTF8AndSize(obj, &n);
    if (!s) throw Failed();
    return parsed(s, n);
  }
  if (Py_TYPE(obj) == g_options || PyType_IsSubtype(Py_TYPE(obj), g_options)) {
    Py_buffer view;
    if (PyObject_GetBuffer(obj, &view, PyBUF_SIMPLE) != 0) throw Failed();
    swb_options o;
    const bool fits = view.len == (Py_ssize_t)sizeof o;
    if (fits) memcpy(&o, view.buf, sizeof o);
    PyBuffer_Release(&view);
    if (fits) return o;
  }
  const int truth = PyObject_IsTrue(obj);
  if (truth < 0) throw Failed();
  if (!truth) return parsed("", 0);  // None and other empty values: the defaults
  PyErr_SetString(PyExc_TypeError, "options must be a string in the reference's spelling or an SwbOptions");
  throw Failed();
}

const at::Tensor &tensor(PyObject *obj, const char *name) {
  if (!THPVariable_Check(obj)) raise_type(name, "must be a CUDA tensor");
  return THPVariable_Unpack(obj);
}

void *device_pointer(const at::Tensor &t, at::ScalarType dtype, const char *name) {
  if (!t.is_cuda()) raise_type(name, "must be a CUDA tensor");
  if (t.scalar_type() != dtype) {
    PyErr_Format(PyExc_TypeError, "%s must have dtype %S, got %S", name, (PyObject *)torch::getTHPDtype(dtype),
                 (PyObject *)torch::getTHPDtype(t.scalar_type()));
    throw Failed();
  }
  if (!t.is_contiguous()) raise_type(name, "must be contiguous");
  return t.data_ptr();
}

void *device_pointer(PyObject *obj, at::ScalarType dtype, const char *name) {
  return device_pointer(tensor(obj, name), dtype, name);
}

int64_t integer(PyObject *obj) {
  const long long v = PyLong_AsLongLong(obj);
  if (v == -1 && PyErr_Occurred()) throw Failed();
  return v;
}

swb_context *context_of(PyObject *obj) {
  if (obj == Py_None) return nullptr;  // a closed context: the library refuses it
  void *p = PyLong_AsVoidPtr(obj);
  if (!p && PyErr_Occurred()) throw Failed();
  return static_cast<swb_context *>(p);
}

void *stream_of(PyObject *device) {
  return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)integer(device)).stream();
}

at::Tensor output(PyObject *given, at::IntArrayRef sizes, at::ScalarType dtype, const at::Tensor &like) {
  if (given != Py_None) return at::Tensor();
  return at::empty(sizes, at::TensorOptions().dtype(dtype).device(like.device()));
}

// Runs `call` without the GIL, turns its status into an exception, returns the output object.
template <typename Call>
PyObject *finish(swb_context *ctx, PyObject *given, at::Tensor &fresh, Call call) {
  int st;
  Py_BEGIN_ALLOW_THREADS
  st = call();
  Py_END_ALLOW_THREADS
  if (st != SWB_OK) raise_status(st, swb_last_error(ctx));
  if (given != Py_None) {
    Py_INCREF(given);
    return given;
  }
  return THPVariable_Wrap(std::move(fresh));
}

template <typename Body>
PyObject *guarded(Py_ssize_t have, Py_ssize_t want, Body body) {
  if (have != want) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, have);
    return nullptr;
  }
  try {
    return body();
  } catch (const Failed &) {
    return nullptr;
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

void require_rank(const at::Tensor &t, int64_t rank, const char *name) {
  if (t.dim() < rank) {
    PyErr_Format(PyExc_IndexError, "%s must have %d dimensions", name, (int)rank);
    throw Failed();
  }
}

// spmv(ctx, device, options, row_ptr, col_idx, val, x, y | None, rows | None)
PyObject *spmv(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded(n, 9, [&]() -> PyObject * {
    swb_context *ctx = context_of(a[0]);
    const swb_options o = options_of(a[2]);
    const at::Tensor &rp = tensor(a[3], "row_ptr"), &val = tensor(a[5], "val"), &x = tensor(a[6], "x");
    const int64_t rows = a[8] == Py_None ? rp.numel() - 1 : integer(a[8]), cols = x.numel(), nnz = val.numel();
    auto *p_rp = (const int32_t *)device_pointer(rp, at::kInt, "row_ptr");
    auto *p_ci = (const int32_t *)device_pointer(a[4], at::kInt, "col_idx");
    auto *p_v = (const float *)device_pointer(val, at::kFloat, "val");
    auto *p_x = (const float *)device_pointer(x, at::kFloat, "x");
    at::Tensor fresh = output(a[7], {rows}, at::kFloat, x);
    auto *p_y = (float *)(fresh.defined() ? fresh.data_ptr() : device_pointer(a[7], at::kFloat, "y"));
    void *s = stream_of(a[1]);
    return finish(ctx, a[7], fresh, [&] { return swb_spmv(ctx, &o, rows, cols, nnz, p_rp, p_ci, p_v, p_x, p_y, s); });
  });
}

// coo_spmv(ctx, device, options, rows, row_idx, col_idx, val, x, y | None)
PyObject *coo_spmv(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded(n, 9, [&]() -> PyObject * {
    swb_context *ctx = context_of(a[0]);
    const swb_options o = options_of(a[2]);
    const int64_t rows = integer(a[3]);
    const at::Tensor &val = tensor(a[6], "val"), &x = tensor(a[7], "x");
    const int64_t cols = x.numel(), nnz = val.numel();
    auto *p_ri = (const int32_t *)device_pointer(a[4], at::kInt, "row_idx");
    auto *p_ci = (const int32_t *)device_pointer(a[5], at::kInt, "col_idx");
    auto *p_v = (const float *)device_pointer(val, at::kFloat, "val");
    auto *p_x = (const float *)device_pointer(x, at::kFloat, "x");
    at::Tensor fresh = output(a[8], {rows}, at::kFloat, x);
    auto *p_y = (float *)(fresh.defined() ? fresh.data_ptr() : device_pointer(a[8], at::kFloat, "y"));
    void *s = stream_of(a[1]);
    return finish(ctx, a[8], fresh,
                  [&] { return swb_coo_spmv(ctx, &o, rows, cols, nnz, p_ri, p_ci, p_v, p_x, p_y, s); });
  });
}

// spmm(ctx, device, options, row_ptr, col_idx, val, B, C | None, rows | None)
PyObject *spmm(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded(n, 9, [&]() -> PyObject * {
    swb_context *ctx = context_of(a[0]);
    const swb_options o = options_of(a[2]);
    const at::Tensor &rp = tensor(a[3], "row_ptr"), &val = tensor(a[5], "val"), &B = tensor(a[6], "B");
    require_rank(B, 2, "B");
    const int64_t rows = a[8] == Py_None ? rp.numel() - 1 : integer(a[8]), cols = B.size(0), rhs = B.size(1),
                  nnz = val.numel();
    auto *p_rp = (const int32_t *)device_pointer(rp, at::kInt, "row_ptr");
    auto *p_ci = (const int32_t *)device_pointer(a[4], at::kInt, "col_idx");
    auto *p_v = (const float *)device_pointer(val, at::kFloat, "val");
    auto *p_B = (const float *)device_pointer(B, at::kFloat, "B");
    at::Tensor fresh = output(a[7], {rows, rhs}, at::kFloat, B);
    auto *p_C = (float *)(fresh.defined() ? fresh.data_ptr() : device_pointer(a[7], at::kFloat, "C"));
    void *s = stream_of(a[1]);
    return finish(ctx, a[7], fresh,
                  [&] { return swb_spmm(ctx, &o, rows, cols, nnz, rhs, p_rp, p_ci, p_v, p_B, p_C, s); });
  });
}

// bsr_spmm(ctx, device, options, block_row_ptr, block_col_idx, block_values, B, block_size, C | None)
PyObject *bsr_spmm(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded(n, 9, [&]() -> PyObject * {
    swb_context *ctx = context_of(a[0]);
    const swb_options o = options_of(a[2]);
    const at::Tensor &brp = tensor(a[3], "block_row_ptr"), &bci = tensor(a[4], "block_col_idx"),
                     &bv = tensor(a[5], "block_values"), &B = tensor(a[6], "B");
    require_rank(B, 2, "B");
    const int64_t bs = integer(a[7]), rows = (brp.numel() - 1) * bs, cols = B.size(0), rhs = B.size(1),
                  nnzb = bci.numel();
    const at::ScalarType dt = bv.scalar_type();
    if (dt != at::kFloat && dt != at::kBFloat16) raise_type("block_values", "must be float32 or bfloat16");
    if (bv.numel() != nnzb * bs * bs) {
      const std::string message =
          "block values size must equal the number of blocks times block_size squared, but got " +
          std::to_string(bv.numel()) + " and " + std::to_string(nnzb) + " blocks";
      raise_status(SWB_ERR_INVALID_SHAPE, message.c_str());
    }
    auto *p_rp = (const int32_t *)device_pointer(brp, at::kInt, "block_row_ptr");
    auto *p_ci = (const int32_t *)device_pointer(bci, at::kInt, "block_col_idx");
    void *p_v = device_pointer(bv, dt, "block_values"), *p_B = device_pointer(B, dt, "B");
    at::Tensor fresh = output(a[8], {rows, rhs}, dt, B);
    void *p_C = fresh.defined() ? fresh.data_ptr() : device_pointer(a[8], dt, "C");
    void *s = stream_of(a[1]);
    return finish(ctx, a[8], fresh, [&] {
      return dt == at::kFloat ? swb_bsr_spmm_f32(ctx, &o, rows, cols, nnzb, bs, rhs, p_rp, p_ci, (const float *)p_v,
                                                 (const float *)p_B, (float *)p_C, s)
                              : swb_bsr_spmm_bf16(ctx, &o, rows, cols, nnzb, bs, rhs, p_rp, p_ci, (const uint16_t *)p_v,
                                                  (const uint16_t *)p_B, (uint16_t *)p_C, s);
    });
  });
}

// ---- products grouped by expert, 8-bit operands ------------------------------------------------------------------------

[[noreturn]] void raise_shape(const std::string &message) { raise_status(SWB_ERR_INVALID_SHAPE, message.c_str()); }

// A tensor of `rank` dimensions on the context's device.
const at::Tensor &operand(PyObject *obj, int64_t rank, int64_t device, const char *name) {
  const at::Tensor &t = tensor(obj, name);
  if (!t.is_cuda()) raise_type(name, "must be a CUDA tensor");
  if (t.get_device() != device) raise_type(name, "must be on the context's device");
  if (t.dim() != rank)
    raise_shape(std::string(name) + " must have " + std::to_string(rank) + " dimensions, but got " + std::to_string(t.dim()));
  return t;
}

void require_sizes(const at::Tensor &t, at::IntArrayRef sizes, const char *name) {
  if (t.sizes() == sizes) return;
  std::string want, got;
  for (int64_t s : sizes) want += (want.empty() ? "" : " x ") + std::to_string(s);
  for (int64_t s : t.sizes()) got += (got.empty() ? "" : " x ") + std::to_string(s);
  raise_shape(std::string(name) + " must be " + want + ", but got " + got);
}

enum class Types { k16Bits, k16BitsOrF32, kFp8 };

int type_code(const at::Tensor &t, const char *name, Types allowed) {
  const bool fp8 = allowed == Types::kFp8;
  switch (t.scalar_type()) {
    case at::kBFloat16: if (!fp8) return SWB_BF16; break;
    case at::kHalf: if (!fp8) return SWB_F16; break;
    case at::kFloat: if (allowed == Types::k16BitsOrF32) return SWB_F32; break;
    case at::kFloat8_e4m3fn: if (fp8) return SWB_E4M3; break;
    case at::kFloat8_e5m2: if (fp8) return SWB_E5M2; break;
    default: break;
  }
  raise_type(name, fp8                           ? "must be float8_e4m3fn or float8_e5m2"
                   : allowed == Types::k16Bits ? "must be bfloat16 or float16"
                                                 : "must be bfloat16, float16 or float32");
}

bool truth(PyObject *obj) {
  const int t = PyObject_IsTrue(obj);
  if (t < 0) throw Failed();
  return t != 0;
}

// The output that the caller gave, checked, or a fresh one.
at::Tensor output_of(PyObject *given, at::IntArrayRef sizes, at::ScalarType dtype, const at::Tensor &like, int64_t device,
                     const char *name) {
  if (given == Py_None) return at::empty(sizes, at::TensorOptions().dtype(dtype).device(like.device()));
  const at::Tensor &t = operand(given, (int64_t)sizes.size(), device, name);
  require_sizes(t, sizes, name);
  device_pointer(t, dtype, name);
  return t;
}

template <typename Call>
void call_library(swb_context *ctx, Call call) {
  int st;
  Py_BEGIN_ALLOW_THREADS
  st = call();
  Py_END_ALLOW_THREADS
  if (st != SWB_OK) raise_status(st, swb_last_error(ctx));
}

PyObject *wrapped(PyObject *given, at::Tensor &t) {
  if (given != Py_None) {
    Py_INCREF(given);
    return given;
  }
  return THPVariable_Wrap(std::move(t));
}

PyObject *pair(PyObject *first, PyObject *second) {
  PyObject *both = first && second ? PyTuple_New(2) : nullptr;
  if (!both) {
    Py_XDECREF(first);
    Py_XDECREF(second);
    throw Failed();
  }
  PyTuple_SET_ITEM(both, 0, first);
  PyTuple_SET_ITEM(both, 1, second);
  return both;
}

// grouped_mm(ctx, device, offsets, A, B, C | None, transpose_b)
PyObject *grouped_mm(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded(n, 7, [&]() -> PyObject * {
    swb_context *ctx = context_of(a[0]);
    const int64_t device = integer(a[1]);
    const at::Tensor &off = operand(a[2], 1, device, "offsets"), &A = operand(a[3], 2, device, "A"),
                     &B = operand(a[4], 3, device, "B");
    const bool tb = truth(a[6]);
    const int64_t rows = A.size(0), inner = A.size(1), groups = B.size(0), cols = B.size(tb ? 1 : 2);
    require_sizes(off, {groups + 1}, "offsets");
    require_sizes(B, {groups, tb ? cols : inner, tb ? inner : cols}, "B");
    const int type = type_code(A, "A", Types::k16Bits);
    auto *p_off = (const int32_t *)device_pointer(off, at::kInt, "offsets");
    void *p_A = device_pointer(A, A.scalar_type(), "A"), *p_B = device_pointer(B, A.scalar_type(), "B");
    at::Tensor C = output_of(a[5], {rows, cols}, A.scalar_type(), A, device, "C");
    void *s = stream_of(a[1]);
    call_library(ctx, [&] {
      return swb_grouped_mm(ctx, type, rows, inner, cols, groups, p_off, p_A, p_B, tb, C.data_ptr(), s);
    });
    return wrapped(a[5], C);
  });
}

// grouped_mm_grad(ctx, device, offsets, A | None, B | None, dC, dA | None, dB | None, transpose_b, need_dA, need_dB): A may be missing where
// dB is not needed, B where dA is not
PyObject *grouped_mm_grad(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded(n, 11, [&]() -> PyObject * {
    swb_context *ctx = context_of(a[0]);
    const int64_t device = integer(a[1]);
    const bool tb = truth(a[8]), need_a = truth(a[9]), need_b = truth(a[10]);
    const bool have_B = need_a || a[4] != Py_None, have_A = need_b || !have_B || a[3] != Py_None;
    const at::Tensor &off = operand(a[2], 1, device, "offsets");
    const at::Tensor *A = have_A ? &operand(a[3], 2, device, "A") : nullptr, *B = have_B ? &operand(a[4], 3, device, "B") : nullptr;
    const at::Tensor &dC = operand(a[5], 2, device, "dC");
    if (off.size(0) < 2) raise_shape("offsets must have at least 2 entries, but got " + std::to_string(off.size(0)));
    const int64_t rows = A ? A->size(0) : dC.size(0), cols = dC.size(1), inner = A ? A->size(1) : B->size(tb ? 2 : 1);
    const int64_t groups = B ? B->size(0) : off.size(0) - 1;
    const at::ScalarType dt = A ? A->scalar_type() : dC.scalar_type();
    require_sizes(off, {groups + 1}, "offsets");
    require_sizes(dC, {rows, cols}, "dC");
    const std::vector<int64_t> a_sizes{rows, inner}, b_sizes{groups, tb ? cols : inner, tb ? inner : cols};
    if (B) require_sizes(*B, b_sizes, "B");
    const int type = A ? type_code(*A, "A", Types::k16Bits) : type_code(dC, "dC", Types::k16Bits);
    auto *p_off = (const int32_t *)device_pointer(off, at::kInt, "offsets");
    void *p_A = A ? device_pointer(*A, dt, "A") : nullptr, *p_B = B ? device_pointer(*B, dt, "B") : nullptr;
    void *p_dC = device_pointer(dC, dt, "dC");
    at::Tensor dA, dB;
    if (need_a) dA = output_of(a[6], a_sizes, dt, dC, device, "dA");
    if (need_b) dB = output_of(a[7], b_sizes, dt, dC, device, "dB");
    void *p_dA = need_a ? dA.data_ptr() : nullptr, *p_dB = need_b ? dB.data_ptr() : nullptr, *s = stream_of(a[1]);
    call_library(ctx, [&] {
      return swb_grouped_mm_grad(ctx, type, rows, inner, cols, groups, p_off, p_A, p_B, p_dC, tb, p_dA, p_dB, s);
    });
    PyObject *first = need_a ? wrapped(a[6], dA) : (Py_INCREF(Py_None), Py_None);
    PyObject *second = need_b ? wrapped(a[7], dB) : (Py_INCREF(Py_None), Py_None);
    return pair(first, second);
  });
}

at::ScalarType fp8_type(PyObject *obj) {
  if (THPDtype_Check(obj)) {
    const at::ScalarType t = reinterpret_cast<THPDtype *>(obj)->scalar_type;
    if (t == at::kFloat8_e4m3fn || t == at::kFloat8_e5m2) return t;
  }
  raise_type("dtype", "must be torch.float8_e4m3fn or torch.float8_e5m2");
}

// fp8_quantize(ctx, device, by_rows, X, Q | None, scales | None, dtype)
PyObject *fp8_quantize(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded(n, 7, [&]() -> PyObject * {
    swb_context *ctx = context_of(a[0]);
    const int64_t device = integer(a[1]);
    const bool by_rows = truth(a[2]);
    const at::Tensor &given = tensor(a[3], "X");
    const at::Tensor &X = operand(a[3], by_rows || given.dim() == 2 ? 2 : 3, device, "X");
    const int64_t d = X.dim(), groups = d == 3 ? X.size(0) : 1, rows = X.size(d - 2), cols = X.size(d - 1);
    const int type = type_code(X, "X", Types::k16BitsOrF32);
    const at::ScalarType out = fp8_type(a[6]);
    void *p_X = device_pointer(X, X.scalar_type(), "X");
    const int64_t rb = (rows + 127) / 128, cb = (cols + 127) / 128;
    const std::vector<int64_t> sizes = by_rows  ? std::vector<int64_t>{cb, rows}
                                       : d == 3 ? std::vector<int64_t>{groups, rb, cb}
                                                : std::vector<int64_t>{rb, cb};
    at::Tensor Q = output_of(a[4], X.sizes(), out, X, device, "Q"), scales = output_of(a[5], sizes, at::kFloat, X, device, "scales");
    void *p_Q = Q.data_ptr(), *s = stream_of(a[1]);
    auto *p_s = (float *)scales.data_ptr();
    const int fp8 = out == at::kFloat8_e5m2 ? SWB_E5M2 : SWB_E4M3;
    call_library(ctx, [&] {
      return by_rows ? swb_fp8_quantize_rows(ctx, type, fp8, rows, cols, p_X, p_Q, p_s, s)
                     : swb_fp8_quantize_blocks(ctx, type, fp8, groups, rows, cols, p_X, p_Q, p_s, s);
    });
    PyObject *first = wrapped(a[4], Q);
    return pair(first, wrapped(a[5], scales));
  });
}

// fp8_product(ctx, device, offsets | None, A, a_scales, B, b_scales, C | None, transpose_b): without offsets B is one matrix
PyObject *fp8_product(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded(n, 9, [&]() -> PyObject * {
    swb_context *ctx = context_of(a[0]);
    const int64_t device = integer(a[1]);
    const bool grouped = a[2] != Py_None, tb = truth(a[8]);
    const int64_t front = grouped ? 1 : 0;
    const at::Tensor &A = operand(a[3], 2, device, "A"), &as = operand(a[4], 2, device, "a_scales"),
                     &B = operand(a[5], 2 + front, device, "B"), &bs = operand(a[6], 2 + front, device, "b_scales");
    const int64_t rows = A.size(0), inner = A.size(1), groups = grouped ? B.size(0) : 1, cols = B.size(front + (tb ? 0 : 1));
    const int64_t kb = (inner + 127) / 128, nb = (cols + 127) / 128;
    std::vector<int64_t> b_sizes{tb ? cols : inner, tb ? inner : cols}, s_sizes{tb ? nb : kb, tb ? kb : nb};
    const int32_t *p_off = nullptr;
    if (grouped) {
      const at::Tensor &off = operand(a[2], 1, device, "offsets");
      require_sizes(off, {groups + 1}, "offsets");
      p_off = (const int32_t *)device_pointer(off, at::kInt, "offsets");
      b_sizes.insert(b_sizes.begin(), groups);
      s_sizes.insert(s_sizes.begin(), groups);
    }
    require_sizes(B, b_sizes, "B");
    require_sizes(as, {kb, rows}, "a_scales");
    require_sizes(bs, s_sizes, "b_scales");
    const int a_type = type_code(A, "A", Types::kFp8), b_type = type_code(B, "B", Types::kFp8);
    void *p_A = device_pointer(A, A.scalar_type(), "A"), *p_B = device_pointer(B, B.scalar_type(), "B");
    auto *p_as = (const float *)device_pointer(as, at::kFloat, "a_scales");
    auto *p_bs = (const float *)device_pointer(bs, at::kFloat, "b_scales");
    at::Tensor C = output_of(a[7], {rows, cols}, at::kBFloat16, A, device, "C");
    auto *p_C = (uint16_t *)C.data_ptr();
    void *s = stream_of(a[1]);
    call_library(ctx, [&] {
      return grouped ? swb_fp8_grouped_mm(ctx, a_type, b_type, rows, inner, cols, groups, p_off, p_A, p_as, p_B, p_bs, tb, p_C, s)
                     : swb_fp8_mm(ctx, a_type, b_type, rows, inner, cols, p_A, p_as, p_B, p_bs, tb, p_C, s);
    });
    return wrapped(a[7], C);
  });
}

// bind(SparseWaveError, SwbOptions): the Python types that the calls above raise and accept
PyObject *bind(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded(n, 2, [&]() -> PyObject * {
    if (!PyType_Check(a[0]) || !PyType_Check(a[1])) raise_type("bind", "needs two types");
    Py_INCREF(a[0]);
    Py_INCREF(a[1]);
    g_error = a[0];
    g_options = (PyTypeObject *)a[1];
    Py_RETURN_NONE;
  });
}

#define SWB_FAST(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {SWB_FAST(spmv), SWB_FAST(coo_spmv), SWB_FAST(spmm), SWB_FAST(bsr_spmm), SWB_FAST(grouped_mm),
                           SWB_FAST(grouped_mm_grad), SWB_FAST(fp8_quantize), SWB_FAST(fp8_product), SWB_FAST(bind),
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "swb_torch", "Device-tensor operator calls over the C ABI.", -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_swb_torch(void) { return PyModule_Create(&g_module); }
