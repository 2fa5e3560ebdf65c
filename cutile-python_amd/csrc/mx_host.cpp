// Native host path of the Python operators (module cutile_amd._mxhost).
//
// A decode-sized product keeps the GPU busy for less than 10 us, while building five ctypes descriptors, asking torch
// for the stream and switching device contexts took about 19 us of Python per operator.  The functions here do the same
// work -- read the tensors, fill in the descriptors, allocate the results from torch's caching allocator, call the C
// ABI of libmxgemm.so -- in one or two microseconds.  They handle the ordinary calls only: anything unusual (another
// device, a dtype or layout that needs a message or the general kernel's rules) returns None before anything is
// enqueued, and ops.py then runs its own path, which validates like the reference and raises its errors.
//
// Scratch comes from the caching allocator on every call and goes back to it when the call returns: blocks are reused
// in stream order, so calls from several threads and streams, and graph captures, need no rule of their own.
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/Context.h>
#include <ATen/Functions.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>

#include <vector>

#include "mxgemm.h"

namespace {

#define MX_FN(name) decltype(&name) p_##name = nullptr
struct Lib {
  MX_FN(mx_gemm);
  MX_FN(mx_gemm_add);
  MX_FN(mx_gemm_workspace_bytes);
  MX_FN(mx_packed_scale_bytes);
  MX_FN(mx_gemm_list);
  MX_FN(mx_gemm_list_workspace_bytes);
  MX_FN(mx_quantize);
  MX_FN(mx_silu_mul_quantize);
  MX_FN(mx_moe_forward);
  MX_FN(mx_moe_forward_workspace_bytes);
  MX_FN(mx_last_error);
  MX_FN(mx_quantize_both);
  MX_FN(mx_gated_gemm);
  MX_FN(mx_gated_gemm_workspace_bytes);
  MX_FN(mx_silu_mul_backward_quantize);
  MX_FN(mx_ffn_saved_bytes);
  MX_FN(mx_ffn_forward);
  MX_FN(mx_ffn_forward_workspace_bytes);
  MX_FN(mx_ffn_backward);
  MX_FN(mx_ffn_backward_workspace_bytes);
  MX_FN(mx_layer_norm);
  MX_FN(mx_layer_norm_quantize);
  MX_FN(mx_layer_norm_backward_workspace_bytes);
  MX_FN(mx_layer_norm_backward);
  MX_FN(mx_adamw_step);
  MX_FN(mx_linear_gemm);
  MX_FN(mx_linear_gemm_workspace_bytes);
  MX_FN(mx_linear_saved_bytes);
  MX_FN(mx_linear_forward);
  MX_FN(mx_linear_forward_workspace_bytes);
  MX_FN(mx_linear_backward);
  MX_FN(mx_linear_backward_workspace_bytes);
} lib;
#undef MX_FN
PyObject* packed_type = nullptr;   // ops.PackedScales
PyObject *s_data, *s_rows, *s_K, *s_operand, *s_layout, *s_batch;

struct NoGil {
  PyThreadState* state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

// MX element format of a tensor given the caller's format argument (None or a str); -1: not for the native path
int elem_format(const at::Tensor& t, PyObject* fmt) {
  const auto dt = t.scalar_type();
  int from_dtype = -1;
  if (dt == at::kFloat8_e4m3fn) from_dtype = MX_E4M3;
  else if (dt == at::kFloat8_e5m2) from_dtype = MX_E5M2;
  else if (dt == at::kFloat4_e2m1fn_x2) from_dtype = MX_E2M1;
  if (fmt == Py_None) return from_dtype;
  if (!PyUnicode_Check(fmt)) return -1;
  int want = -1;
  if (PyUnicode_CompareWithASCIIString(fmt, "e4m3") == 0) want = MX_E4M3;
  else if (PyUnicode_CompareWithASCIIString(fmt, "e5m2") == 0) want = MX_E5M2;
  else if (PyUnicode_CompareWithASCIIString(fmt, "e2m1") == 0) want = MX_E2M1;
  return (want >= 0 && (dt == at::kByte || from_dtype == want)) ? want : -1;
}

inline bool is_e8m0(const at::Tensor& t) {
  return t.scalar_type() == at::kFloat8_e8m0fnu || t.scalar_type() == at::kByte;
}

// descriptor of a tensor of up to 4 dimensions; the extent of `packed` (an FP4 tensor's K axis) counts elements
inline mx_tensor desc(const at::Tensor& t, int dtype, int packed = -1) {
  mx_tensor d;
  d.ptr = t.data_ptr();
  d.dtype = dtype;
  d.ndim = (int32_t)t.dim();
  const auto sz = t.sizes(), st = t.strides();
  for (int i = 0; i < d.ndim; ++i) { d.shape[i] = sz[i]; d.stride[i] = st[i]; }
  if (packed >= 0) d.shape[packed] *= 2;
  d.packed_dim = packed;
  d.reserved = 0;
  return d;
}

inline bool on_current_device(const at::Tensor& t) {
  return t.is_cuda() && t.device().index() == c10::hip::current_device();
}

// a scale argument as descriptor + layout: a 2-D / 3-D / swizzled 4-D E8M0 tensor or a PackedScales made for this
// operand; false: leave it to ops.py
bool scale_desc(PyObject* o, int64_t rows, int64_t K, bool is_b, const at::Device& dev, mx_tensor* d, int32_t* layout) {
  if (THPVariable_Check(o)) {
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!is_e8m0(t) || t.device() != dev || t.dim() < 2 || t.dim() > 4) return false;
    *d = desc(t, MX_E8M0);
    *layout = t.dim() == 4 ? MX_SCALE_SWIZZLE_32_4_4 : MX_SCALE_2D;
    return true;
  }
  if ((PyObject*)Py_TYPE(o) != packed_type) return false;
  PyObject* data = PyObject_GetAttr(o, s_data);
  PyObject* prow = PyObject_GetAttr(o, s_rows);
  PyObject* pk = PyObject_GetAttr(o, s_K);
  PyObject* pop = PyObject_GetAttr(o, s_operand);
  PyObject* pl = PyObject_GetAttr(o, s_layout);
  bool ok = data && prow && pk && pop && pl && THPVariable_Check(data) && PyUnicode_Check(pop);
  if (ok) {
    const at::Tensor& t = THPVariable_Unpack(data);   // kept alive by the PackedScales object
    ok = PyLong_AsLongLong(prow) == rows && PyLong_AsLongLong(pk) == K && t.device() == dev &&
         PyUnicode_CompareWithASCIIString(pop, is_b ? "b" : "a") == 0;
    *d = mx_tensor{t.data_ptr(), MX_E8M0, 2, {rows, K / 32, 0, 0}, {K / 32, 1, 0, 0}, -1, 0};
    *layout = (int32_t)PyLong_AsLong(pl);
  }
  Py_XDECREF(data); Py_XDECREF(prow); Py_XDECREF(pk); Py_XDECREF(pop); Py_XDECREF(pl);
  if (PyErr_Occurred()) { PyErr_Clear(); return false; }
  return ok;
}

// at::empty without the dispatcher (0.47 instead of 0.72 us; a call allocates up to three tensors, a list one per problem),
// unless something has asked to see factory calls (dispatch modes, functorch) or to have new memory filled.
inline at::Tensor device_empty(at::IntArrayRef shape, at::ScalarType t, const at::Device& dev) {
  const c10::impl::LocalDispatchKeySet tls = c10::impl::tls_local_dispatch_key_set();
  if ((tls.included_ - c10::default_included_set).empty() && !at::globalContext().deterministicAlgorithms())
    return at::detail::empty_cuda(shape, t, dev, std::nullopt);
  return at::empty(shape, at::TensorOptions().dtype(t).device(dev));
}

inline void* stream_of(const at::Device& dev) { return (void*)c10::hip::getCurrentHIPStream(dev.index()).stream(); }

inline PyObject* rc_or(int rc, const at::Tensor& t) { return rc == MX_OK ? THPVariable_Wrap(t) : PyLong_FromLong(rc); }

int out_code(at::ScalarType t) { return t == at::kFloat ? MX_F32 : t == at::kBFloat16 ? MX_BF16 : -1; }

// operands of one 2-D product; false: not for the native path
struct Product {
  mx_tensor A, As, B, Bs;
  int32_t la, lb;
  int64_t M, N, K;
};
bool product(PyObject* pa, PyObject* pas, PyObject* pb, PyObject* pbs, PyObject* af, PyObject* bf, Product* p,
             at::Device* dev) {
  if (!THPVariable_Check(pa) || !THPVariable_Check(pb)) return false;
  const at::Tensor &A = THPVariable_Unpack(pa), &B = THPVariable_Unpack(pb);
  if (A.dim() != 2 || B.dim() != 2 || !on_current_device(A) || B.device() != A.device()) return false;
  const int fa = elem_format(A, af), fb = elem_format(B, bf);
  if (fa < 0 || fb < 0) return false;
  if ((fa == MX_E2M1 && A.stride(1) != 1) || (fb == MX_E2M1 && B.stride(0) != 1)) return false;
  p->A = desc(A, fa, fa == MX_E2M1 ? 1 : -1);
  p->B = desc(B, fb, fb == MX_E2M1 ? 0 : -1);
  p->M = p->A.shape[0]; p->K = p->A.shape[1]; p->N = p->B.shape[1];
  if (p->B.shape[0] != p->K) return false;
  *dev = A.device();
  return scale_desc(pas, p->M, p->K, false, *dev, &p->As, &p->la) && scale_desc(pbs, p->N, p->K, true, *dev, &p->Bs, &p->lb);
}

// gemm(A, A_scale, B, B_scale, C | None, out_dtype, a_format, b_format, accumulate, kernel, split_k)
//   -> result tensor, a negative MX_ERR_* code, or None
PyObject* py_gemm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 11) { PyErr_SetString(PyExc_TypeError, "gemm takes 11 arguments"); return nullptr; }
  Product p;
  at::Device dev(at::kCUDA);
  if (!product(a[0], a[1], a[2], a[3], a[6], a[7], &p, &dev)) Py_RETURN_NONE;
  const int accumulate = PyObject_IsTrue(a[8]);
  at::Tensor C;
  if (a[4] != Py_None) {
    if (!THPVariable_Check(a[4])) Py_RETURN_NONE;
    C = THPVariable_Unpack(a[4]);
    if (C.dim() != 2 || C.size(0) != p.M || C.size(1) != p.N || out_code(C.scalar_type()) < 0 || C.device() != dev)
      Py_RETURN_NONE;
  } else {
    if (accumulate || !THPDtype_Check(a[5])) Py_RETURN_NONE;
    const auto t = ((THPDtype*)a[5])->scalar_type;
    if (out_code(t) < 0) Py_RETURN_NONE;
    C = device_empty({p.M, p.N}, t, dev);
  }
  mx_tensor dC = desc(C, out_code(C.scalar_type()));
  mx_gemm_opts o = {sizeof(mx_gemm_opts), accumulate, p.la, p.lb, (int32_t)PyLong_AsLong(a[9]), 32,
                    (int32_t)PyLong_AsLong(a[10]), 0};
  if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
  const int64_t need = lib.p_mx_gemm_workspace_bytes(p.M, p.N, p.K, &o);
  at::Tensor ws;
  if (need > 0) ws = device_empty({need}, at::kByte, dev);
  int rc;
  {
    NoGil nogil;
    rc = lib.p_mx_gemm(&p.A, &p.As, &p.B, &p.Bs, &dC, &o, need > 0 ? ws.data_ptr() : nullptr, need, stream_of(dev));
  }
  if (rc == MX_OK && a[4] != Py_None) { Py_INCREF(a[4]); return a[4]; }
  return rc_or(rc, C);
}

// gemm_list(As, A_scales, Bs, B_scales, Cs | None, out_dtype, kernel) -> list of results, error code, or None
PyObject* py_gemm_list(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 7) { PyErr_SetString(PyExc_TypeError, "gemm_list takes 7 arguments"); return nullptr; }
  auto seq = [](PyObject* o) { return PyList_Check(o) || PyTuple_Check(o); };
  if (!seq(a[0]) || !seq(a[1]) || !seq(a[2]) || !seq(a[3]) || (a[4] != Py_None && !seq(a[4])) || !THPDtype_Check(a[5]))
    Py_RETURN_NONE;
  const Py_ssize_t cnt = PySequence_Fast_GET_SIZE(a[0]);
  for (int i = 1; i < 5; ++i)
    if (a[i] != Py_None && PySequence_Fast_GET_SIZE(a[i]) != cnt) Py_RETURN_NONE;
  const auto out_t = ((THPDtype*)a[5])->scalar_type;
  if (cnt == 0 || out_code(out_t) < 0) Py_RETURN_NONE;
  std::vector<mx_tensor> A(cnt), As(cnt), B(cnt), Bs(cnt), C(cnt);
  std::vector<at::Tensor> outs(cnt), keep;   // keep: the lists may change while the GIL is released
  keep.reserve(4 * cnt);
  at::Device dev(at::kCUDA);
  int32_t la = 0, lb = 0;
  for (Py_ssize_t i = 0; i < cnt; ++i) {
    auto item = [&](int k) { return PySequence_Fast_GET_ITEM(a[k], i); };
    Product p;
    at::Device d(at::kCUDA);
    if (!product(item(0), item(1), item(2), item(3), Py_None, Py_None, &p, &d)) Py_RETURN_NONE;
    if (i > 0 && (p.la != la || p.lb != lb || d != dev)) Py_RETURN_NONE;
    la = p.la; lb = p.lb; dev = d;
    for (int k = 0; k < 4; ++k) {
      if (THPVariable_Check(item(k))) { keep.push_back(THPVariable_Unpack(item(k))); continue; }
      PyObject* data = PyObject_GetAttr(item(k), s_data);   // PackedScales: product() has seen a tensor here
      if (!data) return nullptr;
      if (THPVariable_Check(data)) keep.push_back(THPVariable_Unpack(data));
      Py_DECREF(data);
    }
    if (a[4] != Py_None) {
      if (!THPVariable_Check(item(4))) Py_RETURN_NONE;
      outs[i] = THPVariable_Unpack(item(4));
      if (outs[i].dim() != 2 || outs[i].size(0) != p.M || outs[i].size(1) != p.N ||
          out_code(outs[i].scalar_type()) < 0 || outs[i].device() != dev)
        Py_RETURN_NONE;
    } else {
      outs[i] = device_empty({p.M, p.N}, out_t, dev);
    }
    A[i] = p.A; As[i] = p.As; B[i] = p.B; Bs[i] = p.Bs;
    C[i] = desc(outs[i], out_code(outs[i].scalar_type()));
  }
  mx_gemm_opts o = {sizeof(mx_gemm_opts), 0, la, lb, (int32_t)PyLong_AsLong(a[6]), 32, 0, 0};
  if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
  const int64_t need = lib.p_mx_gemm_list_workspace_bytes((int32_t)cnt, A.data(), B.data(), &o);
  at::Tensor ws;
  if (need > 0) ws = device_empty({need}, at::kByte, dev);
  int rc;
  {
    NoGil nogil;
    rc = lib.p_mx_gemm_list((int32_t)cnt, A.data(), As.data(), B.data(), Bs.data(), C.data(), &o,
                            need > 0 ? ws.data_ptr() : nullptr, need, stream_of(dev));
  }
  if (rc != MX_OK) return PyLong_FromLong(rc);
  PyObject* res = PyList_New(cnt);
  if (!res) return nullptr;
  for (Py_ssize_t i = 0; i < cnt; ++i) {
    PyList_SET_ITEM(res, i, THPVariable_Wrap(outs[i]));   // (a tensor of Cs is the same Python object again)
  }
  return res;
}

// mma(x, x_scale, y, y_scale, acc, x_format, y_format, allow_mixed) -> acc + x @ y (a new tensor), error code, or None.
// Every rule of mma_scaled that could fail is a condition here: what is not the plain block-32 case is left to ops.py.
PyObject* py_mma(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 8) { PyErr_SetString(PyExc_TypeError, "mma takes 8 arguments"); return nullptr; }
  for (int i = 0; i < 5; ++i)
    if (!THPVariable_Check(a[i])) Py_RETURN_NONE;
  const at::Tensor &x = THPVariable_Unpack(a[0]), &xs = THPVariable_Unpack(a[1]), &y = THPVariable_Unpack(a[2]),
                   &ys = THPVariable_Unpack(a[3]), &acc = THPVariable_Unpack(a[4]);
  const int xd = (int)x.dim(), yd = (int)y.dim();
  if ((xd != 2 && xd != 3) || (yd != 2 && yd != 3) || xs.dim() != xd || ys.dim() != yd || !on_current_device(x)) Py_RETURN_NONE;
  const at::Device dev = x.device();
  if (xs.device() != dev || y.device() != dev || ys.device() != dev || acc.device() != dev) Py_RETURN_NONE;
  const int fx = elem_format(x, a[5]), fy = elem_format(y, a[6]);
  if (fx < 0 || fy < 0 || (fx != fy && !PyObject_IsTrue(a[7])) || !is_e8m0(xs) || !is_e8m0(ys)) Py_RETURN_NONE;
  if ((fx == MX_E2M1 && x.stride(-1) != 1) || (fy == MX_E2M1 && y.stride(-2) != 1)) Py_RETURN_NONE;
  mx_tensor dx = desc(x, fx, fx == MX_E2M1 ? xd - 1 : -1), dy = desc(y, fy, fy == MX_E2M1 ? yd - 2 : -1),
            dxs = desc(xs, MX_E8M0), dys = desc(ys, MX_E8M0);
  const int64_t M = dx.shape[xd - 2], K = dx.shape[xd - 1], N = dy.shape[yd - 1];
  const int64_t bx = xd == 3 ? x.size(0) : 1, by = yd == 3 ? y.size(0) : 1, batch = bx > by ? bx : by;
  if (dy.shape[yd - 2] != K || K == 0 || K % 32 != 0 || M == 0 || N == 0 || (bx != by && bx != 1 && by != 1) || bx == 0 || by == 0 ||
      dxs.shape[xd - 2] != M || dxs.shape[xd - 1] != K / 32 || dys.shape[yd - 2] != K / 32 || dys.shape[yd - 1] != N ||
      (xd == 3 && dxs.shape[0] != bx) || (yd == 3 && dys.shape[0] != by))
    Py_RETURN_NONE;
  const bool batched = xd == 3 || yd == 3;
  if (acc.scalar_type() != at::kFloat || !acc.is_contiguous() || acc.dim() != (batched ? 3 : 2) || acc.size(-2) != M ||
      acc.size(-1) != N || (batched && acc.size(0) != batch) || acc.requires_grad())   // (there the result is a clone of acc)
    Py_RETURN_NONE;
  at::Tensor out = device_empty(acc.sizes(), at::kFloat, dev);
  mx_tensor dD = desc(acc, MX_F32), dC = desc(out, MX_F32);
  mx_gemm_opts o = {sizeof(mx_gemm_opts), 0, MX_SCALE_2D, MX_SCALE_2D, MX_KERNEL_AUTO, 32, 0, 0};
  // one product at a time needs its workspace once, a batch in one launch all re-laid scales at once
  const int64_t one = lib.p_mx_gemm_workspace_bytes(M, N, K, &o),
                all = (lib.p_mx_packed_scale_bytes(M, K) + lib.p_mx_packed_scale_bytes(N, K)) * batch, need = one > all ? one : all;
  at::Tensor ws;
  if (need > 0) ws = device_empty({need}, at::kByte, dev);
  int rc;
  {
    NoGil nogil;
    rc = lib.p_mx_gemm_add(&dx, &dxs, &dy, &dys, &dD, &dC, &o, need > 0 ? ws.data_ptr() : nullptr, need, stream_of(dev));
  }
  return rc_or(rc, out);
}

// quantize(x, dtype | str, mode, silu) -> (elements, scales), error code, or None.
// mode: 0 "ceil", 1 "floor"; silu: x is gate | up and silu(gate) * up is what is quantised
PyObject* py_quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 4) { PyErr_SetString(PyExc_TypeError, "quantize takes 4 arguments"); return nullptr; }
  if (!THPVariable_Check(a[0])) Py_RETURN_NONE;
  const at::Tensor& x = THPVariable_Unpack(a[0]);
  const auto xt = x.scalar_type();
  const int xc = xt == at::kFloat ? MX_F32 : xt == at::kBFloat16 ? MX_BF16 : xt == at::kHalf ? MX_F16 : -1;
  int fmt = -1;
  if (THPDtype_Check(a[1])) {
    const auto t = ((THPDtype*)a[1])->scalar_type;
    fmt = t == at::kFloat8_e4m3fn ? MX_E4M3 : t == at::kFloat8_e5m2 ? MX_E5M2 : t == at::kFloat4_e2m1fn_x2 ? MX_E2M1 : -1;
  } else if (PyUnicode_Check(a[1])) {
    if (PyUnicode_CompareWithASCIIString(a[1], "e2m1") == 0) fmt = MX_E2M1;
    else if (PyUnicode_CompareWithASCIIString(a[1], "e4m3") == 0) fmt = MX_E4M3;
    else if (PyUnicode_CompareWithASCIIString(a[1], "e5m2") == 0) fmt = MX_E5M2;
  }
  const int silu = PyObject_IsTrue(a[3]);
  if (fmt < 0 || xc < 0 || x.dim() < 1 || x.dim() > 4 || !on_current_device(x)) Py_RETURN_NONE;
  const int64_t cols = x.size(-1), K = silu ? cols / 2 : cols;
  if (cols == 0 || K % 32 != 0 || K < 32 || (silu && cols % 64 != 0) || x.numel() == 0) Py_RETURN_NONE;
  if (!(x.is_contiguous() || (x.dim() == 2 && x.stride(1) == 1))) Py_RETURN_NONE;
  const at::Device dev = x.device();
  const int64_t rows = x.numel() / cols;
  int64_t shape[4];
  const int nd = (int)x.dim();
  for (int i = 0; i + 1 < nd; ++i) shape[i] = x.size(i);
  shape[nd - 1] = fmt == MX_E2M1 ? K / 2 : K;
  at::Tensor q = device_empty(at::IntArrayRef(shape, nd),
                              fmt == MX_E4M3 ? at::kFloat8_e4m3fn : fmt == MX_E5M2 ? at::kFloat8_e5m2 : at::kByte, dev);
  shape[nd - 1] = K / 32;
  at::Tensor s = device_empty(at::IntArrayRef(shape, nd), at::kFloat8_e8m0fnu, dev);
  mx_tensor dx{x.data_ptr(), xc, 2, {rows, cols, 0, 0}, {nd == 2 ? x.stride(0) : cols, 1, 0, 0}, -1, 0};
  mx_tensor dq{q.data_ptr(), fmt, 2, {rows, K, 0, 0}, {fmt == MX_E2M1 ? K / 2 : K, 1, 0, 0}, fmt == MX_E2M1 ? 1 : -1, 0};
  mx_tensor ds{s.data_ptr(), MX_E8M0, 2, {rows, K / 32, 0, 0}, {K / 32, 1, 0, 0}, -1, 0};
  const int mode = (int)PyLong_AsLong(a[2]);
  int rc;
  {
    NoGil nogil;
    rc = silu ? lib.p_mx_silu_mul_quantize(&dx, &dq, &ds, mode, stream_of(dev)) : lib.p_mx_quantize(&dx, &dq, &ds, mode, stream_of(dev));
  }
  if (rc != MX_OK) return PyLong_FromLong(rc);
  PyObject* res = PyTuple_New(2);
  if (!res) return nullptr;
  PyTuple_SET_ITEM(res, 0, THPVariable_Wrap(q));
  PyTuple_SET_ITEM(res, 1, THPVariable_Wrap(s));
  return res;
}

// scales of a stack of expert weights: a [E, rows, K/32] E8M0 tensor or a PackedScales of it
bool expert_scale_desc(PyObject* o, int64_t E, int64_t rows, int64_t K, const at::Device& dev, mx_tensor* d, int32_t* layout) {
  if (THPVariable_Check(o)) {
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!is_e8m0(t) || t.device() != dev || t.dim() != 3) return false;
    *d = desc(t, MX_E8M0);
    *layout = MX_SCALE_2D;
    return true;
  }
  if ((PyObject*)Py_TYPE(o) != packed_type) return false;
  PyObject* pb = PyObject_GetAttr(o, s_batch);
  const bool ok = pb && PyLong_AsLongLong(pb) == E;
  Py_XDECREF(pb);
  if (PyErr_Occurred()) { PyErr_Clear(); return false; }
  if (!ok || !scale_desc(o, rows, K, true, dev, d, layout) || *layout != MX_SCALE_NATIVE) return false;
  d->ndim = 3;
  d->shape[0] = E; d->shape[1] = rows; d->shape[2] = K / 32;
  d->stride[0] = rows * (K / 32); d->stride[1] = K / 32; d->stride[2] = 1;
  return true;
}

// moe(hidden, hidden_scale, w1, w1_scale, w2, w2_scale, topk_weights, topk_ids, out_dtype, mode, w_format, tile_m)
//   -> result, error code, or None
PyObject* py_moe(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 12) { PyErr_SetString(PyExc_TypeError, "moe takes 12 arguments"); return nullptr; }
  for (int i : {0, 1, 2, 4, 6, 7})
    if (!THPVariable_Check(a[i])) Py_RETURN_NONE;
  const at::Tensor &X = THPVariable_Unpack(a[0]), &Xs = THPVariable_Unpack(a[1]), &W1 = THPVariable_Unpack(a[2]),
                   &W2 = THPVariable_Unpack(a[4]), &wt = THPVariable_Unpack(a[6]), &ids = THPVariable_Unpack(a[7]);
  if (X.dim() != 2 || Xs.dim() != 2 || W1.dim() != 3 || W2.dim() != 3 || ids.dim() != 2 || !on_current_device(X)) Py_RETURN_NONE;
  const at::Device dev = X.device();
  if (Xs.device() != dev || W1.device() != dev || W2.device() != dev || wt.device() != dev || ids.device() != dev) Py_RETURN_NONE;
  const int f1 = elem_format(W1, a[10]), f2 = elem_format(W2, a[10]);
  if (X.scalar_type() != at::kFloat8_e4m3fn || !is_e8m0(Xs) || f1 != f2 || (f1 != MX_E4M3 && f1 != MX_E2M1)) Py_RETURN_NONE;
  if (f1 == MX_E2M1 && (W1.stride(2) != 1 || W2.stride(2) != 1)) Py_RETURN_NONE;
  const int64_t T = X.size(0), topk = ids.size(1), E = W1.size(0);
  if (ids.size(0) != T || T == 0 || topk == 0 || topk > 1 << 20 || !ids.is_contiguous() ||
      (ids.scalar_type() != at::kInt && ids.scalar_type() != at::kLong) || wt.scalar_type() != at::kFloat ||
      !wt.is_contiguous() || wt.numel() != T * topk || !THPDtype_Check(a[8]))
    Py_RETURN_NONE;
  const auto out_t = ((THPDtype*)a[8])->scalar_type;
  if (out_code(out_t) < 0) Py_RETURN_NONE;
  mx_tensor dX = desc(X, MX_E4M3), dXs = desc(Xs, MX_E8M0), dW1 = desc(W1, f1, f1 == MX_E2M1 ? 2 : -1),
            dW2 = desc(W2, f2, f2 == MX_E2M1 ? 2 : -1), dW1s, dW2s;
  const long tile_m = PyLong_AsLong(a[11]);
  if (tile_m == -1 && PyErr_Occurred()) PyErr_Clear();
  if (tile_m <= 0 || tile_m > 0x7FFFFFFF) Py_RETURN_NONE;
  // (the operator's default, 256, leaves the form of the layer to the library)
  mx_gemm_opts o = {sizeof(mx_gemm_opts), 0, 0, 0, MX_KERNEL_AUTO, 32, 0, tile_m == 256 ? 0 : (int32_t)tile_m};
  if (!expert_scale_desc(a[3], E, dW1.shape[1], dW1.shape[2], dev, &dW1s, &o.a_scale_layout) ||
      !expert_scale_desc(a[5], E, dW2.shape[1], dW2.shape[2], dev, &dW2s, &o.b_scale_layout))
    Py_RETURN_NONE;
  at::Tensor out = device_empty({T, dW2.shape[1]}, out_t, dev);
  mx_tensor dO = desc(out, out_code(out_t));
  const int mode = (int)PyLong_AsLong(a[9]);
  const int64_t need = lib.p_mx_moe_forward_workspace_bytes(T, (int32_t)topk, &dW1, &dW2, &o);
  at::Tensor ws = device_empty({need > 0 ? need : 1}, at::kByte, dev);
  int rc;
  {
    NoGil nogil;
    rc = lib.p_mx_moe_forward(&dX, &dXs, &dW1, &dW1s, &dW2, &dW2s, (const float*)wt.data_ptr(), ids.data_ptr(),
                              ids.scalar_type() == at::kLong, (int32_t)topk, &dO, mode, &o, ws.data_ptr(), need, stream_of(dev));
  }
  if (rc == MX_ERR_LAYOUT) Py_RETURN_NONE;   // nothing was enqueued: operands for the single operators
  return rc_or(rc, out);
}

// ---- the feed-forward block that is trained in 8 bits -----------------------------------------------------------------------------
int float_code(at::ScalarType t) { return t == at::kFloat ? MX_F32 : t == at::kBFloat16 ? MX_BF16 : t == at::kHalf ? MX_F16 : -1; }
inline int64_t up32(int64_t n) { return (n + 31) / 32 * 32; }

// a tensor of two or more dimensions as [rows, last axis] with contiguous rows; false: it is no such matrix without a copy
bool matrix(const at::Tensor& t, int dtype, mx_tensor* d) {
  const int nd = (int)t.dim();
  if (nd < 1 || dtype < 0) return false;
  const int64_t cols = t.size(-1);
  if (cols == 0 || t.numel() == 0) return false;
  int64_t ld = cols;
  if (nd == 2 && t.stride(1) == 1 && t.stride(0) >= 0) ld = t.stride(0);
  else if (!t.is_contiguous()) return false;
  *d = mx_tensor{t.data_ptr(), dtype, 2, {t.numel() / cols, cols, 0, 0}, {ld, 1, 0, 0}, -1, 0};
  return true;
}
// room for elements and scales of a [rows, cols] matrix, cols a multiple of 32
struct Codes {
  at::Tensor q, s;
  mx_tensor dq, ds;
  Codes() = default;
  Codes(int64_t rows, int64_t cols, int fmt, const at::Device& dev)
      : q(device_empty({rows, cols}, fmt == MX_E5M2 ? at::kFloat8_e5m2 : at::kFloat8_e4m3fn, dev)),
        s(device_empty({rows, cols / 32}, at::kFloat8_e8m0fnu, dev)), dq(desc(q, fmt)), ds(desc(s, MX_E8M0)) {}
};
int format_of(PyObject* o) {   // an 8-bit format given as dtype or name
  if (THPDtype_Check(o)) {
    const auto t = ((THPDtype*)o)->scalar_type;
    return t == at::kFloat8_e4m3fn ? MX_E4M3 : t == at::kFloat8_e5m2 ? MX_E5M2 : -1;
  }
  if (!PyUnicode_Check(o)) return -1;
  return PyUnicode_CompareWithASCIIString(o, "e4m3") == 0 ? MX_E4M3 : PyUnicode_CompareWithASCIIString(o, "e5m2") == 0 ? MX_E5M2 : -1;
}
PyObject* tuple_of(std::initializer_list<at::Tensor> ts) {
  PyObject* res = PyTuple_New((Py_ssize_t)ts.size());
  if (!res) return nullptr;
  Py_ssize_t i = 0;
  for (const auto& t : ts) {
    PyObject* o = THPVariable_Wrap(t);
    if (!o) { Py_DECREF(res); return nullptr; }
    PyTuple_SET_ITEM(res, i++, o);
  }
  return res;
}

// quantize_both(x, dtype | str, mode) -> (x_q, scale, xt_q, scale_t), error code, or None
PyObject* py_quantize_both(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 3) { PyErr_SetString(PyExc_TypeError, "quantize_both takes 3 arguments"); return nullptr; }
  if (!THPVariable_Check(a[0])) Py_RETURN_NONE;
  const at::Tensor& x = THPVariable_Unpack(a[0]);
  const int fmt = format_of(a[1]);
  mx_tensor dx;
  if (fmt < 0 || !on_current_device(x) || !matrix(x, float_code(x.scalar_type()), &dx) || dx.shape[1] < 32) Py_RETURN_NONE;
  const at::Device dev = x.device();
  const int64_t rows = dx.shape[0], K = dx.shape[1];
  Codes r(rows, up32(K), fmt, dev), t(K, up32(rows), fmt, dev);
  const int mode = (int)PyLong_AsLong(a[2]);
  int rc;
  {
    NoGil nogil;
    rc = lib.p_mx_quantize_both(&dx, &r.dq, &r.ds, &t.dq, &t.ds, mode, stream_of(dev));
  }
  if (rc != MX_OK) return PyLong_FromLong(rc);
  if (x.dim() != 2) {
    auto shape = x.sizes().vec();
    shape.back() = up32(K);
    r.q = r.q.view(shape);
    shape.back() = up32(K) / 32;
    r.s = r.s.view(shape);
  }
  return tuple_of({r.q, r.s, t.q, t.s});
}

// gated(A, A_scale, W, W_scale, a_format, w_format, out_dtype, mode, checkpoint, kernel) -> result or tuple, error code, or None
PyObject* py_gated(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 10) { PyErr_SetString(PyExc_TypeError, "gated takes 10 arguments"); return nullptr; }
  if (!THPVariable_Check(a[0]) || !THPVariable_Check(a[2])) Py_RETURN_NONE;
  const at::Tensor &A = THPVariable_Unpack(a[0]), &W = THPVariable_Unpack(a[2]);
  if (A.dim() != 2 || W.dim() != 2 || !on_current_device(A) || W.device() != A.device()) Py_RETURN_NONE;
  const int fa = elem_format(A, a[4]), fw = elem_format(W, a[5]);
  if (fa < 0 || fw < 0 || A.stride(1) != 1 || W.stride(1) != 1) Py_RETURN_NONE;
  const at::Device dev = A.device();
  const mx_tensor dA = desc(A, fa, fa == MX_E2M1 ? 1 : -1), dW = desc(W, fw, fw == MX_E2M1 ? 1 : -1);
  const int64_t M = dA.shape[0], K = dA.shape[1], N = dW.shape[0], F = N / 2;
  if (M == 0 || K == 0 || dW.shape[1] != K || N == 0 || N % 64 != 0) Py_RETURN_NONE;
  mx_tensor dAs, dWs;
  mx_gemm_opts o = {sizeof(mx_gemm_opts), 0, 0, 0, (int32_t)PyLong_AsLong(a[9]), 32, 0, 0};
  if (!scale_desc(a[1], M, K, false, dev, &dAs, &o.a_scale_layout) || !scale_desc(a[3], N, K, true, dev, &dWs, &o.b_scale_layout)) Py_RETURN_NONE;
  const bool bf16 = THPDtype_Check(a[6]) && ((THPDtype*)a[6])->scalar_type == at::kBFloat16;
  const int fo = bf16 ? MX_BF16 : format_of(a[6]);
  const int mode = (int)PyLong_AsLong(a[7]), keep = PyObject_IsTrue(a[8]);
  if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
  if (fo < 0) Py_RETURN_NONE;
  Codes h, c;
  if (bf16) {
    h.q = device_empty({M, F}, at::kBFloat16, dev);
    h.dq = desc(h.q, MX_BF16);
  } else {
    h = Codes(M, F, fo, dev);
  }
  if (keep) c = Codes(M, N, MX_E4M3, dev);
  const int64_t need = lib.p_mx_gated_gemm_workspace_bytes(M, F, K, &o);
  at::Tensor ws;
  if (need > 0) ws = device_empty({need}, at::kByte, dev);
  int rc;
  {
    NoGil nogil;
    rc = lib.p_mx_gated_gemm(&dA, &dAs, &dW, &dWs, &h.dq, bf16 ? nullptr : &h.ds, keep ? &c.dq : nullptr, keep ? &c.ds : nullptr, mode, &o,
                             need > 0 ? ws.data_ptr() : nullptr, need, stream_of(dev));
  }
  if (rc != MX_OK) return PyLong_FromLong(rc);
  if (bf16) return keep ? tuple_of({h.q, c.q, c.s}) : THPVariable_Wrap(h.q);
  return keep ? tuple_of({h.q, h.s, c.q, c.s}) : tuple_of({h.q, h.s});
}

// silu_backward(dh, gate_up_q, gate_up_scale, mode) -> (d, its scales, dt, .., at, ..), error code, or None
PyObject* py_silu_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 4) { PyErr_SetString(PyExc_TypeError, "silu_backward takes 4 arguments"); return nullptr; }
  for (int i = 0; i < 3; ++i)
    if (!THPVariable_Check(a[i])) Py_RETURN_NONE;
  const at::Tensor &dh = THPVariable_Unpack(a[0]), &gu = THPVariable_Unpack(a[1]), &gus = THPVariable_Unpack(a[2]);
  const at::Device dev = dh.device();
  if (!on_current_device(dh) || gu.device() != dev || gus.device() != dev || dh.dim() != 2 || gu.dim() != 2 || gus.dim() != 2) Py_RETURN_NONE;
  mx_tensor dd, dg, ds;
  if (dh.scalar_type() != at::kBFloat16 || gu.scalar_type() != at::kFloat8_e4m3fn || !is_e8m0(gus) || !matrix(dh, MX_BF16, &dd) ||
      !matrix(gu, MX_E4M3, &dg) || !matrix(gus, MX_E8M0, &ds))
    Py_RETURN_NONE;
  const int64_t M = dd.shape[0], F = dd.shape[1];
  if (F % 32 != 0 || dg.shape[0] != M || dg.shape[1] != 2 * F || ds.shape[0] != M || ds.shape[1] != F / 16 || (uintptr_t)dg.ptr % 8 != 0 ||
      (M > 1 && dg.stride[0] % 8 != 0))
    Py_RETURN_NONE;
  Codes d(M, 2 * F, MX_E4M3, dev), t(2 * F, up32(M), MX_E4M3, dev), act(F, up32(M), MX_E4M3, dev);
  const int mode = (int)PyLong_AsLong(a[3]);
  int rc;
  {
    NoGil nogil;
    rc = lib.p_mx_silu_mul_backward_quantize(&dd, &dg, &ds, &d.dq, &d.ds, &t.dq, &t.ds, &act.dq, &act.ds, mode, stream_of(dev));
  }
  if (rc != MX_OK) return PyLong_FromLong(rc);
  return tuple_of({d.q, d.s, t.q, t.s, act.q, act.s});
}

struct Refused { int rc; };   // by the library, before anything was enqueued
// an input of forward-mode differentiation, which no operator here has: the Python side refuses it
bool has_tangent(std::initializer_list<const at::Tensor*> ts) {
  for (const at::Tensor* t : ts)
    if (t->defined() && t->_fw_grad(0).defined()) return true;
  return false;
}
struct FfnSizes { int64_t T, H, F, Ho; };
// the block's operands as matrices; false: not for the native path
bool ffn_operands(const at::Tensor& x, const at::Tensor& w1, const at::Tensor& w2, mx_tensor* dx, mx_tensor* d1, mx_tensor* d2, FfnSizes* s) {
  if (!on_current_device(x) || w1.device() != x.device() || w2.device() != x.device() || x.dim() < 2 || w1.dim() != 2 || w2.dim() != 2 ||
      out_code(x.scalar_type()) < 0 || out_code(w1.scalar_type()) < 0 || out_code(w2.scalar_type()) < 0)
    return false;
  if (!matrix(x, out_code(x.scalar_type()), dx) || !matrix(w1, out_code(w1.scalar_type()), d1) || !matrix(w2, out_code(w2.scalar_type()), d2)) return false;
  *s = {dx->shape[0], dx->shape[1], d1->shape[0] / 2, d2->shape[0]};
  return d1->shape[0] % 2 == 0 && d1->shape[1] == s->H && d2->shape[1] == s->F && s->H % 32 == 0 && s->F % 32 == 0 && s->Ho % 32 == 0;
}
// y, and where `saved` is given what the backward pass needs
at::Tensor ffn_forward(const at::Tensor& x, const at::Tensor& w1, const at::Tensor& w2, int mode, at::Tensor* saved) {
  mx_tensor dx, d1, d2;
  FfnSizes s;
  if (!ffn_operands(x, w1, w2, &dx, &d1, &d2, &s)) throw Refused{0};
  const at::Device dev = x.device();
  auto shape = x.sizes().vec();
  shape.back() = s.Ho;
  at::Tensor y = device_empty(shape, x.scalar_type(), dev);
  mx_tensor dy{y.data_ptr(), out_code(y.scalar_type()), 2, {s.T, s.Ho, 0, 0}, {s.Ho, 1, 0, 0}, -1, 0};
  const int64_t kept = saved ? lib.p_mx_ffn_saved_bytes(s.T, s.H, s.F, s.Ho) : 0, need = lib.p_mx_ffn_forward_workspace_bytes(s.T, s.H, s.F, s.Ho);
  if (saved) *saved = device_empty({kept}, at::kByte, dev);
  at::Tensor ws = device_empty({need}, at::kByte, dev);
  const int rc = lib.p_mx_ffn_forward(&dx, &d1, &d2, &dy, mode, saved ? saved->data_ptr() : nullptr, kept, ws.data_ptr(), need, stream_of(dev));
  if (rc != MX_OK) throw Refused{rc};
  return y;
}
// dx, dw1, dw2 (undefined where not asked for) from dy [T, Ho]
std::vector<at::Tensor> ffn_backward(const at::Tensor& dy, const at::Tensor& saved, const FfnSizes& s, const at::ScalarType (&types)[3], const bool (&want)[3],
                                     int mode) {
  const at::Device dev = dy.device();
  mx_tensor d{};
  if (!matrix(dy, float_code(dy.scalar_type()), &d)) throw Refused{0};
  const int64_t rows[3] = {s.T, 2 * s.F, s.Ho}, cols[3] = {s.H, s.H, s.F};
  std::vector<at::Tensor> out(3);
  mx_tensor od[3];
  for (int i = 0; i < 3; ++i)
    if (want[i]) {
      out[i] = device_empty({rows[i], cols[i]}, types[i], dev);
      od[i] = desc(out[i], out_code(types[i]));
    }
  const int64_t need = lib.p_mx_ffn_backward_workspace_bytes(s.T, s.H, s.F, s.Ho);
  at::Tensor ws = device_empty({need}, at::kByte, dev);
  const int rc = lib.p_mx_ffn_backward(&d, saved.data_ptr(), saved.numel(), s.H, s.F, want[0] ? &od[0] : nullptr, want[1] ? &od[1] : nullptr,
                                       want[2] ? &od[2] : nullptr, mode, ws.data_ptr(), need, stream_of(dev));
  if (rc != MX_OK) throw Refused{rc};
  return out;
}

struct FeedForward : torch::autograd::Function<FeedForward> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w1, const at::Tensor& w2, int64_t mode) {
    at::Tensor saved;
    at::Tensor y = ffn_forward(x, w1, w2, (int)mode, &saved);
    ctx->save_for_backward({saved});
    ctx->saved_data["x"] = x.sizes().vec();
    ctx->saved_data["sizes"] = std::vector<int64_t>{x.numel() / x.size(-1), x.size(-1), w2.size(1), w2.size(0), mode, (int64_t)x.scalar_type(),
                                                    (int64_t)w1.scalar_type(), (int64_t)w2.scalar_type()};
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const bool again = at::GradMode::is_enabled();
    at::AutoDispatchBelowADInplaceOrView below;
    const auto v = ctx->saved_data["sizes"].toIntVector();
    const at::ScalarType types[3] = {(at::ScalarType)v[5], (at::ScalarType)v[6], (at::ScalarType)v[7]};
    const bool want[3] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->needs_input_grad(2)};
    at::Tensor dy = grads[0].dim() == 2 ? grads[0] : grads[0].reshape({v[0], v[3]});
    if (dy.stride(1) != 1 || dy.stride(0) < 0) dy = dy.contiguous();
    std::vector<at::Tensor> r;
    try {
      r = ffn_backward(dy, ctx->get_saved_variables()[0], {v[0], v[1], v[2], v[3]}, types, want, (int)v[4]);
    } catch (const Refused& e) {
      TORCH_CHECK(false, "gated_feed_forward, backward pass: ", e.rc ? lib.p_mx_last_error() : "unexpected gradient");
    }
    const auto shape = ctx->saved_data["x"].toIntVector();
    if (want[0] && shape.size() != 2) r[0] = r[0].view(shape);
    if (again) {   // asked for a graph of the gradients: there is none, and whoever differentiates them is to be told
      for (at::Tensor& t : r)
        if (t.defined()) t.set_requires_grad(true);
      r = torch::autograd::DelayedError("gated_feed_forward: its gradients cannot be differentiated", 3)(std::move(r));
    }
    r.emplace_back();
    return r;
  }
};

// feed_forward(x, w1, w2, mode, form) -> result, error code, or None.  form 0: y without a backward pass; 1: (y, state for
// feed_forward_backward); 2: y that autograd differentiates, not under graph capture
PyObject* py_feed_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 5) { PyErr_SetString(PyExc_TypeError, "feed_forward takes 5 arguments"); return nullptr; }
  for (int i = 0; i < 3; ++i)
    if (!THPVariable_Check(a[i])) Py_RETURN_NONE;
  const at::Tensor &x = THPVariable_Unpack(a[0]), &w1 = THPVariable_Unpack(a[1]), &w2 = THPVariable_Unpack(a[2]);
  mx_tensor dx, d1, d2;
  FfnSizes s;
  if (!ffn_operands(x, w1, w2, &dx, &d1, &d2, &s)) Py_RETURN_NONE;
  const int mode = (int)PyLong_AsLong(a[3]), form = (int)PyLong_AsLong(a[4]);
  if (form != 1 && has_tangent({&x, &w1, &w2})) Py_RETURN_NONE;
  if (form == 2 && c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None) Py_RETURN_NONE;
  at::Tensor y, saved;
  int rc = MX_OK;
  {
    NoGil nogil;
    try {
      if (form == 2) {
        y = FeedForward::apply(x, w1, w2, (int64_t)mode);
      } else {
        at::AutoDispatchBelowADInplaceOrView below;
        y = ffn_forward(x, w1, w2, mode, form == 1 ? &saved : nullptr);
      }
    } catch (const Refused& e) {
      rc = e.rc;
    }
  }
  if (rc != MX_OK) return PyLong_FromLong(rc);
  return form == 1 ? tuple_of({y, saved}) : THPVariable_Wrap(y);
}

// feed_forward_backward(dy, saved, T, H, F, H_out, x_dtype, w1_dtype, w2_dtype, need_dx, need_dw1, need_dw2, mode)
//   -> [dx [T, H], dw1, dw2] with None where not asked for, error code, or None
PyObject* py_feed_forward_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 13) { PyErr_SetString(PyExc_TypeError, "feed_forward_backward takes 13 arguments"); return nullptr; }
  if (!THPVariable_Check(a[0]) || !THPVariable_Check(a[1])) Py_RETURN_NONE;
  const at::Tensor &dy = THPVariable_Unpack(a[0]), &saved = THPVariable_Unpack(a[1]);
  const FfnSizes s = {PyLong_AsLongLong(a[2]), PyLong_AsLongLong(a[3]), PyLong_AsLongLong(a[4]), PyLong_AsLongLong(a[5])};
  at::ScalarType types[3];
  bool want[3];
  for (int i = 0; i < 3; ++i) {
    if (!THPDtype_Check(a[6 + i])) Py_RETURN_NONE;
    types[i] = ((THPDtype*)a[6 + i])->scalar_type;
    want[i] = PyObject_IsTrue(a[9 + i]) == 1;
    if (out_code(types[i]) < 0) Py_RETURN_NONE;
  }
  const int mode = (int)PyLong_AsLong(a[12]);
  if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
  mx_tensor d;
  if (dy.dim() < 2 || !on_current_device(dy) || saved.device() != dy.device() || !matrix(dy, float_code(dy.scalar_type()), &d) || d.shape[0] != s.T || d.shape[1] != s.Ho ||
      !saved.is_contiguous() || saved.scalar_type() != at::kByte)
    Py_RETURN_NONE;
  std::vector<at::Tensor> r;
  int rc = MX_OK;
  {
    NoGil nogil;
    at::AutoDispatchBelowADInplaceOrView below;
    try {
      r = ffn_backward(dy, saved, s, types, want, mode);
    } catch (const Refused& e) {
      rc = e.rc;
    }
  }
  if (rc != MX_OK) return PyLong_FromLong(rc);
  return tuple_of({r[0], r[1], r[2]});
}

// ---- layer norm ---------------------------------------------------------------------------------------------------------------------
// a weight or bias: undefined, or a contiguous vector of H on the device
bool norm_vector(const at::Tensor& t, int64_t H, const at::Device& dev, mx_tensor* d) {
  if (!t.defined()) return true;
  if (t.dim() != 1 || t.size(0) != H || !t.is_contiguous() || t.device() != dev || float_code(t.scalar_type()) < 0) return false;
  *d = desc(t, float_code(t.scalar_type()));
  return true;
}
// an argument that is a tensor or None; false: neither
bool optional_tensor(PyObject* o, at::Tensor* t) {
  if (o == Py_None) return true;
  if (!THPVariable_Check(o)) return false;
  *t = THPVariable_Unpack(o);
  return true;
}
bool norm_operands(const at::Tensor& x, const at::Tensor& w, const at::Tensor& b, mx_tensor* dx, mx_tensor* dw, mx_tensor* db) {
  return on_current_device(x) && matrix(x, float_code(x.scalar_type()), dx) && norm_vector(w, dx->shape[1], x.device(), dw) &&
         norm_vector(b, dx->shape[1], x.device(), db);
}
mx_tensor rows_of(const at::Tensor& t, int dtype, const mx_tensor& like) {   // a dense tensor as like's matrix
  return mx_tensor{t.data_ptr(), dtype, 2, {like.shape[0], like.shape[1], 0, 0}, {like.shape[1], 1, 0, 0}, -1, 0};
}
at::Tensor norm_forward(const at::Tensor& x, const at::Tensor& w, const at::Tensor& b, double eps, at::Tensor* mean, at::Tensor* rstd) {
  mx_tensor dx, dw, db, dm, dr;
  if (!norm_operands(x, w, b, &dx, &dw, &db)) throw Refused{0};
  const at::Device dev = x.device();
  at::Tensor y = device_empty(x.sizes(), x.scalar_type(), dev);
  mx_tensor dy = rows_of(y, dx.dtype, dx);
  if (mean) {
    *mean = device_empty({dx.shape[0]}, at::kFloat, dev);
    *rstd = device_empty({dx.shape[0]}, at::kFloat, dev);
    dm = desc(*mean, MX_F32);
    dr = desc(*rstd, MX_F32);
  }
  const int rc = lib.p_mx_layer_norm(&dx, w.defined() ? &dw : nullptr, b.defined() ? &db : nullptr, eps, &dy, mean ? &dm : nullptr, mean ? &dr : nullptr,
                                     stream_of(dev));
  if (rc != MX_OK) throw Refused{rc};
  return y;
}
// dx, dweight, dbias (undefined where not asked for)
std::vector<at::Tensor> norm_backward(const at::Tensor& dy, const at::Tensor& x, const at::Tensor& mean, const at::Tensor& rstd, const at::Tensor& w,
                                      const bool (&want)[3], at::ScalarType b_type) {
  mx_tensor dx, dw, db, ddy, o[3];
  if (!norm_operands(x, w, at::Tensor(), &dx, &dw, &db) || dy.device() != x.device() || dy.scalar_type() != x.scalar_type() || !matrix(dy, dx.dtype, &ddy) ||
      ddy.shape[0] != dx.shape[0] || ddy.shape[1] != dx.shape[1])
    throw Refused{0};
  const at::Device dev = x.device();
  for (const at::Tensor* t : {&mean, &rstd})
    if (t->dim() != 1 || t->size(0) != dx.shape[0] || t->scalar_type() != at::kFloat || !t->is_contiguous() || t->device() != dev) throw Refused{0};
  std::vector<at::Tensor> out(3);
  if (want[0]) {
    out[0] = device_empty(x.sizes(), x.scalar_type(), dev);
    o[0] = rows_of(out[0], dx.dtype, dx);
  }
  for (int i = 1; i < 3; ++i)
    if (want[i]) {
      out[i] = device_empty({dx.shape[1]}, i == 2 ? b_type : w.defined() ? w.scalar_type() : at::kFloat, dev);
      o[i] = desc(out[i], float_code(out[i].scalar_type()));
    }
  const int64_t need = want[1] || want[2] ? lib.p_mx_layer_norm_backward_workspace_bytes(dx.shape[0], dx.shape[1]) : 0;
  at::Tensor ws;
  if (need > 0) ws = device_empty({need}, at::kByte, dev);
  mx_tensor dm = desc(mean, MX_F32), dr = desc(rstd, MX_F32);
  const int rc = lib.p_mx_layer_norm_backward(&ddy, &dx, &dm, &dr, w.defined() ? &dw : nullptr, want[0] ? &o[0] : nullptr, want[1] ? &o[1] : nullptr,
                                              want[2] ? &o[2] : nullptr, need > 0 ? ws.data_ptr() : nullptr, need, stream_of(dev));
  if (rc != MX_OK) throw Refused{rc};
  return out;
}
// gradients of a call that was asked for their graph: there is none, and whoever differentiates them is to be told
std::vector<at::Tensor> without_graph(std::vector<at::Tensor> r, const char* what) {
  for (at::Tensor& t : r)
    if (t.defined()) t.set_requires_grad(true);
  const int n = (int)r.size();
  return torch::autograd::DelayedError(what, n)(std::move(r));
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const std::optional<at::Tensor>& ow,
                            const std::optional<at::Tensor>& ob, double eps) {
    const at::Tensor w = ow.value_or(at::Tensor()), b = ob.value_or(at::Tensor());
    at::Tensor mean, rstd, y = norm_forward(x, w, b, eps, &mean, &rstd);
    ctx->save_for_backward({x, w, mean, rstd});
    ctx->saved_data["bias"] = (int64_t)(b.defined() ? b.scalar_type() : at::ScalarType::Undefined);
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const bool again = at::GradMode::is_enabled();
    at::AutoDispatchBelowADInplaceOrView below;
    const auto s = ctx->get_saved_variables();
    const auto b_type = (at::ScalarType)ctx->saved_data["bias"].toInt();
    // (edges are counted over the tensors that there are)
    const bool has_w = s[1].defined(), has_b = b_type != at::ScalarType::Undefined;
    const bool want[3] = {ctx->needs_input_grad(0), has_w && ctx->needs_input_grad(1), has_b && ctx->needs_input_grad(has_w ? 2 : 1)};
    at::Tensor dy = grads[0], x = s[0];
    mx_tensor d;
    if (dy.scalar_type() != x.scalar_type()) dy = dy.to(x.scalar_type());
    if (!matrix(dy, float_code(dy.scalar_type()), &d)) dy = dy.contiguous();
    std::vector<at::Tensor> r;
    try {
      r = norm_backward(dy, x, s[2], s[3], s[1], want, b_type);
    } catch (const Refused& e) {
      TORCH_CHECK(false, "layer_norm, backward pass: ", e.rc ? lib.p_mx_last_error() : "unexpected gradient");
    }
    if (again) r = without_graph(std::move(r), "layer_norm: its gradients cannot be differentiated");
    r.emplace_back();
    return r;
  }
};

// layer_norm(x, weight, bias, eps, form) -> result, error code, or None.  form 0: y; 1: (y, mean, rstd); 2: y that autograd
// differentiates, not under graph capture
PyObject* py_layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 5) { PyErr_SetString(PyExc_TypeError, "layer_norm takes 5 arguments"); return nullptr; }
  at::Tensor w, b;
  if (!THPVariable_Check(a[0]) || !optional_tensor(a[1], &w) || !optional_tensor(a[2], &b)) Py_RETURN_NONE;
  const at::Tensor& x = THPVariable_Unpack(a[0]);
  const double eps = PyFloat_AsDouble(a[3]);
  const int form = (int)PyLong_AsLong(a[4]);
  if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
  mx_tensor dx, dw, db;
  if (!norm_operands(x, w, b, &dx, &dw, &db)) Py_RETURN_NONE;
  if (form != 1 && has_tangent({&x, &w, &b})) Py_RETURN_NONE;
  if (form == 2 && c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None) Py_RETURN_NONE;
  at::Tensor y, mean, rstd;
  int rc = MX_OK;
  {
    NoGil nogil;
    try {
      if (form == 2) {
        const auto optional = [](const at::Tensor& t) { return t.defined() ? std::optional<at::Tensor>(t) : std::nullopt; };
        y = LayerNorm::apply(x, optional(w), optional(b), eps);
      } else {
        at::AutoDispatchBelowADInplaceOrView below;
        y = norm_forward(x, w, b, eps, form == 1 ? &mean : nullptr, &rstd);
      }
    } catch (const Refused& e) {
      rc = e.rc;
    }
  }
  if (rc != MX_OK) return PyLong_FromLong(rc);
  return form == 1 ? tuple_of({y, mean, rstd}) : THPVariable_Wrap(y);
}

// layer_norm_backward(dy, x, mean, rstd, weight, need_dx, need_dweight, need_dbias) -> (dx, dweight, dbias) with None where not asked for,
// error code, or None; dweight and dbias have weight's type (float32 without a weight)
PyObject* py_layer_norm_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 8) { PyErr_SetString(PyExc_TypeError, "layer_norm_backward takes 8 arguments"); return nullptr; }
  for (int i = 0; i < 4; ++i)
    if (!THPVariable_Check(a[i])) Py_RETURN_NONE;
  at::Tensor w;
  if (!optional_tensor(a[4], &w)) Py_RETURN_NONE;
  const at::Tensor &dy = THPVariable_Unpack(a[0]), &x = THPVariable_Unpack(a[1]), &mean = THPVariable_Unpack(a[2]), &rstd = THPVariable_Unpack(a[3]);
  const bool want[3] = {PyObject_IsTrue(a[5]) == 1, PyObject_IsTrue(a[6]) == 1, PyObject_IsTrue(a[7]) == 1};
  std::vector<at::Tensor> r;
  int rc = MX_OK;
  {
    NoGil nogil;
    at::AutoDispatchBelowADInplaceOrView below;
    try {
      r = norm_backward(dy, x, mean, rstd, w, want, w.defined() ? w.scalar_type() : at::kFloat);
    } catch (const Refused& e) {
      rc = e.rc ? e.rc : 1;
    }
  }
  if (rc == 1) Py_RETURN_NONE;
  if (rc != MX_OK) return PyLong_FromLong(rc);
  return tuple_of({r[0], r[1], r[2]});
}

// layer_norm_quantize(x, weight, bias, dtype | str, eps, mode) -> (elements, scales), error code, or None
PyObject* py_layer_norm_quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 6) { PyErr_SetString(PyExc_TypeError, "layer_norm_quantize takes 6 arguments"); return nullptr; }
  at::Tensor w, b;
  if (!THPVariable_Check(a[0]) || !optional_tensor(a[1], &w) || !optional_tensor(a[2], &b)) Py_RETURN_NONE;
  const at::Tensor& x = THPVariable_Unpack(a[0]);
  const int fmt = format_of(a[3]);                     // (8-bit formats)
  const double eps = PyFloat_AsDouble(a[4]);
  const int mode = (int)PyLong_AsLong(a[5]);
  if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
  mx_tensor dx, dw, db;
  if (fmt < 0 || !norm_operands(x, w, b, &dx, &dw, &db) || dx.shape[1] < 32) Py_RETURN_NONE;
  const at::Device dev = x.device();
  Codes c(dx.shape[0], up32(dx.shape[1]), fmt, dev);
  int rc;
  {
    NoGil nogil;
    rc = lib.p_mx_layer_norm_quantize(&dx, w.defined() ? &dw : nullptr, b.defined() ? &db : nullptr, eps, &c.dq, &c.ds, mode, stream_of(dev));
  }
  if (rc != MX_OK) return PyLong_FromLong(rc);
  if (x.dim() != 2) {
    auto shape = x.sizes().vec();
    shape.back() = up32(dx.shape[1]);
    c.q = c.q.view(shape);
    shape.back() /= 32;
    c.s = c.s.view(shape);
  }
  return tuple_of({c.q, c.s});
}

// ---- the linear layer -----------------------------------------------------------------------------------------------------------------
// bias and residual of a result with the sizes `shape` (last: N); false: not for the native path
bool around(const at::Tensor& bias, const at::Tensor& res, at::IntArrayRef shape, const at::Device& dev, mx_tensor* db, mx_tensor* dr) {
  if (!norm_vector(bias, shape.back(), dev, db)) return false;
  return !res.defined() || (res.device() == dev && res.sizes() == shape && matrix(res, float_code(res.scalar_type()), dr));
}

// linear_gemm(A, A_scale, W, W_scale, bias, residual, a_format, w_format, out_dtype, act, kernel) -> result or tuple, error code, or None
PyObject* py_linear_gemm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 11) { PyErr_SetString(PyExc_TypeError, "linear_gemm takes 11 arguments"); return nullptr; }
  at::Tensor bias, res;
  if (!THPVariable_Check(a[0]) || !THPVariable_Check(a[2]) || !optional_tensor(a[4], &bias) || !optional_tensor(a[5], &res)) Py_RETURN_NONE;
  const at::Tensor &A = THPVariable_Unpack(a[0]), &W = THPVariable_Unpack(a[2]);
  if (A.dim() != 2 || W.dim() != 2 || !on_current_device(A) || W.device() != A.device()) Py_RETURN_NONE;
  const int fa = elem_format(A, a[6]), fw = elem_format(W, a[7]);
  if (fa < 0 || fw < 0 || A.stride(1) != 1 || W.stride(1) != 1) Py_RETURN_NONE;
  const at::Device dev = A.device();
  const mx_tensor dA = desc(A, fa, fa == MX_E2M1 ? 1 : -1), dW = desc(W, fw, fw == MX_E2M1 ? 1 : -1);
  const int64_t M = dA.shape[0], K = dA.shape[1], N = dW.shape[0], shape[2] = {M, N};
  if (M == 0 || K == 0 || N == 0 || dW.shape[1] != K) Py_RETURN_NONE;
  mx_tensor dAs, dWs, db, dr;
  mx_gemm_opts o = {sizeof(mx_gemm_opts), 0, 0, 0, (int32_t)PyLong_AsLong(a[10]), 32, 0, 0};
  if (!scale_desc(a[1], M, K, false, dev, &dAs, &o.a_scale_layout) || !scale_desc(a[3], N, K, true, dev, &dWs, &o.b_scale_layout) ||
      !around(bias, res, shape, dev, &db, &dr))
    Py_RETURN_NONE;
  int fo = THPDtype_Check(a[8]) ? out_code(((THPDtype*)a[8])->scalar_type) : -1;
  if (fo < 0) fo = format_of(a[8]);
  const int act = (int)PyLong_AsLong(a[9]);
  if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
  if (fo < 0 || fo == MX_E5M2 || (fo == MX_E4M3 && N % 32 != 0)) Py_RETURN_NONE;
  Codes c;
  if (fo == MX_E4M3) {
    c = Codes(M, N, MX_E4M3, dev);
  } else {
    c.q = device_empty({M, N}, fo == MX_F32 ? at::kFloat : at::kBFloat16, dev);
    c.dq = desc(c.q, fo);
  }
  const int64_t need = lib.p_mx_linear_gemm_workspace_bytes(M, N, K, &o);
  at::Tensor ws;
  if (need > 0) ws = device_empty({need}, at::kByte, dev);
  int rc;
  {
    NoGil nogil;
    rc = lib.p_mx_linear_gemm(&dA, &dAs, &dW, &dWs, bias.defined() ? &db : nullptr, res.defined() ? &dr : nullptr, act, &c.dq, fo == MX_E4M3 ? &c.ds : nullptr,
                              nullptr, &o, need > 0 ? ws.data_ptr() : nullptr, need, stream_of(dev));
  }
  if (rc != MX_OK) return PyLong_FromLong(rc);
  return fo == MX_E4M3 ? tuple_of({c.q, c.s}) : THPVariable_Wrap(c.q);
}

struct LinearSizes { int64_t T, K, N; };
bool linear_operands(const at::Tensor& x, const at::Tensor& w, const at::Tensor& bias, const at::Tensor& res, mx_tensor* dx, mx_tensor* dw, mx_tensor* db,
                     mx_tensor* dr, LinearSizes* s) {
  if (!on_current_device(x) || w.device() != x.device() || x.dim() < 2 || w.dim() != 2 || out_code(x.scalar_type()) < 0 || out_code(w.scalar_type()) < 0 ||
      !matrix(x, out_code(x.scalar_type()), dx) || !matrix(w, out_code(w.scalar_type()), dw))
    return false;
  *s = {dx->shape[0], dx->shape[1], dw->shape[0]};
  if (dw->shape[1] != s->K || s->K % 32 != 0 || s->N % 32 != 0) return false;
  auto shape = x.sizes().vec();
  shape.back() = s->N;
  return around(bias, res, shape, x.device(), db, dr);
}
at::Tensor linear_forward(const at::Tensor& x, const at::Tensor& w, const at::Tensor& bias, const at::Tensor& res, int act, int mode, at::Tensor* saved) {
  mx_tensor dx, dw, db, dr;
  LinearSizes s;
  if (!linear_operands(x, w, bias, res, &dx, &dw, &db, &dr, &s)) throw Refused{0};
  const at::Device dev = x.device();
  auto shape = x.sizes().vec();
  shape.back() = s.N;
  at::Tensor y = device_empty(shape, x.scalar_type(), dev);
  mx_tensor dy{y.data_ptr(), dx.dtype, 2, {s.T, s.N, 0, 0}, {s.N, 1, 0, 0}, -1, 0};
  const int64_t kept = saved ? lib.p_mx_linear_saved_bytes(s.T, s.K, s.N, act) : 0, need = lib.p_mx_linear_forward_workspace_bytes(s.T, s.K, s.N);
  if (saved) *saved = device_empty({kept}, at::kByte, dev);
  at::Tensor ws = device_empty({need}, at::kByte, dev);
  const int rc = lib.p_mx_linear_forward(&dx, &dw, bias.defined() ? &db : nullptr, res.defined() ? &dr : nullptr, act, &dy, mode,
                                         saved ? saved->data_ptr() : nullptr, kept, ws.data_ptr(), need, stream_of(dev));
  if (rc != MX_OK) throw Refused{rc};
  return y;
}
// dx, dw, dbias (undefined where not asked for) from dy [T, N]
std::vector<at::Tensor> linear_backward(at::Tensor dy, const at::Tensor& saved, const LinearSizes& s, const at::ScalarType (&types)[3],
                                        const bool (&want)[3], int act, int mode) {
  const at::Device dev = dy.device();
  mx_tensor d{};
  if (!matrix(dy, float_code(dy.scalar_type()), &d)) throw Refused{0};
  if (s.T > 1 && d.stride[0] > (int64_t)1 << 25) {   // rows farther apart than the library takes them
    dy = dy.contiguous();
    matrix(dy, d.dtype, &d);
  }
  std::vector<at::Tensor> out(3);
  mx_tensor od[3];
  for (int i = 0; i < 3; ++i)
    if (want[i]) {
      out[i] = i == 2 ? device_empty({s.N}, types[i], dev) : device_empty({i == 0 ? s.T : s.N, s.K}, types[i], dev);
      od[i] = desc(out[i], float_code(types[i]));
    }
  const int64_t need = lib.p_mx_linear_backward_workspace_bytes(s.T, s.K, s.N);
  at::Tensor ws = device_empty({need}, at::kByte, dev);
  const int rc = lib.p_mx_linear_backward(&d, saved.data_ptr(), saved.numel(), s.K, act, want[0] ? &od[0] : nullptr, want[1] ? &od[1] : nullptr,
                                          want[2] ? &od[2] : nullptr, mode, ws.data_ptr(), need, stream_of(dev));
  if (rc != MX_OK) throw Refused{rc};
  return out;
}

struct Linear : torch::autograd::Function<Linear> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& bias,
                            const std::optional<at::Tensor>& res, int64_t act, int64_t mode) {
    at::Tensor saved, y = linear_forward(x, w, bias.value_or(at::Tensor()), res.value_or(at::Tensor()), (int)act, (int)mode, &saved);
    ctx->save_for_backward({saved});
    ctx->saved_data["x"] = x.sizes().vec();
    ctx->saved_data["sizes"] = std::vector<int64_t>{x.numel() / x.size(-1), x.size(-1), w.size(0), act, mode, (int64_t)x.scalar_type(), (int64_t)w.scalar_type(),
                                                    bias ? (int64_t)bias->scalar_type() : -1, res ? (int64_t)res->scalar_type() : -1};
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const bool again = at::GradMode::is_enabled();
    const auto v = ctx->saved_data["sizes"].toIntVector();
    const bool has_b = v[7] >= 0, has_r = v[8] >= 0;
    const bool want_r = has_r && ctx->needs_input_grad(has_b ? 3 : 2);
    at::Tensor dr;
    if (want_r) dr = grads[0].to((at::ScalarType)v[8]);   // (recorded, if a graph of the gradients is asked for: this one has one)
    at::AutoDispatchBelowADInplaceOrView below;
    const at::ScalarType types[3] = {(at::ScalarType)v[5], (at::ScalarType)v[6], has_b ? (at::ScalarType)v[7] : at::kFloat};
    // (edges are counted over the tensors that there are)
    const bool want[3] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), has_b && ctx->needs_input_grad(2)};
    at::Tensor dy = grads[0].dim() == 2 ? grads[0] : grads[0].reshape({v[0], v[2]});
    if (dy.stride(1) != 1 || dy.stride(0) < 0) dy = dy.contiguous();
    std::vector<at::Tensor> r(3);
    if (want[0] || want[1] || want[2]) {
      try {
        r = linear_backward(dy, ctx->get_saved_variables()[0], {v[0], v[1], v[2]}, types, want, (int)v[3], (int)v[4]);
      } catch (const Refused& e) {
        TORCH_CHECK(false, "linear, backward pass: ", e.rc ? lib.p_mx_last_error() : "unexpected gradient");
      }
    }
    const auto shape = ctx->saved_data["x"].toIntVector();
    if (want[0] && shape.size() != 2) r[0] = r[0].view(shape);
    if (again) r = without_graph(std::move(r), "linear: its gradients cannot be differentiated");
    r.push_back(dr);
    r.emplace_back();
    r.emplace_back();
    return r;
  }
};

// linear(x, w, bias, residual, act, mode, form) -> result, error code, or None.  form 0: y without a backward pass; 1: (y, state for
// linear_backward); 2: y that autograd differentiates, not under graph capture
PyObject* py_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 7) { PyErr_SetString(PyExc_TypeError, "linear takes 7 arguments"); return nullptr; }
  at::Tensor bias, res;
  if (!THPVariable_Check(a[0]) || !THPVariable_Check(a[1]) || !optional_tensor(a[2], &bias) || !optional_tensor(a[3], &res)) Py_RETURN_NONE;
  const at::Tensor &x = THPVariable_Unpack(a[0]), &w = THPVariable_Unpack(a[1]);
  mx_tensor dx, dw, db, dr;
  LinearSizes s;
  if (!linear_operands(x, w, bias, res, &dx, &dw, &db, &dr, &s)) Py_RETURN_NONE;
  const int act = (int)PyLong_AsLong(a[4]), mode = (int)PyLong_AsLong(a[5]), form = (int)PyLong_AsLong(a[6]);
  if (form != 1 && has_tangent({&x, &w, &bias, &res})) Py_RETURN_NONE;
  if (form == 2 && c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None) Py_RETURN_NONE;
  at::Tensor y, saved;
  int rc = MX_OK;
  {
    NoGil nogil;
    try {
      if (form == 2) {
        const auto optional = [](const at::Tensor& t) { return t.defined() ? std::optional<at::Tensor>(t) : std::nullopt; };
        y = Linear::apply(x, w, optional(bias), optional(res), (int64_t)act, (int64_t)mode);
      } else {
        at::AutoDispatchBelowADInplaceOrView below;
        y = linear_forward(x, w, bias, res, act, mode, form == 1 ? &saved : nullptr);
      }
    } catch (const Refused& e) {
      rc = e.rc;
    }
  }
  if (rc != MX_OK) return PyLong_FromLong(rc);
  return form == 1 ? tuple_of({y, saved}) : THPVariable_Wrap(y);
}

// linear_backward(dy, saved, T, K, N, x_dtype, w_dtype, bias_dtype, need_dx, need_dw, need_dbias, act, mode)
//   -> (dx [T, K], dw, dbias) with None where not asked for, error code, or None
PyObject* py_linear_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 13) { PyErr_SetString(PyExc_TypeError, "linear_backward takes 13 arguments"); return nullptr; }
  if (!THPVariable_Check(a[0]) || !THPVariable_Check(a[1])) Py_RETURN_NONE;
  const at::Tensor &dy = THPVariable_Unpack(a[0]), &saved = THPVariable_Unpack(a[1]);
  const LinearSizes s = {PyLong_AsLongLong(a[2]), PyLong_AsLongLong(a[3]), PyLong_AsLongLong(a[4])};
  at::ScalarType types[3];
  bool want[3];
  for (int i = 0; i < 3; ++i) {
    if (!THPDtype_Check(a[5 + i])) Py_RETURN_NONE;
    types[i] = ((THPDtype*)a[5 + i])->scalar_type;
    want[i] = PyObject_IsTrue(a[8 + i]) == 1;
    if ((i < 2 ? out_code(types[i]) : float_code(types[i])) < 0) Py_RETURN_NONE;
  }
  const int act = (int)PyLong_AsLong(a[11]), mode = (int)PyLong_AsLong(a[12]);
  if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
  mx_tensor d;
  if (dy.dim() < 2 || !on_current_device(dy) || saved.device() != dy.device() || !matrix(dy, float_code(dy.scalar_type()), &d) || d.shape[0] != s.T ||
      d.shape[1] != s.N || !saved.is_contiguous() || saved.scalar_type() != at::kByte)
    Py_RETURN_NONE;
  std::vector<at::Tensor> r;
  int rc = MX_OK;
  {
    NoGil nogil;
    at::AutoDispatchBelowADInplaceOrView below;
    try {
      r = linear_backward(dy, saved, s, types, want, act, mode);
    } catch (const Refused& e) {
      rc = e.rc;
    }
  }
  if (rc != MX_OK) return PyLong_FromLong(rc);
  return tuple_of({r[0], r[1], r[2]});
}

// ---- AdamW --------------------------------------------------------------------------------------------------------------------------
// a number, or a tensor of one element of type `t` on the device; false: neither
bool number_or_tensor(PyObject* o, at::ScalarType t, const at::Device& dev, double* v, const void** at) {
  if (THPVariable_Check(o)) {
    const at::Tensor& x = THPVariable_Unpack(o);
    if (x.scalar_type() != t || x.numel() != 1 || x.device() != dev) return false;
    *at = x.data_ptr();
    return true;
  }
  *v = PyFloat_AsDouble(o);
  if (PyErr_Occurred()) { PyErr_Clear(); return false; }
  return true;
}
inline void written(const at::Tensor& t) {   // behind torch's back: whoever saved it for a backward pass is to be told
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
// adamw(params, grads, states, copies | None, step, lr, beta1, beta2, eps, weight_decay, grad_scale, seed) -> True, error code, or None
PyObject* py_adamw(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 12) { PyErr_SetString(PyExc_TypeError, "adamw takes 12 arguments"); return nullptr; }
  auto seq = [](PyObject* o) { return PyList_Check(o) || PyTuple_Check(o); };
  if (!seq(a[0]) || !seq(a[1]) || !seq(a[2]) || (a[3] != Py_None && !seq(a[3]))) Py_RETURN_NONE;
  const Py_ssize_t cnt = PySequence_Fast_GET_SIZE(a[0]);
  if (cnt == 0 || cnt > 1 << 24) Py_RETURN_NONE;
  for (int i = 1; i < 4; ++i)
    if (a[i] != Py_None && PySequence_Fast_GET_SIZE(a[i]) != cnt) Py_RETURN_NONE;
  std::vector<mx_adamw_tensor> list(cnt);
  // what is written to (parameters, copies, states in tuples, which hold their tensors), and the gradients: the lists may change while the
  // GIL is released
  struct Kept : std::vector<PyObject*> {
    void hold(PyObject* o) { Py_INCREF(o); push_back(o); }
    ~Kept() { for (PyObject* o : *this) Py_DECREF(o); }
  } kept, grads;
  kept.reserve(3 * cnt);
  grads.reserve(cnt);
  at::Device dev(at::kCUDA);
  int bits = 0;
  for (Py_ssize_t i = 0; i < cnt; ++i) {
    auto item = [&](int k) { return PySequence_Fast_GET_ITEM(a[k], i); };
    PyObject* const state = item(2);
    if (!THPVariable_Check(item(0)) || !PyTuple_Check(state) || PyTuple_GET_SIZE(state) != 4) Py_RETURN_NONE;
    const at::Tensor& p = THPVariable_Unpack(item(0));
    if (i == 0) {
      if (!on_current_device(p)) Py_RETURN_NONE;
      dev = p.device();
    }
    mx_adamw_tensor& t = list[i];
    t = mx_adamw_tensor{};
    t.n = p.numel();
    t.param_dtype = out_code(p.scalar_type());
    if (t.param_dtype < 0 || p.device() != dev || !p.is_contiguous()) Py_RETURN_NONE;
    t.grad_dtype = MX_F32;
    if (item(1) == Py_None) { t.n = 0; continue; }      // no gradient: nothing to do
    if (!THPVariable_Check(item(1))) Py_RETURN_NONE;
    const at::Tensor& g = THPVariable_Unpack(item(1));
    if (g.layout() != at::kStrided || g.device() != dev || g.sizes() != p.sizes() || !g.is_contiguous()) Py_RETURN_NONE;
    t.grad_dtype = out_code(g.scalar_type());
    if (t.grad_dtype < 0) Py_RETURN_NONE;
    PyObject* s[4];
    for (int k = 0; k < 4; ++k) s[k] = PyTuple_GET_ITEM(state, k);
    if (!THPVariable_Check(s[0]) || !THPVariable_Check(s[1])) Py_RETURN_NONE;
    const int b = THPVariable_Unpack(s[0]).scalar_type() == at::kFloat ? 32 : 8;
    if (bits != 0 && b != bits) Py_RETURN_NONE;
    bits = b;
    void* at[4] = {};
    for (int k = 0; k < (b == 8 ? 4 : 2); ++k) {
      if (!THPVariable_Check(s[k])) Py_RETURN_NONE;
      const at::Tensor& x = THPVariable_Unpack(s[k]);
      const int64_t want = b == 32 ? t.n : k < 2 ? up32(t.n) : up32(t.n) / 32;
      const auto type = b == 32 ? at::kFloat : k < 2 ? at::kFloat8_e4m3fn : at::kFloat8_e8m0fnu;
      if (x.scalar_type() != type || x.numel() != want || x.device() != dev || !x.is_contiguous()) Py_RETURN_NONE;
      at[k] = x.data_ptr();
    }
    if (b == 32 && (s[2] != Py_None || s[3] != Py_None)) Py_RETURN_NONE;
    t.param = p.data_ptr(); t.grad = g.data_ptr();
    grads.hold(item(1));
    t.exp_avg = at[0]; t.exp_avg_sq = at[1]; t.exp_avg_scale = at[2]; t.exp_avg_sq_scale = at[3];
    kept.hold(item(0));
    kept.hold(state);
    if (a[3] != Py_None && item(3) != Py_None) {
      if (!THPVariable_Check(item(3))) Py_RETURN_NONE;
      const at::Tensor& c = THPVariable_Unpack(item(3));
      if (c.scalar_type() != at::kBFloat16 || c.sizes() != p.sizes() || c.device() != dev || !c.is_contiguous()) Py_RETURN_NONE;
      t.copy = c.data_ptr();
      kept.hold(item(3));
    }
  }
  mx_adamw_opts o = {};
  o.struct_size = sizeof(o);
  o.state_bits = bits ? bits : 32;
  const void *step_at = nullptr, *lr_at = nullptr, *scale_at = nullptr;
  if (THPVariable_Check(a[4])) {
    double unused;
    if (!number_or_tensor(a[4], at::kLong, dev, &unused, &step_at)) Py_RETURN_NONE;
  } else {
    o.step = PyLong_AsLongLong(a[4]);
  }
  if (!number_or_tensor(a[5], at::kFloat, dev, &o.lr, &lr_at) || !number_or_tensor(a[10], at::kFloat, dev, &o.grad_scale, &scale_at)) Py_RETURN_NONE;
  o.beta1 = PyFloat_AsDouble(a[6]); o.beta2 = PyFloat_AsDouble(a[7]); o.eps = PyFloat_AsDouble(a[8]); o.weight_decay = PyFloat_AsDouble(a[9]);
  o.seed = (uint32_t)PyLong_AsUnsignedLongMask(a[11]);
  if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
  o.step_at = (const int64_t*)step_at; o.lr_at = (const float*)lr_at; o.scale_at = (const float*)scale_at;
  int rc;
  {
    NoGil nogil;
    rc = lib.p_mx_adamw_step((int32_t)cnt, list.data(), &o, stream_of(dev));
  }
  if (rc != MX_OK) return PyLong_FromLong(rc);
  for (PyObject* k : kept) {
    if (!PyTuple_Check(k)) written(THPVariable_Unpack(k));
    else
      for (int i = 0; i < (bits == 8 ? 4 : 2); ++i) written(THPVariable_Unpack(PyTuple_GET_ITEM(k, i)));
  }
  Py_RETURN_TRUE;
}

// bind(handle of the loaded libmxgemm.so, PackedScales class)
PyObject* py_bind(PyObject*, PyObject* args) {
  unsigned long long h;
  PyObject* cls;
  if (!PyArg_ParseTuple(args, "KO", &h, &cls)) return nullptr;
#define MX_FN(name)                                                                      \
  if (!(lib.p_##name = (decltype(lib.p_##name))dlsym((void*)h, #name))) {                \
    PyErr_SetString(PyExc_RuntimeError, "libmxgemm.so does not export " #name);          \
    return nullptr;                                                                      \
  }
  MX_FN(mx_gemm)
  MX_FN(mx_gemm_add)
  MX_FN(mx_gemm_workspace_bytes)
  MX_FN(mx_packed_scale_bytes)
  MX_FN(mx_gemm_list)
  MX_FN(mx_gemm_list_workspace_bytes)
  MX_FN(mx_quantize)
  MX_FN(mx_silu_mul_quantize)
  MX_FN(mx_moe_forward)
  MX_FN(mx_moe_forward_workspace_bytes)
  MX_FN(mx_last_error)
  MX_FN(mx_quantize_both)
  MX_FN(mx_gated_gemm)
  MX_FN(mx_gated_gemm_workspace_bytes)
  MX_FN(mx_silu_mul_backward_quantize)
  MX_FN(mx_ffn_saved_bytes)
  MX_FN(mx_ffn_forward)
  MX_FN(mx_ffn_forward_workspace_bytes)
  MX_FN(mx_ffn_backward)
  MX_FN(mx_ffn_backward_workspace_bytes)
  MX_FN(mx_layer_norm)
  MX_FN(mx_layer_norm_quantize)
  MX_FN(mx_layer_norm_backward_workspace_bytes)
  MX_FN(mx_layer_norm_backward)
  MX_FN(mx_adamw_step)
  MX_FN(mx_linear_gemm)
  MX_FN(mx_linear_gemm_workspace_bytes)
  MX_FN(mx_linear_saved_bytes)
  MX_FN(mx_linear_forward)
  MX_FN(mx_linear_forward_workspace_bytes)
  MX_FN(mx_linear_backward)
  MX_FN(mx_linear_backward_workspace_bytes)
#undef MX_FN
  Py_INCREF(cls);
  Py_XDECREF(packed_type);
  packed_type = cls;
  Py_RETURN_NONE;
}

// torch and allocator errors (out of memory, ...) become Python exceptions of the same kind
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  return F(self, a, n);
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"bind", py_bind, METH_VARARGS, nullptr},
    {"gemm", (PyCFunction)(void (*)(void))guarded<py_gemm>, METH_FASTCALL, nullptr},
    {"gemm_list", (PyCFunction)(void (*)(void))guarded<py_gemm_list>, METH_FASTCALL, nullptr},
    {"mma", (PyCFunction)(void (*)(void))guarded<py_mma>, METH_FASTCALL, nullptr},
    {"quantize", (PyCFunction)(void (*)(void))guarded<py_quantize>, METH_FASTCALL, nullptr},
    {"moe", (PyCFunction)(void (*)(void))guarded<py_moe>, METH_FASTCALL, nullptr},
    {"quantize_both", (PyCFunction)(void (*)(void))guarded<py_quantize_both>, METH_FASTCALL, nullptr},
    {"gated", (PyCFunction)(void (*)(void))guarded<py_gated>, METH_FASTCALL, nullptr},
    {"silu_backward", (PyCFunction)(void (*)(void))guarded<py_silu_backward>, METH_FASTCALL, nullptr},
    {"feed_forward", (PyCFunction)(void (*)(void))guarded<py_feed_forward>, METH_FASTCALL, nullptr},
    {"feed_forward_backward", (PyCFunction)(void (*)(void))guarded<py_feed_forward_backward>, METH_FASTCALL, nullptr},
    {"layer_norm", (PyCFunction)(void (*)(void))guarded<py_layer_norm>, METH_FASTCALL, nullptr},
    {"layer_norm_backward", (PyCFunction)(void (*)(void))guarded<py_layer_norm_backward>, METH_FASTCALL, nullptr},
    {"layer_norm_quantize", (PyCFunction)(void (*)(void))guarded<py_layer_norm_quantize>, METH_FASTCALL, nullptr},
    {"linear_gemm", (PyCFunction)(void (*)(void))guarded<py_linear_gemm>, METH_FASTCALL, nullptr},
    {"linear", (PyCFunction)(void (*)(void))guarded<py_linear>, METH_FASTCALL, nullptr},
    {"linear_backward", (PyCFunction)(void (*)(void))guarded<py_linear_backward>, METH_FASTCALL, nullptr},
    {"adamw", (PyCFunction)(void (*)(void))guarded<py_adamw>, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_mxhost", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__mxhost(void) {
  s_data = PyUnicode_InternFromString("data");
  s_rows = PyUnicode_InternFromString("rows");
  s_K = PyUnicode_InternFromString("K");
  s_operand = PyUnicode_InternFromString("operand");
  s_layout = PyUnicode_InternFromString("layout");
  s_batch = PyUnicode_InternFromString("batch");
  return PyModule_Create(&module);
}
