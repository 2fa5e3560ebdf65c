// C ABI of the gated feed-forward block that is trained in 8 bits: argument checks, workspaces and the order of the launches.
// See include/mxgemm.h; kernels in mx_train.hip, products through mx_gemm.
#include <algorithm>

#include "mx_train.h"

using namespace mx;

namespace {

inline int64_t round256(int64_t b) { return (b + 255) & ~(int64_t)255; }
inline int64_t round32(int64_t n) { return (n + 31) / 32 * 32; }
constexpr int64_t kMaxExtent = (int64_t)1 << 30;

// a 2-D tensor [rows, cols] with contiguous rows
int check2d(const mx_tensor* t, const char* name, int64_t rows, int64_t cols) {
  if (!t) return set_error(MX_ERR_INVALID, "%s: null descriptor", name);
  if (t->ndim != 2) return set_error(MX_ERR_SHAPE, "%s: expected 2 dimensions, got %d", name, t->ndim);
  if ((rows >= 0 && t->shape[0] != rows) || (cols >= 0 && t->shape[1] != cols))
    return set_error(MX_ERR_SHAPE, "%s must be [%lld, %lld], got [%lld, %lld]", name, (long long)(rows >= 0 ? rows : t->shape[0]),
                     (long long)(cols >= 0 ? cols : t->shape[1]), (long long)t->shape[0], (long long)t->shape[1]);
  if (t->shape[0] < 0 || t->shape[1] < 0 || t->shape[0] >= kMaxExtent || t->shape[1] >= kMaxExtent)
    return set_error(MX_ERR_SHAPE, "%s: extent out of range", name);
  if (t->stride[0] < 0 || (t->shape[1] > 1 && t->stride[1] != 1))
    return set_error(MX_ERR_LAYOUT, "%s: rows must be contiguous", name);
  if (t->shape[0] > 0 && t->shape[1] > 0 && !t->ptr) return set_error(MX_ERR_INVALID, "%s: null data pointer", name);
  return MX_OK;
}
int check_dtype(const mx_tensor* t, const char* name, bool ok, const char* want) {
  return ok ? MX_OK : set_error(MX_ERR_DTYPE, "%s must be %s (got %d)", name, want, t->dtype);
}
// an output of codes: rows that start at whole `align` bytes and do not overlap
int check_codes(const mx_tensor* t, const char* name, int64_t rows, int64_t cols, int align) {
  if (int rc = check2d(t, name, rows, cols)) return rc;
  if (rows == 0 || cols == 0) return MX_OK;
  if ((uintptr_t)t->ptr % align != 0 || (rows > 1 && (t->stride[0] % align != 0 || t->stride[0] < cols)))
    return set_error(MX_ERR_LAYOUT, "%s: rows must be aligned to %d bytes and apart", name, align);
  return MX_OK;
}
int check_scales(const mx_tensor* t, const char* name, int64_t rows, int64_t blocks) {
  if (int rc = check2d(t, name, rows, blocks)) return rc;
  if (t->dtype != MX_E8M0) return set_error(MX_ERR_DTYPE, "%s must be MX_E8M0", name);
  if (rows > 1 && blocks > 0 && t->stride[0] < blocks) return set_error(MX_ERR_LAYOUT, "%s: rows overlap", name);
  return MX_OK;
}
int check_mode(int32_t scale_mode) {
  return scale_mode == 0 || scale_mode == 1 ? MX_OK : set_error(MX_ERR_INVALID, "scale_mode must be 0 (ceil) or 1 (floor)");
}
inline bool is_float(int d) { return d == MX_F32 || d == MX_BF16 || d == MX_F16; }
inline mx_tensor tensor2d(void* ptr, int dtype, int64_t rows, int64_t cols, int64_t ld) {
  return mx_tensor{ptr, dtype, 2, {rows, cols, 0, 0}, {ld, 1, 0, 0}, -1, 0};
}
inline mx_tensor transposed(const mx_tensor& t) {
  mx_tensor r = t;
  r.shape[0] = t.shape[1]; r.shape[1] = t.shape[0];
  r.stride[0] = t.stride[1]; r.stride[1] = t.stride[0];
  if (t.packed_dim >= 0) r.packed_dim = 1 - t.packed_dim;
  return r;
}
constexpr mx_gemm_opts kPlainOpts = {sizeof(mx_gemm_opts), 0, MX_SCALE_2D, MX_SCALE_2D, MX_KERNEL_AUTO, 32, 0, 0};

// a buffer that is dealt out in pieces of whole 256 bytes
struct Deal {
  uint8_t* base;
  int64_t at = 0;
  uint8_t* take(int64_t bytes) {
    uint8_t* const p = base + at;
    at += round256(bytes);
    return p;
  }
};
int check_room(const char* name, const void* ptr, int64_t given, int64_t need) {
  if (need <= 0) return MX_OK;
  if (!ptr || given < need)
    return set_error(MX_ERR_WORKSPACE, "%s of %lld bytes required, %lld given", name, (long long)need, (long long)(ptr ? given : 0));
  if ((uintptr_t)ptr % 256 != 0) return set_error(MX_ERR_WORKSPACE, "%s must be 256-byte aligned", name);
  return MX_OK;
}

// ---- the gated product --------------------------------------------------------------------------------------------------------
// operands that have been checked; `plain` scale descriptors follow o's layouts
int64_t gated_workspace(int64_t M, int64_t F, int64_t K, const mx_gemm_opts& o) {
  return round256(M * 2 * F * 2) + round256(mx_gemm_workspace_bytes(M, 2 * F, K, &o));
}
int run_gated(const mx_tensor& A, const mx_tensor& As, const mx_tensor& W, const mx_tensor& Ws, const GateOut& out, const mx_gemm_opts& o,
              void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  const int64_t M = A.shape[0], N = W.shape[0];
  if (M > 0)
    if (const int rc = gemm_gated_fused(A, As, W, Ws, out, o, workspace, workspace_bytes, stream); rc != kGatedNotFused) return rc;
  Deal ws = {(uint8_t*)workspace};
  mx_tensor gu = tensor2d(ws.take(M * N * 2), MX_BF16, M, N, N);
  const mx_tensor B = transposed(W), Bs = o.b_scale_layout == MX_SCALE_2D ? transposed(Ws) : Ws;
  if (int rc = mx_gemm(&A, &As, &B, &Bs, &gu, &o, ws.base + ws.at, workspace_bytes - ws.at, stream)) return rc;
  return launch_gate_up(GateUpArgs{(const uint16_t*)gu.ptr, N, M, out}, stream);
}

// ---- the whole block ------------------------------------------------------------------------------------------------------------
struct FfnShape {
  int64_t T, H, F, Ho, Tp;
};
// Few tokens: gate and up, and the activation's gradient, are summed in 32-bit precision (mx_gemm_few.hip).  Where a result differs from its
// definition by more than its own rounding it is by single large elements that took the other neighbour, and the fewer elements the more
// they weigh.  The largest difference of y, dx, dw1 or dw2 in 12 draws, of its norm (rounding to bf16 alone: 0.0017), without that, T x F: 17 x 512
// 0.0097, 33 x 512 0.0068, 64 x 512 0.0051, 100 x 512 0.0044, 40 x 2048 0.0037, 300 x 512 0.0034, 200 x 1024 0.0028, 1000 x 512 0.0026; with it 0.0018.
// us a step, without and with it: 1 and 64 tokens, H x F 4096 x 14336 328 | 349, 389 | 423; 1024 x 2048 49 | 50, 65 | 63; 4096 x 1024
// 57 | 61, 70 | 71; 73 x 4096 x 7168 211 | 224; 256 x 4096 x 512 78 | 72; 512 x 4096 x 1024 96 | 99; 1024 x 1024 x 512 66 | 69.
inline bool few_tokens(const FfnShape& s) { return s.T <= 64 || s.T * s.F <= 524288; }
// scales of an operand whose rows go with the tokens: few rows are multiplied by kernels that read them plain
inline bool native_rows(const FfnShape& s) { return !few_tokens(s); }
inline int64_t scale_bytes(int64_t rows, int64_t K, bool native) { return native ? mx_packed_scale_bytes(rows, K) : rows * (K / 32); }

// what the forward pass leaves for the backward pass
struct FfnSaved {
  uint8_t *xt, *xts, *gu, *gus, *w1t, *w1ts, *w2t, *w2ts;
  int64_t bytes;
};
FfnSaved ffn_saved(uint8_t* base, const FfnShape& s) {
  Deal d = {base};
  FfnSaved r;
  r.xt = d.take(s.H * s.Tp);
  r.xts = d.take(mx_packed_scale_bytes(s.H, s.Tp));
  r.gu = d.take(s.T * 2 * s.F);
  r.gus = d.take(s.T * 2 * s.F / 32);
  r.w1t = d.take(s.H * 2 * s.F);
  r.w1ts = d.take(mx_packed_scale_bytes(s.H, 2 * s.F));
  r.w2t = d.take(s.F * s.Ho);
  r.w2ts = d.take(mx_packed_scale_bytes(s.F, s.Ho));
  r.bytes = d.at;
  return r;
}
mx_gemm_opts layouts(bool a_native, bool b_native) {
  mx_gemm_opts o = kPlainOpts;
  o.a_scale_layout = a_native ? MX_SCALE_NATIVE : MX_SCALE_2D;
  o.b_scale_layout = b_native ? MX_SCALE_NATIVE : MX_SCALE_2D;
  return o;
}
struct FfnForward {
  uint8_t *xq, *xs, *w1, *w1s, *w2, *w2s, *h, *hs, *work;
  int64_t work_bytes, bytes;
};
FfnForward ffn_forward(uint8_t* base, const FfnShape& s) {
  Deal d = {base};
  FfnForward r;
  const bool nat = native_rows(s);
  r.xq = d.take(s.T * s.H);
  r.xs = d.take(scale_bytes(s.T, s.H, nat));
  r.w1 = d.take(2 * s.F * s.H);
  r.w1s = d.take(mx_packed_scale_bytes(2 * s.F, s.H));
  r.w2 = d.take(s.Ho * s.F);
  r.w2s = d.take(mx_packed_scale_bytes(s.Ho, s.F));
  r.h = d.take(s.T * s.F);
  r.hs = d.take(s.T * (s.F / 32));
  const mx_gemm_opts up = layouts(nat, true), down = layouts(false, true);
  r.work_bytes = std::max(gated_workspace(s.T, s.F, s.H, up), mx_gemm_workspace_bytes(s.T, s.Ho, s.F, &down));
  r.work = d.take(r.work_bytes);
  r.bytes = d.at;
  return r;
}
struct FfnBackward {
  uint8_t *dy, *dys, *dyt, *dyts, *dh, *d, *ds, *dt, *dts, *at, *ats, *work;
  bool native_rows, native_act;   // scales of dy and of the activation's gradients
  mx_gemm_opts o_dh, o_dx, o_dw1, o_dw2;
  int64_t work_bytes, bytes;
};
FfnBackward ffn_backward(uint8_t* base, const FfnShape& s) {
  Deal d = {base};
  FfnBackward r;
  const bool nat = native_rows(s), act = s.F % 64 == 0;   // (launch_silu_backward)
  r.native_rows = nat;
  r.native_act = act;
  r.dy = d.take(s.T * s.Ho);
  r.dys = d.take(scale_bytes(s.T, s.Ho, nat));
  r.dyt = d.take(s.Ho * s.Tp);
  r.dyts = d.take(mx_packed_scale_bytes(s.Ho, s.Tp));
  r.dh = d.take(s.T * s.F * 2);
  r.d = d.take(s.T * 2 * s.F);
  r.ds = d.take(scale_bytes(s.T, 2 * s.F, nat && act));
  r.dt = d.take(2 * s.F * s.Tp);
  r.dts = d.take(scale_bytes(2 * s.F, s.Tp, act));
  r.at = d.take(s.F * s.Tp);
  r.ats = d.take(scale_bytes(s.F, s.Tp, act));
  r.o_dh = layouts(nat, true);
  r.o_dx = layouts(nat && act, true);
  r.o_dw1 = layouts(act, true);
  r.o_dw2 = layouts(true, act);
  r.work_bytes = std::max(std::max(mx_gemm_workspace_bytes(s.T, s.F, s.Ho, &r.o_dh), mx_gemm_workspace_bytes(s.T, s.H, 2 * s.F, &r.o_dx)),
                          std::max(mx_gemm_workspace_bytes(2 * s.F, s.H, s.Tp, &r.o_dw1), mx_gemm_workspace_bytes(s.Ho, s.F, s.Tp, &r.o_dw2)));
  if (s.T <= 64) {   // the gradients of both weights in one launch
    const mx_tensor A[2] = {tensor2d(nullptr, MX_E4M3, 2 * s.F, s.Tp, s.Tp), tensor2d(nullptr, MX_E4M3, s.Ho, s.Tp, s.Tp)};
    const mx_tensor B[2] = {transposed(tensor2d(nullptr, MX_E4M3, s.H, s.Tp, s.Tp)), transposed(tensor2d(nullptr, MX_E4M3, s.F, s.Tp, s.Tp))};
    r.work_bytes = std::max(r.work_bytes, mx_gemm_list_workspace_bytes(2, A, B, &r.o_dw1));
  }
  r.work = d.take(r.work_bytes);
  r.bytes = d.at;
  return r;
}
// C [M, N] = A [M, K] B [N, K]^T, E4M3 both
int product(uint8_t* a, uint8_t* as, uint8_t* b, uint8_t* bs, const mx_tensor& C, int64_t M, int64_t N, int64_t K, const mx_gemm_opts& o,
            void* work, int64_t work_bytes, void* stream) {
  const mx_tensor A = tensor2d(a, MX_E4M3, M, K, K), As = tensor2d(as, MX_E8M0, M, K / 32, K / 32);
  const mx_tensor B = transposed(tensor2d(b, MX_E4M3, N, K, K)), Bs = transposed(tensor2d(bs, MX_E8M0, N, K / 32, K / 32));
  mx_tensor c = C;
  return mx_gemm(&A, &As, &B, &Bs, &c, &o, work, work_bytes, stream);
}
BothTensor both(const mx_tensor* x, uint8_t* q, uint8_t* s, int s_kind, uint8_t* qt, uint8_t* st, int st_kind) {
  BothTensor t = {};
  t.rows = (int32_t)x->shape[0]; t.K = (int32_t)x->shape[1];
  t.x = x->ptr; t.x_ld = t.rows > 1 ? x->stride[0] : t.K; t.x_dtype = x->dtype;   // (the pitch of one row is anything)
  const int64_t Kp = round32(t.K), Rp = round32(t.rows);
  t.q = q; t.s = s; t.q_ld = Kp; t.s_ld = Kp / 32; t.s_kind = s_kind;
  t.qt = qt; t.st = st; t.qt_ld = Rp; t.st_ld = Rp / 32; t.st_kind = st_kind;
  return t;
}
int check_ffn(const mx_tensor* x, const mx_tensor* w1, const mx_tensor* w2, const mx_tensor* y, FfnShape& s) {
  if (int rc = check2d(x, "x", -1, -1)) return rc;
  if (int rc = check2d(w1, "w1", -1, x->shape[1])) return rc;
  if (w1->shape[0] % 2 != 0) return set_error(MX_ERR_SHAPE, "w1 must be [2F, H] (gate and up projection), got %lld rows", (long long)w1->shape[0]);
  if (int rc = check2d(w2, "w2", -1, w1->shape[0] / 2)) return rc;
  if (int rc = check2d(y, "y", x->shape[0], w2->shape[0])) return rc;
  s = FfnShape{x->shape[0], x->shape[1], w1->shape[0] / 2, w2->shape[0], round32(x->shape[0])};
  if (s.H % 32 != 0 || s.F % 32 != 0 || s.Ho % 32 != 0 || s.H == 0 || s.F == 0 || s.Ho == 0)
    return set_error(MX_ERR_SHAPE, "H (%lld), F (%lld) and H_out (%lld) must be multiples of 32", (long long)s.H, (long long)s.F, (long long)s.Ho);
  if (int rc = check_dtype(x, "x", is_float(x->dtype), "MX_F32, MX_BF16 or MX_F16")) return rc;
  if (int rc = check_dtype(w1, "w1", is_float(w1->dtype), "MX_F32, MX_BF16 or MX_F16")) return rc;
  if (int rc = check_dtype(w2, "w2", is_float(w2->dtype), "MX_F32, MX_BF16 or MX_F16")) return rc;
  return check_dtype(y, "y", y->dtype == MX_F32 || y->dtype == MX_BF16, "MX_F32 or MX_BF16");
}
// Codes that the products take as operands of less than 2 GiB.
int check_ffn_size(const FfnShape& s) {
  const int64_t lim = (int64_t)1 << 31, rows = std::max(s.T, (int64_t)1), tp = std::max(s.Tp, (int64_t)32);
  if (std::max(rows * std::max(std::max(s.H, s.Ho), 2 * s.F), std::max(std::max(2 * s.F * s.H, s.Ho * s.F), tp * std::max(2 * s.F, std::max(s.H, s.Ho)))) >= lim)
    return set_error(MX_ERR_SHAPE, "feed-forward block: an operand spans 2 GiB or more (T %lld, H %lld, F %lld, H_out %lld)", (long long)s.T, (long long)s.H,
                     (long long)s.F, (long long)s.Ho);
  return MX_OK;
}
}  // namespace

extern "C" {

int mx_quantize_both(const mx_tensor* x, mx_tensor* xq, mx_tensor* scale, mx_tensor* xt, mx_tensor* scale_t, int32_t scale_mode, void* stream) {
  if (int rc = check2d(x, "x", -1, -1)) return rc;
  if (int rc = check_dtype(x, "x", is_float(x->dtype), "MX_F32, MX_BF16 or MX_F16")) return rc;
  const int64_t rows = x->shape[0], K = x->shape[1], Kp = round32(K), Rp = round32(rows);
  if (K < 32)
    return set_error(MX_ERR_SHAPE, "The requested block size 32 is larger than the inner most dimension of the input tensor %lld", (long long)K);
  if (int rc = check_codes(xq, "xq", rows, Kp, 8)) return rc;
  if (int rc = check_scales(scale, "scale", rows, Kp / 32)) return rc;
  if (int rc = check_codes(xt, "xt", K, Rp, 16)) return rc;
  if (int rc = check_scales(scale_t, "scale_t", K, Rp / 32)) return rc;
  if (xq->dtype != xt->dtype || (xq->dtype != MX_E4M3 && xq->dtype != MX_E5M2))
    return set_error(MX_ERR_DTYPE, "xq and xt must both be MX_E4M3 or both MX_E5M2 (got %d, %d)", xq->dtype, xt->dtype);
  if (int rc = check_mode(scale_mode)) return rc;
  BothTensor t = both(x, (uint8_t*)xq->ptr, (uint8_t*)scale->ptr, kScalePlain, (uint8_t*)xt->ptr, (uint8_t*)scale_t->ptr, kScalePlain);
  t.s_ld = scale->stride[0]; t.qt_ld = xt->stride[0]; t.st_ld = scale_t->stride[0];
  if (rows > 1) t.q_ld = xq->stride[0];   // (the kernel tells rows that are not there by their offsets: no row may lie within the first)
  return launch_quantize_both(&t, 1, xq->dtype, scale_mode, (hipStream_t)stream);
}

int64_t mx_gated_gemm_workspace_bytes(int64_t M, int64_t F, int64_t K, const mx_gemm_opts* opts) {
  if (M <= 0 || F <= 0 || K < 0) return 0;   // (an empty sum is a result too, by way of memory)
  return gated_workspace(M, F, K, opts ? *opts : kPlainOpts);
}

int mx_gated_gemm(const mx_tensor* A, const mx_tensor* As, const mx_tensor* W, const mx_tensor* Ws, mx_tensor* out, mx_tensor* out_scale,
                  mx_tensor* gate_up, mx_tensor* gate_up_scale, int32_t scale_mode, const mx_gemm_opts* opts, void* workspace,
                  int64_t workspace_bytes, void* stream) {
  mx_gemm_opts o = opts ? *opts : kPlainOpts;
  if (!A || !As || !W || !Ws) return set_error(MX_ERR_INVALID, "mx_gated_gemm: null descriptor");
  if (A->ndim != 2 || W->ndim != 2) return set_error(MX_ERR_SHAPE, "mx_gated_gemm: A and W must have 2 dimensions");
  for (const mx_tensor* t : {A, W})
    if (t->shape[0] < 0 || t->shape[1] < 0) return set_error(MX_ERR_SHAPE, "mx_gated_gemm: negative extent");
  if (A->shape[1] != W->shape[1])
    return set_error(MX_ERR_SHAPE, "Incompatible matrices: K dimension of A (%lld) must match K dimension of W (%lld)", (long long)A->shape[1],
                     (long long)W->shape[1]);
  const int64_t M = A->shape[0], K = A->shape[1], F = W->shape[0] / 2;
  if (W->shape[0] % 2 != 0) return set_error(MX_ERR_SHAPE, "W must have 2F rows (gate and up projection), got %lld", (long long)W->shape[0]);
  if (F == 0 || F % 32 != 0) return set_error(MX_ERR_SHAPE, "F (%lld) must be a multiple of 32", (long long)F);
  if (M >= kMaxExtent || F >= kMaxExtent / 2 || K >= kMaxExtent) return set_error(MX_ERR_SHAPE, "mx_gated_gemm: extent out of range");
  if (int rc = check_mode(scale_mode)) return rc;
  const struct { const mx_tensor* t; const char* name; int64_t rows, cols; bool plain; } ins[4] = {
      {A, "A", M, K, true}, {W, "W", 2 * F, K, true}, {As, "A_scale", M, K / 32, o.a_scale_layout == MX_SCALE_2D},
      {Ws, "W_scale", 2 * F, K / 32, o.b_scale_layout == MX_SCALE_2D}};
  for (const auto& i : ins) {
    if (i.plain && (i.t->ndim != 2 || i.t->shape[0] != i.rows || i.t->shape[1] != i.cols))
      return set_error(MX_ERR_SHAPE, "%s must be [%lld, %lld]", i.name, (long long)i.rows, (long long)i.cols);
    for (int n = 0; n < i.t->ndim && n < 4; ++n)
      if (i.t->stride[n] < 0) return set_error(MX_ERR_LAYOUT, "%s: negative strides are not supported", i.name);
    if (M > 0 && K > 0 && !i.t->ptr) return set_error(MX_ERR_INVALID, "%s: null data pointer", i.name);
  }
  GateOut g = {};
  if (int rc = check2d(out, "out", M, F)) return rc;
  g.h = out->ptr; g.h_ld = out->stride[0]; g.h_fmt = out->dtype;
  g.F = (int32_t)F; g.scale_mode = scale_mode;
  if (out->dtype == MX_BF16) {
    if (out_scale) return set_error(MX_ERR_INVALID, "out_scale: an MX_BF16 output has none");
    if ((uintptr_t)out->ptr % 16 != 0 || (M > 1 && (out->stride[0] % 8 != 0 || out->stride[0] < F)))
      return set_error(MX_ERR_LAYOUT, "out: rows must be aligned to 16 bytes and apart");
  } else if (out->dtype == MX_E4M3 || out->dtype == MX_E5M2) {
    if (int rc = check_codes(out, "out", M, F, 8)) return rc;
    if (int rc = check_scales(out_scale, "out_scale", M, F / 32)) return rc;
    g.hs = (uint8_t*)out_scale->ptr; g.hs_ld = out_scale->stride[0];
  } else {
    return set_error(MX_ERR_DTYPE, "out must be MX_BF16, MX_E4M3 or MX_E5M2 (got %d)", out->dtype);
  }
  if (!gate_up != !gate_up_scale) return set_error(MX_ERR_INVALID, "gate_up and gate_up_scale go together");
  if (gate_up) {
    if (int rc = check_codes(gate_up, "gate_up", M, 2 * F, 8)) return rc;
    if (int rc = check_scales(gate_up_scale, "gate_up_scale", M, 2 * F / 32)) return rc;
    if (gate_up->dtype != MX_E4M3) return set_error(MX_ERR_DTYPE, "gate_up must be MX_E4M3 (got %d)", gate_up->dtype);
    g.c = (uint8_t*)gate_up->ptr; g.c_ld = gate_up->stride[0];
    g.cs = (uint8_t*)gate_up_scale->ptr; g.cs_ld = gate_up_scale->stride[0];
  }
  o.accumulate = 0;
  if (M > 0)
    if (int rc = check_room("workspace", workspace, workspace_bytes, gated_workspace(M, F, K, o))) return rc;
  return run_gated(*A, *As, *W, *Ws, g, o, workspace, workspace_bytes, (hipStream_t)stream);
}

int mx_silu_mul_backward_quantize(const mx_tensor* dh, const mx_tensor* gate_up, const mx_tensor* gate_up_scale, mx_tensor* d, mx_tensor* d_scale,
                                  mx_tensor* dt, mx_tensor* dt_scale, mx_tensor* at, mx_tensor* at_scale, int32_t scale_mode, void* stream) {
  if (int rc = check2d(dh, "dh", -1, -1)) return rc;
  const int64_t rows = dh->shape[0], F = dh->shape[1], Rp = round32(rows);
  if (dh->dtype != MX_BF16) return set_error(MX_ERR_DTYPE, "dh must be MX_BF16 (got %d)", dh->dtype);
  if (F == 0 || F % 32 != 0) return set_error(MX_ERR_SHAPE, "dh must have a multiple of 32 columns, got %lld", (long long)F);
  if (F >= kMaxExtent / 2) return set_error(MX_ERR_SHAPE, "dh: extent out of range");
  if (int rc = check2d(gate_up, "gate_up", rows, 2 * F)) return rc;
  if (gate_up->dtype != MX_E4M3) return set_error(MX_ERR_DTYPE, "gate_up must be MX_E4M3 (got %d)", gate_up->dtype);
  if ((uintptr_t)gate_up->ptr % 8 != 0 || (rows > 1 && gate_up->stride[0] % 8 != 0))
    return set_error(MX_ERR_LAYOUT, "gate_up: rows must be aligned to 8 bytes");
  if (int rc = check2d(gate_up_scale, "gate_up_scale", rows, 2 * F / 32)) return rc;
  if (gate_up_scale->dtype != MX_E8M0) return set_error(MX_ERR_DTYPE, "gate_up_scale must be MX_E8M0");
  if (int rc = check_codes(d, "d", rows, 2 * F, 8)) return rc;
  if (int rc = check_scales(d_scale, "d_scale", rows, 2 * F / 32)) return rc;
  if (int rc = check_codes(dt, "dt", 2 * F, Rp, 16)) return rc;
  if (int rc = check_scales(dt_scale, "dt_scale", 2 * F, Rp / 32)) return rc;
  if (int rc = check_codes(at, "at", F, Rp, 16)) return rc;
  if (int rc = check_scales(at_scale, "at_scale", F, Rp / 32)) return rc;
  if (d->dtype != MX_E4M3 || dt->dtype != MX_E4M3 || at->dtype != MX_E4M3) return set_error(MX_ERR_DTYPE, "d, dt and at must be MX_E4M3");
  if (int rc = check_mode(scale_mode)) return rc;
  SiluBackwardArgs a = {};
  a.dh = (const uint16_t*)dh->ptr; a.dh_ld = dh->stride[0];
  a.gu = (const uint8_t*)gate_up->ptr; a.gu_ld = gate_up->stride[0];
  a.gus = (const uint8_t*)gate_up_scale->ptr; a.gus_ld = gate_up_scale->stride[0];
  a.d = (uint8_t*)d->ptr; a.d_ld = d->stride[0]; a.ds = (uint8_t*)d_scale->ptr; a.ds_ld = d_scale->stride[0];
  a.dt = (uint8_t*)dt->ptr; a.dt_ld = dt->stride[0]; a.dts = (uint8_t*)dt_scale->ptr; a.dts_ld = dt_scale->stride[0];
  a.at = (uint8_t*)at->ptr; a.at_ld = at->stride[0]; a.ats = (uint8_t*)at_scale->ptr; a.ats_ld = at_scale->stride[0];
  a.rows = (int32_t)rows; a.F = (int32_t)F; a.scale_mode = scale_mode;
  return launch_silu_backward(a, (hipStream_t)stream);
}

int64_t mx_ffn_saved_bytes(int64_t T, int64_t H, int64_t F, int64_t H_out) {
  if (T <= 0 || H <= 0 || F <= 0 || H_out <= 0) return 0;
  return ffn_saved(nullptr, FfnShape{T, H, F, H_out, round32(T)}).bytes;
}
int64_t mx_ffn_forward_workspace_bytes(int64_t T, int64_t H, int64_t F, int64_t H_out) {
  if (T <= 0 || H <= 0 || F <= 0 || H_out <= 0) return 0;
  return ffn_forward(nullptr, FfnShape{T, H, F, H_out, round32(T)}).bytes;
}
int64_t mx_ffn_backward_workspace_bytes(int64_t T, int64_t H, int64_t F, int64_t H_out) {
  if (T <= 0 || H <= 0 || F <= 0 || H_out <= 0) return 0;
  return ffn_backward(nullptr, FfnShape{T, H, F, H_out, round32(T)}).bytes;
}

int mx_ffn_forward(const mx_tensor* x, const mx_tensor* w1, const mx_tensor* w2, mx_tensor* y, int32_t scale_mode, void* saved,
                   int64_t saved_bytes, void* workspace, int64_t workspace_bytes, void* stream) {
  FfnShape s;
  if (int rc = check_ffn(x, w1, w2, y, s)) return rc;
  if (int rc = check_mode(scale_mode)) return rc;
  if (s.T == 0) return MX_OK;
  if (int rc = check_ffn_size(s)) return rc;
  if (s.T > 1 && y->stride[0] < s.Ho) return set_error(MX_ERR_LAYOUT, "y: rows overlap");
  const FfnForward f = ffn_forward((uint8_t*)workspace, s);
  if (int rc = check_room("workspace", workspace, workspace_bytes, f.bytes)) return rc;
  FfnSaved k = {};
  if (saved) {
    k = ffn_saved((uint8_t*)saved, s);
    if (int rc = check_room("saved", saved, saved_bytes, k.bytes)) return rc;
  }
  hipStream_t st = (hipStream_t)stream;
  const bool nat = native_rows(s);
  const BothTensor list[3] = {both(x, f.xq, f.xs, nat ? kScaleNativeA : kScalePlain, k.xt, k.xts, kScaleNativeB),
                              both(w1, f.w1, f.w1s, kScaleNativeB, k.w1t, k.w1ts, kScaleNativeB),
                              both(w2, f.w2, f.w2s, kScaleNativeB, k.w2t, k.w2ts, kScaleNativeB)};
  if (int rc = launch_quantize_both(list, 3, MX_E4M3, scale_mode, st)) return rc;
  GateOut g = {};
  g.h = f.h; g.h_ld = s.F; g.h_fmt = MX_E4M3; g.hs = f.hs; g.hs_ld = s.F / 32;
  g.c = k.gu; g.c_ld = 2 * s.F; g.cs = k.gus; g.cs_ld = 2 * s.F / 32;
  g.F = (int32_t)s.F; g.scale_mode = scale_mode;
  const mx_gemm_opts up = layouts(nat, true), down = layouts(false, true);
  if (few_tokens(s)) {
    FewArgs few = {f.xq, f.xs, f.w1, f.w1s, (uint16_t*)f.work, (int32_t)s.T, (int32_t)(2 * s.F), (int32_t)s.H};
    if (scale_mode) {
      if (int rc = launch_gemm_few_gated(few, g, st)) return rc;
    } else {
      if (int rc = launch_gemm_few(few, st)) return rc;
      if (int rc = launch_gate_up(GateUpArgs{(const uint16_t*)f.work, 2 * s.F, s.T, g}, st)) return rc;
    }
  } else if (int rc = run_gated(tensor2d(f.xq, MX_E4M3, s.T, s.H, s.H), tensor2d(f.xs, MX_E8M0, s.T, s.H / 32, s.H / 32),
                                tensor2d(f.w1, MX_E4M3, 2 * s.F, s.H, s.H), tensor2d(f.w1s, MX_E8M0, 2 * s.F, s.H / 32, s.H / 32), g, up, f.work,
                                f.work_bytes, st)) {
    return rc;
  }
  return product(f.h, f.hs, f.w2, f.w2s, *y, s.T, s.Ho, s.F, down, f.work, f.work_bytes, stream);
}

int mx_ffn_backward(const mx_tensor* dy, const void* saved, int64_t saved_bytes, int64_t H, int64_t F, mx_tensor* dx, mx_tensor* dw1,
                    mx_tensor* dw2, int32_t scale_mode, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check2d(dy, "dy", -1, -1)) return rc;
  if (int rc = check_dtype(dy, "dy", is_float(dy->dtype), "MX_F32, MX_BF16 or MX_F16")) return rc;
  const FfnShape s = {dy->shape[0], H, F, dy->shape[1], round32(dy->shape[0])};
  if (H <= 0 || F <= 0 || H >= kMaxExtent || F >= kMaxExtent / 2 || s.H % 32 != 0 || s.F % 32 != 0 || s.Ho % 32 != 0 || s.Ho == 0)
    return set_error(MX_ERR_SHAPE, "H (%lld), F (%lld) and H_out (%lld) must be multiples of 32", (long long)s.H, (long long)s.F, (long long)s.Ho);
  const struct { mx_tensor* t; const char* name; int64_t rows, cols; } outs[3] = {{dx, "dx", s.T, H}, {dw1, "dw1", 2 * F, H}, {dw2, "dw2", s.Ho, F}};
  for (const auto& o : outs) {
    if (!o.t) continue;
    if (int rc = check2d(o.t, o.name, o.rows, o.cols)) return rc;
    if (int rc = check_dtype(o.t, o.name, o.t->dtype == MX_F32 || o.t->dtype == MX_BF16, "MX_F32 or MX_BF16")) return rc;
    if (o.rows > 1 && o.t->stride[0] < o.cols) return set_error(MX_ERR_LAYOUT, "%s: rows overlap", o.name);
  }
  if (int rc = check_mode(scale_mode)) return rc;
  if (s.T == 0) return set_error(MX_ERR_SHAPE, "mx_ffn_backward: no tokens (the gradients of the weights are zeros)");
  if (int rc = check_ffn_size(s)) return rc;
  if (int rc = check_room("saved", saved, saved_bytes, mx_ffn_saved_bytes(s.T, s.H, s.F, s.Ho))) return rc;
  const FfnBackward b = ffn_backward((uint8_t*)workspace, s);
  if (int rc = check_room("workspace", workspace, workspace_bytes, b.bytes)) return rc;
  const FfnSaved k = ffn_saved((uint8_t*)const_cast<void*>(saved), s);
  hipStream_t st = (hipStream_t)stream;
  const bool to_dh = dx || dw1, act = to_dh || dw2;
  if (!act) return MX_OK;
  const BothTensor t = both(dy, b.dy, b.dys, b.native_rows ? kScaleNativeA : kScalePlain, dw2 ? b.dyt : nullptr, b.dyts, kScaleNativeA);
  if (int rc = launch_quantize_both(&t, 1, MX_E4M3, scale_mode, st)) return rc;
  const mx_tensor dh = tensor2d(b.dh, MX_BF16, s.T, s.F, s.F);
  if (few_tokens(s)) {
    if (int rc = launch_gemm_few(FewArgs{b.dy, b.dys, k.w2t, k.w2ts, (uint16_t*)b.dh, (int32_t)s.T, (int32_t)s.F, (int32_t)s.Ho}, st)) return rc;
  } else if (int rc = product(b.dy, b.dys, k.w2t, k.w2ts, dh, s.T, s.F, s.Ho, b.o_dh, b.work, b.work_bytes, stream)) {
    return rc;
  }
  SiluBackwardArgs a = {};
  a.dh = (const uint16_t*)b.dh; a.dh_ld = s.F;
  a.gu = k.gu; a.gu_ld = 2 * s.F; a.gus = k.gus; a.gus_ld = 2 * s.F / 32;
  a.d = b.d; a.d_ld = 2 * s.F; a.ds = b.ds; a.ds_ld = 2 * s.F / 32;
  a.dt = b.dt; a.dt_ld = s.Tp; a.dts = b.dts; a.dts_ld = s.Tp / 32;
  a.at = b.at; a.at_ld = s.Tp; a.ats = b.ats; a.ats_ld = s.Tp / 32;
  a.rows = (int32_t)s.T; a.F = (int32_t)s.F; a.scale_mode = scale_mode;
  a.ds_kind = b.native_rows && b.native_act ? kScaleNativeA : kScalePlain;
  a.dts_kind = b.native_act ? kScaleNativeA : kScalePlain;
  a.ats_kind = b.native_act ? kScaleNativeB : kScalePlain;
  if (int rc = launch_silu_backward(a, st)) return rc;
  if (dx)
    if (int rc = product(b.d, b.ds, k.w1t, k.w1ts, *dx, s.T, s.H, 2 * s.F, b.o_dx, b.work, b.work_bytes, stream)) return rc;
  // few tokens: the products of the weights' gradients are short and only their output takes time, so both go out in one launch
  if (s.T <= 64 && dw1 && dw2 && b.native_act && dw1->dtype == dw2->dtype) {
    const mx_tensor A[2] = {tensor2d(b.dt, MX_E4M3, 2 * s.F, s.Tp, s.Tp), tensor2d(b.dyt, MX_E4M3, s.Ho, s.Tp, s.Tp)};
    const mx_tensor As[2] = {tensor2d(b.dts, MX_E8M0, 2 * s.F, s.Tp / 32, s.Tp / 32), tensor2d(b.dyts, MX_E8M0, s.Ho, s.Tp / 32, s.Tp / 32)};
    const mx_tensor B[2] = {transposed(tensor2d(k.xt, MX_E4M3, s.H, s.Tp, s.Tp)), transposed(tensor2d(b.at, MX_E4M3, s.F, s.Tp, s.Tp))};
    const mx_tensor Bs[2] = {transposed(tensor2d(k.xts, MX_E8M0, s.H, s.Tp / 32, s.Tp / 32)), transposed(tensor2d(b.ats, MX_E8M0, s.F, s.Tp / 32, s.Tp / 32))};
    mx_tensor C[2] = {*dw1, *dw2};
    return mx_gemm_list(2, A, As, B, Bs, C, &b.o_dw1, b.work, b.work_bytes, stream);
  }
  if (dw1)
    if (int rc = product(b.dt, b.dts, k.xt, k.xts, *dw1, 2 * s.F, s.H, s.Tp, b.o_dw1, b.work, b.work_bytes, stream)) return rc;
  if (dw2)
    if (int rc = product(b.dyt, b.dyts, b.at, b.ats, *dw2, s.Ho, s.F, s.Tp, b.o_dw2, b.work, b.work_bytes, stream)) return rc;
  return MX_OK;
}

}  // extern "C"
