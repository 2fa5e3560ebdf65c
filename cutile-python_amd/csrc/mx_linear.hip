// C ABI of the linear layer on block-scaled operands: argument checks, workspaces and the order of the launches, and the layer's pass
// over a product that went through memory.  See include/mxgemm.h; the epilogue is in mx_linear.h.
#include <algorithm>

#include "mx_check.h"
#include "mx_linear.h"
#include "mx_train.h"

namespace mx {
namespace {

// One pass over fp32 products (of a sum that was split along K, one each): a lane has 8 columns of a row.  Bound: memory (32 x 28672: 3 us, a launch).
template <int KIND>
__global__ __launch_bounds__(256) void linear_pass_kernel(const float* product, const int splits, const int64_t M, const LinearOut o) {
  const int64_t unit = (int64_t)blockIdx.x * 256 + threadIdx.x, per = (o.N + 7) / 8;   // (N % 32 == 0 with codes: four lanes of a wave are a block)
  const int64_t row = unit / per;
  const int col = (int)(unit - row * per) * 8, cols = o.N - col;
  v4f a = {0.f, 0.f, 0.f, 0.f}, b = a;
  if (row < M)
    for (int s = 0; s < splits; ++s) {
      const float* const p = product + ((int64_t)s * M + row) * o.N + col;
      float x[8];
      load_floats<8>(p, MX_F32, 0, cols, 0.f, x);
#pragma unroll
      for (int e = 0; e < 4; ++e) { a[e] += x[e]; b[e] += x[4 + e]; }
    }
  float bias[8];
  linear_bias(o, col, bias);
  FloatsPiece res = {};
  linear_request(o, res, row, col, cols, row < M);
  linear_finish<KIND, false>(o, a, b, bias, res, row, col, cols, row < M, (threadIdx.x & 3) == 0);
}

// sums [parts][N] -> out [N]: a workgroup takes 64 columns, its waves every 16th part
__global__ __launch_bounds__(1024) void column_sums_kernel(const float* partial, const int parts, const int64_t N, void* out, const int out_dtype) {
  __shared__ float red[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t col = (int64_t)blockIdx.x * 64 + lane;
  float s = 0.f;
  if (col < N)
    for (int p = wave; p < parts; p += 16) s += partial[(int64_t)p * N + col];
  red[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || col >= N) return;
#pragma unroll
  for (int k = 1; k < 16; ++k) s += red[k][lane];
  store_float(out, out_dtype, col, s);
}

}  // namespace

int launch_linear_pass(const float* product, int splits, int64_t M, const LinearOut& o, hipStream_t stream) {
  const int64_t blocks = (M * ((o.N + 7) / 8) + 255) / 256;
  if (blocks <= 0) return MX_OK;
  if (blocks > 0x7FFFFFFF) return set_error(MX_ERR_SHAPE, "linear_pass: tensor too large");
  const dim3 grid((unsigned)blocks);
  const int kind = act_kind(o.act);
  const hipError_t e = kind == kActErf       ? launch_kernel(linear_pass_kernel<kActErf>, grid, dim3(256), 0, stream, product, splits, M, o)
                       : kind == kActSigmoid ? launch_kernel(linear_pass_kernel<kActSigmoid>, grid, dim3(256), 0, stream, product, splits, M, o)
                                             : launch_kernel(linear_pass_kernel<kActPlain>, grid, dim3(256), 0, stream, product, splits, M, o);
  if (e != hipSuccess) return set_error(MX_ERR_LAUNCH, "linear_pass_kernel launch: %s", hipGetErrorString(e));
  return MX_OK;
}

int launch_column_sums(const float* partial, int parts, int64_t N, void* out, int out_dtype, hipStream_t stream) {
  const hipError_t e = launch_kernel(column_sums_kernel, dim3((unsigned)((N + 63) / 64)), dim3(1024), 0, stream, partial, parts, N, out, out_dtype);
  if (e != hipSuccess) return set_error(MX_ERR_LAUNCH, "column_sums_kernel launch: %s", hipGetErrorString(e));
  return MX_OK;
}

}  // namespace mx

using namespace mx;

namespace {

constexpr mx_gemm_opts kPlainOpts = {sizeof(mx_gemm_opts), 0, MX_SCALE_2D, MX_SCALE_2D, MX_KERNEL_AUTO, 32, 0, 0};

// bias, residual and activation of a [M, N] result
int check_linear(const mx_tensor* bias, const mx_tensor* residual, int32_t act, int64_t M, int64_t N, LinearOut& o) {
  o.N = (int32_t)N;
  o.act = act;
  if (act < MX_ACT_NONE || act > MX_ACT_SILU) return set_error(MX_ERR_INVALID, "unknown activation %d", act);
  if (bias) {
    if (int rc = check_vector(bias, "bias", N)) return rc;
    o.bias = bias->ptr;
    o.bias_dtype = bias->dtype;
  }
  if (residual) {
    if (int rc = check2d(residual, "residual", M, N)) return rc;
    if (int rc = check_dtype(residual, "residual", is_float(residual->dtype), "MX_F32, MX_BF16 or MX_F16")) return rc;
    o.res = residual->ptr;
    o.r_ld = residual->stride[0];
    o.res_dtype = residual->dtype;
  }
  return MX_OK;
}
int check_apart(const mx_tensor* t, const char* name) {
  return t->shape[0] > 1 && t->stride[0] < t->shape[1] ? set_error(MX_ERR_LAYOUT, "%s: rows overlap", name) : MX_OK;
}
// What no kernel finishes goes through the workspace, some rows at a time (a multiple of 256, which every scale layout can be entered at): the
// product, then the pass.
constexpr int64_t kPassBytes = (int64_t)16 << 20;
int64_t pass_rows(int64_t M, int64_t N) { return std::min(M, std::max(kPassBytes / (N * 4) / 256 * 256, (int64_t)256)); }
mx_gemm_opts pass_opts(const mx_gemm_opts& o) {
  mx_gemm_opts r = o;
  if (r.split_k == 0) r.split_k = 1;
  return r;
}
int64_t linear_workspace(int64_t M, int64_t N, int64_t K, const mx_gemm_opts& o) {
  const mx_gemm_opts po = pass_opts(o);
  const int64_t rows = pass_rows(M, N);
  return std::max(round256(rows * N * 4) + round256(mx_gemm_workspace_bytes(rows, N, K, &po)), mx_gemm_workspace_bytes(M, N, K, &o));
}
int run_linear(const mx_tensor& A, const mx_tensor& As, const mx_tensor& W, const mx_tensor& Ws, const LinearOut& out, const mx_gemm_opts& o, void* workspace,
               int64_t workspace_bytes, hipStream_t stream) {
  const int64_t M = A.shape[0], N = W.shape[0], K = A.shape[1], rows = pass_rows(M, N);
  if (const int rc = gemm_linear_fused(A, As, W, Ws, out, o, workspace, workspace_bytes, stream); rc != kLinearNotFused) return rc;
  const mx_gemm_opts po = pass_opts(o);
  const mx_tensor B = transposed(W), Bs = o.b_scale_layout == MX_SCALE_2D ? transposed(Ws) : Ws;
  for (int64_t m0 = 0; m0 < M; m0 += rows) {
    const int64_t m = std::min(rows, M - m0);
    Deal ws = {(uint8_t*)workspace};
    mx_tensor a = A, as = As, c = tensor2d(ws.take(rows * N * 4), MX_F32, m, N, N);
    a.shape[0] = m;
    a.ptr = (uint8_t*)A.ptr + (A.dtype == MX_E2M1 && A.packed_dim == 0 ? m0 / 2 : m0) * A.stride[0];   // (two rows to a byte, packed along M)
    if (o.a_scale_layout == MX_SCALE_2D || o.a_scale_layout == MX_SCALE_SWIZZLE_32_4_4) {
      as.shape[0] = o.a_scale_layout == MX_SCALE_2D ? m : m / 128;
      as.ptr = (uint8_t*)As.ptr + (o.a_scale_layout == MX_SCALE_2D ? m0 : m0 / 128) * As.stride[0];
    } else {
      as.shape[0] = m;
      as.ptr = (uint8_t*)As.ptr + m0 / 64 * packed_scale_quads(K) * 1024;
    }
    if (int rc = mx_gemm(&a, &as, &B, &Bs, &c, &po, ws.base + ws.at, workspace_bytes - ws.at, stream)) return rc;
    LinearOut l = out;
    l.c = (uint8_t*)out.c + m0 * out.c_ld * (out.c_fmt == MX_F32 ? 4 : out.c_fmt == MX_BF16 ? 2 : 1);
    if (out.s) l.s = out.s + m0 * out.s_ld;
    if (out.pre) l.pre = out.pre + m0 * out.pre_ld;
    if (out.res) l.res = (const uint8_t*)out.res + m0 * out.r_ld * (out.res_dtype == MX_F32 ? 4 : 2);
    if (int rc = launch_linear_pass((const float*)c.ptr, 1, m, l, stream)) return rc;
  }
  return MX_OK;
}

// ---- the trained layer ----------------------------------------------------------------------------------------------------------------
struct LinearShape {
  int64_t T, K, N, Tp;
};
// as in the feed-forward block: P is rounded to bf16 and what is made of it to E4M3 (mx_ffn.hip)
inline bool few_tokens(const LinearShape& s) { return s.T <= 64 || s.T * s.N <= 524288; }
inline int64_t scale_bytes(int64_t rows, int64_t K, bool native) { return native ? mx_packed_scale_bytes(rows, K) : rows * (K / 32); }
mx_gemm_opts layouts(bool a_native, bool b_native) {
  mx_gemm_opts o = kPlainOpts;
  o.a_scale_layout = a_native ? MX_SCALE_NATIVE : MX_SCALE_2D;
  o.b_scale_layout = b_native ? MX_SCALE_NATIVE : MX_SCALE_2D;
  return o;
}
struct LinearSaved {
  uint8_t *xt, *xts, *wt, *wts, *pre;
  int64_t bytes;
};
LinearSaved linear_saved(uint8_t* base, const LinearShape& s, int act) {
  Deal d = {base};
  LinearSaved r;
  r.xt = d.take(s.K * s.Tp);
  r.xts = d.take(mx_packed_scale_bytes(s.K, s.Tp));
  r.wt = d.take(s.K * s.N);
  r.wts = d.take(mx_packed_scale_bytes(s.K, s.N));
  r.pre = d.take(act != MX_ACT_NONE ? s.T * s.N * 2 : 0);
  r.bytes = d.at;
  return r;
}
struct LinearForward {
  uint8_t *xq, *xs, *w, *ws, *work;
  int64_t work_bytes, bytes;
};
LinearForward linear_forward(uint8_t* base, const LinearShape& s) {
  Deal d = {base};
  LinearForward r;
  r.xq = d.take(s.T * s.K);
  r.xs = d.take(scale_bytes(s.T, s.K, !few_tokens(s)));
  r.w = d.take(s.N * s.K);
  r.ws = d.take(mx_packed_scale_bytes(s.N, s.K));
  const mx_gemm_opts o = layouts(true, true);
  r.work_bytes = few_tokens(s) ? 0 : linear_workspace(s.T, s.N, s.K, o);
  r.work = d.take(r.work_bytes);
  r.bytes = d.at;
  return r;
}
struct LinearBackward {
  uint8_t *d, *ds, *dt, *dts, *sums, *work;
  bool native_rows;
  mx_gemm_opts o_dx, o_dw;
  int64_t work_bytes, bytes;
};
LinearBackward linear_backward(uint8_t* base, const LinearShape& s) {
  Deal d = {base};
  LinearBackward r;
  r.native_rows = !few_tokens(s);
  r.d = d.take(s.T * s.N);
  r.ds = d.take(scale_bytes(s.T, s.N, r.native_rows));
  r.dt = d.take(s.N * s.Tp);
  r.dts = d.take(mx_packed_scale_bytes(s.N, s.Tp));
  r.sums = d.take((s.T + 127) / 128 * s.N * 4);
  r.o_dx = layouts(r.native_rows, true);
  r.o_dw = layouts(true, true);
  r.work_bytes = std::max(mx_gemm_workspace_bytes(s.T, s.K, s.N, &r.o_dx), mx_gemm_workspace_bytes(s.N, s.K, s.Tp, &r.o_dw));
  r.work = d.take(r.work_bytes);
  r.bytes = d.at;
  return r;
}
int check_size(const LinearShape& s) {
  const int64_t lim = (int64_t)1 << 31, tp = std::max(s.Tp, (int64_t)32);
  if (std::max(tp * std::max(s.K, s.N), s.N * s.K) >= lim)
    return set_error(MX_ERR_SHAPE, "linear layer: an operand spans 2 GiB or more (T %lld, K %lld, N %lld)", (long long)s.T, (long long)s.K, (long long)s.N);
  return MX_OK;
}
int check_extents(int64_t K, int64_t N) {
  if (K <= 0 || N <= 0 || K >= kMaxExtent || N >= kMaxExtent || K % 32 != 0 || N % 32 != 0)
    return set_error(MX_ERR_SHAPE, "K (%lld) and N (%lld) must be multiples of 32", (long long)K, (long long)N);
  return MX_OK;
}
// C [M, N] = A [M, K] B [N, K]^T, E4M3 both
int product(uint8_t* a, uint8_t* as, uint8_t* b, uint8_t* bs, const mx_tensor& C, int64_t M, int64_t N, int64_t K, const mx_gemm_opts& o, void* work,
            int64_t work_bytes, void* stream) {
  const mx_tensor A = tensor2d(a, MX_E4M3, M, K, K), As = tensor2d(as, MX_E8M0, M, K / 32, K / 32);
  const mx_tensor B = transposed(tensor2d(b, MX_E4M3, N, K, K)), Bs = transposed(tensor2d(bs, MX_E8M0, N, K / 32, K / 32));
  mx_tensor c = C;
  return mx_gemm(&A, &As, &B, &Bs, &c, &o, work, work_bytes, stream);
}
BothTensor both(const mx_tensor* x, uint8_t* q, uint8_t* s, int s_kind, uint8_t* qt, uint8_t* st, int st_kind) {
  BothTensor t = {};
  t.rows = (int32_t)x->shape[0]; t.K = (int32_t)x->shape[1];
  t.x = x->ptr; t.x_ld = t.rows > 1 ? x->stride[0] : t.K; t.x_dtype = x->dtype;   // (the pitch of one row is anything)
  t.q = q; t.s = s; t.q_ld = t.K; t.s_ld = t.K / 32; t.s_kind = s_kind;
  t.qt = qt; t.st = st; t.qt_ld = round32(t.rows); t.st_ld = t.qt_ld / 32; t.st_kind = st_kind;
  return t;
}

}  // namespace

extern "C" {

int64_t mx_linear_gemm_workspace_bytes(int64_t M, int64_t N, int64_t K, const mx_gemm_opts* opts) {
  if (M <= 0 || N <= 0 || K < 0) return 0;
  return linear_workspace(M, N, K, opts ? *opts : kPlainOpts);
}

int mx_linear_gemm(const mx_tensor* A, const mx_tensor* As, const mx_tensor* W, const mx_tensor* Ws, const mx_tensor* bias, const mx_tensor* residual,
                   int32_t activation, mx_tensor* out, mx_tensor* out_scale, mx_tensor* pre, const mx_gemm_opts* opts, void* workspace,
                   int64_t workspace_bytes, void* stream) {
  mx_gemm_opts o = opts ? *opts : kPlainOpts;
  if (!A || !As || !W || !Ws) return set_error(MX_ERR_INVALID, "mx_linear_gemm: null descriptor");
  if (A->ndim != 2 || W->ndim != 2) return set_error(MX_ERR_SHAPE, "mx_linear_gemm: A and W must have 2 dimensions");
  for (const mx_tensor* t : {A, W})
    if (t->shape[0] < 0 || t->shape[1] < 0) return set_error(MX_ERR_SHAPE, "mx_linear_gemm: negative extent");
  if (A->shape[1] != W->shape[1])
    return set_error(MX_ERR_SHAPE, "Incompatible matrices: K dimension of A (%lld) must match K dimension of W (%lld)", (long long)A->shape[1],
                     (long long)W->shape[1]);
  const int64_t M = A->shape[0], K = A->shape[1], N = W->shape[0];
  if (M >= kMaxExtent || N >= kMaxExtent || K >= kMaxExtent) return set_error(MX_ERR_SHAPE, "mx_linear_gemm: extent out of range");
  if (o.block_size != 32) return set_error(MX_ERR_INVALID, "mx_linear_gemm: block_size must be 32 (got %d)", o.block_size);
  const struct { const mx_tensor* t; const char* name; int64_t rows, cols; bool plain; } ins[4] = {
      {A, "A", M, K, true}, {W, "W", N, K, true}, {As, "A_scale", M, K / 32, o.a_scale_layout == MX_SCALE_2D},
      {Ws, "W_scale", N, K / 32, o.b_scale_layout == MX_SCALE_2D}};
  for (const auto& i : ins) {
    if (i.plain && (i.t->ndim != 2 || i.t->shape[0] != i.rows || i.t->shape[1] != i.cols))
      return set_error(MX_ERR_SHAPE, "%s must be [%lld, %lld]", i.name, (long long)i.rows, (long long)i.cols);
    for (int n = 0; n < i.t->ndim && n < 4; ++n)
      if (i.t->stride[n] < 0) return set_error(MX_ERR_LAYOUT, "%s: negative strides are not supported", i.name);
    if (M > 0 && N > 0 && K > 0 && !i.t->ptr) return set_error(MX_ERR_INVALID, "%s: null data pointer", i.name);
  }
  LinearOut l = {};
  if (int rc = check_linear(bias, residual, activation, M, N, l)) return rc;
  if (int rc = check2d(out, "out", M, N)) return rc;
  l.c = out->ptr; l.c_ld = out->stride[0]; l.c_fmt = out->dtype;
  if (out->dtype == MX_BF16 || out->dtype == MX_F32) {
    if (out_scale) return set_error(MX_ERR_INVALID, "out_scale: only an MX_E4M3 output has one");
    if (int rc = check_apart(out, "out")) return rc;
  } else if (out->dtype == MX_E4M3) {
    if (N % 32 != 0) return set_error(MX_ERR_SHAPE, "N (%lld) must be a multiple of 32 for an MX_E4M3 output", (long long)N);
    if (int rc = check_codes(out, "out", M, N, 8)) return rc;
    if (int rc = check_scales(out_scale, "out_scale", M, N / 32)) return rc;
    l.s = (uint8_t*)out_scale->ptr; l.s_ld = out_scale->stride[0];
  } else {
    return set_error(MX_ERR_DTYPE, "out must be MX_F32, MX_BF16 or MX_E4M3 (got %d)", out->dtype);
  }
  if (pre) {
    if (int rc = check2d(pre, "pre", M, N)) return rc;
    if (pre->dtype != MX_BF16) return set_error(MX_ERR_DTYPE, "pre must be MX_BF16 (got %d)", pre->dtype);
    if (int rc = check_apart(pre, "pre")) return rc;
    l.pre = (uint16_t*)pre->ptr; l.pre_ld = pre->stride[0];
  }
  if (M == 0 || N == 0) return MX_OK;
  if (M == 1) {   // (the pitch of one row is anything)
    l.c_ld = l.pre_ld = l.r_ld = (N + 7) / 8 * 8;
    l.s_ld = N / 32;
  }
  o.accumulate = 0;
  if (int rc = check_room("workspace", workspace, workspace_bytes, linear_workspace(M, N, K, o))) return rc;
  return run_linear(*A, *As, *W, *Ws, l, o, workspace, workspace_bytes, (hipStream_t)stream);
}

int64_t mx_linear_saved_bytes(int64_t T, int64_t K, int64_t N, int32_t activation) {
  if (T <= 0 || K <= 0 || N <= 0) return 0;
  return linear_saved(nullptr, LinearShape{T, K, N, round32(T)}, activation).bytes;
}
int64_t mx_linear_forward_workspace_bytes(int64_t T, int64_t K, int64_t N) {
  if (T <= 0 || K <= 0 || N <= 0) return 0;
  return linear_forward(nullptr, LinearShape{T, K, N, round32(T)}).bytes;
}
int64_t mx_linear_backward_workspace_bytes(int64_t T, int64_t K, int64_t N) {
  if (T <= 0 || K <= 0 || N <= 0) return 0;
  return linear_backward(nullptr, LinearShape{T, K, N, round32(T)}).bytes;
}

int mx_linear_forward(const mx_tensor* x, const mx_tensor* w, const mx_tensor* bias, const mx_tensor* residual, int32_t activation, mx_tensor* y,
                      int32_t scale_mode, void* saved, int64_t saved_bytes, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check2d(x, "x", -1, -1)) return rc;
  if (int rc = check2d(w, "w", -1, x->shape[1])) return rc;
  const LinearShape s = {x->shape[0], x->shape[1], w->shape[0], round32(x->shape[0])};
  if (int rc = check2d(y, "y", s.T, s.N)) return rc;
  if (int rc = check_extents(s.K, s.N)) return rc;
  if (int rc = check_dtype(x, "x", is_float(x->dtype), "MX_F32, MX_BF16 or MX_F16")) return rc;
  if (int rc = check_dtype(w, "w", is_float(w->dtype), "MX_F32, MX_BF16 or MX_F16")) return rc;
  if (int rc = check_dtype(y, "y", y->dtype == MX_F32 || y->dtype == MX_BF16, "MX_F32 or MX_BF16")) return rc;
  LinearOut l = {};
  if (int rc = check_linear(bias, residual, activation, s.T, s.N, l)) return rc;
  if (int rc = check_mode(scale_mode)) return rc;
  if (s.T == 0) return MX_OK;
  if (int rc = check_size(s)) return rc;
  if (int rc = check_apart(y, "y")) return rc;
  const LinearForward f = linear_forward((uint8_t*)workspace, s);
  if (int rc = check_room("workspace", workspace, workspace_bytes, f.bytes)) return rc;
  LinearSaved k = {};
  if (saved) {
    k = linear_saved((uint8_t*)saved, s, activation);
    if (int rc = check_room("saved", saved, saved_bytes, k.bytes)) return rc;
  }
  hipStream_t st = (hipStream_t)stream;
  const bool few = few_tokens(s);
  const BothTensor list[2] = {both(x, f.xq, f.xs, few ? kScalePlain : kScaleNativeA, k.xt, k.xts, kScaleNativeB),
                              both(w, f.w, f.ws, kScaleNativeB, k.wt, k.wts, kScaleNativeB)};
  if (int rc = launch_quantize_both(list, 2, MX_E4M3, scale_mode, st)) return rc;
  l.c = y->ptr; l.c_ld = y->stride[0]; l.c_fmt = y->dtype;
  if (activation != MX_ACT_NONE) { l.pre = (uint16_t*)k.pre; l.pre_ld = s.N; }
  if (few) return launch_gemm_few_linear(FewArgs{f.xq, f.xs, f.w, f.ws, nullptr, (int32_t)s.T, (int32_t)s.N, (int32_t)s.K}, l, st);
  return run_linear(tensor2d(f.xq, MX_E4M3, s.T, s.K, s.K), tensor2d(f.xs, MX_E8M0, s.T, s.K / 32, s.K / 32), tensor2d(f.w, MX_E4M3, s.N, s.K, s.K),
                  tensor2d(f.ws, MX_E8M0, s.N, s.K / 32, s.K / 32), l, layouts(true, true), f.work, f.work_bytes, st);
}

int mx_linear_backward(const mx_tensor* dy, const void* saved, int64_t saved_bytes, int64_t K, int32_t activation, mx_tensor* dx, mx_tensor* dw,
                       mx_tensor* dbias, int32_t scale_mode, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check2d(dy, "dy", -1, -1)) return rc;
  if (int rc = check_dtype(dy, "dy", is_float(dy->dtype), "MX_F32, MX_BF16 or MX_F16")) return rc;
  const LinearShape s = {dy->shape[0], K, dy->shape[1], round32(dy->shape[0])};
  if (int rc = check_extents(s.K, s.N)) return rc;
  if (activation < MX_ACT_NONE || activation > MX_ACT_SILU) return set_error(MX_ERR_INVALID, "unknown activation %d", activation);
  const struct { mx_tensor* t; const char* name; int64_t rows, cols; } outs[2] = {{dx, "dx", s.T, K}, {dw, "dw", s.N, K}};
  for (const auto& o : outs) {
    if (!o.t) continue;
    if (int rc = check2d(o.t, o.name, o.rows, o.cols)) return rc;
    if (int rc = check_dtype(o.t, o.name, o.t->dtype == MX_F32 || o.t->dtype == MX_BF16, "MX_F32 or MX_BF16")) return rc;
    if (int rc = check_apart(o.t, o.name)) return rc;
  }
  if (dbias)
    if (int rc = check_vector(dbias, "dbias", s.N)) return rc;
  if (int rc = check_mode(scale_mode)) return rc;
  if (s.T > 1 && dy->stride[0] > (int64_t)1 << 25) return set_error(MX_ERR_LAYOUT, "dy: rows lie more than 2^25 elements apart");
  if (s.T == 0) return set_error(MX_ERR_SHAPE, "mx_linear_backward: no tokens (the gradients of w and bias are zeros)");
  if (int rc = check_size(s)) return rc;
  if (int rc = check_room("saved", saved, saved_bytes, mx_linear_saved_bytes(s.T, s.K, s.N, activation))) return rc;
  const LinearBackward b = linear_backward((uint8_t*)workspace, s);
  if (int rc = check_room("workspace", workspace, workspace_bytes, b.bytes)) return rc;
  if (!dx && !dw && !dbias) return MX_OK;
  const LinearSaved k = linear_saved((uint8_t*)const_cast<void*>(saved), s, activation);
  hipStream_t st = (hipStream_t)stream;
  ActBackwardArgs a = {};
  a.dy = dy->ptr; a.dy_ld = s.T > 1 ? dy->stride[0] : s.N; a.dy_dtype = dy->dtype;
  if (activation != MX_ACT_NONE) { a.pre = (const uint16_t*)k.pre; a.pre_ld = s.N; }
  a.act = activation; a.scale_mode = scale_mode;
  a.rows = (int32_t)s.T; a.N = (int32_t)s.N;
  if (dx) { a.d = b.d; a.d_ld = s.N; a.ds = b.ds; a.ds_ld = s.N / 32; a.ds_kind = b.native_rows ? kScaleNativeA : kScalePlain; }
  if (dw) { a.dt = b.dt; a.dt_ld = s.Tp; a.dts = b.dts; a.dts_ld = s.Tp / 32; a.dts_kind = kScaleNativeA; }
  if (dbias) a.partial = (float*)b.sums;
  if (int rc = launch_act_backward(a, st)) return rc;
  if (dbias)
    if (int rc = launch_column_sums((const float*)b.sums, (int)((s.T + 127) / 128), s.N, dbias->ptr, dbias->dtype, st)) return rc;
  if (dx)
    if (int rc = product(b.d, b.ds, k.wt, k.wts, *dx, s.T, s.K, s.N, b.o_dx, b.work, b.work_bytes, stream)) return rc;
  if (dw)
    if (int rc = product(b.dt, b.dts, k.xt, k.xts, *dw, s.N, s.K, s.Tp, b.o_dw, b.work, b.work_bytes, stream)) return rc;
  return MX_OK;
}

}  // extern "C"
