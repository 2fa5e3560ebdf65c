// What becomes of the columns of a product in a linear layer: act(product + bias) + residual, rounded or MX-quantised, and
// optionally product + bias itself for the backward pass.
//
// Activations, with the hardware's 2^x and reciprocal (a few units in the last place of 32 bits):
//   silu       x s(x),  s(z) = 1 / (1 + exp(-z))
//   gelu_tanh  x s(2 c (x + 0.044715 x^3)),  c = sqrt(2 / pi): the same form, its argument x (k1 + k3 x^2)
//   gelu       x P(X < x) = max(x, 0) - |x| q(|x|),  q(a) = erfc(a / sqrt 2) / 2 = exp(-a^2 / 2) t (c1 + c2 t + .. + c7 t^6) with t = 1 / (1 + 0.35 a):
//              fitted to 2.6e-7 of the value up to a = 7 (3.5e-5 up to 12.75, where x q is 2e-36, 4.4e-5 up to 14)
// Each is within 2e-6 + 2.5e-7 |z| of its value (gelu beyond 7: the fit's error more), exp(-|z|) the exponential in it: z is off by its roundings and
// those of its constants, by 2.3e-7 of it at most (gelu_tanh), and so is the exponential, relatively, by that much.  Where 1 / (1 + exp(-z)) or q is below
// 2^-126 it is zero: so may be numbers below 2e-36.
// Bound, in a large product: this arithmetic, which little of the product runs beside (8192 x 14336 x 4096 on the ping-pong kernel, to bf16: plain
// product 338 us, bias 348, silu 368, gelu 390); in a small one the launch (1 x 8192 x 2048: 4.8 and 5.1 to 5.5).
// Far out a factor is 0 or 1, and x ends at -126 in front of it: -inf makes -0 of silu and gelu (inf times 0 is NaN; x^2 ends at 1e30 for
// the same reason, k3 is 0 for silu).  A NaN is NaN.
#pragma once
#include "mx_gated.h"
#include "mx_rows.h"

namespace mx {

struct LinearOut {
  void* c;                             // [rows][N]: bf16, fp32 or E4M3 codes (the floor rule, N % 32 == 0)
  uint8_t* s;                          // [rows][N / 32]
  uint16_t* pre;                       // bf16 [rows][N] or null: product + bias
  const void *bias, *res;              // [N], [rows][N]; either may be null
  int64_t c_ld, s_ld, pre_ld, r_ld;    // elements; bytes of codes and scales
  int32_t N, c_fmt, bias_dtype, res_dtype, act;
};
constexpr float kLog2E = 1.44269504f;

// activations of one kind share code: what differs are two constants
enum { kActPlain = 0, kActSigmoid = 1, kActErf = 2 };
inline int act_kind(int act) { return act == MX_ACT_GELU ? kActErf : act == MX_ACT_SILU || act == MX_ACT_GELU_TANH ? kActSigmoid : kActPlain; }

__device__ __forceinline__ float sigmoid_of(float z2) {   // 1 / (1 + 2^-z2)
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-z2));
}
// erfc(a / sqrt 2) / 2 of a >= 0; x2 = a^2
__device__ __forceinline__ float upper_tail(float a, float x2) {
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.35f, a, 1.0f)), e = __builtin_amdgcn_exp2f(x2 * (-0.5f * kLog2E));
  float p = 0.04749621718155301f;
  p = __builtin_fmaf(p, t, -0.19578235176913694f);
  p = __builtin_fmaf(p, t, 0.22907965550534493f);
  p = __builtin_fmaf(p, t, -0.005667519383105447f);
  p = __builtin_fmaf(p, t, 0.14949177971864963f);
  p = __builtin_fmaf(p, t, 0.13548805371821698f);
  p = __builtin_fmaf(p, t, 0.13989429034358855f);
  return p * t * e;
}
// k1, k3 of an activation of the sigmoid kind, times log2 e
__device__ __forceinline__ void sigmoid_constants(int act, float& k1, float& k3) {
  k1 = act == MX_ACT_SILU ? kLog2E : 1.5957691216f * kLog2E;
  k3 = act == MX_ACT_SILU ? 0.f : 1.5957691216f * 0.044715f * kLog2E;
}
// (maximum, which keeps NaN, and the median in the place of fmax and fmin: for those what comes from another block of code is made canonical
// first, an instruction each)
template <int KIND>
__device__ __forceinline__ void activate(float (&v)[8], int act) {
  if constexpr (KIND == kActPlain) {
    const float least = act == MX_ACT_RELU ? 0.f : -__builtin_inff();
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = __builtin_elementwise_maximum(v[e], least);   // (keeps NaN)
  } else if constexpr (KIND == kActSigmoid) {
    float k1, k3;
    sigmoid_constants(act, k1, k3);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = __builtin_elementwise_maximum(v[e], -126.0f) * sigmoid_of(v[e] * __builtin_fmaf(fminf(v[e] * v[e], 1e30f), k3, k1));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = __builtin_fabsf(v[e]);
      v[e] = __builtin_fmaf(-__builtin_amdgcn_fmed3f(a, 0.f, 126.0f), upper_tail(a, v[e] * v[e]), __builtin_elementwise_maximum(v[e], 0.f));
    }
  }
}
// the activation's derivative (d/dx x s(f(x)) = s + x f'(x) s (1 - s); d/dx x P = P + x exp(-x^2 / 2) / sqrt(2 pi)); NaN for NaN
template <int KIND>
__device__ __forceinline__ float act_slope(float x, int act) {
  if constexpr (KIND == kActPlain) return x > 0.f ? 1.0f : x <= 0.f ? 0.f : x;   // (relu: with no activation nobody asks)
  const float c = __builtin_amdgcn_fmed3f(x, -126.0f, 126.0f), x2 = x * x;
  if constexpr (KIND == kActErf) {
    const float q = upper_tail(__builtin_fabsf(x), x2);
    return __builtin_fmaf(c, 0.3989422804f * __builtin_amdgcn_exp2f(x2 * (-0.5f * kLog2E)), x > 0.f ? 1.0f - q : q);
  }
  float k1, k3;
  sigmoid_constants(act, k1, k3);
  const float s = sigmoid_of(x * __builtin_fmaf(fminf(x2, 1e30f), k3, k1));
  const float slope = __builtin_fmaf(c * c, 3.0f * k3, k1) * (1.0f / kLog2E);   // f'(x)
  return __builtin_fmaf(c * s, (1.0f - s) * slope, s);
}

// eight numbers of a row as they lie in memory (fp32: two pieces), to be asked for ahead of their use
struct FloatsPiece { u4 lo, hi; };
__device__ __forceinline__ void request_floats(const void* p, int dtype, int64_t at, int n, FloatsPiece& r) {
  if (dtype == MX_F32) {
    r.lo = load_piece<MX_F32>(p, at, n);
    r.hi = load_piece<MX_F32>(p, at + 4, n - 4);
  } else {
    r.lo = load_piece<MX_BF16>(p, at, n);
  }
}
__device__ __forceinline__ void floats_of(const FloatsPiece& p, int dtype, float (&v)[8]) {
  if (dtype == MX_F32) {
    float x[4], y[4];
    unpack_piece<MX_F32>(p.lo, x);
    unpack_piece<MX_F32>(p.hi, y);
#pragma unroll
    for (int e = 0; e < 4; ++e) { v[e] = x[e]; v[4 + e] = y[e]; }
  } else if (dtype == MX_BF16) {
    unpack_piece<MX_BF16>(p.lo, v);
  } else {
    unpack_piece<MX_F16>(p.lo, v);
  }
}
__device__ __forceinline__ void linear_request(const LinearOut& o, FloatsPiece& r, int64_t row, int col, int cols, bool live) {
  if (o.res) request_floats((const uint8_t*)o.res + row * o.r_ld * (o.res_dtype == MX_F32 ? 4 : 2), o.res_dtype, col, live ? cols : 0, r);
}
__device__ __forceinline__ void linear_add(const LinearOut& o, const FloatsPiece& p, float (&v)[8]) {
  if (!o.res) return;
  float r[8];
  floats_of(p, o.res_dtype, r);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] += r[e];
}

// scale of the block that four lanes hold (LANES16: l ^ 16, l ^ 32, else 4 n .. 4 n + 3), and its byte
template <bool LANES16>
__device__ __forceinline__ float linear_scale(const float (&v)[8], uint32_t& byte) {
  float m = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = __builtin_elementwise_maximum(m, __builtin_fabsf(v[e]));   // (keeps NaN: block_quantize's scale and zeros)
  const BlockScale s = block_scale<MX_E4M3, true>(LANES16 ? max_xor_16_32(magnitude(m)) : max_quad(magnitude(m)));
  byte = s.byte;
  return s.scale;
}

// Columns col .. col + 7 of row `row`, of which `cols` (1 to 8; anything less: none) exist; a, b: the product.  live: the row exists.
// With codes four lanes hold a block's 32 columns, scale_lane one of them.
template <int KIND, bool LANES16>
__device__ __forceinline__ void linear_finish(const LinearOut& o, const v4f& a, const v4f& b, const float (&bias)[8], const FloatsPiece& res, int64_t row, int col,
                                              int cols, bool live, bool scale_lane) {
  const bool in = live && cols > 0;
  float v[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = a[e] + bias[e];
    v[4 + e] = b[e] + bias[4 + e];
  }
  auto put16 = [&](uint16_t* p) { store8_edge<uint16_t>(p, (v4f){v[0], v[1], v[2], v[3]}, (v4f){v[4], v[5], v[6], v[7]}, cols); };
  if (o.pre && in) put16(o.pre + row * o.pre_ld + col);
  activate<KIND>(v, o.act);
  linear_add(o, res, v);
  if (o.c_fmt == MX_BF16) {
    if (in) put16((uint16_t*)o.c + row * o.c_ld + col);
  } else if (o.c_fmt == MX_F32) {
    if (in) store8_edge<float>((float*)o.c + row * o.c_ld + col, (v4f){v[0], v[1], v[2], v[3]}, (v4f){v[4], v[5], v[6], v[7]}, cols);
  } else {
    uint32_t byte;
    const float scale = linear_scale<LANES16>(v, byte);
    // (the mode is set back behind the store: before it, the compiler takes the conversions down to the store, out of the mode)
    saturate_conversions(true);
    const u2 c = {encode4<MX_E4M3>(v[0], v[1], v[2], v[3], scale), encode4<MX_E4M3>(v[4], v[5], v[6], v[7], scale)};
    if (in) {
      *(u2*)((uint8_t*)o.c + row * o.c_ld + col) = c;
      if (scale_lane) o.s[row * o.s_ld + col / 32] = (uint8_t)byte;
    }
    saturate_conversions(false);
  }
}
// the same with the kind chosen here, where one place finishes all that a wave has
template <bool LANES16>
__device__ __forceinline__ void linear_finish_any(const LinearOut& o, const v4f& a, const v4f& b, const float (&bias)[8], const FloatsPiece& res, int64_t row, int col,
                                                  int cols, bool live, bool scale_lane) {
  if (o.act == MX_ACT_GELU) linear_finish<kActErf, LANES16>(o, a, b, bias, res, row, col, cols, live, scale_lane);
  else if (o.act == MX_ACT_SILU || o.act == MX_ACT_GELU_TANH) linear_finish<kActSigmoid, LANES16>(o, a, b, bias, res, row, col, cols, live, scale_lane);
  else linear_finish<kActPlain, LANES16>(o, a, b, bias, res, row, col, cols, live, scale_lane);
}

// What a wave's row tiles of the ping-pong kernel leave by: everything through buffer descriptors, whose range takes the place of comparisons
// with the last row; columns that are not there have an offset beyond it.  bf16 or fp32 (CODES false) or E4M3 out, a bf16 residual or, CODES false, an fp32
// one, rows of whole 16-byte pieces (codes: of 8), each tensor less than 2 GiB, the rows behind it that a tile reaches included (their offsets must not
// come round): linear_is_plain().
inline bool linear_is_plain(const LinearOut& o, int64_t M) {
  const int64_t lim = (int64_t)1 << 31;
  auto fine = [&](const void* p, int64_t ld, int size, int align) { return !p || ((uintptr_t)p % align == 0 && ld * size % align == 0 && (M + 256) * ld * size < lim); };
  const bool codes = o.c_fmt == MX_E4M3, r32 = o.res_dtype == MX_F32;
  const bool out = codes ? fine(o.c, o.c_ld, 1, 8) && fine(o.s, o.s_ld, 1, 1) : fine(o.c, o.c_ld, o.c_fmt == MX_F32 ? 4 : 2, 16);
  return o.N % 8 == 0 && out && fine(o.pre, o.pre_ld, 2, 16) && (!o.res || ((o.res_dtype == MX_BF16 || (r32 && !codes)) && fine(o.res, o.r_ld, r32 ? 4 : 2, 16)));
}
__device__ __forceinline__ void linear_bias(const LinearOut& o, int col, float (&bias)[8]) { load_floats<8>(o.bias, o.bias_dtype, col, o.N - col, 0.f, bias); }

// the product's kernels with this epilogue: MX_KERNEL_MFMA_PINGPONG, MX_KERNEL_MFMA_128x128 (one K range), MX_KERNEL_STREAM
int launch_gemm_pingpong_linear(const GemmArgs& g, const LinearOut& o, hipStream_t stream);
struct T128Args;
int launch_gemm_t128_linear(const T128Args& g, const LinearOut& o, hipStream_t stream);
struct StreamArgs;
int launch_gemm_stream_linear(const StreamArgs& a, const LinearOut& o, hipStream_t stream);
// a product on the kernel that mx_gemm would take, with its workspace; kLinearNotFused: on none of these (nothing enqueued)
constexpr int kLinearNotFused = 3;
int gemm_linear_fused(const mx_tensor& A, const mx_tensor& As, const mx_tensor& W, const mx_tensor& Ws, const LinearOut& out, const mx_gemm_opts& o,
                      void* workspace, int64_t workspace_bytes, hipStream_t stream);

// fp32 products [splits][M][N], added in their order, to the layer's output (mx_linear.hip); splits may be zero
int launch_linear_pass(const float* product, int splits, int64_t M, const LinearOut& o, hipStream_t stream);

// gradient through the activation, quantised along rows and columns, with the bias's gradient (mx_linear.hip)
struct ActBackwardArgs {
  const void* dy;
  const uint16_t* pre;                 // bf16; null: no activation
  uint8_t *d, *ds, *dt, *dts;          // d or dt may be null
  float* partial;                      // [rows / 128, rounded up][N] or null: no bias gradient
  int64_t dy_ld, pre_ld, d_ld, ds_ld, dt_ld, dts_ld;
  int32_t rows, N, dy_dtype, act, scale_mode, ds_kind, dts_kind;
  int32_t tiles_k, tiles;              // filled in by the launcher
};
int launch_act_backward(const ActBackwardArgs& a, hipStream_t stream);
int launch_column_sums(const float* partial, int parts, int64_t N, void* out, int out_dtype, hipStream_t stream);

}  // namespace mx
