// What becomes of the columns of a product in a linear layer: act(product + bias) + residual, rounded or MX-quantised, and
// optionally product + bias itself for the backward pass.
//
// Activations, with the hardware's 2^x and reciprocal (a few units in the last place of 32 bits):
//   silu       x s(x),  s(z) = 1 / (1 + exp(-z))
//   gelu_tanh  x s(2 c (x + 0.044715 x^3)),  c = sqrt(2 / pi): the same form, its argument x (k1 + k3 x^2)
//   gelu       x P(X < x) = max(x, 0) - |x| q(|x|),  q(a) = erfc(a / sqrt 2) / 2 = exp(-a^2 / 2) t (c1 + c2 t + .. + c7 t^6) with t = 1 / (1 + 0.35 a):
//              fitted to 2.6e-7 of the value up to a = 7 (4e-5 up to 14, where q is 1e-44); exp's argument rounds to 1e-6 there
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
    for (int e = 0; e < 8; ++e) v[e] = fmaxf(v[e], -126.0f) * sigmoid_of(v[e] * __builtin_fmaf(fminf(v[e] * v[e], 1e30f), k3, k1));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = __builtin_fabsf(v[e]);
      v[e] = __builtin_fmaf(-fminf(a, 126.0f), upper_tail(a, v[e] * v[e]), fmaxf(v[e], 0.f));
    }
  }
}
// the activation's derivative (d/dx x s(f(x)) = s + x f'(x) s (1 - s); d/dx x P = P + x exp(-x^2 / 2) / sqrt(2 pi)); NaN for NaN
__device__ __forceinline__ float act_slope(float x, int act) {
  if (act == MX_ACT_NONE) return 1.0f;
  if (act == MX_ACT_RELU) return x > 0.f ? 1.0f : x <= 0.f ? 0.f : x;
  const float c = __builtin_amdgcn_fmed3f(x, -126.0f, 126.0f), x2 = x * x;
  if (act == MX_ACT_GELU) {
    const float q = upper_tail(__builtin_fabsf(x), x2);
    return __builtin_fmaf(c, 0.3989422804f * __builtin_amdgcn_exp2f(x2 * (-0.5f * kLog2E)), x > 0.f ? 1.0f - q : q);
  }
  float k1, k3;
  sigmoid_constants(act, k1, k3);
  const float s = sigmoid_of(x * __builtin_fmaf(fminf(x2, 1e30f), k3, k1));
  const float slope = __builtin_fmaf(c * c, 3.0f * k3, k1) * (1.0f / kLog2E);   // f'(x)
  return __builtin_fmaf(c * s, (1.0f - s) * slope, s);
}

// Columns col .. col + 7 of row `row`, of which `cols` (1 to 8; anything less: none) exist; a, b: the product.  live: the row exists.
// With codes the four lanes l ^ 16, l ^ 32 (LANES16) or 4 n .. 4 n + 3 hold a block's 32 columns, scale_lane one of them.
template <int KIND, bool LANES16>
__device__ __forceinline__ void linear_finish(const LinearOut& o, const v4f& a, const v4f& b, const float (&bias)[8], int64_t row, int col, int cols, bool live,
                                              bool scale_lane) {
  const bool in = live && cols > 0;
  float v[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = a[e] + bias[e];
    v[4 + e] = b[e] + bias[4 + e];
  }
  if (o.pre && in)
    store8_edge<uint16_t>(o.pre + row * o.pre_ld + col, (v4f){v[0], v[1], v[2], v[3]}, (v4f){v[4], v[5], v[6], v[7]}, cols);
  activate<KIND>(v, o.act);
  if (o.res && in) {
    float r[8];
    load_floats<8>((const uint8_t*)o.res + row * o.r_ld * (o.res_dtype == MX_F32 ? 4 : 2), o.res_dtype, col, cols, 0.f, r);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += r[e];
  }
  const v4f lo = {v[0], v[1], v[2], v[3]}, hi = {v[4], v[5], v[6], v[7]};
  if (o.c_fmt == MX_BF16) {
    if (in) store8_edge<uint16_t>((uint16_t*)o.c + row * o.c_ld + col, lo, hi, cols);
  } else if (o.c_fmt == MX_F32) {
    if (in) store8_edge<float>((float*)o.c + row * o.c_ld + col, lo, hi, cols);
  } else {
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = __builtin_elementwise_maximum(m, __builtin_fabsf(v[e]));   // (keeps NaN: block_quantize's scale and zeros)
    const uint32_t am = LANES16 ? max_xor_16_32(magnitude(m)) : max_quad(magnitude(m));
    const BlockScale s = block_scale<MX_E4M3, true>(am);
    saturate_conversions(true);
    const u2 c = {encode4<MX_E4M3>(v[0], v[1], v[2], v[3], s.scale), encode4<MX_E4M3>(v[4], v[5], v[6], v[7], s.scale)};
    saturate_conversions(false);
    if (in) {
      *(u2*)((uint8_t*)o.c + row * o.c_ld + col) = c;
      if (scale_lane) o.s[row * o.s_ld + col / 32] = (uint8_t)s.byte;
    }
  }
}
__device__ __forceinline__ void linear_bias(const LinearOut& o, int col, float (&bias)[8]) { load_floats<8>(o.bias, o.bias_dtype, col, o.N - col, 0.f, bias); }

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
