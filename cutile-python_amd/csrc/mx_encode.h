// MX encoding of values in registers by the hardware conversions alone: what the kernels that quantise tiles share.  The codes and
// scales are those of encode_block (mx_quant.h) to the bit, but for the sign of NaN.
#pragma once
#include "mx_quant.h"

namespace mx {

typedef uint32_t u2 __attribute__((ext_vector_type(2)));

// ---- maxima over lanes ------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t umin(uint32_t a, uint32_t b) { return a < b ? a : b; }
__device__ __forceinline__ uint32_t max_quad(uint32_t m) {            // lanes 4 n .. 4 n + 3
  m = umax(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xF, 0xF, true));
  return umax(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xF, 0xF, true));
}
__device__ __forceinline__ uint32_t max_xor_8(uint32_t m) {           // lanes l, l ^ 8: a rotation of the 16-lane row by 8
  return umax(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x128, 0xF, 0xF, true));
}
__device__ __forceinline__ uint32_t max_xor_16_32(uint32_t m) {       // lanes l, l ^ 16, l ^ 32, l ^ 48
  const auto a = __builtin_amdgcn_permlane32_swap(m, m, false, false);
  m = umax(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(m, m, false, false);
  return umax(b[0], b[1]);
}
// Maxima of eight columns over lanes l, l ^ 16, l ^ 32, l ^ 48, of which every lane gets two: half of the columns go away with each
// exchange.  r[e] is column e + own_column(lane); spread_columns hands what has been made of them back to all four lanes.
__device__ __forceinline__ int own_column(int lane) { return (lane >> 4 & 1) * 2 + (lane >> 5) * 4; }
__device__ __forceinline__ void max_columns(const uint32_t (&m)[8], uint32_t (&r)[2]) {
  uint32_t t[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const auto a = __builtin_amdgcn_permlane32_swap(m[e], m[e + 4], false, false);
    t[e] = umax(a[0], a[1]);
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const auto a = __builtin_amdgcn_permlane16_swap(t[e], t[e + 2], false, false);
    r[e] = umax(a[0], a[1]);
  }
}
__device__ __forceinline__ void spread_columns(const float (&s)[2], float (&all)[8]) {
  uint32_t t[4];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const uint32_t v = __builtin_bit_cast(uint32_t, s[e]);
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    t[e] = a[0];
    t[e + 2] = a[1];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const auto a = __builtin_amdgcn_permlane32_swap(t[e], t[e], false, false);
    all[e] = __builtin_bit_cast(float, (uint32_t)a[0]);
    all[e + 4] = __builtin_bit_cast(float, (uint32_t)a[1]);
  }
}
__device__ __forceinline__ uint32_t magnitude(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7FFFFFFFu; }

// ---- encoding ---------------------------------------------------------------------------------------------------------------
// The scale of a block whose largest magnitude has the bits `am`, as the hardware conversions take it and as a byte.  They read
// the exponent field of the scale, 0 as 2^-127, and with saturate_conversions() they give the codes of encode_block for every
// finite value and scale, subnormal ones included, and for infinities under the floor rule (compared with the integer encoders over all 255
// exponents of amax, both formats, 2^20 values each).  What is left to encode_block: odd_block().
struct BlockScale {
  float scale;
  uint32_t byte;
};
template <int FMT, bool FLOOR>
__device__ __forceinline__ BlockScale block_scale(uint32_t am) {
  constexpr uint32_t EMAX = FMT == MX_E4M3 ? 8 : 15;
  BlockScale b;
  if constexpr (FLOOR) {
    b.byte = __builtin_elementwise_sub_sat(am >> 23, EMAX);
    b.scale = __builtin_bit_cast(float, b.byte << 23);
  } else {
    const uint32_t t = __builtin_bit_cast(uint32_t, fmaxf(__fdiv_rn(__builtin_bit_cast(float, am), 448.0f), 1e-12f));
    b.byte = (t >> 23) + ((t & 0x7FFFFFu) ? 1 : 0);   // (88 or more)
    b.scale = __builtin_bit_cast(float, b.byte << 23);
  }
  return b;
}
// Mode bit FP16_OVFL of the wave: conversions to 8-bit formats end at the largest finite number instead of NaN or infinity (NaN
// stays), and so do conversions to bf16.  (The ceiling rule never gets there.)  Instructions do not move across a write of that register; what the
// compiler has not made instructions yet it may, down to the only place that uses it.
__device__ __forceinline__ void saturate_conversions(bool on = true) {
  if (on) __builtin_amdgcn_s_setreg(1 | 23 << 6, 1);
  else __builtin_amdgcn_s_setreg(1 | 23 << 6, 0);
}
// Whether the largest amax that a lane has seen belongs to a block that differs: NaN, whose sign the conversions don't keep, and
// under the ceiling rule infinity, where the scale is NaN and finite elements become zeros.
template <bool FLOOR>
__device__ __forceinline__ bool odd_block(uint32_t most) { return FLOOR ? most > 0x7F800000u : most >= 0x7F800000u; }
// four values of a block as codes, lowest byte first
template <int FMT>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, float scale) {
  typedef short s2 __attribute__((ext_vector_type(2)));
  s2 r = {0, 0};
  if constexpr (FMT == MX_E4M3) {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, a, b, scale, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, c, d, scale, true);
  } else {
    r = __builtin_amdgcn_cvt_scalef32_pk_bf8_f32(r, a, b, scale, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_bf8_f32(r, c, d, scale, true);
  }
  return __builtin_bit_cast(uint32_t, r);
}
template <int N>
__device__ inline void encode_slow(const float* v, uint32_t am, int fmt, int scale_mode, uint32_t* packed, uint32_t& byte) {
  uint32_t code[N];
  uint8_t sb;
  encode_block<N>(v, am, fmt, scale_mode, code, sb);
#pragma unroll
  for (int h = 0; h < N / 4; ++h) packed[h] = code[4 * h] | (code[4 * h + 1] << 8) | (code[4 * h + 2] << 16) | (code[4 * h + 3] << 24);
  byte = sb;
}

// m or |a|, the larger; passes over NaN (three of them are one instruction)
__device__ __forceinline__ float fmax_abs(float m, float a) { return __builtin_fmaxf(m, __builtin_fabsf(a)); }

}  // namespace mx
