// What becomes of the gate and up columns that a wave's matrix instructions leave in its lanes (GateOut, mx_common.h).
#pragma once
#include "mx_encode.h"
#include "mx_gemm_tile.h"   // store8_full

namespace mx {

// one MX block's eight values of this lane: codes (E4M3, the floor rule) and scale byte.  NaN counts as more than infinity, as in encode_block: the
// scale is 2^120 and what is finite beside it zero.
__device__ __forceinline__ u2 gated_encode(const float (&v)[8], uint32_t& byte) {
  float m = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = __builtin_elementwise_maximum(m, __builtin_fabsf(v[e]));   // (keeps NaN; two of them are one instruction)
  const BlockScale b = block_scale<MX_E4M3, true>(max_xor_16_32(magnitude(m)));
  byte = b.byte;
  return (u2){encode4<MX_E4M3>(v[0], v[1], v[2], v[3], b.scale), encode4<MX_E4M3>(v[4], v[5], v[6], v[7], b.scale)};
}
struct Ungated {};

// Row `row` (of C, if live), columns col .. col + 7 of gate and up (HALVES: col .. col + 3 and col + 16 .. col + 19).  (The floor rule, bf16 or E4M3: with the other rule and format
// beside them the eight copies of this in a kernel are more than the instruction cache; such calls go through memory.)
// The saturating mode is on for the 8-bit conversions only: with it conversions to bf16 end at the largest finite number too, which is not how gate,
// up and a bf16 result are rounded, and the scaled MFMA takes NaN elements and scales for numbers.  (gate and up are rounded for h, which both branches
// use, so they stay in front of it.  1531 x 4096 -> 14336 to E4M3 149.9 -> 151.5 us, others the same; all rows rounded first and the mode set
// once 150.7, but 8192 rows to bf16 696 -> 709.)
template <bool HALVES = false>
__device__ __forceinline__ void gated_store(const GateOut& o, const v4f (&acc)[4], int64_t row, int col, bool live, bool scale_lane) {
  auto put = [](uint8_t* p, const u2& c) {
    if constexpr (HALVES) {
      *(uint32_t*)p = c[0];
      *(uint32_t*)(p + 16) = c[1];
    } else {
      *(u2*)p = c;
    }
  };
  float g[8], u[8], h[8];
  typedef float f2 __attribute__((ext_vector_type(2)));
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int k = 0; k < 4; ++k) {                        // through bf16, the precision of the activation between the projections
    const uint32_t pg = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){acc[k / 2][2 * (k & 1)], acc[k / 2][2 * (k & 1) + 1]}, b2));
    const uint32_t pu = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){acc[2 + k / 2][2 * (k & 1)], acc[2 + k / 2][2 * (k & 1) + 1]}, b2));
    g[2 * k] = __builtin_bit_cast(float, pg << 16);
    g[2 * k + 1] = __builtin_bit_cast(float, pg & 0xFFFF0000u);
    u[2 * k] = __builtin_bit_cast(float, pu << 16);
    u[2 * k + 1] = __builtin_bit_cast(float, pu & 0xFFFF0000u);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)   // (the hardware's 2^x and reciprocal: a few units in the last place.  Below -126 the reciprocal is 0, which -inf is no factor for)
    h[e] = fmaxf(g[e], -126.0f) * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * g[e])) * u[e];
  if (o.h_fmt == MX_BF16) {
    uint16_t* const p = (uint16_t*)o.h + row * o.h_ld + col;
    if constexpr (HALVES) {
      if (live)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          typedef __bf16 b4 __attribute__((ext_vector_type(4)));
          *(b4*)(p + 16 * k) = __builtin_convertvector((v4f){h[4 * k], h[4 * k + 1], h[4 * k + 2], h[4 * k + 3]}, b4);
        }
    } else if (live) {
      store8_full<uint16_t>(p, (v4f){h[0], h[1], h[2], h[3]}, (v4f){h[4], h[5], h[6], h[7]});
    }
  }
  if (o.h_fmt == MX_BF16 && !o.c) return;
  saturate_conversions(true);
  if (o.h_fmt != MX_BF16) {
    uint32_t byte;
    const u2 c = gated_encode(h, byte);
    if (live) {
      put((uint8_t*)o.h + row * o.h_ld + col, c);
      if (scale_lane) o.hs[row * o.hs_ld + col / 32] = (uint8_t)byte;
    }
  }
  if (o.c) {
    uint32_t bg, bu;
    const u2 cg = gated_encode(g, bg), cu = gated_encode(u, bu);
    if (live) {
      uint8_t* const c = o.c + row * o.c_ld + col;
      put(c, cg);
      put(c + o.F, cu);
      if (scale_lane) {
        uint8_t* const cs = o.cs + row * o.cs_ld + col / 32;
        cs[0] = (uint8_t)bg;
        cs[o.F / 32] = (uint8_t)bu;
      }
    }
  }
  saturate_conversions(false);
}

}  // namespace mx
