// Kernels of the gated feed-forward block that is trained in 8 bits (mx_train.hip) and what they are given.
#pragma once
#include "mx_common.h"

namespace mx {

// where a block's scale byte goes: [rows][blocks], or one of the layouts that the products read (mx_common.h)
enum { kScalePlain = 0, kScaleNativeA = 1, kScaleNativeB = 2 };

// quantisation of one matrix along its rows (q, s) and, transposed, along its columns (qt, st); either pair may be null
struct BothTensor {
  const void* x;
  int64_t x_ld;                      // elements
  uint8_t *q, *s, *qt, *st;
  int64_t q_ld, s_ld, qt_ld, st_ld;  // bytes; s_ld, st_ld of plain scales
  int32_t rows, K, x_dtype;
  int32_t s_kind, st_kind;           // kScale*
  // filled in by the launcher
  int32_t first, tiles, tiles_k, once, near;
};
constexpr int kBothMax = 3;
struct BothArgs {
  BothTensor t[kBothMax];
  int32_t n, scale_mode;
};
// up to kBothMax matrices, all quantised to `fmt` (MX_E4M3, MX_E5M2): one launch per run of equal x_dtype
int launch_quantize_both(const BothTensor* list, int n, int fmt, int scale_mode, hipStream_t stream);

// [g|u] (bf16 [rows, 2 F]) -> silu(g) * u, as bf16 or quantised, and optionally [g|u] quantised to E4M3
struct GateUpArgs {
  const uint16_t* gu;
  int64_t gu_ld, rows;
  GateOut out;
};
int launch_gate_up(const GateUpArgs& a, hipStream_t stream);

// E4M3 products of few rows in 32-bit precision (mx_gemm_few.hip): rows without gaps, X's scales plain, W's native (operand B)
struct FewArgs {
  const uint8_t *X, *Xs, *W, *Ws;
  uint16_t* C;                       // bf16 [M, N]; gated: not used
  int32_t M, N, K;                   // N and K multiples of 32
};
int launch_gemm_few(const FewArgs& a, hipStream_t stream);
int launch_gemm_few_gated(const FewArgs& a, const GateOut& o, hipStream_t stream);   // N = 2 F; the floor rule, E4M3 out

// dh and the checkpoint [g|u] -> d[g|u] quantised along rows and columns, silu(g) * u along columns (all E4M3)
struct SiluBackwardArgs {
  const uint16_t* dh;                // bf16
  const uint8_t *gu, *gus;
  uint8_t *d, *ds, *dt, *dts, *at, *ats;
  int64_t dh_ld, gu_ld, gus_ld, d_ld, ds_ld, dt_ld, dts_ld, at_ld, ats_ld;
  int32_t rows, F, scale_mode;
  int32_t ds_kind, dts_kind, ats_kind;   // kScale*; other than plain only with F % 64 == 0
  int32_t tiles_k;                       // filled in by the launcher
};
int launch_silu_backward(const SiluBackwardArgs& a, hipStream_t stream);

}  // namespace mx
