// E4M3 products of few rows that are rounded again: C[M, N] = X[M, K] W[N, K]^T in training steps of the feed-forward block.
//
// The scaled MFMA aligns the products of an instruction with some 18 bits below the largest: 1.5e-5 of a sum's norm, whatever K.  With
// many tokens that is far below the roundings around it.  With few, a result that is rounded to bf16 and to E4M3 behind it (gate,
// up, the activation's gradient) may be one of the large ones that carry a norm, and its other neighbour is 2^-4 of it away: a step of one token,
// 1024 x 2048, was 0.0055 of dw1's norm off now and then.  Here elements and scales become bf16 numbers, which is exact but for quantised
// numbers below bf16's smallest (the least code and scale are 2^-136) and for 2^128, to which the ceiling rule rounds floats just below it, and v_mfma_f32_16x16x32_bf16 sums them to 1e-7.
//
// Bound: reading W once.  A load instruction takes 128 bytes, a K-step of four MX blocks, of eight rows; the wave's corner of LDS hands lane
// (c, g) the 32 bytes of row c's block g, whose scale in the native layout is its own (without that, 16 rows x 16 bytes an instruction,
// a step of one token through 4096 x 1024 took 68 us in place of 61).  A bf16 instruction takes eight elements of each of the four
// blocks.  Two K-steps are in flight in registers, eight waves split K and add up in LDS.  Any K % 32 == 0.
#include "mx_gated.h"
#include "mx_train.h"

namespace mx {
namespace {

typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
constexpr int kFewWaves = 8;

// eight elements, two dwords, times the power of two 2^(scale byte - 127)
__device__ __forceinline__ bf8 to_bf16(int lo, int hi, float scale) {
  const bf2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return (bf8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// A workgroup: up to 32 rows of X and four 16-row tiles of W, the 64 rows of group u, or with GATED 32 gate rows and the 32 up rows of the
// same columns.  Beyond 32 rows workgroups share W: ids 8 apart, which are on one XCD.
template <int MT, bool GATED>
__global__ __launch_bounds__(kFewWaves * 64) void few_kernel(const FewArgs a, const GateOut o) {
  __shared__ v4f red[kFewWaves * MT * 4 * 64];         // [wave][row tile][tile][lane]; before, 4 KiB a wave to sort operands in
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, gq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), id = blockIdx.x;
  const int slabs = (a.M + 31) / 32, u = slabs > 1 ? id / (8 * slabs) * 8 + id % 8 : id, m0 = slabs > 1 ? id / 8 % slabs * 32 : 0;
  if (GATED ? 32 * u >= o.F : 64 * u >= a.N) return;   // uniform: the grid is rounded up
  const int K = a.K, steps = (K + 127) / 128, KQ = (steps + 3) / 4;
  const int s0 = wave * steps / kFewWaves, s1 = (wave + 1) * steps / kFewWaves;
  const __amdgpu_buffer_rsrc_t rsX = make_rsrc(a.X, (uint32_t)(a.M * K)), rsXs = make_rsrc(a.Xs, (uint32_t)(a.M * (K / 32)));
  const __amdgpu_buffer_rsrc_t rsW = make_rsrc(a.W, (uint32_t)((int64_t)a.N * K)), rsWs = make_rsrc(a.Ws, (uint32_t)(packed_scale_dwords(a.N, K) * 4));
  uint32_t xo[MT][2], xso[MT], wo[4][2], wso[2], shift[4];
  const int lrow = lane >> 3, lcol = (lane & 7) * 16;  // of a load instruction's eight rows
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = m0 + 16 * i;
#pragma unroll
    for (int h = 0; h < 2; ++h) xo[i][h] = m + 8 * h + lrow < a.M ? (uint32_t)((m + 8 * h + lrow) * K + lcol) : kOobOffset;
    xso[i] = m + r < a.M ? (uint32_t)((m + r) * (K / 32) + gq) : kOobOffset;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int first = GATED ? 32 * u + (j / 2) * o.F : 64 * u + 32 * (j / 2);   // of the 32 rows that tiles j & ~1, j | 1 are
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int n = first + 4 * (j % 2) + bperm_lane_off(8 * h + lrow);
      wo[j][h] = n < a.N ? (uint32_t)n * (uint32_t)K + lcol : kOobOffset;
    }
    shift[j] = 8 * (first / 32 % 2 * 2 + j % 2);
    if (j % 2 == 0) wso[j / 2] = first < a.N ? (uint32_t)(first / 64 * KQ * 1024 + lane * 16) : kOobOffset;
  }
  struct Step {
    v4i x[MT][2], w[4][2];
    uint32_t xs[MT], ws[2];
  };
  auto load = [&](int s, Step& t) {                    // K-step s; beyond the wave's or K's end zeros
    const bool live = s < s1, in = live && 128 * s + lcol < K;
#pragma unroll
    for (int g = 0; g < 2; ++g) t.ws[g] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rsWs, live ? wso[g] : kOobOffset, (s >> 2) * 1024 + (s & 3) * 4, 0);
#pragma unroll
    for (int i = 0; i < MT; ++i) t.xs[i] = __builtin_amdgcn_raw_buffer_load_b8(rsXs, live && 128 * s + 32 * gq < K ? xso[i] : kOobOffset, 4 * s, 0);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) t.x[i][h] = __builtin_amdgcn_raw_buffer_load_b128(rsX, in ? xo[i][h] : kOobOffset, 128 * s, 0);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) t.w[j][h] = __builtin_amdgcn_raw_buffer_load_b128(rsW, in ? wo[j][h] : kOobOffset, 128 * s, 0);
  };
  v4f acc[MT][4] = {};
  // tile of 16 rows x 128 bytes as loaded -> the lane's 32 bytes of it, by way of 2 KiB of LDS (chunks swizzled by row; LDS serves a wave in order)
  uint8_t* const scr = (uint8_t*)red + wave * 4096;
  auto sorted = [&](int slot, const v4i (&in)[2], v4i (&out)[2]) {
    uint8_t* const p = scr + slot * 2048;
#pragma unroll
    for (int h = 0; h < 2; ++h) *(v4i*)(p + (8 * h + lrow) * 128 + (((lane & 7) ^ lrow) << 4)) = in[h];
#pragma unroll
    for (int h = 0; h < 2; ++h) out[h] = *(const v4i*)(p + r * 128 + (((2 * gq + h) ^ (r & 7)) << 4));
  };
  auto multiply = [&](const Step& t) {
    bf8 x[MT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      v4i v[2];
      sorted(i & 1, t.x[i], v);
#pragma unroll
      for (int q = 0; q < 4; ++q) x[i][q] = to_bf16(v[q >> 1][2 * (q & 1)], v[q >> 1][2 * (q & 1) + 1], __builtin_bit_cast(float, t.xs[i] << 23));
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float scale = __builtin_bit_cast(float, (t.ws[j / 2] >> shift[j] & 0xFF) << 23);
      v4i v[2];
      sorted(j & 1, t.w[j], v);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const bf8 w = to_bf16(v[q >> 1][2 * (q & 1)], v[q >> 1][2 * (q & 1) + 1], scale);
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, x[i][q], acc[i][j], 0, 0, 0);
      }
    }
  };
  Step t[2];
  load(s0, t[0]);
  for (int s = s0; s < s1; s += 2) {
    load(s + 1, t[1]);
    multiply(t[0]);
    load(s + 2, t[0]);
    multiply(t[1]);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) red[((wave * MT + i) * 4 + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  // ---- the ranges of K, added in their order -----------------------------------------------------------------------
  if (wave >= MT) return;
  const int row = m0 + 16 * wave + r;
  v4f v[4] = {};
  for (int k = 0; k < kFewWaves; ++k)
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += red[((k * MT + wave) * 4 + j) * 64 + lane];
  if constexpr (GATED) {
    gated_store(o, v, row, 32 * u + 8 * gq, row < a.M, gq == 0);
  } else {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int n = 64 * u + 32 * p + 8 * gq;
      if (row < a.M && n < a.N) store8_full<uint16_t>(a.C + (int64_t)row * a.N + n, v[2 * p], v[2 * p + 1]);
    }
  }
}

template <bool GATED>
int launch(const FewArgs& a, const GateOut& o, int units, hipStream_t stream) {
  const int slabs = (a.M + 31) / 32, blocks = slabs > 1 ? (units + 7) / 8 * 8 * slabs : units;
  const hipError_t e = a.M <= 16 ? launch_kernel(few_kernel<1, GATED>, dim3((unsigned)blocks), dim3(kFewWaves * 64), 0, stream, a, o)
                                 : launch_kernel(few_kernel<2, GATED>, dim3((unsigned)blocks), dim3(kFewWaves * 64), 0, stream, a, o);
  if (e != hipSuccess) return set_error(MX_ERR_LAUNCH, "few_kernel launch: %s", hipGetErrorString(e));
  return MX_OK;
}

}  // namespace

// (operands of less than 2 GiB, checked by the callers)
int launch_gemm_few(const FewArgs& a, hipStream_t stream) { return launch<false>(a, GateOut{}, (a.N + 63) / 64, stream); }
int launch_gemm_few_gated(const FewArgs& a, const GateOut& o, hipStream_t stream) { return launch<true>(a, o, o.F / 32, stream); }

}  // namespace mx
