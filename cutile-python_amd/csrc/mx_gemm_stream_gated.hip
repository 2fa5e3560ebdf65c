// Gated product of few rows (decode): the weights streamed through registers as in mx_gemm_stream.h, silu(gate) * up and its
// quantisation in the epilogue.
//
// Bound: reading W once.  A wave takes 32 gate rows and the 32 up rows that belong to them, four 16-row tiles, and a range of K; the
// ranges of a workgroup's waves meet in LDS, where a lane then finds gate and up of eight columns, and the four lanes l ^ 16, l ^ 32
// an MX block.  Workgroups of four waves: two of them fit on a CU, one's start and output beside the other's stream; with eight
// waves 4096 x 4096 (K x F) FP8 takes 10.5 us in place of 8.8, 8192 x 14336 48 in place of 38.
// One row: 2048 x 7168 FP8 7.2 us (29 MB of W and 1 of scales, 4.2 TB/s; a launch alone is about 3), 8192 x 14336 38 us (235 MB, 6.2 TB/s).
#include "mx_gated.h"
#include "mx_gemm_stream.h"

namespace mx {
namespace {

constexpr int kGatedWaves = 4;

template <class C>
__global__ __launch_bounds__(C::WAVES * 64, 2) void stream_gated_kernel(const StreamArgs a, const GateOut o) {
  constexpr int NT = C::NT, MT = C::MT;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem_generic[];
  lds_u8* const smem = (lds_u8*)smem_generic;
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, gq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kq = wave % a.kw, nw = wave / a.kw, nwv = C::WAVES / a.kw;
  const int u = blockIdx.x * nwv + nw;               // unit: 32 columns
  const int KQ = (a.K + 511) / 512;
  const int Q0 = kq * KQ / a.kw, Q1 = (kq + 1) * KQ / a.kw;
  const int half[2] = {32 * u, o.F + 32 * u};        // first row of tiles 0, 1 and of tiles 2, 3
  const bool in = half[0] < o.F;

  StreamWave w;
  w.rsX = make_rsrc(a.X, (uint32_t)((int64_t)(a.M - 1) * a.ldx + a.K));
  w.rsXs = make_rsrc(a.Xs, (uint32_t)((int64_t)(a.M - 1) * a.ldxs + a.K / 32));
  w.rsW = make_rsrc(a.W, (uint32_t)((int64_t)(a.N - 1) * a.ldw + (int64_t)a.K * (C::WF == MX_E2M1 ? 1 : 2) / 2));
  w.rsWs = C::PACKED ? make_rsrc(a.Ws, (uint32_t)(packed_scale_dwords(a.N, a.K) * 4))
                     : make_rsrc(a.Ws, (uint32_t)((int64_t)(a.N - 1) * a.ldws + a.K / 32));
  uint32_t xvo[2 * MT], xso[MT], wvo[2 * NT], wso[C::NSW];
  int j0[2];
#pragma unroll
  for (int q = 0; q < 2 * MT; ++q) {
    const int m = 8 * q + (lane >> 3);
    xvo[q] = m < a.M ? (uint32_t)(m * a.ldx + stream_x_col(q, lane)) : kOobOffset;
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = 16 * i + r;
    xso[i] = m < a.M ? (uint32_t)(m * a.ldxs) : kOobOffset;
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int base = half[j / 2] + 4 * (j % 2);
#pragma unroll
    for (int h = 0; h < 2; ++h) wvo[2 * j + h] = in ? (uint32_t)((base + bperm_lane_off(8 * h + (lane >> 3))) * a.ldw + (lane & 7) * 16) : kOobOffset;
    if constexpr (!C::PACKED) wso[j] = in ? (uint32_t)((base + bperm_lane_off(r)) * a.ldws) : kOobOffset;
  }
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    j0[g] = half[g] / 32 % 2 * 2;
    if constexpr (C::PACKED) wso[g] = in ? (uint32_t)(half[g] / 64 * KQ * 1024 + lane * 16) : kOobOffset;
  }
  v4f acc[MT][NT];
  stream_products<C>(w, smem + wave * C::WAVE_BYTES, xvo, xso, wvo, wso, j0, Q0, Q1, (a.K + 127) / 128, acc);

  // ---- the K ranges meet in LDS, added in their order ------------------------------------------------------------
  __syncthreads();
  typedef __attribute__((address_space(3))) v4f lds_v4f;
  lds_v4f* const red = (lds_v4f*)smem;               // [nw][kq][i][j][lane]
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) red[((nw * a.kw + kq) * (MT * NT) + i * NT + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  for (int it = wave; it < nwv * MT; it += C::WAVES) {   // uniform per wave
    const int i = it % MT, wv = it / MT;
    v4f v[4] = {};
    for (int k = 0; k < a.kw; ++k)
#pragma unroll
      for (int h = 0; h < 4; ++h) v[h] += red[((wv * a.kw + k) * (MT * NT) + i * NT + h) * 64 + lane];
    const int col = 32 * (blockIdx.x * nwv + wv) + 8 * gq, row = 16 * i + r;
    if (col < o.F) gated_store(o, v, row, col, row < a.M, gq == 0);   // uniform: F is a multiple of 32
  }
}

template <class C>
int launch(const StreamArgs& a, const GateOut& o, int blocks, hipStream_t stream) {
  auto kern = stream_gated_kernel<C>;
  static int attr_done = 0;   // benign race: the attribute call is idempotent
  if (!attr_done) {
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS_BYTES);
    if (e != hipSuccess) return set_error(MX_ERR_LAUNCH, "hipFuncSetAttribute(%d bytes LDS): %s", C::LDS_BYTES, hipGetErrorString(e));
    attr_done = 1;
  }
  const hipError_t e = launch_kernel(kern, dim3((unsigned)blocks), dim3(C::WAVES * 64), C::LDS_BYTES, stream, a, o);
  if (e != hipSuccess) return set_error(MX_ERR_LAUNCH, "stream_gated_kernel launch: %s", hipGetErrorString(e));
  return MX_OK;
}

template <int XF, int WF, int MT, bool PACKED>
int launch_p(const StreamArgs& a, const GateOut& o, int blocks, hipStream_t stream) {
  if (stream_loads_once(a.N, WF == MX_E2M1 ? a.K / 2 : a.K, a.ldw, (uint64_t)a.W, 1))
    return launch<StreamCfg<XF, WF, 4, MT, PACKED, kGatedWaves, true, true>>(a, o, blocks, stream);
  return launch<StreamCfg<XF, WF, 4, MT, PACKED, kGatedWaves, true>>(a, o, blocks, stream);
}
template <int XF, int WF>
int launch_m(const StreamArgs& a, const GateOut& o, int blocks, hipStream_t stream) {
  if (a.M <= 16) return a.ws_packed ? launch_p<XF, WF, 1, true>(a, o, blocks, stream) : launch_p<XF, WF, 1, false>(a, o, blocks, stream);
  return a.ws_packed ? launch_p<XF, WF, 2, true>(a, o, blocks, stream) : launch_p<XF, WF, 2, false>(a, o, blocks, stream);
}

}  // namespace

int launch_gemm_stream_gated(const StreamArgs& a0, const GateOut& o, hipStream_t stream) {
  StreamArgs a = a0;
  if (a.M < 1 || a.M > kStreamGatedRows || a.N != 2 * o.F || o.F % 32 != 0) return set_error(MX_ERR_SHAPE, "gated stream kernel: unsupported sizes");
  if (const char* why = stream_issue(a)) return set_error(MX_ERR_LAYOUT, "gated stream kernel: %s", why);
  // as many K ranges as there are, up to a wave each: the most waves, hence the most of W in flight
  const int KQ = (a.K + 511) / 512;
  a.kw = KQ >= 4 ? 4 : KQ >= 2 ? 2 : 1;
  const int nwv = kGatedWaves / a.kw, blocks = (o.F / 32 + nwv - 1) / nwv;
#define MX_CASE(XF, WF) \
  if (a.x_fmt == XF && a.w_fmt == WF) return launch_m<XF, WF>(a, o, blocks, stream);
  MX_CASE(MX_E4M3, MX_E4M3)
  MX_CASE(MX_E4M3, MX_E2M1)
  MX_CASE(MX_E5M2, MX_E5M2)
  MX_CASE(MX_E5M2, MX_E2M1)
#undef MX_CASE
  return set_error(MX_ERR_DTYPE, "gated stream kernel: unsupported element format pair (%d, %d)", a.x_fmt, a.w_fmt);
}

}  // namespace mx
