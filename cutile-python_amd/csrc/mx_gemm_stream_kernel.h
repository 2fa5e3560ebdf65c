// The weight-streaming kernel of plain products and of linear layers, and its launch (mx_gemm_stream.hip, mx_gemm_stream_linear.hip).
#pragma once
#include "mx_gemm_stream.h"
#include "mx_linear.h"

namespace mx {
namespace {

// Workgroup of C::WAVES waves: kw K ranges x WAVES / kw units of NT tiles.  m_tiles row tiles of 16 MT rows are neighbours in
// dispatch order on the same XCD (workgroup ids go round-robin over 8 XCDs), so W is read from memory once.
// Out: Ungated (C) or LinearOut: bias, activation and residual of a linear layer (mx_linear.h; not with NT of 1 where
// the result is quantised: a lane has four columns then, a workgroup perhaps sixteen).
template <class C, class Out>
__global__ __launch_bounds__(C::WAVES * 64) void stream_kernel(const StreamArgs a, const Out o) {
  constexpr bool LINEAR = std::is_same<Out, LinearOut>::value;
  constexpr int NT = C::NT, MT = C::MT;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem_generic[];
  lds_u8* const smem = (lds_u8*)smem_generic;
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, gq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kq = wave % a.kw, nw = wave / a.kw, nwv = C::WAVES / a.kw;
  int unit0 = blockIdx.x, mt = 0;
  if (a.m_tiles > 1) {
    const int per = 8 * a.m_tiles, hi = unit0 / per, in = unit0 % per;
    mt = in / 8;
    unit0 = hi * 8 + in % 8;
    if (unit0 >= a.units) return;   // uniform: the grid is rounded up to whole rows of 8
  }
  const int m0 = mt * 16 * MT;
  const int u = unit0 * nwv + nw;                    // unit of NT tiles
  const int G = u * NT / 4, j0[1] = {u * NT % 4};
  const int KQ = (a.K + 511) / 512;
  const int Q0 = kq * KQ / a.kw, Q1 = (kq + 1) * KQ / a.kw;

  StreamWave w;
  w.rsX = make_rsrc(a.X, (uint32_t)((int64_t)(a.M - 1) * a.ldx + a.K));
  w.rsXs = make_rsrc(a.Xs, (uint32_t)((int64_t)(a.M - 1) * a.ldxs + a.K / 32));
  w.rsW = make_rsrc(a.W, (uint32_t)((int64_t)(a.N - 1) * a.ldw + (int64_t)a.K * (C::WF == MX_E2M1 ? 1 : 2) / 2));
  w.rsWs = C::PACKED ? make_rsrc(a.Ws, (uint32_t)(packed_scale_dwords(a.N, a.K) * 4))
                     : make_rsrc(a.Ws, (uint32_t)((int64_t)(a.N - 1) * a.ldws + a.K / 32));
  uint32_t xvo[2 * MT], xso[MT], wvo[2 * NT], wso[C::NSW];
#pragma unroll
  for (int q = 0; q < 2 * MT; ++q) {
    const int m = m0 + 8 * q + (lane >> 3);
    xvo[q] = m < a.M ? (uint32_t)(m * a.ldx + stream_x_col(q, lane)) : kOobOffset;
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = m0 + 16 * i + r;
    xso[i] = m < a.M ? (uint32_t)(m * a.ldxs) : kOobOffset;
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int n = 64 * G + bperm_row(j0[0] + j, r);
    if constexpr (!C::PACKED) wso[j] = n < a.N ? (uint32_t)(n * a.ldws) : kOobOffset;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int nl = 64 * G + bperm_row(j0[0] + j, 8 * h + (lane >> 3));
      wvo[2 * j + h] = nl < a.N ? (uint32_t)(nl * a.ldw + (lane & 7) * 16) : kOobOffset;
    }
  }
  if constexpr (C::PACKED) wso[0] = 64 * G < a.N ? (uint32_t)(G * KQ * 1024 + lane * 16) : kOobOffset;

  v4f acc[MT][NT];
  stream_products<C>(w, smem + wave * C::WAVE_BYTES, xvo, xso, wvo, wso, j0, Q0, Q1, (a.K + 127) / 128, acc);

  // item = (unit, row tile, tile pair) of the workgroup; lane (c, g) of tile j holds row c, columns
  // bperm_tile_off(j) + 8 g .. + 3 of the group, so a pair of tiles is 8 consecutive outputs of a lane
  constexpr int JP = NT >= 2 ? 2 : 1;
  auto item = [&](int it, int& m, int& n) {
    const int jp = it % (NT / JP), i = it / (NT / JP) % MT, t0 = (unit0 * nwv + it / (NT / JP) / MT) * NT + jp * JP;   // t0: first tile of the item
    n = 64 * (t0 / 4) + bperm_tile_off(t0 % 4) + 8 * gq;
    m = m0 + 16 * i + r;
  };
  // a linear layer's bias and residual of the wave's first item (as a rule its only one) are on their way while the K ranges meet
  FloatsPiece bias = {}, res = {};
  auto request = [&](int it) {
    if constexpr (LINEAR) {
      int m, n;
      item(it, m, n);
      const int cols = JP == 1 && a.N - n > 4 ? 4 : a.N - n;
      if (o.bias) request_floats(o.bias, o.bias_dtype, n, cols, bias);
      linear_request(o, res, m, n, cols, m < a.M);
    }
  };
  if (wave < nwv * MT * (NT / JP)) request(wave);

  // ---- the K ranges meet in LDS, added in their order ------------------------------------------------------------
  __syncthreads();
  typedef __attribute__((address_space(3))) v4f lds_v4f;
  lds_v4f* const red = (lds_v4f*)smem;               // [nw][kq][i][j][lane]
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) red[((nw * a.kw + kq) * (MT * NT) + i * NT + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  for (int it = wave; it < nwv * MT * (NT / JP); it += C::WAVES) {   // uniform per wave
    const int jp = it % (NT / JP), i = it / (NT / JP) % MT, wv = it / (NT / JP) / MT;
    v4f v[2] = {};
    for (int k = 0; k < a.kw; ++k)
#pragma unroll
      for (int h = 0; h < JP; ++h) v[h] += red[((wv * a.kw + k) * (MT * NT) + i * NT + jp * JP + h) * 64 + lane];
    int m, n;
    item(it, m, n);
    int cols = a.N - n;
    if (JP == 1 && cols > 4) cols = 4;
    if constexpr (LINEAR) {
      float b[8] = {};
      if (o.bias) floats_of(bias, o.bias_dtype, b);
      linear_finish_any<true>(o, v[0], v[1], b, res, m, n, cols, m < a.M, gq == 0);
      if (it + C::WAVES < nwv * MT * (NT / JP)) request(it + C::WAVES);
    } else if (m < a.M && cols > 0) {
      if (a.c_dtype == MX_F32) {
        float* p = (float*)a.C + (int64_t)m * a.ldc + n;
        if (a.accumulate) add8_edge<float>(p, v[0], v[1], cols);
        store8_edge<float>(p, v[0], v[1], cols);
      } else {
        uint16_t* p = (uint16_t*)a.C + (int64_t)m * a.ldc + n;
        if (a.accumulate) add8_edge<uint16_t>(p, v[0], v[1], cols);
        store8_edge<uint16_t>(p, v[0], v[1], cols);
      }
    }
  }
}

// Waves of a workgroup: with 64 rows of X a stage of FP4 weights is 16 KiB of X, of which two for each of 8 waves do not fit
// into LDS.
constexpr int stream_waves(int mt, int w_fmt) { return mt == 4 && w_fmt == MX_E2M1 ? 4 : 8; }

template <class C, class Out>
int launch(const StreamArgs& a, const Out& o, int blocks, hipStream_t stream) {
  auto kern = stream_kernel<C, Out>;
  static int attr_done = 0;   // benign race: the attribute call is idempotent
  if (!attr_done) {
    hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS_BYTES);
    if (e != hipSuccess)
      return set_error(MX_ERR_LAUNCH, "hipFuncSetAttribute(%d bytes LDS): %s", C::LDS_BYTES, hipGetErrorString(e));
    attr_done = 1;
  }
  hipError_t e = launch_kernel(kern, dim3((unsigned)blocks), dim3(C::WAVES * 64), C::LDS_BYTES, stream, a, o);
  if (e != hipSuccess) return set_error(MX_ERR_LAUNCH, "stream_kernel launch: %s", hipGetErrorString(e));
  return MX_OK;
}

template <int XF, int WF, int NT, int MT, class Out>
int launch_p(const StreamArgs& a, const Out& o, int blocks, hipStream_t stream) {
  constexpr int W = stream_waves(MT, WF);
  if constexpr (NT == 4)
    if (stream_loads_once(a.N, WF == MX_E2M1 ? a.K / 2 : a.K, a.ldw, (uint64_t)a.W, a.m_tiles))
      return a.ws_packed ? launch<StreamCfg<XF, WF, NT, MT, true, W, false, true>>(a, o, blocks, stream)
                         : launch<StreamCfg<XF, WF, NT, MT, false, W, false, true>>(a, o, blocks, stream);
  return a.ws_packed ? launch<StreamCfg<XF, WF, NT, MT, true, W>>(a, o, blocks, stream)
                     : launch<StreamCfg<XF, WF, NT, MT, false, W>>(a, o, blocks, stream);
}
template <int XF, int WF, int NT, class Out>
int launch_m(const StreamArgs& a, const Out& o, int mt, int blocks, hipStream_t stream) {
  return mt == 1 ? launch_p<XF, WF, NT, 1>(a, o, blocks, stream)
         : mt == 2 ? launch_p<XF, WF, NT, 2>(a, o, blocks, stream) : launch_p<XF, WF, NT, 4>(a, o, blocks, stream);
}

}  // namespace
}  // namespace mx
