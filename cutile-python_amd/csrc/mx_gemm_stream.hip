// Launches of the weight-streaming kernel (mx_gemm_stream.h) for plain products.
#include "mx_gemm_stream_kernel.h"

namespace mx {

bool stream_supports(int x_fmt, int w_fmt) {
  return (x_fmt == MX_E4M3 && (w_fmt == MX_E4M3 || w_fmt == MX_E2M1)) ||
         (x_fmt == MX_E5M2 && (w_fmt == MX_E5M2 || w_fmt == MX_E2M1));
}

// How the waves of a workgroup split the problem: kw K ranges x waves / kw units of nt tiles; M in tiles of 16 mt rows.  The
// cost that is minimised is a wave's K-quads times what a K-step of it moves (nt tiles of W, the rows of X), plus a
// start-up per workgroup, for every round of workgroups over the 256 CUs: X is fetched once per unit, so wide units
// save traffic, but a second, partly filled round costs more (28672 x 8192 FP4 at 4 rows: 224 workgroups 28 us, 448
// 33.6 us; 14336 x 8192 FP8 at 64 rows: 224 of 4 tiles 34 us, 448 of 2 45 us).
// (tiles of a 64-row group interleave its rows, so groups are covered whole; `least`: of nt, 2 where a lane has to have eight columns)
StreamPlan stream_plan(int64_t M, int64_t N, int64_t K, int w_fmt, int least) {
  StreamPlan p = {};
  // FP4 weights for 33 .. 64 rows: one row tile of 64 (four waves) once the weights have 8192 rows to share out, which
  // reads them once (28672 x 8192: 64 rows 52.6 -> 44.8 us, 48 rows 47.9 -> 41.7; 14336 x 4096, 40 rows 16.1 -> 15.0);
  // with fewer, two tiles of 32 have the waves that it lacks (4096 x 14336, 64 rows: 17.8 against 21.5)
  p.mt = M <= 16 ? 1 : M <= 32 ? 2 : w_fmt != MX_E2M1 ? 4 : M <= 64 && N >= 8192 ? 4 : 2;
  const int waves = stream_waves(p.mt, w_fmt);   // (half as many waves have twice the bandwidth each)
  p.m_tiles = (int)((M + 16 * p.mt - 1) / (16 * p.mt));
  const int tiles = (int)((N + 63) / 64 * 4), KQ = (int)((K + 511) / 512);
  const float wb = w_fmt == MX_E2M1 ? 1.f : 2.f, xb = (M < 16 * p.mt ? M : 16 * p.mt) / 16.f;
  p.cost = 1e30f;
  for (int n = 4; n >= least; n >>= 1)
    for (int kw = waves; kw >= 1; kw >>= 1) {
      if (kw > 1 && kw > KQ) continue;
      const int units = (tiles + n * (waves / kw) - 1) / (n * (waves / kw));
      const int64_t rounds = ((int64_t)units * p.m_tiles + 255) / 256;
      const float t = rounds * ((KQ + kw - 1) / kw * (n * wb + xb) * waves / 8.f + 3.f);
      if (t < p.cost) { p.cost = t; p.nt = n; p.kw = kw; p.units = units; }
    }
  return p;
}

// Rows may overlap (a row pitch of zero is a broadcast row): the descriptors end behind the last row's last byte.
const char* stream_issue(const StreamArgs& a) {
  if (!stream_supports(a.x_fmt, a.w_fmt)) return "it takes 8-bit A with FP4 B or B of A's format";
  if (a.K < 128 || a.K % 128 != 0) return "K is not a multiple of 128";
  if ((((uintptr_t)a.X | (uintptr_t)a.W | (uintptr_t)a.ldx | (uintptr_t)a.ldw) % 16) != 0)
    return "A and B must have 16-byte aligned rows";
  if ((((uintptr_t)a.Xs | (uintptr_t)a.ldxs) % 4) != 0) return "A_scale must have 4-byte aligned rows";
  if (a.ws_packed ? ((uintptr_t)a.Ws % 16) != 0 : (((uintptr_t)a.Ws | (uintptr_t)a.ldws) % 4) != 0)
    return "B_scale must be 16-byte aligned (packed) or have 4-byte aligned rows";
  // lane offsets are 32-bit, and 2^31 marks what does not exist
  auto fits = [](int64_t rows, int64_t pitch, int64_t row) {
    return rows * pitch < (int64_t)1 << 31 && (rows - 1) * pitch + row < (int64_t)1 << 31;
  };
  if (!fits(a.M, a.ldx, a.K) || !fits(a.N, a.ldw, a.w_fmt == MX_E2M1 ? a.K / 2 : a.K)) return "A or B spans 2 GiB or more";
  if (!fits(a.M, a.ldxs, a.K / 32) ||
      !(a.ws_packed ? fits(1, 0, packed_scale_dwords(a.N, a.K) * 4) : fits(a.N, a.ldws, a.K / 32)))
    return "A_scale or B_scale spans 2 GiB or more";
  return nullptr;
}

int launch_gemm_stream(const StreamArgs& a0, hipStream_t stream) {
  StreamArgs a = a0;
  if (a.M < 1 || a.N < 1) return set_error(MX_ERR_SHAPE, "stream kernel: no rows");
  if (const char* why = stream_issue(a)) return set_error(MX_ERR_LAYOUT, "stream kernel: %s", why);
  const StreamPlan p = stream_plan(a.M, a.N, a.K, a.w_fmt);
  const int mt = p.mt, nt = p.nt;
  a.m_tiles = p.m_tiles; a.kw = p.kw; a.units = p.units;
  const int blocks = a.m_tiles > 1 ? (a.units + 7) / 8 * 8 * a.m_tiles : a.units;
#define MX_CASE(XF, WF)                                                                       \
  if (a.x_fmt == XF && a.w_fmt == WF)                                                         \
    return nt == 4 ? launch_m<XF, WF, 4>(a, Ungated{}, mt, blocks, stream)                               \
           : nt == 2 ? launch_m<XF, WF, 2>(a, Ungated{}, mt, blocks, stream) : launch_m<XF, WF, 1>(a, Ungated{}, mt, blocks, stream);
  MX_CASE(MX_E4M3, MX_E4M3)
  MX_CASE(MX_E4M3, MX_E2M1)
  MX_CASE(MX_E5M2, MX_E5M2)
  MX_CASE(MX_E5M2, MX_E2M1)
#undef MX_CASE
  return MX_ERR_DTYPE;
}

}  // namespace mx
