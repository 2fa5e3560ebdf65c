// Launches of the weight-streaming kernel for linear layers: bias, activation and residual where the K ranges meet.
#include "mx_gemm_stream_kernel.h"

namespace mx {

int launch_gemm_stream_linear(const StreamArgs& a0, const LinearOut& o, hipStream_t stream) {
  StreamArgs a = a0;
  if (a.M < 1 || a.N < 1) return set_error(MX_ERR_SHAPE, "stream kernel: no rows");
  if (const char* why = stream_issue(a)) return set_error(MX_ERR_LAYOUT, "stream kernel: %s", why);
  const StreamPlan p = stream_plan(a.M, a.N, a.K, a.w_fmt, o.c_fmt == MX_E4M3 ? 2 : 1);   // (1 x 8192 x 2048: units of one tile 4.8 us, of two 6.0)
  a.m_tiles = p.m_tiles; a.kw = p.kw; a.units = p.units;
  const int blocks = a.m_tiles > 1 ? (a.units + 7) / 8 * 8 * a.m_tiles : a.units;
#define MX_CASE(XF, WF) \
  if (a.x_fmt == XF && a.w_fmt == WF) return p.nt == 4 ? launch_m<XF, WF, 4>(a, o, p.mt, blocks, stream) : p.nt == 2 ? launch_m<XF, WF, 2>(a, o, p.mt, blocks, stream) \
                                                                                   : launch_m<XF, WF, 1>(a, o, p.mt, blocks, stream);
  MX_CASE(MX_E4M3, MX_E4M3)
  MX_CASE(MX_E4M3, MX_E2M1)
  MX_CASE(MX_E5M2, MX_E5M2)
  MX_CASE(MX_E5M2, MX_E2M1)
#undef MX_CASE
  return set_error(MX_ERR_DTYPE, "stream kernel: unsupported element format pair (%d, %d)", a.x_fmt, a.w_fmt);
}

}  // namespace mx
