// Layer norm (mx_norm.hip): forward with its MX quantisation, backward with the gradients of weight and bias.
#pragma once
#include "mx_common.h"

namespace mx {

struct NormArgs {
  const void *x, *w, *b;             // [rows][H]; [H] or null
  void* y;                           // [rows][H] of x's type, or codes (MX_E2M1: two per byte)
  uint8_t* s;                        // scales of the codes
  float *mean, *rstd;                // [rows] or null
  int64_t x_ld, y_ld, s_ld;          // elements; bytes of codes and scales
  int32_t rows, H, x_dtype, w_dtype, b_dtype;
  int32_t fmt, scale_mode;           // of the codes; fmt -1: y
  float eps;
};
int launch_layer_norm(const NormArgs& a, hipStream_t stream);

struct NormBackwardArgs {
  const void *dy, *x, *w;            // w may be null
  const float *mean, *rstd;
  void *dx, *dw, *db;                // each may be null
  float* partial;                    // rows of dw and db, one for each workgroup: norm_backward_bytes()
  int64_t dy_ld, x_ld, dx_ld;
  int32_t rows, H, x_dtype, w_dtype, dw_dtype, db_dtype;
};
int64_t norm_backward_bytes(int64_t rows, int64_t H);
int launch_layer_norm_backward(const NormBackwardArgs& a, hipStream_t stream);

}  // namespace mx
