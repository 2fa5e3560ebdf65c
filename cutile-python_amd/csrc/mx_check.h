// Checks of the C entries' descriptors that several translation units share.
#pragma once
#include "mx_common.h"

namespace mx {

inline int64_t round256(int64_t b) { return (b + 255) & ~(int64_t)255; }
inline int64_t round32(int64_t n) { return (n + 31) / 32 * 32; }
constexpr int64_t kMaxExtent = (int64_t)1 << 30;

// a 2-D tensor [rows, cols] with contiguous rows
inline int check2d(const mx_tensor* t, const char* name, int64_t rows, int64_t cols) {
  if (!t) return set_error(MX_ERR_INVALID, "%s: null descriptor", name);
  if (t->ndim != 2) return set_error(MX_ERR_SHAPE, "%s: expected 2 dimensions, got %d", name, t->ndim);
  if ((rows >= 0 && t->shape[0] != rows) || (cols >= 0 && t->shape[1] != cols))
    return set_error(MX_ERR_SHAPE, "%s must be [%lld, %lld], got [%lld, %lld]", name, (long long)(rows >= 0 ? rows : t->shape[0]),
                     (long long)(cols >= 0 ? cols : t->shape[1]), (long long)t->shape[0], (long long)t->shape[1]);
  if (t->shape[0] < 0 || t->shape[1] < 0 || t->shape[0] >= kMaxExtent || t->shape[1] >= kMaxExtent)
    return set_error(MX_ERR_SHAPE, "%s: extent out of range", name);
  if (t->stride[0] < 0 || (t->shape[1] > 1 && t->stride[1] != 1))
    return set_error(MX_ERR_LAYOUT, "%s: rows must be contiguous", name);
  if (t->shape[0] > 0 && t->shape[1] > 0 && !t->ptr) return set_error(MX_ERR_INVALID, "%s: null data pointer", name);
  return MX_OK;
}
inline int check_dtype(const mx_tensor* t, const char* name, bool ok, const char* want) {
  return ok ? MX_OK : set_error(MX_ERR_DTYPE, "%s must be %s (got %d)", name, want, t->dtype);
}
// an output of codes: rows that start at whole `align` bytes and do not overlap
inline int check_codes(const mx_tensor* t, const char* name, int64_t rows, int64_t cols, int align) {
  if (int rc = check2d(t, name, rows, cols)) return rc;
  if (rows == 0 || cols == 0) return MX_OK;
  if ((uintptr_t)t->ptr % align != 0 || (rows > 1 && (t->stride[0] % align != 0 || t->stride[0] < cols)))
    return set_error(MX_ERR_LAYOUT, "%s: rows must be aligned to %d bytes and apart", name, align);
  return MX_OK;
}
inline int check_scales(const mx_tensor* t, const char* name, int64_t rows, int64_t blocks) {
  if (int rc = check2d(t, name, rows, blocks)) return rc;
  if (t->dtype != MX_E8M0) return set_error(MX_ERR_DTYPE, "%s must be MX_E8M0", name);
  if (rows > 1 && blocks > 0 && t->stride[0] < blocks) return set_error(MX_ERR_LAYOUT, "%s: rows overlap", name);
  return MX_OK;
}
inline int check_mode(int32_t scale_mode) {
  return scale_mode == 0 || scale_mode == 1 ? MX_OK : set_error(MX_ERR_INVALID, "scale_mode must be 0 (ceil) or 1 (floor)");
}
inline bool is_float(int d) { return d == MX_F32 || d == MX_BF16 || d == MX_F16; }
inline mx_tensor tensor2d(void* ptr, int dtype, int64_t rows, int64_t cols, int64_t ld) {
  return mx_tensor{ptr, dtype, 2, {rows, cols, 0, 0}, {ld, 1, 0, 0}, -1, 0};
}
inline mx_tensor transposed(const mx_tensor& t) {
  mx_tensor r = t;
  r.shape[0] = t.shape[1]; r.shape[1] = t.shape[0];
  r.stride[0] = t.stride[1]; r.stride[1] = t.stride[0];
  if (t.packed_dim >= 0) r.packed_dim = 1 - t.packed_dim;
  return r;
}
// a buffer that is dealt out in pieces of whole 256 bytes
struct Deal {
  uint8_t* base;
  int64_t at = 0;
  uint8_t* take(int64_t bytes) {
    uint8_t* const p = base + at;
    at += round256(bytes);
    return p;
  }
};
inline int check_room(const char* name, const void* ptr, int64_t given, int64_t need) {
  if (need <= 0) return MX_OK;
  if (!ptr || given < need)
    return set_error(MX_ERR_WORKSPACE, "%s of %lld bytes required, %lld given", name, (long long)need, (long long)(ptr ? given : 0));
  if ((uintptr_t)ptr % 256 != 0) return set_error(MX_ERR_WORKSPACE, "%s must be 256-byte aligned", name);
  return MX_OK;
}
// a vector of `n` contiguous floats of any kind
inline int check_vector(const mx_tensor* t, const char* name, int64_t n) {
  if (t->ndim != 1 || t->shape[0] != n) return set_error(MX_ERR_SHAPE, "%s must be [%lld]", name, (long long)n);
  if (n > 1 && t->stride[0] != 1) return set_error(MX_ERR_LAYOUT, "%s must be contiguous", name);
  if (!is_float(t->dtype)) return set_error(MX_ERR_DTYPE, "%s must be MX_F32, MX_BF16 or MX_F16 (got %d)", name, t->dtype);
  if (n > 0 && !t->ptr) return set_error(MX_ERR_INVALID, "%s: null data pointer", name);
  return MX_OK;
}

}  // namespace mx
