// Rows of 16-, 32-bit floats in 16-byte pieces, at any element alignment: loads, stores and sums over lanes, for kernels that hold
// rows in registers.
#pragma once
#include "mx_encode.h"
#include "mx_gemm_tile.h"   // u4_any

namespace mx {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
template <int T> constexpr int kPiece = T == MX_F32 ? 4 : 8;   // elements of a piece
template <int T> constexpr int kSize = T == MX_F32 ? 4 : 2;

// Elements at .. at + kPiece - 1 of a row, of which the first n exist (global memory takes 16-byte loads at any element); the others are zero.
template <int T>
__device__ __forceinline__ u4 load_piece(const void* row, int64_t at, int n) {
  u4 r = {0, 0, 0, 0};
  const uint8_t* const p = (const uint8_t*)row + at * kSize<T>;
  if (n >= kPiece<T>) {
    const u4_any v = *(const u4_any*)p;
    r = (u4){v[0], v[1], v[2], v[3]};
  } else if (kPiece<T> == 8 && n == 4) {
    const u2_any v = *(const u2_any*)p;
    r[0] = v[0];
    r[1] = v[1];
  } else if (n > 0) {
#pragma unroll
    for (int e = 0; e < kPiece<T>; ++e) {
      if (e >= n) continue;
      if constexpr (T == MX_F32) r[e] = ((const uint32_t*)p)[e];
      else r[e / 2] |= (uint32_t)((const uint16_t*)p)[e] << (16 * (e & 1));
    }
  }
  return r;
}
template <int T>
__device__ __forceinline__ void unpack_piece(const u4& r, float (&v)[kPiece<T>]) {
#pragma unroll
  for (int e = 0; e < kPiece<T>; ++e) {
    if constexpr (T == MX_F32) v[e] = __builtin_bit_cast(float, (uint32_t)r[e]);   // (of the element itself the compiler takes the first)
    else if constexpr (T == MX_BF16) v[e] = __builtin_bit_cast(float, e & 1 ? r[e / 2] & 0xFFFF0000u : r[e / 2] << 16);
    else v[e] = (float)__builtin_bit_cast(_Float16, (uint16_t)(r[e / 2] >> (16 * (e & 1))));
  }
}
// rounded to nearest even
template <int T>
__device__ __forceinline__ u4 pack_piece(const float (&v)[kPiece<T>]) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  u4 r;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (T == MX_F32) r[k] = __builtin_bit_cast(uint32_t, v[k]);
    else if constexpr (T == MX_BF16) r[k] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){v[2 * k], v[2 * k + 1]}, b2));
    else r[k] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * k]) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * k + 1]) << 16;
  }
  return r;
}
template <int T>
__device__ __forceinline__ void store_piece(void* row, int64_t at, int n, const u4& r) {
  uint8_t* const p = (uint8_t*)row + at * kSize<T>;
  if (n >= kPiece<T>) {
    *(u4_any*)p = (u4_any){r[0], r[1], r[2], r[3]};
  } else if (n > 0) {
#pragma unroll
    for (int e = 0; e < kPiece<T>; ++e) {
      if (e >= n) continue;
      if constexpr (T == MX_F32) ((uint32_t*)p)[e] = r[e];
      else ((uint16_t*)p)[e] = (uint16_t)(r[e / 2] >> (16 * (e & 1)));
    }
  }
}
// N elements (4 or 8) of a vector of any float type (`p` null: `fill`), zeros where they do not exist
template <int N>
__device__ __forceinline__ void load_floats(const void* p, int dtype, int64_t at, int n, float fill, float (&v)[N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = p || e >= n ? 0.f : fill;
  if (!p) return;
  if (dtype == MX_F32) {
#pragma unroll
    for (int h = 0; h < N / 4; ++h) {
      float f[4];
      unpack_piece<MX_F32>(load_piece<MX_F32>(p, at + 4 * h, n - 4 * h), f);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * h + e] = f[e];
    }
  } else {
    // (a piece of eight where only four are wanted: the others may not exist)
    const u4 r = load_piece<MX_BF16>(p, at, n < N ? n : N == 8 ? 8 : 4);
    float f[8];
    if (dtype == MX_BF16) unpack_piece<MX_BF16>(r, f);
    else unpack_piece<MX_F16>(r, f);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = f[e];
  }
}
__device__ __forceinline__ void store_float(void* p, int dtype, int64_t at, float v) {
  if (dtype == MX_F32) ((float*)p)[at] = v;
  else if (dtype == MX_BF16) ((uint16_t*)p)[at] = f32_to_bf16(v);
  else ((_Float16*)p)[at] = (_Float16)v;
}

// sum over the wave, in every lane, in the same order for every lane
__device__ __forceinline__ float wave_sum(float v) {
  auto dpp = [](float x, auto c) { return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), decltype(c)::value, 0xF, 0xF, true)); };
  v += dpp(v, std::integral_constant<int, 0xB1>{});    // l ^ 1
  v += dpp(v, std::integral_constant<int, 0x4E>{});    // l ^ 2
  v += dpp(v, std::integral_constant<int, 0x141>{});   // mirrored within 8
  v += dpp(v, std::integral_constant<int, 0x140>{});   // mirrored within 16
  const auto a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
  v = __builtin_bit_cast(float, (uint32_t)a[0]) + __builtin_bit_cast(float, (uint32_t)a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
  return __builtin_bit_cast(float, (uint32_t)b[0]) + __builtin_bit_cast(float, (uint32_t)b[1]);
}

}  // namespace mx
