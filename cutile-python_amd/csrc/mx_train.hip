// Kernels of the gated feed-forward block that is trained in 8 bits: quantisation along both axes of a matrix, the activation
// between the projections with its checkpoint, and the activation's backward pass.  What they quantise follows encode_block
// (mx_quant.h) to the bit.
#include "mx_quant.h"
#include "mx_train.h"

namespace mx {
namespace {

typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));

// ---- maxima over lanes ------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t max_quad(uint32_t m) {            // lanes 4 n .. 4 n + 3
  m = umax(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xF, 0xF, true));
  return umax(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xF, 0xF, true));
}
__device__ __forceinline__ uint32_t max_xor_8(uint32_t m) {           // lanes l, l ^ 8: a rotation of the 16-lane row by 8
  return umax(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x128, 0xF, 0xF, true));
}
__device__ __forceinline__ uint32_t max_xor_16_32(uint32_t m) {       // lanes l, l ^ 16, l ^ 32, l ^ 48
  const auto a = __builtin_amdgcn_permlane32_swap(m, m, false, false);
  m = umax(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(m, m, false, false);
  return umax(b[0], b[1]);
}
__device__ __forceinline__ uint32_t magnitude(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7FFFFFFFu; }

// ---- encoding ---------------------------------------------------------------------------------------------------------------
// What the hardware conversions need of a block whose largest magnitude has the bits `am`: its scale, as a number and as a byte,
// and the bound that saturation clamps to.  ok = false: a block for encode_block (subnormal or non-finite amax, extreme scale).
struct BlockScale {
  float scale, lim;
  uint32_t byte;
  bool ok;
};
template <int FMT>
__device__ __forceinline__ BlockScale block_scale(uint32_t am, bool floor_mode) {
  constexpr int EMAX = FMT == MX_E4M3 ? 8 : 15;
  constexpr float FMAX = FMT == MX_E4M3 ? 448.0f : 57344.0f;
  BlockScale b;
  int se;
  if (floor_mode) {
    se = (int)(am >> 23) - 127 - EMAX;
  } else {
    const uint32_t t = __builtin_bit_cast(uint32_t, fmaxf(__fdiv_rn(__builtin_bit_cast(float, am), 448.0f), 1e-12f));
    se = (int)(t >> 23) - 127 + ((t & 0x7FFFFFu) ? 1 : 0);
  }
  b.ok = am == 0 || (am >= 0x00800000u && am < 0x7F800000u && se > -127 && se < 120);
  b.byte = am == 0 && floor_mode ? 0u : (uint32_t)(se + 127);
  b.scale = am == 0 ? 1.0f : __builtin_bit_cast(float, (uint32_t)(se + 127) << 23);   // (a block of zeros is zeros at any scale)
  b.lim = floor_mode ? __fmul_rn(FMAX, b.scale) : __builtin_inff();
  return b;
}
// four values of a block as codes, lowest byte first
template <int FMT>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, const BlockScale& s) {
  typedef short s2 __attribute__((ext_vector_type(2)));
  a = __builtin_amdgcn_fmed3f(a, -s.lim, s.lim);
  b = __builtin_amdgcn_fmed3f(b, -s.lim, s.lim);
  c = __builtin_amdgcn_fmed3f(c, -s.lim, s.lim);
  d = __builtin_amdgcn_fmed3f(d, -s.lim, s.lim);
  s2 r = {0, 0};
  if constexpr (FMT == MX_E4M3) {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, a, b, s.scale, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, c, d, s.scale, true);
  } else {
    r = __builtin_amdgcn_cvt_scalef32_pk_bf8_f32(r, a, b, s.scale, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_bf8_f32(r, c, d, s.scale, true);
  }
  return __builtin_bit_cast(uint32_t, r);
}
template <int N>
__device__ inline void encode_slow(const float* v, uint32_t am, int fmt, int scale_mode, uint32_t* packed, uint32_t& byte) {
  uint32_t code[N];
  uint8_t sb;
  encode_block<N>(v, am, fmt, scale_mode, code, sb);
#pragma unroll
  for (int h = 0; h < N / 4; ++h) packed[h] = code[4 * h] | (code[4 * h + 1] << 8) | (code[4 * h + 2] << 16) | (code[4 * h + 3] << 24);
  byte = sb;
}

// Scale bytes [rows of the tile][4 blocks] of a 128-row tile, from LDS to where they belong: row0, block0 = first row and block
// of the tile; rows, blocks = of the whole matrix.  Bytes outside of the matrix are 127 in LDS, which is what the native layouts
// are padded with (rows to 64, blocks to 16).
__device__ __forceinline__ void store_scales_128(const uint32_t* lds, uint8_t* s, int64_t ld, int kind, int64_t row0, int64_t rows,
                                                 int64_t block0, int64_t blocks) {
  if (threadIdx.x >= 128) return;
  const int tid = threadIdx.x;
  if (kind == kScalePlain) {
    const int64_t row = row0 + tid;
    if (row >= rows || block0 >= blocks) return;
    const uint32_t w = lds[tid];
    uint8_t* const p = s + row * ld + block0;
    if (block0 + 4 <= blocks && (((uintptr_t)p) & 3) == 0) *(uint32_t*)p = w;
    else
      for (int k = 0; k < 4; ++k)
        if (block0 + k < blocks) p[k] = (uint8_t)(w >> (8 * k));
  } else {
    const int64_t G = row0 / 64 + (tid >> 6), quads = (blocks + 15) / 16;
    if (G >= (rows + 63) / 64) return;
    const int l = tid & 63, c = l & 15, g = l >> 4;
    uint32_t w = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int r = (tid & 64) + (kind == kScaleNativeB ? bperm_row(b, c) : 16 * b + c);
      w |= (lds[r] >> (8 * g) & 0xFF) << (8 * b);
    }
    ((uint32_t*)s)[((G * quads + block0 / 16) * 64 + l) * 4 + (block0 / 4) % 4] = w;
  }
}

// ================================================================================================================================
// Quantisation along both axes
// ================================================================================================================================
// Bound: one pass over the input (2 or 4 bytes an element) and two over codes.  A workgroup takes 128 x 128 elements, so that what it
// writes of a row, and of a column, is one line of 128 codes; a wave takes 32 rows, a lane 8 x 8 elements (rows 8 (lane / 16) ..,
// columns 8 (lane % 16) ..), all loaded before the first is used.  The maximum of 32 elements of a row is then over four neighbouring
// lanes, of a column over the lane's rows and lanes l ^ 16, l ^ 32, without LDS; each lane has 8 codes in sequence in both
// directions.  The transposed codes pass through LDS (16-byte chunks, swizzled by column).
template <int SRC>
__device__ __forceinline__ float load_one(const void* x, int64_t at) {
  if constexpr (SRC == MX_F32) return ((const float*)x)[at];
  else if constexpr (SRC == MX_BF16) return bf16_to_f32(((const uint16_t*)x)[at]);
  else return (float)((const _Float16*)x)[at];
}

template <int SRC, int FMT>
__global__ __launch_bounds__(256) void quantize_both_kernel(const BothArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t tile[128 * 128];
  __shared__ uint32_t srow[128], scol[128];
  int which = 0;
#pragma unroll
  for (int k = 1; k < kBothMax; ++k)
    if (k < a.n && (int)blockIdx.x >= a.t[k].first) which = k;
  const BothTensor& t = a.t[which];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, rg = lane >> 4, cg = lane & 15;
  const int at = blockIdx.x - t.first, tr = at / t.tiles_k;
  const int64_t r0 = (int64_t)tr * 128, k0 = (int64_t)(at - tr * t.tiles_k) * 128;
  const int64_t rows = t.rows, K = t.K, Kpad = (K + 31) / 32 * 32, Rpad = (rows + 31) / 32 * 32;
  const bool floor_mode = a.scale_mode != 0;
  if (tid < 128) srow[tid] = scol[tid] = 0x7F7F7F7Fu;
  __syncthreads();
  uint8_t* const srow_b = (uint8_t*)srow;
  uint8_t* const scol_b = (uint8_t*)scol;
  if (r0 < rows && k0 < Kpad) {                       // (else: padding of native scales only)
    const int64_t row = r0 + 32 * wave + 8 * rg, col = k0 + 8 * cg;   // of the lane's first element
    float v[8][8];
    if (t.vec && col + 8 <= K) {
      v4i raw[8][SRC == MX_F32 ? 2 : 1];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint8_t* const p = (const uint8_t*)t.x + ((row + i < rows ? row + i : rows - 1) * t.x_ld + col) * (SRC == MX_F32 ? 4 : 2);
#pragma unroll
        for (int h = 0; h < (SRC == MX_F32 ? 2 : 1); ++h) raw[i][h] = *(const v4i*)(p + 16 * h);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          if constexpr (SRC == MX_F32) {
            v[i][h] = __builtin_bit_cast(float, (uint32_t)raw[i][0][h]);
            v[i][4 + h] = __builtin_bit_cast(float, (uint32_t)raw[i][1][h]);
          } else if constexpr (SRC == MX_BF16) {
            v[i][2 * h] = __builtin_bit_cast(float, (uint32_t)raw[i][0][h] << 16);
            v[i][2 * h + 1] = __builtin_bit_cast(float, (uint32_t)raw[i][0][h] & 0xFFFF0000u);
          } else {
            v[i][2 * h] = (float)__builtin_bit_cast(_Float16, (uint16_t)(uint32_t)raw[i][0][h]);
            v[i][2 * h + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)((uint32_t)raw[i][0][h] >> 16));
          }
        }
        if (row + i >= rows) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[i][e] = 0.f;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[i][e] = 0.f;
          if (row + i < rows && col + e < K) v[i][e] = load_one<SRC>(t.x, (row + i) * t.x_ld + col + e);
        }
    }
    uint32_t again_row = 0, again_col = 0;            // blocks that encode_block takes, from memory
    if (t.q) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint32_t am = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) am = umax(am, magnitude(v[i][e]));
        const BlockScale b = block_scale<FMT>(max_quad(am), floor_mode);
        const bool live = row + i < rows && col < Kpad;
        const u2 c = {encode4<FMT>(v[i][0], v[i][1], v[i][2], v[i][3], b), encode4<FMT>(v[i][4], v[i][5], v[i][6], v[i][7], b)};
        if (live && b.ok) {
          *(u2*)(t.q + (row + i) * t.q_ld + col) = c;
          if ((lane & 3) == 0) srow_b[(32 * wave + 8 * rg + i) * 4 + (cg >> 2)] = (uint8_t)b.byte;
        }
        if (live && !b.ok) again_row |= 1u << i;
      }
    }
    // transposed: the lane's codes of column 8 cg + e are 8 of that column's 128 bytes
    auto place = [&](int e, u2 c) {
      *(u2*)(tile + (8 * cg + e) * 128 + (((2 * wave + (rg >> 1)) ^ (cg & 7)) << 4) + (rg & 1) * 8) = c;
    };
    if (t.qt) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        uint32_t am = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) am = umax(am, magnitude(v[i][e]));
        const BlockScale b = block_scale<FMT>(max_xor_16_32(am), floor_mode);
        const bool live = r0 + 32 * wave < rows && col + e < K;
        const u2 c = {encode4<FMT>(v[0][e], v[1][e], v[2][e], v[3][e], b), encode4<FMT>(v[4][e], v[5][e], v[6][e], v[7][e], b)};
        if (live && b.ok) {
          place(e, c);
          if (rg == 0) scol_b[(8 * cg + e) * 4 + wave] = (uint8_t)b.byte;
        }
        if (live && !b.ok) again_col |= 1u << e;
      }
    }
    if (again_row) {                                   // (the four lanes of a block agree)
      for (int i = 0; i < 8; ++i) {
        if (!(again_row >> i & 1)) continue;
        float w[8];
        uint32_t am = 0, c[2], byte;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          w[e] = col + e < K ? load_one<SRC>(t.x, (row + i) * t.x_ld + col + e) : 0.f;
          am = umax(am, magnitude(w[e]));
        }
        encode_slow<8>(w, max_quad(am), FMT, a.scale_mode, c, byte);
        *(u2*)(t.q + (row + i) * t.q_ld + col) = (u2){c[0], c[1]};
        if ((lane & 3) == 0) srow_b[(32 * wave + 8 * rg + i) * 4 + (cg >> 2)] = (uint8_t)byte;
      }
    }
    if (again_col) {                                   // (the lanes l ^ 16, l ^ 32 of a block agree)
      for (int e = 0; e < 8; ++e) {
        if (!(again_col >> e & 1)) continue;
        float w[8];
        uint32_t am = 0, c[2], byte;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          w[i] = row + i < rows ? load_one<SRC>(t.x, (row + i) * t.x_ld + col + e) : 0.f;
          am = umax(am, magnitude(w[i]));
        }
        encode_slow<8>(w, max_xor_16_32(am), FMT, a.scale_mode, c, byte);
        place(e, (u2){c[0], c[1]});
        if (rg == 0) scol_b[(8 * cg + e) * 4 + wave] = (uint8_t)byte;
      }
    }
  }
  __syncthreads();
  if (t.qt && r0 < rows) {
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int c = n * 32 + (tid >> 3), j = tid & 7;
      if (k0 + c < K && r0 + 16 * j < Rpad)
        *(u4*)(t.qt + (k0 + c) * t.qt_ld + r0 + 16 * j) = *(const u4*)(tile + c * 128 + ((j ^ (c >> 3 & 7)) << 4));
    }
  }
  if (t.q) store_scales_128(srow, t.s, t.s_ld, t.s_kind, r0, rows, k0 / 32, Kpad / 32);
  if (t.qt) store_scales_128(scol, t.st, t.st_ld, t.st_kind, k0, K, r0 / 32, Rpad / 32);
}

// ================================================================================================================================
// The activation between the projections
// ================================================================================================================================
// One pass over bf16 [g|u]: a lane has 8 columns of both.  Bound: memory (4 bytes read, 1 to 4 written an element of h).
__device__ __forceinline__ void unpack_bf16(const v4i& t, float (&v)[8]) {
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    v[2 * h] = __builtin_bit_cast(float, (uint32_t)t[h] << 16);
    v[2 * h + 1] = __builtin_bit_cast(float, (uint32_t)t[h] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void store_row_block(const float (&v)[8], int fmt, int scale_mode, uint8_t* q, uint8_t* s, bool scale_lane) {
  uint32_t am = 0, c[2], byte;
#pragma unroll
  for (int e = 0; e < 8; ++e) am = umax(am, magnitude(v[e]));
  am = max_quad(am);
  const BlockScale b = fmt == MX_E4M3 ? block_scale<MX_E4M3>(am, scale_mode != 0) : block_scale<MX_E5M2>(am, scale_mode != 0);
  if (b.ok) {
    if (fmt == MX_E4M3) {
      c[0] = encode4<MX_E4M3>(v[0], v[1], v[2], v[3], b);
      c[1] = encode4<MX_E4M3>(v[4], v[5], v[6], v[7], b);
    } else {
      c[0] = encode4<MX_E5M2>(v[0], v[1], v[2], v[3], b);
      c[1] = encode4<MX_E5M2>(v[4], v[5], v[6], v[7], b);
    }
    byte = b.byte;
  } else {
    encode_slow<8>(v, am, fmt, scale_mode, c, byte);
  }
  *(u2*)q = (u2){c[0], c[1]};
  if (scale_lane) *s = (uint8_t)byte;
}

__global__ __launch_bounds__(256) void gate_up_kernel(const GateUpArgs a) {
  const int64_t unit = (int64_t)blockIdx.x * 256 + threadIdx.x, per = a.F / 8;   // (32 columns are four lanes of a wave)
  const int64_t row = unit / per, col = (unit - row * per) * 8;
  if (row >= a.rows) return;
  const uint16_t* const p = a.gu + row * a.gu_ld + col;
  float g[8], u[8], h[8];
  unpack_bf16(*(const v4i*)p, g);
  unpack_bf16(*(const v4i*)(p + a.F), u);
#pragma unroll
  for (int e = 0; e < 8; ++e) h[e] = silu_mul_f32(g[e], u[e]);
  const bool first = (threadIdx.x & 3) == 0;
  if (a.h_fmt == MX_BF16) {
    u4 w;
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = (uint32_t)f32_to_bf16(h[2 * k]) | ((uint32_t)f32_to_bf16(h[2 * k + 1]) << 16);
    *(u4*)((uint16_t*)a.h + row * a.h_ld + col) = w;
  } else {
    store_row_block(h, a.h_fmt, a.scale_mode, (uint8_t*)a.h + row * a.h_ld + col, a.hs + row * a.hs_ld + col / 32, first);
  }
  if (a.c) {
    uint8_t* const c = a.c + row * a.c_ld + col;
    uint8_t* const cs = a.cs + row * a.cs_ld + col / 32;
    store_row_block(g, MX_E4M3, a.scale_mode, c, cs, first);
    store_row_block(u, MX_E4M3, a.scale_mode, c + a.F, cs + a.F / 32, first);
  }
}

// ================================================================================================================================
// The activation's backward pass
// ================================================================================================================================
//   s = 1 / (1 + exp(-g));  du = dh g s;  dg = dh u s (1 + g (1 - s));  a = g s u
// g and u are the checkpoint's values.  d[g|u] goes out quantised along the rows (for the product with w1) and along the columns
// (for the gradient of w1), a along the columns (for the gradient of w2; the forward pass kept no copy of it, which saves 8.25 bits per element from
// one pass to the other for one multiplication here).
// Bound: memory, 4.06 bytes read and 5.16 written an element of dh.  A workgroup takes 128 rows x 64 columns, a wave 32 rows, a lane 4 rows
// x 8 columns (rows 4 (lane / 8) .., columns 8 (lane % 8) ..): the three results of a lane, 96 numbers, stay in registers until
// their columns' maxima are known.
__device__ __forceinline__ void silu_backward(float dh, float g, float u, float& dg, float& du, float& a) {
  // exp through the hardware's 2^x and a reciprocal: a few units in the last place, against the 2^-4 of what follows
  const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * g));
  const float gs = g * s;
  a = gs * u;
  du = dh * gs;
  dg = dh * u * s * (1.0f + g * (1.0f - s));
}

__global__ __launch_bounds__(256) void silu_backward_kernel(const SiluBackwardArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t tile[3][64 * 128];   // codes along columns: dg, du, a
  __shared__ uint8_t srow[2][128 * 2], scol[3][64 * 4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, rg = lane >> 3, cg = lane & 7;
  const int tr = blockIdx.x / a.tiles_k;
  const int64_t r0 = (int64_t)tr * 128, k0 = (int64_t)(blockIdx.x - tr * a.tiles_k) * 64;
  const int64_t rows = a.rows, F = a.F, Rpad = (rows + 31) / 32 * 32;
  const bool floor_mode = a.scale_mode != 0;
  if (tid < 128) ((uint32_t*)srow)[tid] = 0x7F7F7F7Fu;
  if (tid < 192) ((uint32_t*)scol)[tid] = 0x7F7F7F7Fu;
  __syncthreads();
  if (r0 < rows) {
    const int64_t row = r0 + 32 * wave + 4 * rg, col = k0 + 8 * cg;
    const bool col_in = col < F;
    float v[3][4][8];
    // four rows at a time are requested before the first is used
    v4i rdh[4];
    u2 rg_[4], ru[4];
    uint32_t sg[4], su[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t r = row + i < rows ? row + i : rows - 1, c = col_in ? col : 0;
      const uint16_t* const p = a.dh + r * a.dh_ld + c;
      if (a.vec) rdh[i] = *(const v4i*)p;
      else
#pragma unroll
        for (int h = 0; h < 4; ++h) rdh[i][h] = (int)((uint32_t)p[2 * h] | ((uint32_t)p[2 * h + 1] << 16));
      rg_[i] = *(const u2*)(a.gu + r * a.gu_ld + c);
      ru[i] = *(const u2*)(a.gu + r * a.gu_ld + F + c);
      sg[i] = a.gus[r * a.gus_ld + c / 32];
      su[i] = a.gus[r * a.gus_ld + (F + c) / 32];
    }
    uint32_t again = 0;   // bits 0 - 3: rows of dg, 4 - 7: rows of du, 8 + 8 o ..: columns of result o
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float dh[8];
      unpack_bf16(rdh[i], dh);
      const float fg = decode_e8m0(sg[i]), fu = decode_e8m0(su[i]);
      const bool live = row + i < rows && col_in;
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const f2 pg = (h & 1) ? __builtin_amdgcn_cvt_pk_f32_fp8((int)rg_[i][h >> 1], true) : __builtin_amdgcn_cvt_pk_f32_fp8((int)rg_[i][h >> 1], false);
        const f2 pu = (h & 1) ? __builtin_amdgcn_cvt_pk_f32_fp8((int)ru[i][h >> 1], true) : __builtin_amdgcn_cvt_pk_f32_fp8((int)ru[i][h >> 1], false);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int e = 2 * h + q;
          silu_backward(dh[e], pg[q] * fg, pu[q] * fu, v[0][i][e], v[1][i][e], v[2][i][e]);
          if (!live) v[0][i][e] = v[1][i][e] = v[2][i][e] = 0.f;
        }
      }
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        uint32_t am = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) am = umax(am, magnitude(v[o][i][e]));
        const BlockScale b = block_scale<MX_E4M3>(max_quad(am), floor_mode);
        const float (&w)[8] = v[o][i];
        const u2 c = {encode4<MX_E4M3>(w[0], w[1], w[2], w[3], b), encode4<MX_E4M3>(w[4], w[5], w[6], w[7], b)};
        if (live && b.ok) {
          *(u2*)(a.d + (row + i) * a.d_ld + o * F + col) = c;
          if ((lane & 3) == 0) srow[o][(32 * wave + 4 * rg + i) * 2 + (cg >> 2)] = (uint8_t)b.byte;
        }
        if (live && !b.ok) again |= 1u << (4 * o + i);
      }
    }
    auto place = [&](int o, int e, uint32_t c) {
      *(uint32_t*)(tile[o] + (8 * cg + e) * 128 + (((2 * wave + (rg >> 2)) ^ cg) << 4) + (rg & 3) * 4) = c;
    };
    const bool block_in = r0 + 32 * wave < rows && col_in;
#pragma unroll
    for (int o = 0; o < 3; ++o) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        uint32_t am = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) am = umax(am, magnitude(v[o][i][e]));
        const BlockScale b = block_scale<MX_E4M3>(max_xor_16_32(max_xor_8(am)), floor_mode);
        const uint32_t c = encode4<MX_E4M3>(v[o][0][e], v[o][1][e], v[o][2][e], v[o][3][e], b);
        if (block_in && b.ok) {
          place(o, e, c);
          if (rg == 0) scol[o][(8 * cg + e) * 4 + wave] = (uint8_t)b.byte;
        }
        if (block_in && !b.ok) again |= 1u << (8 + 8 * o + e);
      }
    }
    if (again) {   // blocks for encode_block: computed again from memory (the lanes of a block agree)
      auto value = [&](int o, int64_t r, int64_t c) {
        if (r >= rows) return 0.f;
        const float fg = decode_e8m0(a.gus[r * a.gus_ld + c / 32]), fu = decode_e8m0(a.gus[r * a.gus_ld + (F + c) / 32]);
        float dg, du, ac;
        silu_backward(bf16_to_f32(a.dh[r * a.dh_ld + c]), __builtin_amdgcn_cvt_pk_f32_fp8(a.gu[r * a.gu_ld + c], false)[0] * fg,
                      __builtin_amdgcn_cvt_pk_f32_fp8(a.gu[r * a.gu_ld + F + c], false)[0] * fu, dg, du, ac);
        return o == 0 ? dg : o == 1 ? du : ac;
      };
      for (int n = 0; n < 8; ++n) {
        if (!(again >> n & 1)) continue;
        const int o = n >> 2, i = n & 3;
        float w[8];
        uint32_t am = 0, c[2], byte;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          w[e] = value(o, row + i, col + e);
          am = umax(am, magnitude(w[e]));
        }
        encode_slow<8>(w, max_quad(am), MX_E4M3, a.scale_mode, c, byte);
        *(u2*)(a.d + (row + i) * a.d_ld + o * F + col) = (u2){c[0], c[1]};
        if ((lane & 3) == 0) srow[o][(32 * wave + 4 * rg + i) * 2 + (cg >> 2)] = (uint8_t)byte;
      }
      for (int n = 8; n < 32; ++n) {
        if (!(again >> n & 1)) continue;
        const int o = (n >> 3) - 1, e = n & 7;
        float w[4];
        uint32_t am = 0, c[1], byte;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[i] = value(o, row + i, col + e);
          am = umax(am, magnitude(w[i]));
        }
        encode_slow<4>(w, max_xor_16_32(max_xor_8(am)), MX_E4M3, a.scale_mode, c, byte);
        place(o, e, c[0]);
        if (rg == 0) scol[o][(8 * cg + e) * 4 + wave] = (uint8_t)byte;
      }
    }
  }
  __syncthreads();
  if (r0 < rows) {
#pragma unroll
    for (int n = 0; n < 6; ++n) {
      const int o = n >> 1, c = (n & 1) * 32 + (tid >> 3), j = tid & 7;
      if (k0 + c < F && r0 + 16 * j < Rpad) {
        const u4 w = *(const u4*)(tile[o] + c * 128 + ((j ^ (c >> 3)) << 4));
        uint8_t* const p = o == 2 ? a.at + (k0 + c) * a.at_ld : a.dt + (o * F + k0 + c) * a.dt_ld;
        *(u4*)(p + r0 + 16 * j) = w;
      }
    }
  }
  // ---- scales along the rows: [128][2 blocks] of dg and du -------------------------------------------------------------------
  const int64_t blocks = 2 * F / 32, quads = (blocks + 15) / 16;
  if (a.ds_kind == kScalePlain) {
    const int o = tid >> 7, r = tid & 127;
    if (r0 + r < rows)
      for (int k = 0; k < 2; ++k)
        if (k0 + 32 * k < F) a.ds[(r0 + r) * a.ds_ld + (o * F + k0) / 32 + k] = srow[o][r * 2 + k];
  } else {
    // a dword (lane c of a block, group of 64 rows): o = matrix, h = group of the tile, k = block
    const int c = tid & 15, k = tid >> 4 & 1, h = tid >> 5 & 1, o = tid >> 6 & 1;
    const int64_t G = r0 / 64 + h, kb = (o * F + k0) / 32 + k, groups = (rows + 63) / 64;
    auto dword = [&](int64_t block) { return ((G * quads + block / 16) * 64 + (block & 3) * 16 + c) * 4 + (block >> 2 & 3); };
    if (tid < 128 && G < groups) {
      uint32_t w = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b)
        w |= (uint32_t)srow[o][(64 * h + (a.ds_kind == kScaleNativeB ? bperm_row(b, c) : 16 * b + c)) * 2 + k] << (8 * b);
      ((uint32_t*)a.ds)[dword(kb)] = w;
      // the last tile of the row also fills the quad up
      if (k0 + 64 >= F && o == 1)
        for (int64_t block = blocks + k; block < quads * 16; block += 2) ((uint32_t*)a.ds)[dword(block)] = 0x7F7F7F7Fu;
    }
  }
  // ---- scales along the columns: [64][4 blocks] of dg, du, a ------------------------------------------------------------------
  const int64_t cblocks = Rpad / 32, cquads = (cblocks + 15) / 16, cb0 = r0 / 32;
  if (tid < 192) {
    const int o = tid >> 6, l = tid & 63;
    const int kind = o == 2 ? a.ats_kind : a.dts_kind;
    uint8_t* const s = o == 2 ? a.ats : a.dts;
    const int64_t base = o == 1 ? F : 0;               // row of dt
    if (kind == kScalePlain) {
      if (k0 + l < F) {
        uint8_t* const p = s + (base + k0 + l) * (o == 2 ? a.ats_ld : a.dts_ld) + cb0;
        for (int k = 0; k < 4; ++k)
          if (cb0 + k < cblocks) p[k] = scol[o][l * 4 + k];
      }
    } else if (cb0 < cquads * 16) {
      const int c = l & 15, g = l >> 4;
      const int64_t G = (base + k0) / 64;
      uint32_t w = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b)
        w |= (uint32_t)scol[o][(kind == kScaleNativeB ? bperm_row(b, c) : 16 * b + c) * 4 + g] << (8 * b);
      ((uint32_t*)s)[((G * cquads + cb0 / 16) * 64 + l) * 4 + (cb0 / 4) % 4] = w;
    }
  }
}

template <int SRC, int FMT>
hipError_t launch_both(const BothArgs& a, int64_t blocks, hipStream_t stream) {
  return launch_kernel(quantize_both_kernel<SRC, FMT>, dim3((unsigned)blocks), dim3(256), 0, stream, a);
}

}  // namespace

int launch_quantize_both(const BothTensor* list, int n, int fmt, int scale_mode, hipStream_t stream) {
  for (int i = 0; i < n;) {
    BothArgs a = {};
    a.scale_mode = scale_mode;
    const int dtype = list[i].x_dtype, esz = dtype == MX_F32 ? 4 : 2;
    int64_t blocks = 0;
    for (; i < n && a.n < kBothMax && list[i].x_dtype == dtype; ++i) {
      BothTensor t = list[i];
      if (t.rows <= 0 || t.K <= 0) continue;
      // native scales are filled up to whole K-quads (512 elements along the blocks), also where there are no elements
      const int64_t rows = t.qt && t.st_kind != kScalePlain ? (t.rows + 511ll) / 512 * 512 : t.rows;
      const int64_t cols = t.q && t.s_kind != kScalePlain ? (t.K + 511ll) / 512 * 512 : (t.K + 31ll) / 32 * 32;
      t.vec = (((uintptr_t)t.x | (uintptr_t)(t.x_ld * esz)) & 15) == 0;
      t.first = (int32_t)blocks;
      t.tiles_k = (int32_t)((cols + 127) / 128);
      blocks += (rows + 127) / 128 * t.tiles_k;
      if (blocks > 0x7FFFFFFF) return set_error(MX_ERR_SHAPE, "quantize_both: tensor too large");
      a.t[a.n++] = t;
    }
    if (blocks == 0) continue;
    hipError_t e = hipSuccess;
#define MX_CASE(SRC, FMT) if (dtype == SRC && fmt == FMT) e = launch_both<SRC, FMT>(a, blocks, stream);
    MX_CASE(MX_BF16, MX_E4M3)
    MX_CASE(MX_BF16, MX_E5M2)
    MX_CASE(MX_F32, MX_E4M3)
    MX_CASE(MX_F32, MX_E5M2)
    MX_CASE(MX_F16, MX_E4M3)
    MX_CASE(MX_F16, MX_E5M2)
#undef MX_CASE
    if (e != hipSuccess) return set_error(MX_ERR_LAUNCH, "quantize_both_kernel launch: %s", hipGetErrorString(e));
  }
  return MX_OK;
}

int launch_gate_up(const GateUpArgs& a, hipStream_t stream) {
  const int64_t blocks = (a.rows * (a.F / 8) + 255) / 256;
  if (blocks <= 0) return MX_OK;
  if (blocks > 0x7FFFFFFF) return set_error(MX_ERR_SHAPE, "gate_up: tensor too large");
  const hipError_t e = launch_kernel(gate_up_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, a);
  if (e != hipSuccess) return set_error(MX_ERR_LAUNCH, "gate_up_kernel launch: %s", hipGetErrorString(e));
  return MX_OK;
}

int launch_silu_backward(const SiluBackwardArgs& args, hipStream_t stream) {
  SiluBackwardArgs a = args;
  if (a.rows <= 0 || a.F <= 0) return MX_OK;
  a.vec = (((uintptr_t)a.dh | (uintptr_t)(a.dh_ld * 2)) & 15) == 0;
  a.tiles_k = (a.F + 63) / 64;
  const bool native = a.dts_kind != kScalePlain || a.ats_kind != kScalePlain;
  const int64_t rows = native ? (a.rows + 511ll) / 512 * 512 : a.rows, blocks = (rows + 127) / 128 * a.tiles_k;
  if (blocks > 0x7FFFFFFF) return set_error(MX_ERR_SHAPE, "silu_backward: tensor too large");
  const hipError_t e = launch_kernel(silu_backward_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, a);
  if (e != hipSuccess) return set_error(MX_ERR_LAUNCH, "silu_backward_kernel launch: %s", hipGetErrorString(e));
  return MX_OK;
}

}  // namespace mx
