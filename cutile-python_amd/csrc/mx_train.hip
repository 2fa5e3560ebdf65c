// Kernels of the gated feed-forward block that is trained in 8 bits: quantisation along both axes of a matrix, the activation
// between the projections with its checkpoint, and the activation's backward pass.  What they quantise follows encode_block
// (mx_quant.h) to the bit, but for blocks with a NaN or, under the ceiling rule, an infinity in silu_backward_kernel.
#include <type_traits>

#include "mx_encode.h"
#include "mx_gemm_tile.h"   // make_rsrc, kOobOffset
#include "mx_load_once.h"
#include "mx_train.h"

namespace mx {
namespace {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));

// Tile (tr, tk) of a workgroup: groups of ROWS tile rows, walked column by column.  Workgroup ids are dealt round-robin to the 8 XCDs,
// each with its own L2; XCD: an XCD takes neighbouring tiles instead.
template <int ROWS, bool XCD>
__device__ __forceinline__ void tile_of(uint32_t id, uint32_t n, uint32_t tiles_k, uint32_t& tr, uint32_t& tk) {
  if constexpr (XCD) {
    const uint32_t per = n >> 3, rest = n & 7, x = id & 7;
    id = x * per + (x < rest ? x : rest) + (id >> 3);
  }
  const uint32_t group = id / (ROWS * tiles_k), first = group * ROWS, in = id - first * tiles_k, left = n / tiles_k - first;
  const uint32_t rows = left < ROWS ? left : ROWS;
  tk = in / rows;
  tr = first + in - tk * rows;
}

// Scale bytes [rows of the tile][4 blocks] of a 128-row tile, from LDS to where they belong: row0, block0 = first row and block
// of the tile; rows, blocks = of the whole matrix; tid = 0 .. 127.  The native layouts are padded with 127 (rows to 64, blocks to 16).
__device__ __forceinline__ void store_scales(const uint32_t* lds, uint8_t* s, int64_t ld, int kind, int tid, int64_t row0, int64_t rows,
                                             int64_t block0, int64_t blocks) {
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
      const uint32_t byte = block0 + g < blocks && row0 + r < rows ? lds[r] >> (8 * g) & 0xFF : 127u;
      w |= byte << (8 * b);
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
//
// PLAIN: aligned rows of whole blocks that do not overlap, tiles of less than 2 GiB.  Loads and stores then go through buffer
// descriptors of the tile, whose range takes the place of every comparison with the matrix's ends, and magnitudes of 16-bit input
// are compared two at a time as they lie in memory.  The vector ALUs are what the rest of the time is spent on otherwise: with
// the comparisons, 64-bit addresses and the scale rule decided per block 8192 x 8192 bf16 took 56 us, now 48 (5.6 TB/s); a copy of
// 2 GiB reaches 5.1 TB/s, where what was just written is in no cache, and this kernel 4.4 of 32768 x 14336.
template <int SRC>
__device__ __forceinline__ float load_one(const void* x, int64_t at) {
  if constexpr (SRC == MX_F32) return ((const float*)x)[at];
  else if constexpr (SRC == MX_BF16) return bf16_to_f32(((const uint16_t*)x)[at]);
  else return (float)((const _Float16*)x)[at];
}
// bits of a float from the bits of a magnitude in SRC
template <int SRC>
__device__ __forceinline__ uint32_t widen(uint32_t m) {
  if constexpr (SRC == MX_BF16) return m << 16;
  else return __builtin_bit_cast(uint32_t, (float)__builtin_bit_cast(_Float16, (uint16_t)m));
}
typedef uint16_t h2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pk_max(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(h2, a), __builtin_bit_cast(h2, b)));
}
// max_columns of columns 2 h, 2 h + 1 in m[h]: the lane's two in one register
__device__ __forceinline__ uint32_t pk_max_columns(const uint32_t (&m)[4]) {
  const auto a = __builtin_amdgcn_permlane32_swap(m[0], m[2], false, false), b = __builtin_amdgcn_permlane32_swap(m[1], m[3], false, false);
  const auto c = __builtin_amdgcn_permlane16_swap(pk_max(a[0], a[1]), pk_max(b[0], b[1]), false, false);
  return pk_max(c[0], c[1]);
}

template <int SRC, int FMT, bool FLOOR, bool PLAIN>
__global__ __launch_bounds__(256) void quantize_both_kernel(const BothArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t tile[128 * 128];
  __shared__ uint32_t srow[128], scol[128];
  constexpr int ESZ = SRC == MX_F32 ? 4 : 2, NL = SRC == MX_F32 ? 2 : 1;
  int which = 0;
#pragma unroll
  for (int k = 1; k < kBothMax; ++k)
    if (k < a.n && (int)blockIdx.x >= a.t[k].first) which = k;
  const BothTensor t = a.t[which];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, rg = lane >> 4, cg = lane & 15;
  uint32_t tr, tk;
  if (t.near) tile_of<2, true>(blockIdx.x - t.first, t.tiles, t.tiles_k, tr, tk);
  else tile_of<1, false>(blockIdx.x - t.first, t.tiles, t.tiles_k, tr, tk);
  const int64_t r0 = (int64_t)tr * 128, k0 = (int64_t)tk * 128;
  const int64_t rows = t.rows, K = t.K, Kpad = (K + 31) / 32 * 32, Rpad = (rows + 31) / 32 * 32;
  uint8_t* const srow_b = (uint8_t*)srow;
  uint8_t* const scol_b = (uint8_t*)scol;
  if constexpr (FLOOR) saturate_conversions();
  const bool inside = r0 < rows && k0 < Kpad;         // (else: padding of native scales only)
  if (inside && r0 + 32 * wave < rows) {              // (waves without rows have nothing to do)
    const int64_t row = r0 + 32 * wave + 8 * rg, col = k0 + 8 * cg;   // of the lane's first element
    const int n_rows = rows - r0 < 128 ? (int)(rows - r0) : 128, n_cols = Kpad - k0 < 128 ? (int)(Kpad - k0) : 128;
    float v[8][8];
    uint32_t mag[8][4];                               // PLAIN, 16-bit input: magnitudes as they lie in memory
    if constexpr (PLAIN) {
      const uint32_t pitch = (uint32_t)(t.x_ld * ESZ);
      const __amdgpu_buffer_rsrc_t rs = make_rsrc((const uint8_t*)t.x + (r0 * t.x_ld + k0) * ESZ, (n_rows - 1) * pitch + n_cols * ESZ);
      uint32_t vo = 8 * cg < n_cols ? (32 * wave + 8 * rg) * pitch + 8 * cg * ESZ : kOobOffset;
      v4i raw[8][NL];
      auto load = [&](auto once) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
          for (int h = 0; h < NL; ++h) raw[i][h] = __builtin_amdgcn_raw_buffer_load_b128(rs, vo + 16 * h, 0, decltype(once)::value);
          vo += pitch;
        }
      };
      if (t.once) load(std::integral_constant<int, kLoadOnce>{});
      else load(std::integral_constant<int, 0>{});
#pragma unroll
      for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          if constexpr (SRC == MX_F32) {
            v[i][h] = __builtin_bit_cast(float, (uint32_t)raw[i][0][h]);
            v[i][4 + h] = __builtin_bit_cast(float, (uint32_t)raw[i][NL - 1][h]);
          } else if constexpr (SRC == MX_BF16) {
            v[i][2 * h] = __builtin_bit_cast(float, (uint32_t)raw[i][0][h] << 16);
            v[i][2 * h + 1] = __builtin_bit_cast(float, (uint32_t)raw[i][0][h] & 0xFFFF0000u);
          } else {
            v[i][2 * h] = (float)__builtin_bit_cast(_Float16, (uint16_t)(uint32_t)raw[i][0][h]);
            v[i][2 * h + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)((uint32_t)raw[i][0][h] >> 16));
          }
          mag[i][h] = (uint32_t)raw[i][0][h] & 0x7FFF7FFFu;
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
    uint32_t most = 0;
    // (scale bytes are written by all lanes of a block, the same byte to the same place: a branch around each costs more)
    if (t.q) {
      const __amdgpu_buffer_rsrc_t rq = make_rsrc(t.q + r0 * t.q_ld + k0, PLAIN ? (uint32_t)((n_rows - 1) * t.q_ld + n_cols) : 0u);
      uint32_t qo = 8 * cg < n_cols ? (32 * wave + 8 * rg) * (uint32_t)t.q_ld + 8 * cg : kOobOffset;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint32_t am = 0;
        if constexpr (PLAIN && SRC != MX_F32) {
          const uint32_t m = pk_max(pk_max(mag[i][0], mag[i][1]), pk_max(mag[i][2], mag[i][3]));
          am = widen<SRC>(max_quad(umax(m & 0xFFFF, m >> 16)));
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) am = umax(am, magnitude(v[i][e]));
          am = max_quad(am);
        }
        most = umax(most, am);
        const BlockScale b = block_scale<FMT, FLOOR>(am);
        const u2 c = {encode4<FMT>(v[i][0], v[i][1], v[i][2], v[i][3], b.scale), encode4<FMT>(v[i][4], v[i][5], v[i][6], v[i][7], b.scale)};
        if constexpr (PLAIN) {
          __builtin_amdgcn_raw_buffer_store_b64(c, rq, qo, 0, 0);
          qo += (uint32_t)t.q_ld;
        } else if (row + i < rows && col < Kpad) {
          *(u2*)(t.q + (row + i) * t.q_ld + col) = c;
        }
        srow_b[(32 * wave + 8 * rg + i) * 4 + (cg >> 2)] = (uint8_t)b.byte;
      }
    }
    // transposed: the lane's codes of column 8 cg + e are 8 of that column's 128 bytes
    auto place = [&](int e, u2 c) {
      *(u2*)(tile + (8 * cg + e) * 128 + (((2 * wave + (rg >> 1)) ^ (cg & 7)) << 4) + (rg & 1) * 8) = c;
    };
    if (t.qt) {
      uint32_t own[2];
      if constexpr (PLAIN && SRC != MX_F32) {
        uint32_t m[4];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          m[h] = mag[0][h];
#pragma unroll
          for (int i = 1; i < 8; ++i) m[h] = pk_max(m[h], mag[i][h]);
        }
        const uint32_t r = pk_max_columns(m);
        own[0] = widen<SRC>(r & 0xFFFF);
        own[1] = widen<SRC>(r >> 16);
      } else {
        uint32_t m[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          m[e] = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) m[e] = umax(m[e], magnitude(v[i][e]));
        }
        max_columns(m, own);
      }
      float scale[2], s[8];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        most = umax(most, own[e]);
        const BlockScale b = block_scale<FMT, FLOOR>(own[e]);
        scale[e] = b.scale;
        scol_b[(8 * cg + own_column(lane) + e) * 4 + wave] = (uint8_t)b.byte;
      }
      spread_columns(scale, s);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        place(e, (u2){encode4<FMT>(v[0][e], v[1][e], v[2][e], v[3][e], s[e]), encode4<FMT>(v[4][e], v[5][e], v[6][e], v[7][e], s[e])});
    }
    if (__builtin_amdgcn_ballot_w64(odd_block<FLOOR>(most))) {   // a wave with such a block does all of its blocks again, from memory
#pragma unroll 1
      for (int i = 0; t.q && i < 8; ++i) {
        float w[8];
        uint32_t am = 0, c[2], byte;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          w[e] = row + i < rows && col + e < K ? load_one<SRC>(t.x, (row + i) * t.x_ld + col + e) : 0.f;
          am = umax(am, magnitude(w[e]));
        }
        encode_slow<8>(w, max_quad(am), FMT, a.scale_mode, c, byte);
        if (row + i < rows && col < Kpad) *(u2*)(t.q + (row + i) * t.q_ld + col) = (u2){c[0], c[1]};
        if ((lane & 3) == 0) srow_b[(32 * wave + 8 * rg + i) * 4 + (cg >> 2)] = (uint8_t)byte;
      }
#pragma unroll 1
      for (int e = 0; t.qt && e < 8; ++e) {
        float w[8];
        uint32_t am = 0, c[2], byte;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          w[i] = row + i < rows && col + e < K ? load_one<SRC>(t.x, (row + i) * t.x_ld + col + e) : 0.f;
          am = umax(am, magnitude(w[i]));
        }
        encode_slow<8>(w, max_xor_16_32(am), FMT, a.scale_mode, c, byte);
        place(e, (u2){c[0], c[1]});
        if (rg == 0) scol_b[(8 * cg + e) * 4 + wave] = (uint8_t)byte;
      }
    }
  }
  __syncthreads();
  if (inside) {
    if (t.qt) {
      const int m_cols = K - k0 < 128 ? (int)(K - k0) : 128, m_rows = Rpad - r0 < 128 ? (int)(Rpad - r0) : 128;   // of the transposed tile
      const __amdgpu_buffer_rsrc_t rt = make_rsrc(t.qt + k0 * t.qt_ld + r0, PLAIN ? (uint32_t)((m_cols - 1) * t.qt_ld + m_rows) : 0u);
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int c = n * 32 + (tid >> 3), j = tid & 7;
        const u4 w = *(const u4*)(tile + c * 128 + ((j ^ (c >> 3 & 7)) << 4));
        if constexpr (PLAIN) __builtin_amdgcn_raw_buffer_store_b128(w, rt, 16 * j < m_rows ? c * (uint32_t)t.qt_ld + 16 * j : kOobOffset, 0, 0);
        else if (c < m_cols && 16 * j < m_rows) *(u4*)(t.qt + (k0 + c) * t.qt_ld + r0 + 16 * j) = w;
      }
    }
  }
  if (tid >= 128) {
    if (t.q) store_scales(srow, t.s, t.s_ld, t.s_kind, tid - 128, r0, rows, k0 / 32, Kpad / 32);
  } else if (t.qt) {
    store_scales(scol, t.st, t.st_ld, t.st_kind, tid, k0, K, r0 / 32, Rpad / 32);
  }
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
template <int FMT, bool FLOOR>
__device__ __forceinline__ void store_row_block(const float (&v)[8], uint8_t* q, uint8_t* s, bool scale_lane) {
  uint32_t am = 0, c[2], byte;
#pragma unroll
  for (int e = 0; e < 8; ++e) am = umax(am, magnitude(v[e]));
  am = max_quad(am);
  const BlockScale b = block_scale<FMT, FLOOR>(am);
  if (!odd_block<FLOOR>(am)) {
    c[0] = encode4<FMT>(v[0], v[1], v[2], v[3], b.scale);
    c[1] = encode4<FMT>(v[4], v[5], v[6], v[7], b.scale);
    byte = b.byte;
  } else {
    encode_slow<8>(v, am, FMT, FLOOR, c, byte);
  }
  *(u2*)q = (u2){c[0], c[1]};
  if (scale_lane) *s = (uint8_t)byte;
}

// OUT: MX_BF16, MX_E4M3 or MX_E5M2
template <int OUT, bool FLOOR>
__global__ __launch_bounds__(256) void gate_up_kernel(const GateUpArgs a) {
  const GateOut& o = a.out;
  if constexpr (FLOOR) saturate_conversions();
  const int64_t unit = (int64_t)blockIdx.x * 256 + threadIdx.x, per = o.F / 8;   // (32 columns are four lanes of a wave)
  const int64_t row = unit / per, col = (unit - row * per) * 8;
  if (row >= a.rows) return;
  const uint16_t* const p = a.gu + row * a.gu_ld + col;
  float g[8], u[8], h[8];
  unpack_bf16(*(const v4i*)p, g);
  unpack_bf16(*(const v4i*)(p + o.F), u);
#pragma unroll
  for (int e = 0; e < 8; ++e) h[e] = silu_mul_f32(g[e], u[e]);
  const bool first = (threadIdx.x & 3) == 0;
  if constexpr (OUT == MX_BF16) {
    u4 w;
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = (uint32_t)f32_to_bf16(h[2 * k]) | ((uint32_t)f32_to_bf16(h[2 * k + 1]) << 16);
    *(u4*)((uint16_t*)o.h + row * o.h_ld + col) = w;
  } else {
    store_row_block<OUT, FLOOR>(h, (uint8_t*)o.h + row * o.h_ld + col, o.hs + row * o.hs_ld + col / 32, first);
  }
  if (o.c) {
    uint8_t* const c = o.c + row * o.c_ld + col;
    uint8_t* const cs = o.cs + row * o.cs_ld + col / 32;
    store_row_block<MX_E4M3, FLOOR>(g, c, cs, first);
    store_row_block<MX_E4M3, FLOOR>(u, c + o.F, cs + o.F / 32, first);
  }
}

// ================================================================================================================================
// The activation's backward pass
// ================================================================================================================================
//   s = 1 / (1 + exp(-g));  du = dh g s;  dg = dh u s (1 + g (1 - s));  a = g s u
// g and u are the checkpoint's values.  d[g|u] goes out quantised along the rows (for the product with w1) and along the columns
// (for the gradient of w1), a along the columns (for the gradient of w2; the forward pass kept no copy of it, which saves 8.25 bits per element from
// one pass to the other for one multiplication here).
// Bound: memory, 4.06 bytes read and 5.16 written an element of dh.  A workgroup takes 128 rows x 128 columns (whole lines both
// ways), a wave 32 x 64, a lane 4 rows x 8 columns (rows 4 (lane / 8) .., columns 8 (lane % 8) ..), one result after the other: 32
// numbers that stay in registers until their rows' and columns' maxima are known, beside g s, which the second and the third are
// made of.  4096 x 14336: 109 us where every call writes the same memory, 123 (4.4 TB/s) where it is another; a copy of 2 GiB reaches
// 5.1 TB/s, and the difference goes into eight streams of one line a row each.
// g -> g s and s (1 + g (1 - s)) = s + g s (1 - s); exp through the hardware's 2^x and a reciprocal: within 2^-18 of the value (2^-17 for g below -32,
// where rounding -1.44 g counts), of the terms where they cancel (g near -1.28), against the 2^-4 of what follows.  1 - s, not s + g s - g s s: that is 1 + g - g for a large g, 0 in place of 1
// from 2^24 on.  s is 0 or 1 far out, and g ends at numbers that such an s multiplies without a NaN (-126, below which s is 0; the largest float for
// a code and scale beyond it); a NaN comes back through s.
__device__ __forceinline__ void silu_slope(float g, float& gs, float& slope) {
  const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * g));
  gs = __builtin_amdgcn_fmed3f(g, -126.0f, 3.4028234664e38f) * s;
  slope = __builtin_fmaf(gs, 1.0f - s, s);
}

// Loads and stores through descriptors of the tile, as in quantize_both_kernel (the launcher's rule; PLAIN false: any pitch).
// ONCE: dh and the checkpoint are loaded non-temporally (as the quantiser's input, mx_load_once.h).
template <bool FLOOR, bool PLAIN, bool ONCE>
__global__ __launch_bounds__(512, 4) void silu_backward_kernel(const SiluBackwardArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t tile[3][128 * 128];   // codes along columns: dg, du, a
  __shared__ uint32_t srow[2][128], scol[3][128];      // their scales, four blocks a row
  __shared__ uint32_t sin[2][128];                     // scales of g and u
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6 & 3, half = tid >> 8, rg = lane >> 3, cg = lane & 7;
  const int64_t rows = a.rows, F = a.F, Rpad = (rows + 31) / 32 * 32;
  const int lr = 32 * wave + 4 * rg, lc = 64 * half + 8 * cg;    // of the lane's first element, in the tile
  if constexpr (FLOOR) saturate_conversions();
  // ---- the lane's inputs, of the tile that begins at (r0, k0): zeros outside of the matrix -------------------------------------
  v4i rdh[4];
  u2 rgt[4], rup[4];
  // at: 0 (gate), F (up).  PLAIN: 1 KiB of eight rows at a time into tile[o], 16-byte chunks swizzled by row / 4: a wave needs half lines
  // only, and a line that two waves load non-temporally, half each, is fetched twice (4096 x 14336: 334 MB in place of 239,
  // 142 us in place of 123; loaded plainly 134).
  auto load_gate_or_up = [&](int64_t r0, int64_t k0, int o, u2 (&q)[4]) {
    const int n_rows = rows - r0 < 128 ? (int)(rows - r0) : 128, n_cols = F - k0 < 128 ? (int)(F - k0) : 128;
    const int64_t at = o * F;
    if constexpr (PLAIN) {
      const uint32_t pg = (uint32_t)a.gu_ld;
      const __amdgpu_buffer_rsrc_t rs = make_rsrc(a.gu + r0 * a.gu_ld + at + k0, (uint32_t)((n_rows - 1) * pg + n_cols));
      const int w8 = __builtin_amdgcn_readfirstlane(tid >> 6);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int row = 16 * w8 + 8 * j + (lane >> 3), col = ((lane & 7) ^ (row >> 2 & 7)) * 16;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)((lds_u8*)tile[o] + (16 * w8 + 8 * j) * 128), 16,
                                                 row < n_rows && col < n_cols ? row * pg + col : kOobOffset, 0, 0, ONCE ? kLoadOnce : 0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        q[i] = (u2){0, 0};
        if (lr + i < n_rows && lc < n_cols) q[i] = *(const u2*)(a.gu + (r0 + lr + i) * a.gu_ld + at + k0 + lc);
      }
    }
  };
  auto load_dh = [&](int64_t r0, int64_t k0) {
    const int n_rows = rows - r0 < 128 ? (int)(rows - r0) : 128;
    const bool col_in = k0 + lc < F;
    if constexpr (PLAIN) {
      const uint32_t pd = (uint32_t)(a.dh_ld * 2);
      const __amdgpu_buffer_rsrc_t rs = make_rsrc(a.dh + r0 * a.dh_ld + k0, (uint32_t)((n_rows - 1) * pd + (F - k0) * 2));
#pragma unroll
      for (int i = 0; i < 4; ++i)
        rdh[i] = __builtin_amdgcn_raw_buffer_load_b128(rs, (col_in && lr + i < n_rows ? 0 : kOobOffset) | ((lr + i) * pd + lc * 2), 0, ONCE ? kLoadOnce : 0);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        rdh[i] = (v4i){0, 0, 0, 0};
        if (lr + i >= n_rows || !col_in) continue;
        const uint16_t* const p = a.dh + (r0 + lr + i) * a.dh_ld + k0 + lc;
#pragma unroll
        for (int h = 0; h < 4; ++h) rdh[i][h] = (int)((uint32_t)p[2 * h] | ((uint32_t)p[2 * h + 1] << 16));
      }
    }
  };
  uint32_t tr, tk;
  tile_of<8, true>(blockIdx.x, gridDim.x, a.tiles_k, tr, tk);
  const int64_t r0 = (int64_t)tr * 128, k0 = (int64_t)tk * 128;
  const int n_rows = rows - r0 < 128 ? (int)(rows - r0) : 128, n_cols = F - k0 < 128 ? (int)(F - k0) : 128, m_rows = Rpad - r0 < 128 ? (int)(Rpad - r0) : 128;
  if (r0 < rows) {                                     // (else: padding of native scales only)
    const int64_t row = r0 + lr, col = k0 + lc;
    const bool col_in = lc < n_cols;
    // the four blocks' scales of a row of g or u at a time: by the byte, each lane its own, they were as many requests as the codes
    // (4096 x 14336 152 -> 145 us)
    uint32_t scales = 0;
    const int so = tid >> 7 & 1, sr = tid & 127;
    if (tid < 256 && sr < n_rows) {
      const uint8_t* const p = a.gus + (r0 + sr) * a.gus_ld + (so * F + k0) / 32;
      if (n_cols == 128 && ((uintptr_t)p & 3) == 0) scales = *(const uint32_t*)p;
      else
        for (int k = 0; k < n_cols / 32; ++k) scales |= (uint32_t)p[k] << (8 * k);
    }
    __builtin_amdgcn_sched_barrier(0);
    load_gate_or_up(r0, k0, 0, rgt);
    load_gate_or_up(r0, k0, 1, rup);
    // (what the wait below may leave in flight are the four loads of dh, requested last)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    load_dh(r0, k0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    if (tid < 256) sin[so][sr] = scales;
    if constexpr (PLAIN) {
      __builtin_amdgcn_s_waitcnt(0x0F70 | 4);          // the wave's share of g and u is in LDS
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");   // (a fence would wait for dh as well)
    } else {
      __syncthreads();
    }
    if constexpr (PLAIN) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = (lr + i) * 128 + ((4 * half + (cg >> 1)) ^ rg) * 16 + (cg & 1) * 8;
        rgt[i] = *(const u2*)(tile[0] + at);
        rup[i] = *(const u2*)(tile[1] + at);
      }
      __syncthreads();                                 // codes along columns go there
    }
    if (lr - 4 * rg < n_rows) {                        // (waves without rows have nothing to do)
      auto scale_in = [&](int o, int i) { return (uint32_t)((const uint8_t*)sin[o])[(lr + i) * 4 + lc / 32]; };
      const __amdgpu_buffer_rsrc_t rd = make_rsrc(a.d + r0 * a.d_ld + k0, PLAIN ? (uint32_t)((n_rows - 1) * a.d_ld + F + n_cols) : 0u);
      // (The maxima pass over NaN: it is NaN among codes of its block's other values, where encode_block gives zeros under the floor rule and NaN
      // under the ceiling rule.  An infinity under the ceiling rule has the scale NaN as there, and other codes.)
      // one result at a time, 32 numbers of a lane: out along the rows (dg, du), then along the columns
      auto row_out = [&](int o, const float (&v)[4][8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float m = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) m = fmax_abs(m, v[i][e]);
          const BlockScale b = block_scale<MX_E4M3, FLOOR>(max_quad(__builtin_bit_cast(uint32_t, m)));
          const float (&w)[8] = v[i];
          const u2 c = {encode4<MX_E4M3>(w[0], w[1], w[2], w[3], b.scale), encode4<MX_E4M3>(w[4], w[5], w[6], w[7], b.scale)};
          if constexpr (PLAIN) {
            const uint32_t in = col_in && lr + i < n_rows ? 0 : kOobOffset;
            __builtin_amdgcn_raw_buffer_store_b64(c, rd, in | ((lr + i) * (uint32_t)a.d_ld + o * (uint32_t)F + lc), 0, 0);
          } else if (row + i < rows && col_in) {
            *(u2*)(a.d + (row + i) * a.d_ld + o * F + col) = c;
          }
          ((uint8_t*)srow[o])[(lr + i) * 4 + lc / 32] = (uint8_t)b.byte;
        }
      };
      auto place = [&](int o, int e, uint32_t c) {
        *(uint32_t*)(tile[o] + (lc + e) * 128 + (((2 * wave + (rg >> 2)) ^ cg) << 4) + (rg & 3) * 4) = c;
      };
      auto col_out = [&](int o, const float (&v)[4][8]) {
        uint32_t m[8], own[2];
        float scale[2], s[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          m[e] = __builtin_bit_cast(uint32_t, fmax_abs(fmax_abs(fmax_abs(__builtin_fabsf(v[0][e]), v[1][e]), v[2][e]), v[3][e]));
        max_columns(m, own);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const BlockScale b = block_scale<MX_E4M3, FLOOR>(max_xor_8(own[e]));
          scale[e] = b.scale;
          ((uint8_t*)scol[o])[(lc + own_column(lane) + e) * 4 + wave] = (uint8_t)b.byte;
        }
        spread_columns(scale, s);
#pragma unroll
        for (int e = 0; e < 8; ++e) place(o, e, encode4<MX_E4M3>(v[0][e], v[1][e], v[2][e], v[3][e], s[e]));
      };
      // (zeros out of range make zeros: 2^-127 * 0, 0 * 0.5)
      auto decoded = [](const u2& c, uint32_t byte, float (&out)[8]) {
        const float scale = __builtin_bit_cast(float, byte << 23);   // (the conversion takes the exponent: 0 is 2^-127, 255 NaN)
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const f2 p = (h & 1) ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c[h >> 1], scale, true) : __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c[h >> 1], scale, false);
          out[2 * h] = p[0];
          out[2 * h + 1] = p[1];
        }
      };
      float v[4][8], gs[4][8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float g[8];
        decoded(rgt[i], scale_in(0, i), g);
#pragma unroll
        for (int e = 0; e < 8; ++e) silu_slope(g[e], gs[i][e], v[i][e]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float dh[8], u[8];
        unpack_bf16(rdh[i], dh);
        decoded(rup[i], scale_in(1, i), u);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = dh[e] * u[e] * v[i][e];
      }
      row_out(0, v);
      col_out(0, v);
      // (the next result is not begun before, and the inputs are unpacked again for it: more waves on a SIMD)
      auto again = [&]() {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(rup[i]));
      };
#pragma unroll
      for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(rdh[i]));
      again();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float dh[8];
        unpack_bf16(rdh[i], dh);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = dh[e] * gs[i][e];
      }
      row_out(1, v);
      col_out(1, v);
      again();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float u[8];
        decoded(rup[i], scale_in(1, i), u);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = gs[i][e] * u[e];
      }
      col_out(2, v);
    }
    __syncthreads();
    // (whole lines that are not merged with others': not kept in the caches, 16384 x 14336 634 -> 570 us, 4096 x 14336 139 -> 125)
#pragma unroll
    for (int n = 0; n < 6; ++n) {
      const int o = n >> 1, c = (n & 1) * 64 + (tid >> 3), j = tid & 7;
      if (c < n_cols && 16 * j < m_rows) {
        const u4 w = *(const u4*)(tile[o] + c * 128 + ((j ^ (c >> 3 & 7)) << 4));
        uint8_t* const p = o == 2 ? a.at + (k0 + c) * a.at_ld : a.dt + (o * F + k0 + c) * a.dt_ld;
        __builtin_nontemporal_store(w, (u4*)(p + r0 + 16 * j));
      }
    }
  }
  // ---- scales: rows of dg and du, whose blocks begin at 0 and F / 32 of a row of d ... ------------------------------------------
  const int64_t blocks = 2 * F / 32, quads = (blocks + 15) / 16;
  if (a.ds_kind == kScalePlain) {
    const int o = tid >> 7 & 1, r = tid & 127;
    if (tid < 256 && r < n_rows) {
      uint8_t* const p = a.ds + (r0 + r) * a.ds_ld + (o * F + k0) / 32;
      if (n_cols == 128 && ((uintptr_t)p & 3) == 0) *(uint32_t*)p = srow[o][r];
      else
        for (int k = 0; k < n_cols / 32; ++k) p[k] = (uint8_t)(srow[o][r] >> (8 * k));
    }
  } else {
    // a dword (lane c of a block, group of 64 rows): o = matrix, h = group of the tile, k = block
    const int c = tid & 15, k = tid >> 4 & 3, h = tid >> 6 & 1, o = tid >> 7 & 1;
    const int64_t G = r0 / 64 + h, kb = (o * F + k0) / 32 + k, groups = (rows + 63) / 64;
    auto dword = [&](int64_t block) { return ((G * quads + block / 16) * 64 + (block & 3) * 16 + c) * 4 + (block >> 2 & 3); };
    if (tid < 256 && G < groups) {
      uint32_t w = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int r = 64 * h + (a.ds_kind == kScaleNativeB ? bperm_row(b, c) : 16 * b + c);
        w |= (r < n_rows ? srow[o][r] >> (8 * k) & 0xFF : 127u) << (8 * b);
      }
      if (32 * k < n_cols) ((uint32_t*)a.ds)[dword(kb)] = w;
      // the last tile of the row also fills the quad up
      if (k0 + 128 >= F && o == 1)
        for (int64_t block = blocks + k; block < quads * 16; block += 4) ((uint32_t*)a.ds)[dword(block)] = 0x7F7F7F7Fu;
    }
  }
  // ---- ... and columns of dg, du, a ---------------------------------------------------------------------------------------------
  if (tid < 384) {
    const int o = tid >> 7;
    // (128 columns from F + k0 on are whole groups of 64 rows of dt: native scales are for F % 64 == 0 only)
    const int64_t base = o == 1 ? F : 0;
    store_scales(scol[o], o == 2 ? a.ats : a.dts, o == 2 ? a.ats_ld : a.dts_ld, o == 2 ? a.ats_kind : a.dts_kind, tid & 127, base + k0, base + F, r0 / 32,
                 Rpad / 32);
  }
}

template <int SRC, int FMT, bool PLAIN>
hipError_t launch_both(const BothArgs& a, int64_t blocks, hipStream_t stream) {
  const dim3 grid((unsigned)blocks);
  if (a.scale_mode) return launch_kernel(quantize_both_kernel<SRC, FMT, true, PLAIN>, grid, dim3(256), 0, stream, a);
  return launch_kernel(quantize_both_kernel<SRC, FMT, false, PLAIN>, grid, dim3(256), 0, stream, a);
}
// a matrix that PLAIN instances take
bool both_is_plain(const BothTensor& t) {
  const int64_t esz = t.x_dtype == MX_F32 ? 4 : 2, lim = (int64_t)1 << 31;
  return t.K % 32 == 0 && t.x_ld >= t.K && (((uintptr_t)t.x | (uintptr_t)(t.x_ld * esz)) & 15) == 0 && 128 * t.x_ld * esz < lim &&
         (!t.q || 128 * t.q_ld < lim) && (!t.qt || 128 * t.qt_ld < lim);
}

}  // namespace

int launch_quantize_both(const BothTensor* list, int n, int fmt, int scale_mode, hipStream_t stream) {
  for (int i = 0; i < n;) {
    BothArgs a = {};
    a.scale_mode = scale_mode;
    const int dtype = list[i].x_dtype;
    const bool plain = both_is_plain(list[i]);
    int64_t blocks = 0;
    for (; i < n && a.n < kBothMax && list[i].x_dtype == dtype && both_is_plain(list[i]) == plain; ++i) {
      BothTensor t = list[i];
      if (t.rows <= 0 || t.K <= 0) continue;
      // native scales are filled up to whole K-quads (512 elements along the blocks), also where there are no elements
      const int64_t rows = t.qt && t.st_kind != kScalePlain ? (t.rows + 511ll) / 512 * 512 : t.rows;
      const int64_t cols = t.q && t.s_kind != kScalePlain ? (t.K + 511ll) / 512 * 512 : (t.K + 31ll) / 32 * 32;
      t.first = (int32_t)blocks;
      t.tiles_k = (int32_t)((cols + 127) / 128);
      const int64_t tiles = (rows + 127) / 128 * t.tiles_k;
      blocks += tiles;
      if (blocks > 0x7FFFFFFF) return set_error(MX_ERR_SHAPE, "quantize_both: tensor too large");
      t.tiles = (int32_t)tiles;
      t.once = quantize_loads_once((int64_t)t.rows * t.K);
      // An XCD takes neighbouring tiles, by two rows of tiles, so that lines of scales meet in its L2.  us, row by row over all XCDs and so: bf16
      // 4096 x 14336 46.4 | 43.6, 8192 x 8192 50.2 | 48.7, 28672 x 4096 97 | 94, 16384 x 8192 123 | 109, 16384 x 14336 221 | 199;
      // fp32 4096 x 4096 20.7 | 19.4, 8192 x 8192 76 | 78; but 32768 x 14336 437 | 469, 32768 x 14464 428 | 501.  Not of a number of elements alone:
      // 32896 x 14336 502 | 443, 13 % lost here.
      t.near = (int64_t)t.rows * t.K < (int64_t)1 << 28;
      a.t[a.n++] = t;
    }
    if (blocks == 0) continue;
    hipError_t e = hipSuccess;
#define MX_CASE(SRC, FMT) \
    if (dtype == SRC && fmt == FMT) e = plain ? launch_both<SRC, FMT, true>(a, blocks, stream) : launch_both<SRC, FMT, false>(a, blocks, stream);
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
  const int64_t blocks = (a.rows * (a.out.F / 8) + 255) / 256;
  if (blocks <= 0) return MX_OK;
  if (blocks > 0x7FFFFFFF) return set_error(MX_ERR_SHAPE, "gate_up: tensor too large");
  hipError_t e = hipSuccess;
#define MX_CASE(OUT, FLOOR) \
  if (a.out.h_fmt == OUT && (a.out.scale_mode != 0) == FLOOR) e = launch_kernel(gate_up_kernel<OUT, FLOOR>, dim3((unsigned)blocks), dim3(256), 0, stream, a);
  MX_CASE(MX_BF16, true)
  MX_CASE(MX_BF16, false)
  MX_CASE(MX_E4M3, true)
  MX_CASE(MX_E4M3, false)
  MX_CASE(MX_E5M2, true)
  MX_CASE(MX_E5M2, false)
#undef MX_CASE
  if (e != hipSuccess) return set_error(MX_ERR_LAUNCH, "gate_up_kernel launch: %s", hipGetErrorString(e));
  return MX_OK;
}

int launch_silu_backward(const SiluBackwardArgs& args, hipStream_t stream) {
  SiluBackwardArgs a = args;
  if (a.rows <= 0 || a.F <= 0) return MX_OK;
  a.tiles_k = (a.F + 127) / 128;
  const bool native = a.dts_kind != kScalePlain || a.ats_kind != kScalePlain;
  const int64_t rows = native ? (a.rows + 511ll) / 512 * 512 : a.rows, blocks = (rows + 127) / 128 * a.tiles_k;
  if (blocks > 0x7FFFFFFF) return set_error(MX_ERR_SHAPE, "silu_backward: tensor too large");
  const int64_t lim = (int64_t)1 << 31;
  const bool plain = (((uintptr_t)a.dh | (uintptr_t)(a.dh_ld * 2) | (uintptr_t)a.gu | (uintptr_t)a.gu_ld) & 15) == 0 &&   // (F % 32 == 0)
                     a.dh_ld >= a.F && a.gu_ld >= 2 * a.F && a.gus_ld >= a.F / 16 && 128 * a.dh_ld * 2 < lim && 128 * a.gu_ld < lim && 128 * a.gus_ld < lim && 128 * a.d_ld < lim;
  const dim3 grid((unsigned)blocks);
  const bool once = quantize_loads_once((int64_t)a.rows * a.F);
  hipError_t e = hipSuccess;
#define MX_CASE(FLOOR, PLAIN, ONCE) \
  if ((a.scale_mode != 0) == FLOOR && plain == PLAIN && (plain && once) == ONCE) \
    e = launch_kernel(silu_backward_kernel<FLOOR, PLAIN, ONCE>, grid, dim3(512), 0, stream, a);
  MX_CASE(true, true, true)
  MX_CASE(true, true, false)
  MX_CASE(true, false, false)
  MX_CASE(false, true, true)
  MX_CASE(false, true, false)
  MX_CASE(false, false, false)
#undef MX_CASE
  if (e != hipSuccess) return set_error(MX_ERR_LAUNCH, "silu_backward_kernel launch: %s", hipGetErrorString(e));
  return MX_OK;
}

}  // namespace mx
