// Layer norm: forward, with its result rounded or MX-quantised, and backward with the gradients of weight and bias.
//
//   mean = sum x / H,  rstd = 1 / sqrt(sum (x - mean)^2 / H + eps),  y = (x - mean) rstd w + b
//   h = dy w,  xhat = (x - mean) rstd:  dx = rstd (h - mean(h) - xhat mean(h xhat)),  dw = sum_rows dy xhat,  db = sum_rows dy
//
// Bound: memory.  A row stays in the registers of its threads, a wave's up to 1024 elements, those of two to sixteen waves beyond, so that it is read once
// and the second moment is that of the differences from the mean (of x^2 - mean^2 nothing is left where the mean is large).  Threads
// keep their columns for all of their rows: weight and bias are loaded once, and the gradients of both are summed in
// registers; each workgroup leaves one row of partial sums, which a second launch adds up in their order.
#include <algorithm>
#include <type_traits>

#include "mx_check.h"
#include "mx_gemm_pp.h"   // num_cus
#include "mx_norm.h"
#include "mx_rows.h"

namespace mx {
namespace {

// Sums over the GT threads of a row, in every thread; `slot` alternates between two from one sum to the next (so that one barrier is
// enough: who is two sums ahead has passed the barrier in between).
template <int GT, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float* red, int& slot) {
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = wave_sum(v[k]);
  if constexpr (GT > 64) {
    constexpr int W = GT / 64;
    float* const r = red + slot * N * W;               // [N][waves of the row]
    slot ^= 1;
    const int wave = threadIdx.x % GT >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < N; ++k) r[k * W + wave] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) s += r[k * W + w];
      v[k] = s;
    }
  }
}

// what a row's result becomes.  E4M3 under the floor rule has an instance of its own, by the hardware's conversions alone
// (1531 x 8192, calls one after another on inputs that are in no cache: 13.9 us; by the ceiling rule, with encode_block, 17.2, E5M2 17.7): the
// other formats and the ceiling rule share encode_block.
enum { kNormFloats, kNormE4M3, kNormCodes };

// codes and scale byte of a piece whose block's other elements are in the neighbouring lanes (OUT kNormE4M3: conversions saturate)
template <int T, int OUT>
__device__ __forceinline__ void store_codes(const NormArgs& a, int64_t row, int piece, const float (&v)[kPiece<T>]) {
  constexpr int E = kPiece<T>, LPB = 32 / E;
  uint32_t am = 0, code[E];
  uint8_t byte;
#pragma unroll
  for (int e = 0; e < E; ++e) am = umax(am, magnitude(v[e]));
  am = max_quad(am);
  if constexpr (LPB == 8) am = umax(am, (uint32_t)__builtin_amdgcn_mov_dpp((int)am, 0x141, 0xF, 0xF, true));
  if constexpr (OUT == kNormE4M3) {
    const BlockScale b = block_scale<MX_E4M3, true>(am);
    if (piece * E >= (a.H + 31) / 32 * 32) return;
    uint8_t* const q = (uint8_t*)a.y + row * a.y_ld + piece * E;
    if constexpr (E == 8) *(u2*)q = (u2){encode4<MX_E4M3>(v[0], v[1], v[2], v[3], b.scale), encode4<MX_E4M3>(v[4], v[5], v[6], v[7], b.scale)};
    else *(uint32_t*)q = encode4<MX_E4M3>(v[0], v[1], v[2], v[3], b.scale);
    if (piece % LPB == 0) a.s[row * a.s_ld + piece / LPB] = (uint8_t)b.byte;
    return;
  }
  encode_block<E>(v, am, a.fmt, a.scale_mode, code, byte);
  if (piece * E >= (a.H + 31) / 32 * 32) return;
  uint8_t* const q = (uint8_t*)a.y + row * a.y_ld + (a.fmt == MX_E2M1 ? piece * E / 2 : piece * E);
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (a.fmt == MX_E2M1) w[0] |= code[e] << (4 * e);
    else w[e / 4] |= code[e] << (8 * (e % 4));
  }
  if (a.fmt == MX_E2M1) {
    if constexpr (E == 8) *(uint32_t*)q = w[0];
    else *(uint16_t*)q = (uint16_t)w[0];
  } else if constexpr (E == 8) {
    *(u2*)q = (u2){w[0], w[1]};
  } else {
    *(uint32_t*)q = w[0];
  }
  if (piece % LPB == 0) a.s[row * a.s_ld + piece / LPB] = byte;
}

// GT threads to a row, S * 8 elements to a thread.  16384 x 4096 bf16: 47 us, 5.7 TB/s; 1531 x 8192 to E4M3 12.7 us, of which a launch is 3.
template <int T, int S, int GT, int OUT>
__global__ __launch_bounds__(GT == 64 ? 256 : GT) void norm_kernel(const NormArgs a) {
  constexpr bool CODES = OUT != kNormFloats;
  constexpr int E = kPiece<T>, V = S * 8 / E, WG = GT == 64 ? 256 : GT, GPW = WG / GT;
  __shared__ float red[GT > 64 ? 2 * GT / 64 : 1];
  const int t = threadIdx.x % GT, H = a.H;
  const float count = (float)H;
  int slot = 0;
  if constexpr (OUT == kNormE4M3) saturate_conversions();
  float w[V][E], b[V][E];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int at = (t + i * GT) * E;
    load_floats<E>(a.w, a.w_dtype, at, H - at, 1.f, w[i]);
    load_floats<E>(a.b, a.b_dtype, at, H - at, 0.f, b[i]);
  }
  auto load = [&](int64_t row, u4 (&raw)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int at = (t + i * GT) * E;
      raw[i] = load_piece<T>((const uint8_t*)a.x + row * a.x_ld * kSize<T>, at, row < a.rows ? H - at : 0);
    }
  };
  u4 raw[V];
  const int64_t step = (int64_t)gridDim.x * GPW;
  int64_t row = (int64_t)blockIdx.x * GPW + threadIdx.x / GT;
  load(row, raw);
  for (; row < a.rows; row += step) {                  // (a row of more than one wave has the workgroup to itself: uniform)
    float v[V][E], sum[1] = {0.f};
#pragma unroll
    for (int i = 0; i < V; ++i) {
      unpack_piece<T>(raw[i], v[i]);
#pragma unroll
      for (int e = 0; e < E; ++e) sum[0] += v[i][e];
    }
    load(row + step, raw);
    row_sums<GT>(sum, red, slot);
    const float mean = sum[0] / count;
    sum[0] = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int n = H - (t + i * GT) * E;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        v[i][e] = e < n ? v[i][e] - mean : 0.f;
        sum[0] = __builtin_fmaf(v[i][e], v[i][e], sum[0]);
      }
    }
    row_sums<GT>(sum, red, slot);
    const float rstd = 1.0f / __builtin_sqrtf(sum[0] / count + a.eps);
    if (t == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int at = (t + i * GT) * E;
#pragma unroll
      for (int e = 0; e < E; ++e) v[i][e] = !CODES || at + e < H ? __builtin_fmaf(v[i][e] * rstd, w[i][e], b[i][e]) : 0.f;
      if constexpr (CODES) store_codes<T, OUT>(a, row, t + i * GT, v[i]);
      else store_piece<T>((uint8_t*)a.y + row * a.y_ld * kSize<T>, at, H - at, pack_piece<T>(v[i]));
    }
  }
}

// rows that do not fit into a workgroup's registers: read three times, from L2 after the first (1024 x 32768 bf16 43 us; with 32 elements to a
// thread, which spill, 49)
constexpr int kLongThreads = 1024;
template <int T, int OUT>
__global__ __launch_bounds__(kLongThreads) void norm_long_kernel(const NormArgs a) {
  constexpr bool CODES = OUT != kNormFloats;
  constexpr int E = kPiece<T>;
  __shared__ float red[2 * kLongThreads / 64];
  const int H = a.H, pieces = ((H + 31) / 32 * 32) / E;
  const float count = (float)H;
  int slot = 0;
  if constexpr (OUT == kNormE4M3) saturate_conversions();
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const uint8_t* const x = (const uint8_t*)a.x + row * a.x_ld * kSize<T>;
    float sum[1] = {0.f}, v[E];
    for (int p = threadIdx.x; p * E < H; p += kLongThreads) {
      unpack_piece<T>(load_piece<T>(x, (int64_t)p * E, H - p * E), v);
#pragma unroll
      for (int e = 0; e < E; ++e) sum[0] += v[e];
    }
    row_sums<kLongThreads>(sum, red, slot);
    const float mean = sum[0] / count;
    sum[0] = 0.f;
    for (int p = threadIdx.x; p * E < H; p += kLongThreads) {
      unpack_piece<T>(load_piece<T>(x, (int64_t)p * E, H - p * E), v);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float d = p * E + e < H ? v[e] - mean : 0.f;
        sum[0] = __builtin_fmaf(d, d, sum[0]);
      }
    }
    row_sums<kLongThreads>(sum, red, slot);
    const float rstd = 1.0f / __builtin_sqrtf(sum[0] / count + a.eps);
    if (threadIdx.x == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
    // (whole waves stay together: the lanes of a block exchange its maximum)
    for (int p0 = 0; p0 < pieces; p0 += kLongThreads) {
      const int p = p0 + threadIdx.x, n = H - p * E;
      float w[E], b[E];
      unpack_piece<T>(load_piece<T>(x, (int64_t)p * E, n), v);
      load_floats<E>(a.w, a.w_dtype, (int64_t)p * E, n, 1.f, w);
      load_floats<E>(a.b, a.b_dtype, (int64_t)p * E, n, 0.f, b);
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = e < n ? __builtin_fmaf((v[e] - mean) * rstd, w[e], b[e]) : 0.f;
      if constexpr (CODES) store_codes<T, OUT>(a, row, p, v);
      else store_piece<T>((uint8_t*)a.y + row * a.y_ld * kSize<T>, (int64_t)p * E, n, pack_piece<T>(v));
    }
  }
}

// ================================================================================================================================
// Backward
// ================================================================================================================================
constexpr int kBackThreads = 512;

// 16384 x 4096 bf16: 87 us, 4.6 TB/s
template <int T, int S, int GT>
__global__ __launch_bounds__(kBackThreads) void norm_backward_kernel(const NormBackwardArgs a) {
  constexpr int E = kPiece<T>, V = S * 8 / E, GPW = kBackThreads / GT, W = GT / 64;
  __shared__ float red[GPW * 2 * 2 * W];
  __shared__ float part[GPW > 1 ? GPW * GT * E : 1];
  const int t = threadIdx.x % GT, g = threadIdx.x / GT, H = a.H;
  const float count = (float)H;
  int slot = 0;
  float w[V][E], dw[V][E] = {}, db[V][E] = {};
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int at = (t + i * GT) * E;
    load_floats<E>(a.w, a.w_dtype, at, H - at, 1.f, w[i]);
  }
  u4 rx[V], rd[V];
  float mean = 0.f, rstd = 0.f;
  auto load = [&](int64_t row) {
    const bool live = row < a.rows;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int at = (t + i * GT) * E;
      rx[i] = load_piece<T>((const uint8_t*)a.x + row * a.x_ld * kSize<T>, at, live ? H - at : 0);
      rd[i] = load_piece<T>((const uint8_t*)a.dy + row * a.dy_ld * kSize<T>, at, live ? H - at : 0);
    }
    mean = live ? a.mean[row] : 0.f;
    rstd = live ? a.rstd[row] : 0.f;
  };
  const int64_t step = (int64_t)gridDim.x * GPW;
  int64_t row0 = (int64_t)blockIdx.x * GPW;
  load(row0 + g);
  for (; row0 < a.rows; row0 += step) {                // uniform: rows beyond the last are zeros
    const int64_t row = row0 + g;
    float h[V][E], xh[V][E], sum[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int n = H - (t + i * GT) * E;
      float d[E];
      unpack_piece<T>(rx[i], xh[i]);
      unpack_piece<T>(rd[i], d);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        xh[i][e] = e < n ? (xh[i][e] - mean) * rstd : 0.f;   // (the mean of a row far from zero times rstd may be infinite)
        db[i][e] += d[e];
        dw[i][e] = __builtin_fmaf(d[e], xh[i][e], dw[i][e]);
        h[i][e] = d[e] * w[i][e];
        sum[0] += h[i][e];
        sum[1] = __builtin_fmaf(h[i][e], xh[i][e], sum[1]);
      }
    }
    const float r = rstd;
    load(row + step);
    row_sums<GT>(sum, red + g * 4 * W, slot);
    if (a.dx && row < a.rows) {
      const float c0 = sum[0] / count, c1 = sum[1] / count;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int at = (t + i * GT) * E;
#pragma unroll
        for (int e = 0; e < E; ++e) h[i][e] = r * (h[i][e] - c0 - xh[i][e] * c1);
        store_piece<T>((uint8_t*)a.dx + row * a.dx_ld * kSize<T>, at, H - at, pack_piece<T>(h[i]));
      }
    }
  }
  if (!a.dw && !a.db) return;
  // the workgroup's rows, group by group
  auto out = [&](int which, float (&v)[V][E]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (GPW > 1) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e) part[(g * E + e) * GT + t] = v[i][e];
        __syncthreads();
        if (g == 0) {
#pragma unroll
          for (int k = 1; k < GPW; ++k)
#pragma unroll
            for (int e = 0; e < E; ++e) v[i][e] += part[(k * E + e) * GT + t];
        }
      }
      const int at = (t + i * GT) * E;
      if (g == 0) store_piece<MX_F32>(a.partial + ((int64_t)blockIdx.x * 2 + which) * H, at, H - at, (u4){__builtin_bit_cast(uint32_t, v[i][0]), __builtin_bit_cast(uint32_t, v[i][1]),
                  __builtin_bit_cast(uint32_t, v[i][2]), __builtin_bit_cast(uint32_t, v[i][3])});
      if constexpr (E == 8)
        if (g == 0) store_piece<MX_F32>(a.partial + ((int64_t)blockIdx.x * 2 + which) * H, at + 4, H - at - 4, (u4){__builtin_bit_cast(uint32_t, v[i][4]),
                    __builtin_bit_cast(uint32_t, v[i][5]), __builtin_bit_cast(uint32_t, v[i][6]), __builtin_bit_cast(uint32_t, v[i][7])});
    }
  };
  if (a.dw) out(0, dw);
  if (a.db) out(1, db);
}

// long rows: dx row by row (x and dy read twice) ...
template <int T>
__global__ __launch_bounds__(kLongThreads) void norm_backward_long_kernel(const NormBackwardArgs a) {
  constexpr int E = kPiece<T>;
  __shared__ float red[2 * 2 * kLongThreads / 64];
  const int H = a.H;
  const float count = (float)H;
  int slot = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const uint8_t *const x = (const uint8_t*)a.x + row * a.x_ld * kSize<T>, *const dy = (const uint8_t*)a.dy + row * a.dy_ld * kSize<T>;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float sum[2] = {0.f, 0.f}, xh[E], h[E], w[E];
    auto piece = [&](int p) {
      const int n = H - p * E;
      unpack_piece<T>(load_piece<T>(x, (int64_t)p * E, n), xh);
      unpack_piece<T>(load_piece<T>(dy, (int64_t)p * E, n), h);
      load_floats<E>(a.w, a.w_dtype, (int64_t)p * E, n, 1.f, w);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        xh[e] = e < n ? (xh[e] - mean) * rstd : 0.f;   // (as above)
        h[e] *= w[e];
      }
    };
    for (int p = threadIdx.x; p * E < H; p += kLongThreads) {
      piece(p);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        sum[0] += h[e];
        sum[1] = __builtin_fmaf(h[e], xh[e], sum[1]);
      }
    }
    row_sums<kLongThreads>(sum, red, slot);
    const float c0 = sum[0] / count, c1 = sum[1] / count;
    for (int p = threadIdx.x; p * E < H; p += kLongThreads) {
      piece(p);
#pragma unroll
      for (int e = 0; e < E; ++e) h[e] = rstd * (h[e] - c0 - xh[e] * c1);
      store_piece<T>((uint8_t*)a.dx + row * a.dx_ld * kSize<T>, (int64_t)p * E, H - p * E, pack_piece<T>(h));
    }
  }
}
// ... and the columns' sums: a thread keeps its columns for its workgroup's rows
template <int T>
__global__ __launch_bounds__(256) void norm_columns_kernel(const NormBackwardArgs a) {
  constexpr int E = kPiece<T>;
  const int H = a.H, at = ((int)blockIdx.x * 256 + threadIdx.x) * E, n = H - at;
  if (n <= 0) return;
  float dw[E] = {}, db[E] = {};
#pragma unroll 4
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float mean = a.mean[row], rstd = a.rstd[row];
    float x[E], d[E];
    unpack_piece<T>(load_piece<T>((const uint8_t*)a.x + row * a.x_ld * kSize<T>, at, n), x);
    unpack_piece<T>(load_piece<T>((const uint8_t*)a.dy + row * a.dy_ld * kSize<T>, at, n), d);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      db[e] += d[e];
      dw[e] = __builtin_fmaf(d[e], (x[e] - mean) * rstd, dw[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (e >= n) continue;
    float* const p = a.partial + (int64_t)blockIdx.y * 2 * H + at + e;
    p[0] = dw[e];
    p[H] = db[e];
  }
}

// Partial sums [parts][2][H] -> dw, db.  A workgroup takes 64 columns of one of them, its waves every 16th part.
__global__ __launch_bounds__(1024) void norm_reduce_kernel(const NormBackwardArgs a, const int parts) {
  __shared__ float red[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, which = blockIdx.y;
  const int64_t col = (int64_t)blockIdx.x * 64 + lane;
  void* const out = which ? a.db : a.dw;
  if (!out) return;
  float s = 0.f;
  if (col < a.H)
    for (int p = wave; p < parts; p += 16) s += a.partial[((int64_t)p * 2 + which) * a.H + col];
  red[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || col >= a.H) return;
#pragma unroll
  for (int k = 1; k < 16; ++k) s += red[k][lane];
  store_float(out, which ? a.db_dtype : a.dw_dtype, col, s);
}

// S and the threads of a row by its length: 16 elements to a thread.  (With 32, fewer threads and fewer barriers, or 8 up to 8192, full occupancy:
// 1531 x 8192 to E4M3 13.9 us, 16.2 and 14.2; fp32 8192 x 2048 25.5, 30.0 and 23.9; bf16 16384 x 4096 46.0, 47.7 and 47.4; inputs that are in no cache.)
template <typename F>
bool by_length(int64_t H, F&& f) {
#define MX_CASE(MOST, S, GT) \
  if (H <= MOST) { f(std::integral_constant<int, S>{}, std::integral_constant<int, GT>{}); return true; }
  MX_CASE(512, 1, 64)
  MX_CASE(1024, 2, 64)
  MX_CASE(2048, 2, 128)
  MX_CASE(4096, 2, 256)
  MX_CASE(8192, 2, 512)
  MX_CASE(16384, 2, 1024)
#undef MX_CASE
  return false;
}

template <int T, int OUT>
hipError_t run_norm(const NormArgs& a, hipStream_t stream) {
  hipError_t e = hipSuccess;
  const int64_t cus = num_cus();
  const bool held = by_length((a.H + 31ll) / 32 * 32, [&](auto s, auto gt) {
    constexpr int S = decltype(s)::value, GT = decltype(gt)::value, WG = GT == 64 ? 256 : GT, GPW = WG / GT;
    const auto kern = norm_kernel<T, S, GT, OUT>;
    static int held = 0;                               // workgroups that a CU holds at once (benign race: always the same)
    if (!held && (hipOccupancyMaxActiveBlocksPerMultiprocessor(&held, kern, WG, 0) != hipSuccess || held < 1)) held = 1;
    // as many rows to every workgroup: 1531 rows of 8192 in 511 workgroups of three instead of 1024 of one or two
    const int64_t groups = (a.rows + GPW - 1) / GPW, rounds = (groups + cus * held - 1) / (cus * held);
    e = launch_kernel(kern, dim3((unsigned)((groups + rounds - 1) / rounds)), dim3(WG), 0, stream, a);
  });
  if (!held) e = launch_kernel(norm_long_kernel<T, OUT>, dim3((unsigned)std::min<int64_t>(a.rows, 2 * cus)), dim3(kLongThreads), 0, stream, a);
  return e;
}

// Longest row of norm_backward_kernel.  (fp32 rows beyond 8192 do not fit into registers: 2048 x 16384 took 170 us so.)
template <int T> constexpr int64_t kBackHeld = T == MX_F32 ? 8192 : 16384;
int64_t back_parts(int64_t rows, int64_t H) {
  const int64_t per = H <= 1024 ? 8 : H <= 2048 ? 4 : H <= 4096 ? 2 : 1;
  return std::min<int64_t>((rows + per - 1) / per, num_cus());
}
// partial sums of norm_columns_kernel: a thousand workgroups or two, eight rows at least to each
int64_t column_parts(int64_t rows, int64_t H) { return std::min<int64_t>({back_parts(rows, H), (rows + 7) / 8, std::max<int64_t>(((int64_t)2 << 20) / H, 1)}); }
template <int T>
hipError_t run_backward(const NormBackwardArgs& a, hipStream_t stream) {
  const int64_t parts = a.H <= kBackHeld<T> ? back_parts(a.rows, a.H) : column_parts(a.rows, a.H);
  hipError_t e = hipSuccess;
  auto held = [&](auto s, auto gt) {
    constexpr int S = decltype(s)::value, GT = decltype(gt)::value;
    e = launch_kernel(norm_backward_kernel<T, S, GT>, dim3((unsigned)parts), dim3(kBackThreads), 0, stream, a);
  };
  using std::integral_constant;
  if (a.H <= 512) held(integral_constant<int, 1>{}, integral_constant<int, 64>{});
  else if (a.H <= 1024) held(integral_constant<int, 2>{}, integral_constant<int, 64>{});
  else if (a.H <= 2048) held(integral_constant<int, 2>{}, integral_constant<int, 128>{});
  else if (a.H <= 4096) held(integral_constant<int, 2>{}, integral_constant<int, 256>{});
  else if (a.H <= 8192) held(integral_constant<int, 2>{}, integral_constant<int, 512>{});
  else if (a.H <= kBackHeld<T>) {
    if constexpr (T != MX_F32) held(integral_constant<int, 4>{}, integral_constant<int, 512>{});
  } else {
    if (a.dx) e = launch_kernel(norm_backward_long_kernel<T>, dim3((unsigned)std::min<int64_t>(a.rows, 2 * num_cus())), dim3(kLongThreads), 0, stream, a);
    if (e == hipSuccess && (a.dw || a.db)) {
      const int64_t per = 256 * kPiece<T>;
      e = launch_kernel(norm_columns_kernel<T>, dim3((unsigned)((a.H + per - 1) / per), (unsigned)parts), dim3(256), 0, stream, a);
    }
  }
  if (e == hipSuccess && (a.dw || a.db)) e = launch_kernel(norm_reduce_kernel, dim3((unsigned)((a.H + 63) / 64), 2), dim3(1024), 0, stream, a, (int)parts);
  return e;
}

}  // namespace

int launch_layer_norm(const NormArgs& a, hipStream_t stream) {
  if (a.rows <= 0) return MX_OK;
  const bool e4m3 = a.fmt == MX_E4M3 && a.scale_mode != 0;
  hipError_t e = hipSuccess;
#define MX_CASE(T) \
  if (a.x_dtype == T) e = a.fmt < 0 ? run_norm<T, kNormFloats>(a, stream) : e4m3 ? run_norm<T, kNormE4M3>(a, stream) : run_norm<T, kNormCodes>(a, stream);
  MX_CASE(MX_F32)
  MX_CASE(MX_BF16)
  MX_CASE(MX_F16)
#undef MX_CASE
  if (e != hipSuccess) return set_error(MX_ERR_LAUNCH, "norm_kernel launch: %s", hipGetErrorString(e));
  return MX_OK;
}

int64_t norm_backward_bytes(int64_t rows, int64_t H) { return rows <= 0 || H <= 0 ? 0 : round256(back_parts(rows, H) * 2 * H * 4); }

int launch_layer_norm_backward(const NormBackwardArgs& a, hipStream_t stream) {
  if (a.rows <= 0) return MX_OK;
  hipError_t e = hipSuccess;
#define MX_CASE(T) \
  if (a.x_dtype == T) e = run_backward<T>(a, stream);
  MX_CASE(MX_F32)
  MX_CASE(MX_BF16)
  MX_CASE(MX_F16)
#undef MX_CASE
  if (e != hipSuccess) return set_error(MX_ERR_LAUNCH, "norm_backward_kernel launch: %s", hipGetErrorString(e));
  return MX_OK;
}

}  // namespace mx

using namespace mx;

namespace {
// x [rows, H] and its parameters
int check_norm(const mx_tensor* x, const mx_tensor* weight, const mx_tensor* bias) {
  if (int rc = check2d(x, "x", -1, -1)) return rc;
  if (int rc = check_dtype(x, "x", is_float(x->dtype), "MX_F32, MX_BF16 or MX_F16")) return rc;
  if (x->shape[1] < 1) return set_error(MX_ERR_SHAPE, "x must have at least one column");
  if (weight)
    if (int rc = check_vector(weight, "weight", x->shape[1])) return rc;
  if (bias)
    if (int rc = check_vector(bias, "bias", x->shape[1])) return rc;
  return MX_OK;
}
int check_stats(const mx_tensor* t, const char* name, int64_t rows) {
  if (int rc = check_vector(t, name, rows)) return rc;
  return t->dtype == MX_F32 ? MX_OK : set_error(MX_ERR_DTYPE, "%s must be MX_F32 (got %d)", name, t->dtype);
}
int check_result(const mx_tensor* t, const char* name, const mx_tensor* x) {
  if (int rc = check2d(t, name, x->shape[0], x->shape[1])) return rc;
  if (t->dtype != x->dtype) return set_error(MX_ERR_DTYPE, "%s must have the type of x", name);
  if (t->shape[0] > 1 && t->stride[0] < t->shape[1]) return set_error(MX_ERR_LAYOUT, "%s: rows overlap", name);
  return MX_OK;
}
NormArgs norm_args(const mx_tensor* x, const mx_tensor* weight, const mx_tensor* bias, double eps) {
  NormArgs a = {};
  a.x = x->ptr; a.x_ld = x->stride[0]; a.x_dtype = x->dtype;
  a.rows = (int32_t)x->shape[0]; a.H = (int32_t)x->shape[1];
  if (weight) { a.w = weight->ptr; a.w_dtype = weight->dtype; }
  if (bias) { a.b = bias->ptr; a.b_dtype = bias->dtype; }
  a.eps = (float)eps;
  a.fmt = -1;
  return a;
}
int check_eps(double eps) {
  return eps >= 0.0 && eps <= 3.4e38 ? MX_OK : set_error(MX_ERR_INVALID, "eps must be a number of at least zero");
}
}  // namespace

extern "C" {

int mx_layer_norm(const mx_tensor* x, const mx_tensor* weight, const mx_tensor* bias, double eps, mx_tensor* y, mx_tensor* mean, mx_tensor* rstd,
                  void* stream) {
  if (int rc = check_norm(x, weight, bias)) return rc;
  if (int rc = check_eps(eps)) return rc;
  if (int rc = check_result(y, "y", x)) return rc;
  NormArgs a = norm_args(x, weight, bias, eps);
  if (mean) {
    if (int rc = check_stats(mean, "mean", x->shape[0])) return rc;
    a.mean = (float*)mean->ptr;
  }
  if (rstd) {
    if (int rc = check_stats(rstd, "rstd", x->shape[0])) return rc;
    a.rstd = (float*)rstd->ptr;
  }
  a.y = y->ptr; a.y_ld = y->stride[0];
  return launch_layer_norm(a, (hipStream_t)stream);
}

int mx_layer_norm_quantize(const mx_tensor* x, const mx_tensor* weight, const mx_tensor* bias, double eps, mx_tensor* xq, mx_tensor* scale,
                           int32_t scale_mode, void* stream) {
  if (int rc = check_norm(x, weight, bias)) return rc;
  if (int rc = check_eps(eps)) return rc;
  const int64_t rows = x->shape[0], H = x->shape[1], Hp = round32(H);
  if (H < 32)
    return set_error(MX_ERR_SHAPE, "The requested block size 32 is larger than the inner most dimension of the input tensor %lld", (long long)H);
  if (!xq) return set_error(MX_ERR_INVALID, "xq: null descriptor");
  if (xq->dtype != MX_E4M3 && xq->dtype != MX_E5M2 && xq->dtype != MX_E2M1) return set_error(MX_ERR_DTYPE, "xq must be an MX element format (got %d)", xq->dtype);
  mx_tensor q = *xq;
  if (q.dtype == MX_E2M1) {
    if (q.ndim != 2 || q.packed_dim != 1) return set_error(MX_ERR_LAYOUT, "xq must be packed along H");
    if (q.shape[1] != Hp) return set_error(MX_ERR_SHAPE, "xq must be [%lld, %lld]", (long long)rows, (long long)Hp);
    q.shape[1] = Hp / 2;
  }
  if (int rc = check_codes(&q, "xq", rows, q.dtype == MX_E2M1 ? Hp / 2 : Hp, q.dtype == MX_E2M1 ? 4 : 8)) return rc;
  if (int rc = check_scales(scale, "scale", rows, Hp / 32)) return rc;
  if (int rc = check_mode(scale_mode)) return rc;
  NormArgs a = norm_args(x, weight, bias, eps);
  a.y = q.ptr; a.y_ld = q.stride[0]; a.fmt = q.dtype; a.scale_mode = scale_mode;
  a.s = (uint8_t*)scale->ptr; a.s_ld = scale->stride[0];
  return launch_layer_norm(a, (hipStream_t)stream);
}

int64_t mx_layer_norm_backward_workspace_bytes(int64_t rows, int64_t H) { return norm_backward_bytes(rows, H); }

int mx_layer_norm_backward(const mx_tensor* dy, const mx_tensor* x, const mx_tensor* mean, const mx_tensor* rstd, const mx_tensor* weight, mx_tensor* dx,
                           mx_tensor* dweight, mx_tensor* dbias, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check_norm(x, weight, nullptr)) return rc;
  const int64_t rows = x->shape[0], H = x->shape[1];
  if (int rc = check2d(dy, "dy", rows, H)) return rc;
  if (dy->dtype != x->dtype) return set_error(MX_ERR_DTYPE, "dy must have the type of x");
  if (!mean || !rstd) return set_error(MX_ERR_INVALID, "mean and rstd of the forward pass are needed");
  if (int rc = check_stats(mean, "mean", rows)) return rc;
  if (int rc = check_stats(rstd, "rstd", rows)) return rc;
  NormBackwardArgs a = {};
  if (dx) {
    if (int rc = check_result(dx, "dx", x)) return rc;
    a.dx = dx->ptr; a.dx_ld = dx->stride[0];
  }
  if (dweight) {
    if (int rc = check_vector(dweight, "dweight", H)) return rc;
    a.dw = dweight->ptr; a.dw_dtype = dweight->dtype;
  }
  if (dbias) {
    if (int rc = check_vector(dbias, "dbias", H)) return rc;
    a.db = dbias->ptr; a.db_dtype = dbias->dtype;
  }
  if (rows == 0 && (dweight || dbias)) return set_error(MX_ERR_SHAPE, "mx_layer_norm_backward: no rows (the gradients of weight and bias are zeros)");
  if (dweight || dbias)
    if (int rc = check_room("workspace", workspace, workspace_bytes, norm_backward_bytes(rows, H))) return rc;
  a.dy = dy->ptr; a.dy_ld = dy->stride[0];
  a.x = x->ptr; a.x_ld = x->stride[0]; a.x_dtype = x->dtype;
  a.mean = (const float*)mean->ptr; a.rstd = (const float*)rstd->ptr;
  if (weight) { a.w = weight->ptr; a.w_dtype = weight->dtype; }
  a.partial = (float*)workspace;
  a.rows = (int32_t)rows; a.H = (int32_t)H;
  if (!dx && !dweight && !dbias) return MX_OK;
  return launch_layer_norm_backward(a, (hipStream_t)stream);
}

}  // extern "C"
