// AdamW over many tensors at once, states in 32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,  p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Bound: memory, 28 bytes an element (fp32 parameters, gradients and states) down to 10.1 (bf16, 8-bit states); 117 M elements of 16.1
// bytes (fp32 parameters with bf16 copies and gradients, 8-bit states) 370 us, 5.1 TB/s.  A workgroup takes
// kChunk elements of one tensor; which tensor, it finds in a table in the kernel's arguments, so that nothing is copied to the
// device and a launch serves kTensors of them.
//
// 8-bit states are the library's MXFP8: E4M3 elements, one power of two for 32 of them, the least that keeps the largest within 448.  (Not
// the floor rule, which ends between 448 and 512: a state that grows by a part in a thousand a step would stay there for good.)  Of v the
// root is kept, which has half as many octaves.  With b2 = 0.999 a step changes a root by far less than the 2^-3 between E4M3 numbers: rounded to
// nearest it would never move.  Both states are rounded up or down at random instead, up with the chance that the value's place between
// its neighbours gives (16 bits of it), so that their means are right.  The random bits are a hash of seed, step, tensor and
// element: two multiplications between shifted exclusive ors, enough for a rounding, and the same on every call with the same
// arguments.  A root above zero is stored as the least number of its block at least: a state of zero beside a first moment that is not
// would make a step of m / eps.
#include <algorithm>
#include <cmath>
#include <utility>
#include <vector>

#include "mx_check.h"
#include "mx_rows.h"

namespace mx {
namespace {

constexpr int kTensors = 54, kThreads = 256, kChunk = 4096;
struct AdamTensor {
  void* p;
  const void* g;
  void *m, *v;
  uint8_t *ms, *vs;
  uint16_t* copy;
  int64_t n;
};
struct AdamArgs {
  AdamTensor t[kTensors];
  int32_t first[kTensors];           // chunk
  int32_t index[kTensors];           // place in the caller's list
  int32_t count;
  uint32_t seed;
  float b1, c1, b2, c2, eps;         // c1 = 1 - b1, c2 = 1 - b2
  float keep, rate, root;            // 1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  float scale;                       // of the gradients
  // where lr, the step or the gradients' scale are on the device: the host's values are not used, `keep`, `rate` and `root` are made here
  float lr, decay, log_b1, log_b2;
  int64_t step;
  const float *lr_at, *scale_at;
  const int64_t* step_at;
};
static_assert(sizeof(AdamArgs) <= 4096, "kernel arguments");

__host__ __device__ __forceinline__ uint32_t mix(uint32_t x) {
  x ^= x >> 16;
  x *= 0x9E3779B1u;   // 2^32 over the golden ratio, the nearest prime (Knuth's multiplicative hashing)
  x ^= x >> 15;
  x *= 0xBB67AE85u;   // the fraction of sqrt(3)
  return x ^ x >> 16;
}

// |x| of a block's element over its scale, 448 at most, to an E4M3 number: up with the chance of bits / 2^16
__device__ __forceinline__ float round_e4m3(float x, uint32_t bits) {
  const float a = __builtin_fabsf(x), tiny = a < 0x1p-6f ? 0x1p-6f : 0.f;   // (the grid below 2^-6 is that of 2^-6 .. 2^-5)
  const uint32_t u = (__builtin_bit_cast(uint32_t, a + tiny) + (bits << 4)) & 0xFFF00000u;
  const float r = fminf(__builtin_bit_cast(float, u), 448.f) - tiny;
  return __builtin_copysignf(a != a ? a : r, x);
}
// eight elements of a state (32 in four lanes) as codes; returns the block's scale byte
template <bool ROOT>
__device__ __forceinline__ uint32_t store_state(const float (&v)[8], const uint32_t (&bits)[8], u2& code) {
  uint32_t am = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) am = umax(am, magnitude(v[e]));
  // 2^(floor(log2 amax) - 8), twice that beyond 1.75 of a power of two.  248 at most: the inverse is a normal number
  const uint32_t byte = __builtin_elementwise_sub_sat((max_quad(am) + 0x1FFFFFu) >> 23, 8u);
  const float inv = __builtin_bit_cast(float, (254u - byte) << 23);
  float q[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    q[e] = round_e4m3(v[e] * inv, bits[e]);
    if (ROOT && v[e] > 0.f) q[e] = fmaxf(q[e], 0x1p-9f);
  }
  code = (u2){encode4<MX_E4M3>(q[0], q[1], q[2], q[3], 1.0f), encode4<MX_E4M3>(q[4], q[5], q[6], q[7], 1.0f)};
  return byte;
}
__device__ __forceinline__ void load_state(u2 c, uint32_t byte, float (&v)[8]) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  const float scale = __builtin_bit_cast(float, byte << 23);
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    const f2 p = (h & 1) ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c[h >> 1], scale, true) : __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c[h >> 1], scale, false);
    v[2 * h] = p[0];
    v[2 * h + 1] = p[1];
  }
}
template <int T>
__device__ __forceinline__ void load8(const void* p, int64_t at, int n, float (&v)[8]) {
  if constexpr (T == MX_F32) {
    float a[4], b[4];
    unpack_piece<MX_F32>(load_piece<MX_F32>(p, at, n), a);
    unpack_piece<MX_F32>(load_piece<MX_F32>(p, at + 4, n - 4), b);
#pragma unroll
    for (int e = 0; e < 4; ++e) { v[e] = a[e]; v[4 + e] = b[e]; }
  } else {
    unpack_piece<T>(load_piece<T>(p, at, n), v);
  }
}
template <int T>
__device__ __forceinline__ void store8(void* p, int64_t at, int n, const float (&v)[8]) {
  if constexpr (T == MX_F32) {
    store_piece<MX_F32>(p, at, n, pack_piece<MX_F32>({v[0], v[1], v[2], v[3]}));
    store_piece<MX_F32>(p, at + 4, n - 4, pack_piece<MX_F32>({v[4], v[5], v[6], v[7]}));
  } else {
    store_piece<T>(p, at, n, pack_piece<T>(v));
  }
}

template <int P, int G, bool SMALL>
__global__ __launch_bounds__(kThreads) void adamw_kernel(const AdamArgs a) {
  const int lane = threadIdx.x & 63;
  const uint64_t upto = __builtin_amdgcn_ballot_w64(lane < a.count && a.first[lane < kTensors ? lane : 0] <= (int)blockIdx.x);
  const int which = 63 - __builtin_clzll(upto);        // (the first tensor's first chunk is 0)
  const AdamTensor& t = a.t[which];
  const int64_t chunk = (int64_t)((int)blockIdx.x - a.first[which]) * kChunk, n = t.n;
  float keep = a.keep, rate = a.rate, root = a.root, gs = a.scale;
  if (a.lr_at || a.step_at) {
    const float lr = a.lr_at ? *a.lr_at : a.lr, step = (float)(a.step_at ? *a.step_at : a.step);
    keep = 1.f - lr * a.decay;
    rate = lr / -expm1f(step * a.log_b1);
    root = 1.f / __builtin_sqrtf(-expm1f(step * a.log_b2));
  }
  if (a.scale_at) gs = *a.scale_at;
  uint32_t key = 0;
  if constexpr (SMALL) {
    key = mix(mix(a.seed) ^ (uint32_t)(a.step_at ? *a.step_at : a.step)) ^ (uint32_t)a.index[which];
    key = mix(mix(key) ^ (uint32_t)(chunk >> 32));
  }
#pragma unroll
  for (int i = 0; i < kChunk / (8 * kThreads); ++i) {
    const int64_t at = chunk + (i * kThreads + threadIdx.x) * 8;
    const int left = n - at < 8 ? (int)(n - at) : 8;   // (zero or less: beyond the end)
    const int64_t block = at >> 5;
    const bool there = block * 32 < n;                 // the lane's block has elements
    float p[8], g[8], m[8], v[8];
    load8<P>(t.p, at, left, p);
    load8<G>(t.g, at, left, g);
    if constexpr (SMALL) {
      u2 cm = {0, 0}, cv = {0, 0};
      uint32_t bm = 0, bv = 0;
      if (there) {
        cm = *(const u2*)((const uint8_t*)t.m + at);
        cv = *(const u2*)((const uint8_t*)t.v + at);
        bm = t.ms[block];
        bv = t.vs[block];
      }
      load_state(cm, bm, m);
      load_state(cv, bv, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        m[e] = e < left ? m[e] : 0.f;
        v[e] = e < left ? v[e] * v[e] : 0.f;
      }
    } else {
      load8<MX_F32>(t.m, at, left, m);
      load8<MX_F32>(t.v, at, left, v);
    }
    float r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = g[e] * gs;
      {
        // (rounded one by one, like the formula in separate operations: what lies on the border of two codes is then on the same side)
#pragma clang fp contract(off)
        m[e] = a.b1 * m[e] + a.c1 * x;
        v[e] = a.b2 * v[e] + a.c2 * x * x;
      }
      r[e] = __builtin_sqrtf(v[e]);
      p[e] = __builtin_fmaf(p[e], keep, -(rate * m[e] / __builtin_fmaf(r[e], root, a.eps)));
    }
    store8<P>(t.p, at, left, p);
    if (t.copy) store8<MX_BF16>(t.copy, at, left, p);
    if constexpr (SMALL) {
      uint32_t lo[8], hi[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t w = mix(key + (uint32_t)(at + e));
        lo[e] = w & 0xFFFF;
        hi[e] = w >> 16;
      }
      u2 cm, cv;
      const uint32_t bm = store_state<false>(m, lo, cm), bv = store_state<true>(r, hi, cv);
      if (there) {
        *(u2*)((uint8_t*)t.m + at) = cm;
        *(u2*)((uint8_t*)t.v + at) = cv;
        if ((lane & 3) == 0) {
          t.ms[block] = (uint8_t)bm;
          t.vs[block] = (uint8_t)bv;
        }
      }
    } else {
      store8<MX_F32>(t.m, at, left, m);
      store8<MX_F32>(t.v, at, left, v);
    }
  }
}

template <int P, int G>
hipError_t launch(const AdamArgs& a, int64_t chunks, bool small, hipStream_t stream) {
  return small ? launch_kernel(adamw_kernel<P, G, true>, dim3((unsigned)chunks), dim3(kThreads), 0, stream, a)
               : launch_kernel(adamw_kernel<P, G, false>, dim3((unsigned)chunks), dim3(kThreads), 0, stream, a);
}

typedef std::vector<std::pair<uintptr_t, uintptr_t>> Ranges;
// Of the ranges in the lists, two with one another (1), or one with one of `read` (2), which may overlap among themselves.  (The lists are sorted and
// joined.)
int overlap(Ranges (&lists)[6], Ranges& read) {
  for (Ranges& l : lists)
    if (!std::is_sorted(l.begin(), l.end())) std::sort(l.begin(), l.end());
  std::sort(lists, lists + 6);   // by their first range, empty ones in front
  Ranges all;
  size_t total = 0;
  for (const Ranges& l : lists) total += l.size();
  all.reserve(total);
  for (const Ranges& l : lists) {
    const size_t mid = all.size();
    all.insert(all.end(), l.begin(), l.end());
    if (mid > 0 && mid < all.size() && all[mid] < all[mid - 1]) std::inplace_merge(all.begin(), all.begin() + mid, all.end());
  }
  for (size_t i = 1; i < all.size(); ++i)
    if (all[i].first < all[i - 1].second) return 1;
  if (!std::is_sorted(read.begin(), read.end())) std::sort(read.begin(), read.end());
  size_t k = 0;
  for (const auto& r : read) {
    while (k < all.size() && all[k].second <= r.first) ++k;
    if (k < all.size() && all[k].first < r.second) return 2;
  }
  return 0;
}
int check_adamw(int32_t count, const mx_adamw_tensor* list, const mx_adamw_opts& o) {
  if (o.state_bits != 8 && o.state_bits != 32) return set_error(MX_ERR_INVALID, "states have 8 or 32 bits (got %d)", o.state_bits);
  auto within = [](double x, double lo, double hi) { return x >= lo && x <= hi; };   // (not NaN)
  if (!o.lr_at && !within(o.lr, 0.0, 3e38)) return set_error(MX_ERR_INVALID, "the learning rate must be a number of at least zero (got %g)", o.lr);
  if (!within(o.beta1, 0.0, 1.0) || !within(o.beta2, 0.0, 1.0) || o.beta1 == 1.0 || o.beta2 == 1.0)
    return set_error(MX_ERR_INVALID, "betas must be at least 0 and less than 1 (got %g, %g)", o.beta1, o.beta2);
  if (!within(o.eps, 0.0, 3e38)) return set_error(MX_ERR_INVALID, "eps must be a number of at least zero (got %g)", o.eps);
  if (!within(o.weight_decay, 0.0, 3e38)) return set_error(MX_ERR_INVALID, "the weight decay must be a number of at least zero (got %g)", o.weight_decay);
  if (!o.step_at && o.step < 1) return set_error(MX_ERR_INVALID, "steps are counted from 1 (got %lld)", (long long)o.step);
  if (!o.scale_at && !within(o.grad_scale, -3e38, 3e38)) return set_error(MX_ERR_INVALID, "the gradients' scale must be a number");
  // What is written, a list for each kind: as a rule ascending, as its tensors were allocated.  (200 tensors: a step takes 28 us of host time, with
  // all of it sorted at once 40.)
  Ranges written[6], read;
  read.reserve((size_t)count + 3);
  auto reads = [&](const void* p, int64_t bytes) {
    if (p) read.emplace_back((uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes);
  };
  reads(o.lr_at, 4);
  reads(o.step_at, 8);
  reads(o.scale_at, 4);
  for (int k = 0; k < (o.state_bits == 8 ? 6 : 4); ++k) written[k].reserve(count);
  for (int32_t i = 0; i < count; ++i) {
    const mx_adamw_tensor& t = list[i];
    if (t.n < 0) return set_error(MX_ERR_SHAPE, "tensor %d: negative extent", i);
    if ((t.param_dtype != MX_F32 && t.param_dtype != MX_BF16) || (t.grad_dtype != MX_F32 && t.grad_dtype != MX_BF16))
      return set_error(MX_ERR_DTYPE, "tensor %d: parameters and gradients must be MX_F32 or MX_BF16 (got %d, %d)", i, t.param_dtype, t.grad_dtype);
    if (t.n == 0) continue;
    const bool small = o.state_bits == 8;
    if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq || (small && (!t.exp_avg_scale || !t.exp_avg_sq_scale)))
      return set_error(MX_ERR_INVALID, "tensor %d: null data pointer", i);
    if ((t.n + kChunk - 1) / kChunk > 0x7FFFFFFF) return set_error(MX_ERR_SHAPE, "tensor %d: too large", i);
    if ((uintptr_t)t.param % (t.param_dtype == MX_F32 ? 4 : 2) || (uintptr_t)t.grad % (t.grad_dtype == MX_F32 ? 4 : 2) ||
        ((uintptr_t)t.exp_avg | (uintptr_t)t.exp_avg_sq) % (small ? 8 : 4) || (uintptr_t)t.copy % 2)
      return set_error(MX_ERR_LAYOUT, "tensor %d: misaligned", i);
    const int64_t state = small ? round32(t.n) : t.n * 4;
    auto writes = [&](int k, const void* p, int64_t bytes) {
      if (p) written[k].emplace_back((uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes);
    };
    reads(t.grad, t.n * (t.grad_dtype == MX_F32 ? 4 : 2));
    writes(0, t.param, t.n * (t.param_dtype == MX_F32 ? 4 : 2));
    writes(1, t.exp_avg, state);
    writes(2, t.exp_avg_sq, state);
    writes(3, t.copy, t.n * 2);
    if (small) {
      writes(4, t.exp_avg_scale, state / 32);
      writes(5, t.exp_avg_sq_scale, state / 32);
    }
  }
  const int bad = overlap(written, read);
  if (bad == 1) return set_error(MX_ERR_INVALID, "parameters, states and copies must not overlap (is a tensor listed twice?)");
  return bad ? set_error(MX_ERR_INVALID, "parameters, states and copies must not overlap a gradient, nor a step, rate or scale that the kernel reads") : MX_OK;
}

}  // namespace
}  // namespace mx

using namespace mx;

extern "C" int mx_adamw_step(int32_t count, const mx_adamw_tensor* tensors, const mx_adamw_opts* opts, void* stream) try {
  if (count < 0) return set_error(MX_ERR_INVALID, "mx_adamw_step: negative count");
  if (!opts) return set_error(MX_ERR_INVALID, "mx_adamw_step: no options");
  if (opts->struct_size != (int32_t)sizeof(mx_adamw_opts)) return set_error(MX_ERR_INVALID, "mx_adamw_step: options of another version");
  if (count > 0 && !tensors) return set_error(MX_ERR_INVALID, "mx_adamw_step: null tensor array");
  const mx_adamw_opts& o = *opts;
  if (int rc = check_adamw(count, tensors, o)) return rc;
  AdamArgs a = {};
  a.seed = o.seed;
  a.b1 = (float)o.beta1; a.c1 = (float)(1.0 - o.beta1); a.b2 = (float)o.beta2; a.c2 = (float)(1.0 - o.beta2); a.eps = (float)o.eps;
  a.scale = (float)o.grad_scale;
  a.keep = (float)(1.0 - o.lr * o.weight_decay);
  a.rate = (float)(o.lr / (1.0 - std::pow(o.beta1, (double)o.step)));
  a.root = (float)(1.0 / std::sqrt(1.0 - std::pow(o.beta2, (double)o.step)));
  a.lr = (float)o.lr; a.decay = (float)o.weight_decay; a.log_b1 = (float)std::log(o.beta1); a.log_b2 = (float)std::log(o.beta2);
  a.step = o.step; a.lr_at = o.lr_at; a.step_at = o.step_at; a.scale_at = o.scale_at;
  for (const int P : {MX_F32, MX_BF16})
    for (const int G : {MX_F32, MX_BF16}) {
      int64_t chunks = 0;
      a.count = 0;
      auto flush = [&]() {
        if (a.count == 0) return (int)MX_OK;
        const bool small = o.state_bits == 8;
        hipStream_t st = (hipStream_t)stream;
        const hipError_t e = P == MX_F32 ? (G == MX_F32 ? launch<MX_F32, MX_F32>(a, chunks, small, st) : launch<MX_F32, MX_BF16>(a, chunks, small, st))
                                         : (G == MX_F32 ? launch<MX_BF16, MX_F32>(a, chunks, small, st) : launch<MX_BF16, MX_BF16>(a, chunks, small, st));
        chunks = 0;
        a.count = 0;
        return e == hipSuccess ? (int)MX_OK : set_error(MX_ERR_LAUNCH, "adamw_kernel launch: %s", hipGetErrorString(e));
      };
      for (int32_t i = 0; i < count; ++i) {
        const mx_adamw_tensor& t = tensors[i];
        if (t.n == 0 || t.param_dtype != P || t.grad_dtype != G) continue;
        const int64_t more = (t.n + kChunk - 1) / kChunk;
        if (a.count == kTensors || chunks + more > 0x7FFFFFFF)
          if (int rc = flush()) return rc;
        a.t[a.count] = {t.param, t.grad, t.exp_avg, t.exp_avg_sq, (uint8_t*)t.exp_avg_scale, (uint8_t*)t.exp_avg_sq_scale, (uint16_t*)t.copy, t.n};
        a.first[a.count] = (int32_t)chunks;
        a.index[a.count++] = i;
        chunks += more;
      }
      if (int rc = flush()) return rc;
    }
  return MX_OK;
} catch (const std::bad_alloc&) {   // (the list of ranges)
  return set_error(MX_ERR_INVALID, "mx_adamw_step: out of host memory");
}
