// pccl_optim_kernels.h -- device code of the optimizer-side operators of
// libpccl_hip.so (gfx950).  Included by pccl_optim.hip only.
//
// Everything here is bound by HBM (0.3-1 flop per byte): the kernels are
// organised so that every byte moves once, in accesses of a wave that are
// contiguous, and the arithmetic of an element stays in registers.
//
// A workgroup is one wave of 64 lanes wherever lanes do not need each other
// beyond it, and a lane holds 4 consecutive elements: one wave covers 256
// elements, which is also a block of the 8-bit form, so a block's maximum is a
// reduction inside a wave and needs neither LDS nor a barrier.
//
// The same source is compiled for the host by the tests, where a launch runs
// the kernel thread by thread.  Code in which lanes work together is therefore
// written over a small array of lanes: one entry on the device (the lane
// itself), all of them on the host, where the first thread of a group does the
// work of the whole group.
#ifndef PCCL_OPTIM_KERNELS_H
#define PCCL_OPTIM_KERNELS_H

#include <cmath>
#include <cstddef>
#include <cstdint>

#include "pccl_optim.h"

namespace pccl_optim_kernels {

constexpr int kWave = 64;
constexpr int kVec = 4;                     // elements of a lane
constexpr int kBlock = kWave * kVec;        // elements of a wave, and of a block of the 8-bit form
static_assert(kBlock == PCCL_OPTIM_BLOCK, "a wave holds one block");

// Tensors of one launch: their addresses travel in the kernel arguments, which
// are kept below 4 KiB.
constexpr int kAdamSegs = 64;               // 52 bytes each
constexpr int kAdam8Segs = 56;              // 68 bytes each
constexpr int kNormSegs = 64;
constexpr int kBlockSegs = 64;

constexpr float kCodeMax = 448.0f;              // largest finite e4m3 value
constexpr float kCodeMin = 0x1p-9f;             // smallest positive one
constexpr float kCodeNormal = 0x1p-6f;          // smallest with a full mantissa
constexpr float kAmaxFloor = 0x1p-100f;         // keeps 1 / scale finite for blocks of zeros and denormals

// ---------------------------------------------------------------------------
// lanes
// ---------------------------------------------------------------------------
#if defined(__HIP_DEVICE_COMPILE__)
constexpr bool kHostRun = false;
constexpr int kLaneSlots = 1;
template <class F> __device__ __forceinline__ void each_lane(F&& f) { f(0, (int)(threadIdx.x & (kWave - 1))); }
#else
constexpr bool kHostRun = true;
constexpr int kLaneSlots = kWave;
template <class F> __device__ __forceinline__ void each_lane(F&& f) { for (int l = 0; l < kWave; ++l) f(l, l); }
#endif

// Largest of an unsigned value over the wave, in every lane.  Six DPP steps
// (shifts within rows of 16, then the row results handed on), no LDS.
__device__ __forceinline__ uint32_t wave_max(const uint32_t* lanes) {
#if defined(__HIP_DEVICE_COMPILE__)
  uint32_t x = lanes[0];
#define PCCL_DPP_MAX(ctrl)                                                                            \
  {                                                                                                   \
    const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, 0xf, 0xf, true);        \
    x = y > x ? y : x;                                                                                \
  }
  PCCL_DPP_MAX(0x111)   // row_shr:1
  PCCL_DPP_MAX(0x112)   // row_shr:2
  PCCL_DPP_MAX(0x114)   // row_shr:4
  PCCL_DPP_MAX(0x118)   // row_shr:8
  PCCL_DPP_MAX(0x142)   // row_bcast:15
  PCCL_DPP_MAX(0x143)   // row_bcast:31
#undef PCCL_DPP_MAX
  return (uint32_t)__builtin_amdgcn_readlane((int)x, kWave - 1);
#else
  uint32_t x = 0;
  for (int l = 0; l < kWave; ++l) x = lanes[l] > x ? lanes[l] : x;
  return x;
#endif
}

// The tensor that work item `item` belongs to: start[] holds the first item of
// each of the `count` <= 64 tensors, in rising order from 0.  Every lane
// compares one entry; the number of starts at or below the item is the answer.
__device__ __forceinline__ int find_segment(const uint32_t* start, int count, uint32_t item) {
  if (count == 1) return 0;
#if defined(__HIP_DEVICE_COMPILE__)
  const int lane = (int)(threadIdx.x & (kWave - 1));
  const uint64_t at = __builtin_amdgcn_ballot_w64(lane < count && start[lane < count ? lane : 0] <= item);
  return __builtin_popcountll(at) - 1;
#else
  int s = 0;
  while (s + 1 < count && start[s + 1] <= item) ++s;
  return s;
#endif
}

// ---------------------------------------------------------------------------
// elements: four consecutive ones at any address that suits the element type.
// gfx950 takes vector accesses at any alignment; a tensor that starts in the
// middle of a flat buffer runs in the same code as an aligned one.
// ---------------------------------------------------------------------------
typedef uint32_t u32x4a __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2a __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32a __attribute__((aligned(1)));

// NT: with the non-temporal hint (the alignment belongs to the pointed-to type, so these are not one template)
template <bool NT> __device__ __forceinline__ u32x4a load16(const void* p) {
  if constexpr (NT) return __builtin_nontemporal_load((const u32x4a*)p);
  else return *(const u32x4a*)p;
}
template <bool NT> __device__ __forceinline__ u32x2a load8(const void* p) {
  if constexpr (NT) return __builtin_nontemporal_load((const u32x2a*)p);
  else return *(const u32x2a*)p;
}
template <bool NT> __device__ __forceinline__ void store16(void* p, u32x4a v) {
  if constexpr (NT) __builtin_nontemporal_store(v, (u32x4a*)p);
  else *(u32x4a*)p = v;
}
template <bool NT> __device__ __forceinline__ void store8(void* p, u32x2a v) {
  if constexpr (NT) __builtin_nontemporal_store(v, (u32x2a*)p);
  else *(u32x2a*)p = v;
}

struct F32 {
  typedef float elem;
  static constexpr bool kNone = false;
  template <bool NT> static __device__ __forceinline__ void load4(const void* p, size_t i, float* x) {
    const u32x4a w = load16<NT>((const elem*)p + i);
    x[0] = __uint_as_float(w.x); x[1] = __uint_as_float(w.y); x[2] = __uint_as_float(w.z); x[3] = __uint_as_float(w.w);
  }
  template <bool NT> static __device__ __forceinline__ void store4(void* p, size_t i, const float* x) {
    const u32x4a w = {__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
    store16<NT>((elem*)p + i, w);
  }
  static __device__ __forceinline__ float load1(const void* p, size_t i) { return ((const elem*)p)[i]; }
  static __device__ __forceinline__ void store1(void* p, size_t i, float x) { ((elem*)p)[i] = x; }
};

// T: __bf16 or _Float16; the conversions round to nearest even
template <class T> struct Half {
  typedef T elem;
  static constexpr bool kNone = false;
  typedef T x4 __attribute__((ext_vector_type(4)));
  typedef float f4 __attribute__((ext_vector_type(4)));
  template <bool NT> static __device__ __forceinline__ void load4(const void* p, size_t i, float* x) {
    const u32x2a w = load8<NT>((const elem*)p + i);
    x4 h;
    __builtin_memcpy(&h, &w, 8);
    const f4 f = __builtin_convertvector(h, f4);
    x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
  }
  template <bool NT> static __device__ __forceinline__ void store4(void* p, size_t i, const float* x) {
    const f4 f = {x[0], x[1], x[2], x[3]};
    const x4 h = __builtin_convertvector(f, x4);
    u32x2a w;
    __builtin_memcpy(&w, &h, 8);
    store8<NT>((elem*)p + i, w);
  }
  static __device__ __forceinline__ float load1(const void* p, size_t i) { return (float)((const elem*)p)[i]; }
  static __device__ __forceinline__ void store1(void* p, size_t i, float x) { ((elem*)p)[i] = (elem)x; }
};
typedef Half<__bf16> BF16;
typedef Half<_Float16> F16;

struct None {   // no copy
  static constexpr bool kNone = true;
  template <bool NT> static __device__ __forceinline__ void store4(void*, size_t, const float*) {}
  static __device__ __forceinline__ void store1(void*, size_t, float) {}
};

// Elements [i, i + 4) of a tensor of n; what lies behind its end is 0 and is
// not stored.
template <class T, bool NT> __device__ __forceinline__ void load_upto4(const void* p, size_t i, size_t n, float* x) {
  if (i + kVec <= n) { T::template load4<NT>(p, i, x); return; }
  for (int e = 0; e < kVec; ++e) x[e] = i + e < n ? T::load1(p, i + e) : 0.0f;
}
template <class T, bool NT> __device__ __forceinline__ void store_upto4(void* p, size_t i, size_t n, const float* x) {
  if (i + kVec <= n) { T::template store4<NT>(p, i, x); return; }
  for (int e = 0; e < kVec; ++e) if (i + e < n) T::store1(p, i + e, x[e]);
}

// ---------------------------------------------------------------------------
// e4m3 codes, four in a word
// ---------------------------------------------------------------------------
__device__ __forceinline__ void decode4(uint32_t w, float* x) {
#if defined(__HIP_DEVICE_COMPILE__)
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  x[0] = lo[0]; x[1] = lo[1]; x[2] = hi[0]; x[3] = hi[1];
#else
  for (int e = 0; e < 4; ++e) {
    const uint32_t c = (w >> (8 * e)) & 0xff, mag = c & 0x7f;
    const float a = mag == 0x7f ? std::nanf("") : mag < 8 ? (float)mag * 0x1p-9f
                                                          : std::ldexp(1.0f + (float)(mag & 7) / 8, (int)(mag >> 3) - 7);
    x[e] = c & 0x80 ? -a : a;
  }
#endif
}

// |x| <= 448 (1 + 2^-20) or NaN: nothing here overflows
__device__ __forceinline__ uint32_t encode4(const float* x) {
#if defined(__HIP_DEVICE_COMPILE__)
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], w, true);
#else
  uint32_t w = 0;
  for (int e = 0; e < 4; ++e) {
    const float a = std::fabs(x[e]);
    uint32_t c;
    if (!(a == a)) c = 0x7f;
    else {
      int ex = 0;
      std::frexp(a, &ex);
      if (a == 0 || ex < -5) ex = -5;
      const int q = (int)std::nearbyint(std::ldexp(a, 4 - ex));   // in units of the last place
      c = ex == -5 ? (uint32_t)q : (uint32_t)(q + ((ex + 5) << 3));
    }
    w |= (c | (std::signbit(x[e]) ? 0x80u : 0u)) << (8 * e);
  }
  return w;
#endif
}

// A 32-bit multiply-xorshift mix; the multipliers are from Chris Wellons'
// public-domain search for mixes of this form with low bias.
__device__ __forceinline__ uint32_t mix32(uint32_t x) {
  x ^= x >> 16; x *= 0x7feb352du;
  x ^= x >> 15; x *= 0x846ca68bu;
  return x ^ (x >> 16);
}
__device__ __forceinline__ uint32_t noise_key(uint32_t seed, uint64_t step) { return mix32(mix32(seed) + (uint32_t)step); }
__device__ __forceinline__ uint32_t noise(uint32_t key, uint64_t index) {
  return mix32((uint32_t)index + key + (uint32_t)(index >> 32) * 0x9e3779b1u);
}

// y, |y| <= 448 (1 + 2^-20), to one of the two e4m3 values next to it, the upper
// one with the probability of its nearness: 16 random bits are added to the 20
// mantissa bits that e4m3 drops, which are then cut off.  Below 2^-6 the codes
// are 2^-9 apart, as they are just above it, so the value is moved up there and
// back.  The result is exactly a code.  NaN stays NaN (a carry out of its
// mantissa is kept out by the test).
__device__ __forceinline__ float round_stochastic(float y, uint32_t u16) {
  const float a = std::fabs(y);
  const float shift = a < kCodeNormal ? kCodeNormal : 0.0f;
  const uint32_t cut = (__float_as_uint(a + shift) + (u16 << 4)) & 0xfff00000u;
  const float q = __uint_as_float(cut) - shift;
  return std::copysign(a <= kCodeMax * 1.001f ? (q > kCodeMax ? kCodeMax : q) : y, y);
}

struct BlockScale { float scale, inv; };

// From the largest |x| of a block, as bits (NaN is above infinity there, and
// comes out as NaN).
__device__ __forceinline__ BlockScale block_scale(uint32_t amax_bits) {
  float a = __uint_as_float(amax_bits);
  a = a < kAmaxFloor ? kAmaxFloor : a;
  BlockScale s;
  s.scale = a / kCodeMax;
  s.inv = 1.0f / s.scale;
  return s;
}

__device__ __forceinline__ uint32_t amax4(const float* x) {
  uint32_t a = 0;
  for (int e = 0; e < kVec; ++e) {
    const uint32_t b = __float_as_uint(x[e]) & 0x7fffffffu;
    a = b > a ? b : a;
  }
  return a;
}

// A root other than 0 keeps at least the smallest code.
__device__ __forceinline__ float lift_root(float r, float y) { return r > 0.0f && y < kCodeMin ? kCodeMin : y; }

__device__ __forceinline__ void store_codes(void* p, size_t i, size_t n, uint32_t w) {
  if (i + kVec <= n) { *(u32a*)((uint8_t*)p + i) = w; return; }
  for (int e = 0; e < kVec; ++e) if (i + e < n) ((uint8_t*)p)[i + e] = (uint8_t)(w >> (8 * e));
}
__device__ __forceinline__ uint32_t load_codes(const void* p, size_t i, size_t n) {
  if (i + kVec <= n) return *(const u32a*)((const uint8_t*)p + i);
  uint32_t w = 0;
  for (int e = 0; e < kVec; ++e) if (i + e < n) w |= (uint32_t)((const uint8_t*)p)[i + e] << (8 * e);
  return w;
}

// ---------------------------------------------------------------------------
// AdamW
// ---------------------------------------------------------------------------
// The scalars of a step.  The host fills in the fp32 ones from lr and step; if
// either lives in device memory the kernel computes them again, in 64 bits.
struct Hyper {
  float beta1, one_minus_beta1, beta2, one_minus_beta2, eps;
  float grad_scale, max_norm;
  float lr_decay;        // lr * weight_decay
  float step_size;       // lr / (1 - beta1^t)
  float inv_root_bias;   // 1 / sqrt(1 - beta2^t)
  int skip_nonfinite, stochastic;
  uint32_t seed;
  uint64_t step;
  double lr, beta1_d, beta2_d, weight_decay;
  const float* lr_dev;
  const int64_t* step_dev;
  const float* norm;
};

// base^n by squaring: the error is n roundings of 2^-53 at most, and n base^n is bounded
__device__ __forceinline__ double int_power(double base, uint64_t n) {
  double r = 1.0;
  for (; n; n >>= 1) {
    if (n & 1) r *= base;
    base *= base;
  }
  return r;
}

// Everything that depends on lr and t, in 64 bits: 1 - beta^t loses up to ten bits to cancellation
__device__ __forceinline__ void fill_schedule(Hyper& h, double lr, uint64_t t) {
  h.lr_decay = (float)(lr * h.weight_decay);
  h.step_size = (float)(lr / (1.0 - int_power(h.beta1_d, t)));
  h.inv_root_bias = (float)(1.0 / sqrt(1.0 - int_power(h.beta2_d, t)));
}

// Completes the scalars from device memory; false if the step is skipped.
__device__ __forceinline__ bool finish_hyper(Hyper& h) {
  if (h.norm) {
    const float norm = *h.norm;
    if (h.skip_nonfinite && !(std::fabs(norm) <= 3.402823466e38f)) return false;
    if (h.max_norm > 0.0f) {
      const float c = h.max_norm / (norm * std::fabs(h.grad_scale) + 1e-6f);
      h.grad_scale *= c >= 1.0f ? 1.0f : c;      // a NaN norm gives NaN gradients
    }
  }
  if (h.lr_dev || h.step_dev) {
    if (h.step_dev) {
      const int64_t t = *h.step_dev;
      h.step = t < 1 ? 1 : (uint64_t)t;
    }
    fill_schedule(h, h.lr_dev ? (double)*h.lr_dev : h.lr, h.step);
  }
  return true;
}

// One element.  Returns sqrt(v), which the 8-bit form stores.
__device__ __forceinline__ float adamw_element(const Hyper& h, float& p, float g, float& m, float& v) {
  g *= h.grad_scale;
  m = h.beta1 * m + h.one_minus_beta1 * g;
  v = h.beta2 * v + h.one_minus_beta2 * (g * g);
  const float root = sqrtf(v);
  const float update = m / (root * h.inv_root_bias + h.eps);
  p -= h.lr_decay * p + h.step_size * update;   // the two small terms first: 1 - lr * decay would round them away
  return root;
}

struct AdamTable {
  void* p[kAdamSegs];
  const void* g[kAdamSegs];
  void* m[kAdamSegs];
  void* v[kAdamSegs];
  void* c[kAdamSegs];
  size_t n[kAdamSegs];
  uint32_t start[kAdamSegs];   // first workgroup of each tensor
};

// Moments in 32 bits: one wave per U * 256 elements.
template <class P, class G, class C, int U, bool NT>
__global__ __launch_bounds__(kWave) void k_adamw(AdamTable t, int count, Hyper h) {
  const int s = find_segment(t.start, count, blockIdx.x);
  const size_t n = t.n[s];
  const size_t base = (size_t)(blockIdx.x - t.start[s]) * (U * kBlock) + (threadIdx.x & (kWave - 1)) * kVec;
  if (!finish_hyper(h)) return;
  float p[U][kVec], g[U][kVec], m[U][kVec], v[U][kVec];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const size_t i = base + u * kBlock;
    load_upto4<P, NT>(t.p[s], i, n, p[u]);
    load_upto4<G, NT>(t.g[s], i, n, g[u]);
    load_upto4<F32, NT>(t.m[s], i, n, m[u]);
    load_upto4<F32, NT>(t.v[s], i, n, v[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const size_t i = base + u * kBlock;
#pragma unroll
    for (int e = 0; e < kVec; ++e) adamw_element(h, p[u][e], g[u][e], m[u][e], v[u][e]);
    store_upto4<P, NT>(t.p[s], i, n, p[u]);
    store_upto4<F32, NT>(t.m[s], i, n, m[u]);
    store_upto4<F32, NT>(t.v[s], i, n, v[u]);
    if constexpr (!C::kNone) store_upto4<C, NT>(t.c[s], i, n, p[u]);
  }
}

struct Adam8Table {
  void* p[kAdam8Segs];
  const void* g[kAdam8Segs];
  void* m[kAdam8Segs];         // codes of the first moment
  void* r[kAdam8Segs];         // codes of the root of the second
  float* ms[kAdam8Segs];
  float* rs[kAdam8Segs];
  void* c[kAdam8Segs];
  size_t n[kAdam8Segs];
  uint32_t start[kAdam8Segs];
};

// Moments in 8 bits: one wave per block.
template <class P, class G, class C, bool NT>
__global__ __launch_bounds__(kWave) void k_adamw8(Adam8Table t, int count, Hyper h) {
  if (kHostRun && threadIdx.x) return;
  const int s = find_segment(t.start, count, blockIdx.x);
  const size_t n = t.n[s], block = blockIdx.x - t.start[s];
  if (!finish_hyper(h)) return;
  const float ms = t.ms[s][block], rs = t.rs[s][block];
  float m[kLaneSlots][kVec], r[kLaneSlots][kVec];
  uint32_t ma[kLaneSlots], ra[kLaneSlots];
  each_lane([&](int k, int lane) {
    const size_t i = block * kBlock + lane * kVec;
    float p[kVec], g[kVec];
    load_upto4<P, NT>(t.p[s], i, n, p);
    load_upto4<G, NT>(t.g[s], i, n, g);
    decode4(load_codes(t.m[s], i, n), m[k]);
    decode4(load_codes(t.r[s], i, n), r[k]);
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      m[k][e] *= ms;
      const float old = r[k][e] * rs;
      float v = old * old;
      r[k][e] = adamw_element(h, p[e], g[e], m[k][e], v);
    }
    store_upto4<P, NT>(t.p[s], i, n, p);
    if constexpr (!C::kNone) store_upto4<C, NT>(t.c[s], i, n, p);
    ma[k] = amax4(m[k]);
    ra[k] = amax4(r[k]);
  });
  const BlockScale mb = block_scale(wave_max(ma)), rb = block_scale(wave_max(ra));
  const uint32_t key = noise_key(h.seed, h.step);
  each_lane([&](int k, int lane) {
    const size_t i = block * kBlock + lane * kVec;
    float y[kVec], z[kVec];
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      y[e] = m[k][e] * mb.inv;
      z[e] = lift_root(r[k][e], r[k][e] * rb.inv);
    }
    if (h.stochastic) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const uint32_t bits = noise(key, i + e);
        y[e] = round_stochastic(y[e], bits & 0xffffu);
        z[e] = round_stochastic(z[e], bits >> 16);
      }
    }
    store_codes(t.m[s], i, n, encode4(y));
    store_codes(t.r[s], i, n, encode4(z));
    if (lane == 0) { t.ms[s][block] = mb.scale; t.rs[s][block] = rb.scale; }
  });
}

// ---------------------------------------------------------------------------
// 8-bit blocks
// ---------------------------------------------------------------------------
struct BlocksTable {
  void* codes[kBlockSegs];
  float* scales[kBlockSegs];
  void* x[kBlockSegs];
  size_t n[kBlockSegs];
  uint32_t start[kBlockSegs];
};

template <class T, bool NT>
__global__ __launch_bounds__(kWave) void k_quantize(BlocksTable t, int count, int root) {
  if (kHostRun && threadIdx.x) return;
  const int s = find_segment(t.start, count, blockIdx.x);
  const size_t n = t.n[s], block = blockIdx.x - t.start[s];
  float x[kLaneSlots][kVec];
  uint32_t a[kLaneSlots];
  each_lane([&](int k, int lane) {
    load_upto4<T, NT>(t.x[s], block * kBlock + lane * kVec, n, x[k]);
    if (root)
      for (int e = 0; e < kVec; ++e) x[k][e] = sqrtf(x[k][e]);
    a[k] = amax4(x[k]);
  });
  const BlockScale b = block_scale(wave_max(a));
  each_lane([&](int k, int lane) {
    float y[kVec];
    for (int e = 0; e < kVec; ++e) {
      y[e] = x[k][e] * b.inv;
      if (root) y[e] = lift_root(x[k][e], y[e]);
    }
    store_codes(t.codes[s], block * kBlock + lane * kVec, n, encode4(y));
    if (lane == 0) t.scales[s][block] = b.scale;
  });
}

template <class T, bool NT>
__global__ __launch_bounds__(kWave) void k_dequantize(BlocksTable t, int count, int root) {
  const int s = find_segment(t.start, count, blockIdx.x);
  const size_t n = t.n[s], block = blockIdx.x - t.start[s];
  const size_t i = block * kBlock + (threadIdx.x & (kWave - 1)) * kVec;
  const float scale = t.scales[s][block];
  float x[kVec];
  decode4(load_codes(t.codes[s], i, n), x);
  for (int e = 0; e < kVec; ++e) {
    x[e] *= scale;
    if (root) x[e] *= x[e];
  }
  store_upto4<T, NT>(t.x[s], i, n, x);
}

// ---------------------------------------------------------------------------
// gradient norm
// ---------------------------------------------------------------------------
constexpr int kNormThreads = 256;
constexpr int kNormUnroll = 4;
constexpr int kNormTile = kNormThreads * kVec * kNormUnroll;     // elements of a work item

struct NormTable {
  const void* x[kNormSegs];
  size_t n[kNormSegs];
  uint32_t start[kNormSegs];
};

// Sum over the threads of a workgroup, in a fixed order; valid in thread 0.
// `part`: the thread's own value on the device, all threads' on the host.
template <int T>
__device__ __forceinline__ double group_sum(const double* part) {
#if defined(__HIP_DEVICE_COMPILE__)
  __shared__ double waves[T / kWave];
  double x = part[0];
  for (int d = kWave / 2; d; d >>= 1) x += __shfl_xor(x, d);
  if constexpr (T == kWave) return x;
  if ((threadIdx.x & (kWave - 1)) == 0) waves[threadIdx.x / kWave] = x;
  __syncthreads();
  double sum = 0;
  if (threadIdx.x == 0)
    for (int w = 0; w < T / kWave; ++w) sum += waves[w];
  return sum;
#else
  double sum = 0;
  for (int k = 0; k < T; ++k) sum += part[k];
  return sum;
#endif
}

// One partial sum per workgroup, which walks the work items gridDim.x apart.
// FINAL: the only workgroup of the whole norm; it writes the result itself.
template <class T, bool NT, bool FINAL>
__global__ __launch_bounds__(kNormThreads) void k_sum_squares(NormTable t, int count, uint32_t items, double* part, float* out) {
  if (kHostRun && threadIdx.x) return;
  constexpr int kSlots = kHostRun ? kNormThreads : 1;
  double sum[kSlots];
  for (int k = 0; k < kSlots; ++k) {
    const int thread = kHostRun ? k : (int)threadIdx.x;
    double acc = 0;
    for (uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
      const int s = find_segment(t.start, count, item);
      const size_t n = t.n[s];
      const size_t base = (size_t)(item - t.start[s]) * kNormTile + (size_t)thread * kVec;
      float x[kNormUnroll][kVec];
#pragma unroll
      for (int u = 0; u < kNormUnroll; ++u) load_upto4<T, NT>(t.x[s], base + u * (kNormThreads * kVec), n, x[u]);
#pragma unroll
      for (int u = 0; u < kNormUnroll; ++u)
#pragma unroll
        for (int e = 0; e < kVec; ++e) acc += (double)x[u][e] * (double)x[u][e];
    }
    sum[k] = acc;
  }
  const double total = group_sum<kNormThreads>(sum);
  if (threadIdx.x == 0) {
    if constexpr (FINAL) out[0] = (float)sqrt(total);
    else part[blockIdx.x] = total;
  }
}

__global__ __launch_bounds__(kNormThreads) void k_norm_join(const double* part, uint32_t count, float* out) {
  if (kHostRun && threadIdx.x) return;
  constexpr int kSlots = kHostRun ? kNormThreads : 1;
  double sum[kSlots];
  for (int k = 0; k < kSlots; ++k) {
    double acc = 0;
    for (uint32_t i = kHostRun ? k : threadIdx.x; i < count; i += kNormThreads) acc += part[i];
    sum[k] = acc;
  }
  const double total = group_sum<kNormThreads>(sum);
  if (threadIdx.x == 0) out[0] = (float)sqrt(total);
}

}  // namespace pccl_optim_kernels

#endif  // PCCL_OPTIM_KERNELS_H
