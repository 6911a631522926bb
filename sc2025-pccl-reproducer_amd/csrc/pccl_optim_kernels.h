// pccl_optim_kernels.h -- device code of the optimizer-side operators of
// libpccl_hip.so (gfx950).  Included by pccl_optim.hip only.
//
// Everything here is bound by HBM (0.3-6 flop per byte): the kernels are
// organised so that every byte moves once, in accesses of a wave that are
// contiguous, and the arithmetic of an element stays in registers.  For scale:
// on MI355X a copy kernel moves 6.7 TB/s, a kernel that only reads 7.4-7.5, and
// the smallest launch takes 2-3 us.
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

constexpr float kCodeMax = 448.0f;              // largest finite e4m3 value
constexpr float kCodeMin = 0x1p-9f;             // smallest positive one
constexpr float kCodeNormal = 0x1p-6f;          // smallest with a full mantissa
constexpr uint32_t kFloorBits = 0x0d800000u;    // 2^-100: keeps 1 / scale finite for blocks of zeros and denormals

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

// A value that the caller knows to be the same in all lanes, for the compiler
__device__ __forceinline__ uint32_t wave_uniform(uint32_t x) {
#if defined(__HIP_DEVICE_COMPILE__)
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)x);
#else
  return x;
#endif
}

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

// ---------------------------------------------------------------------------
// the tensors of a launch
// ---------------------------------------------------------------------------
// start[] holds the first work item of each tensor, in rising order from 0.  The
// table travels in the kernel arguments, which are kept below 4 KiB, or lies in
// device memory, where one launch then serves up to kTableMax tensors.
template <class E, int CAP> struct Table {
  typedef E entry;
  static constexpr int kInline = CAP;
  E e[CAP];
  uint32_t start[CAP];
};
constexpr int kTableMax = kWave * kWave;

struct AdamEntry { void* p; const void* g; void* m; void* v; void* c; size_t n; };
struct Adam8Entry { void* p; const void* g; void* m; void* r; float* ms; float* rs; void* c; size_t n; };
struct BlocksEntry { void* codes; float* scales; void* x; size_t n; };
struct NormEntry { const void* x; size_t n; };
typedef Table<AdamEntry, 64> AdamTable;
typedef Table<Adam8Entry, 56> Adam8Table;
typedef Table<BlocksEntry, 104> BlocksTable;
typedef Table<NormEntry, 192> NormTable;

// Both places are read through the constant address space, i.e. by scalar loads:
// nothing writes a table while a kernel runs.
#if defined(__HIP_DEVICE_COMPILE__)
#define PCCL_CONSTANT __attribute__((address_space(4)))
#define PCCL_GLOBAL __attribute__((address_space(1)))
#else
#define PCCL_CONSTANT
#define PCCL_GLOBAL
#endif
// Addresses read from a table are said to be of global memory: to the compiler
// they could be anything, and it would use flat accesses.
typedef PCCL_GLOBAL char* gptr;
typedef const PCCL_GLOBAL char* cgptr;

template <class E> struct View {
  const PCCL_CONSTANT E* e;
  const PCCL_CONSTANT uint32_t* start;
};

// The table is the kernel's FIRST argument, i.e. at the start of its arguments.
template <class T> __device__ __forceinline__ View<typename T::entry> view_of(const T& args, const void* dev, int count) {
  typedef typename T::entry E;
#if defined(__HIP_DEVICE_COMPILE__)
  typedef const PCCL_CONSTANT char* bytes;
  const bytes in_args = (bytes)__builtin_amdgcn_kernarg_segment_ptr(), in_memory = (bytes)(uintptr_t)dev;
  const bytes entries = dev ? in_memory : in_args;
  return {(const PCCL_CONSTANT E*)entries,
          (const PCCL_CONSTANT uint32_t*)(entries + (dev ? (size_t)count * sizeof(E) : offsetof(T, start)))};
#else
  if (!dev) return {args.e, args.start};
  return {(const E*)dev, (const uint32_t*)((const char*)dev + (size_t)count * sizeof(E))};
#endif
}

// The tensor that a work item belongs to: every lane compares one start, and the
// number of those at or below the item is the answer; above 64 tensors first
// among every 64th.
template <class E> __device__ __forceinline__ int find_segment(const View<E>& v, int count, uint32_t item) {
  if (count == 1) return 0;
#if defined(__HIP_DEVICE_COMPILE__)
  const int lane = (int)(threadIdx.x & (kWave - 1));
  int base = 0;
  if (count > kWave) {
    const int at = lane * kWave;
    base = (__builtin_popcountll(__builtin_amdgcn_ballot_w64(at < count && v.start[at < count ? at : 0] <= item)) - 1) * kWave;
  }
  const int at = base + lane;
  return base + __builtin_popcountll(__builtin_amdgcn_ballot_w64(at < count && v.start[at < count ? at : 0] <= item)) - 1;
#else
  int s = 0;
  while (s + 1 < count && v.start[s + 1] <= item) ++s;
  return s;
#endif
}

// Workgroup i runs on accelerator die i % 8, and each die has an L2 of its own.
// Work items that write a few bytes of a cache line each (the scales of their
// blocks) are handed out in runs of 64 to one die, so that a line is put
// together in one L2 and not written to memory in parts by eight: k_quantize of
// 128 Mi elements 66.6 -> 63.6 us (bf16), 105 -> 101 us (fp32).
constexpr uint32_t kXcds = 8, kXcdRun = 64;
__device__ __forceinline__ uint32_t xcd_run(uint32_t b, uint32_t total) {
  const uint32_t r = b % (kXcds * kXcdRun), base = b - r;
  return base + kXcds * kXcdRun <= total ? base + r % kXcds * kXcdRun + r / kXcds : b;
}

// ---------------------------------------------------------------------------
// elements: four consecutive ones at any address that suits the element type.
// gfx950 takes vector accesses at any alignment; a tensor that starts in the
// middle of a flat buffer runs in the same code as an aligned one.
// ---------------------------------------------------------------------------
typedef uint32_t u32x4a __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2a __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32a __attribute__((aligned(1)));

// NT: with the non-temporal hint (the alignment belongs to the pointed-to type, so these are not one template)
template <bool NT> __device__ __forceinline__ u32x4a load16(cgptr p) {
  if constexpr (NT) return __builtin_nontemporal_load((const PCCL_GLOBAL u32x4a*)p);
  else return *(const PCCL_GLOBAL u32x4a*)p;
}
template <bool NT> __device__ __forceinline__ u32x2a load8(cgptr p) {
  if constexpr (NT) return __builtin_nontemporal_load((const PCCL_GLOBAL u32x2a*)p);
  else return *(const PCCL_GLOBAL u32x2a*)p;
}
template <bool NT> __device__ __forceinline__ uint32_t load4b(cgptr p) {
  if constexpr (NT) return __builtin_nontemporal_load((const PCCL_GLOBAL u32a*)p);
  else return *(const PCCL_GLOBAL u32a*)p;
}
template <bool NT> __device__ __forceinline__ void store16(gptr p, u32x4a v) {
  if constexpr (NT) __builtin_nontemporal_store(v, (PCCL_GLOBAL u32x4a*)p);
  else *(PCCL_GLOBAL u32x4a*)p = v;
}
template <bool NT> __device__ __forceinline__ void store8(gptr p, u32x2a v) {
  if constexpr (NT) __builtin_nontemporal_store(v, (PCCL_GLOBAL u32x2a*)p);
  else *(PCCL_GLOBAL u32x2a*)p = v;
}
template <bool NT> __device__ __forceinline__ void store4b(gptr p, uint32_t v) {
  if constexpr (NT) __builtin_nontemporal_store(v, (PCCL_GLOBAL u32a*)p);
  else *(PCCL_GLOBAL u32a*)p = v;
}

// The elements [lo, hi) of a work item that are its tensor's.  A work item is
// addressed by its first element (the same for the whole wave, so it stays in
// scalar registers) and 32-bit places relative to it.
struct Span { uint32_t lo, hi; };
__device__ __forceinline__ bool whole4(uint32_t i, Span s) { return i >= s.lo && i + kVec <= s.hi; }
__device__ __forceinline__ bool inside(uint32_t i, Span s) { return i >= s.lo && i < s.hi; }

// i: place relative to p, in elements
struct F32 {
  typedef float elem;
  static constexpr bool kNone = false;
  typedef u32x4a raw;      // four elements as they lie in memory
  template <bool NT> static __device__ __forceinline__ raw load4(cgptr p, uint32_t i) { return load16<NT>(p + i * 4u); }
  static __device__ __forceinline__ raw load_some(cgptr p, uint32_t i, Span s) {
    raw w = {0, 0, 0, 0};
    const PCCL_GLOBAL uint32_t* q = (const PCCL_GLOBAL uint32_t*)p + i;
    if (inside(i, s)) w.x = q[0];
    if (inside(i + 1, s)) w.y = q[1];
    if (inside(i + 2, s)) w.z = q[2];
    if (inside(i + 3, s)) w.w = q[3];
    return w;
  }
  static __device__ __forceinline__ void widen(raw w, float* x) {
    x[0] = __uint_as_float(w.x); x[1] = __uint_as_float(w.y); x[2] = __uint_as_float(w.z); x[3] = __uint_as_float(w.w);
  }
  template <bool NT> static __device__ __forceinline__ void store4(gptr p, uint32_t i, const float* x) {
    const u32x4a w = {__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
    store16<NT>(p + i * 4u, w);
  }
  static __device__ __forceinline__ void store1(gptr p, uint32_t i, float x) { ((PCCL_GLOBAL elem*)p)[i] = x; }
};

// T: __bf16 or _Float16; the conversions round to nearest even
template <class T> struct Half {
  typedef T elem;
  static constexpr bool kNone = false;
  typedef T x4 __attribute__((ext_vector_type(4)));
  typedef float f4 __attribute__((ext_vector_type(4)));
  typedef u32x2a raw;
  template <bool NT> static __device__ __forceinline__ raw load4(cgptr p, uint32_t i) { return load8<NT>(p + i * 2u); }
  static __device__ __forceinline__ raw load_some(cgptr p, uint32_t i, Span s) {
    raw w = {0, 0};
    const PCCL_GLOBAL uint16_t* q = (const PCCL_GLOBAL uint16_t*)p + i;
    if (inside(i, s)) w.x = q[0];
    if (inside(i + 1, s)) w.x |= (uint32_t)q[1] << 16;
    if (inside(i + 2, s)) w.y = q[2];
    if (inside(i + 3, s)) w.y |= (uint32_t)q[3] << 16;
    return w;
  }
  static __device__ __forceinline__ void widen(raw w, float* x) {
    x4 h;
    __builtin_memcpy(&h, &w, 8);
    const f4 f = __builtin_convertvector(h, f4);
    x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
  }
  template <bool NT> static __device__ __forceinline__ void store4(gptr p, uint32_t i, const float* x) {
    const f4 f = {x[0], x[1], x[2], x[3]};
    const x4 h = __builtin_convertvector(f, x4);
    u32x2a w;
    __builtin_memcpy(&w, &h, 8);
    store8<NT>(p + i * 2u, w);
  }
  static __device__ __forceinline__ void store1(gptr p, uint32_t i, float x) { ((PCCL_GLOBAL elem*)p)[i] = (elem)x; }
};
typedef Half<__bf16> BF16;
typedef Half<_Float16> F16;

struct None {   // no copy
  static constexpr bool kNone = true;
};

// Elements [i, i + 4) of an item; those outside the span are 0 and are not
// stored.  FULL: the caller knows that all four are inside.
template <class T, bool NT, bool FULL> __device__ __forceinline__ typename T::raw load_upto4(cgptr p, uint32_t i, Span s) {
  return FULL || whole4(i, s) ? T::template load4<NT>(p, i) : T::load_some(p, i, s);
}
template <class T, bool NT, bool FULL> __device__ __forceinline__ void store_upto4(gptr p, uint32_t i, Span s, const float* x) {
  if (FULL || whole4(i, s)) { T::template store4<NT>(p, i, x); return; }
  for (int e = 0; e < kVec; ++e) if (inside(i + e, s)) T::store1(p, i + e, x[e]);
}

// Address of an element of a tensor, `at` possibly before its start
__device__ __forceinline__ gptr element(const void* p, ptrdiff_t at, size_t bytes) {
  return (gptr)((uintptr_t)p + (uintptr_t)at * bytes);
}

// The smaller of the two.  In halves: the compiler has left a 64-bit comparison
// of this form in the vector unit and its selection in the scalar unit, which
// then read a condition that nobody had set.
__device__ __forceinline__ uint32_t at_most(size_t rest, uint32_t size) {
  const uint32_t low = (uint32_t)rest;
  return (uint32_t)((uint64_t)rest >> 32) != 0 || low > size ? size : low;
}

// What a work item of `size` elements that starts at element `first` of n has of its tensor
__device__ __forceinline__ Span span_of(size_t first, size_t n, uint32_t size) { return {0, at_most(n - first, size)}; }

// f(true_type) for a work item that lies whole in its tensor, which runs without
// a bound check, f(false_type) for the last one.  The choice is the same for the
// whole wave.
template <bool V> struct Full { static constexpr bool value = V; };
template <class F> __device__ __forceinline__ void with_bounds(bool full, F&& f) {
  if (full) f(Full<true>());
  else f(Full<false>());
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

// To nearest, ties to even.  |x| <= 448 (1 + 2^-20): nothing here overflows.  (A
// block with an inf or NaN has a scale that is not finite: its codes do not
// matter.)
__device__ __forceinline__ uint32_t encode4(const float* x) {
#if defined(__HIP_DEVICE_COMPILE__)
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], w, true);
#else
  uint32_t w = 0;
  for (int e = 0; e < 4; ++e) {
    const float a = std::fabs(x[e]);
    uint32_t c = 0x7f;
    if (a < 480.0f) {
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

// A value that a carry would take out of the codes: 448 times 1 + 2^-20
__device__ __forceinline__ float clamp_code(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_fmed3f(x, -kCodeMax, kCodeMax);
#else
  return x > kCodeMax ? kCodeMax : x < -kCodeMax ? -kCodeMax : x;
#endif
}

// |x| <= 448.  To one of the two codes next to x, the upper one (in magnitude) with the
// probability of its nearness: the 16 random bits in the upper half of each
// bits[e] are added to the 20 mantissa bits that e4m3 drops, which are then cut
// off; below 2^-6, where the codes are 2^-9 apart, to x in units of that.  It is
// what v_cvt_sr_fp8_f32 does with its second operand's upper 20 bits (checked on
// MI355X against this description for 4 million values and random numbers).
__device__ __forceinline__ uint32_t encode4_stochastic(const float* x, const uint32_t* bits) {
  uint32_t w = 0;
#if defined(__HIP_DEVICE_COMPILE__)
  w = (uint32_t)__builtin_amdgcn_cvt_sr_fp8_f32(x[0], (int)bits[0], (int)w, 0);
  w = (uint32_t)__builtin_amdgcn_cvt_sr_fp8_f32(x[1], (int)bits[1], (int)w, 1);
  w = (uint32_t)__builtin_amdgcn_cvt_sr_fp8_f32(x[2], (int)bits[2], (int)w, 2);
  w = (uint32_t)__builtin_amdgcn_cvt_sr_fp8_f32(x[3], (int)bits[3], (int)w, 3);
#else
  float y[kVec];
  for (int e = 0; e < 4; ++e) {
    const float a = std::fabs(x[e]), shift = a < kCodeNormal ? kCodeNormal : 0.0f;
    const float q = __uint_as_float((__float_as_uint(a + shift) + (bits[e] >> 12)) & 0xfff00000u) - shift;
    y[e] = std::copysign(q, x[e]);
  }
  w = encode4(y);
#endif
  return w;
}

// A 32-bit multiply-xorshift mix; the multipliers are from Chris Wellons'
// public-domain search for mixes of this form with low bias.
__device__ __forceinline__ uint32_t mix32(uint32_t x) {
  x ^= x >> 16; x *= 0x7feb352du;
  x ^= x >> 15; x *= 0x846ca68bu;
  return x ^ (x >> 16);
}
__device__ __forceinline__ uint32_t noise_key(uint32_t seed, uint64_t step) { return mix32(mix32(seed) + (uint32_t)step); }
// 32 random bits for an element of the block that starts at `first` (a multiple
// of 256, so the upper half of the index is that of the whole block)
__device__ __forceinline__ uint32_t noise(uint32_t key, size_t first, uint32_t i) {
  return mix32((uint32_t)first + key + (uint32_t)((uint64_t)first >> 32) * 0x9e3779b1u + i);
}

struct BlockScale { float scale, inv; };
constexpr float kInvCodeMax = 1.0f / kCodeMax;

// 1 / x for a normal x whose reciprocal is normal: the hardware's, which is not the
// rounded one for 11 % of all x, and one Newton step, after which it is (compared
// on MI355X for all mantissas).
__device__ __forceinline__ float reciprocal(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
  const float r = __builtin_amdgcn_rcpf(x);
  return __builtin_fmaf(__builtin_fmaf(-x, r, 1.0f), r, r);
#else
  return 1.0f / x;
#endif
}

// From the largest |x| of a block, as bits.  The comparison is one of integers,
// in which NaN is above infinity, so that either becomes the scale.  The product
// with 1 / 448 is the quotient or one unit beside it, and x * inv within two units of
// x / scale.  The format is defined by these products: they are what a plain form
// in elementary operations gives on the GPU, where torch divides by a number in
// this way, so that states agree bit for bit.  Rounded quotients were built and
// taken back: they move single codes, half way between two and so no nearer (error
// of 128 Mi bf16 values 0.0031 either way), and cost 1-2 % of k_quantize.
__device__ __forceinline__ BlockScale block_scale(uint32_t amax_bits) {
  BlockScale s;
  s.scale = __uint_as_float(amax_bits > kFloorBits ? amax_bits : kFloorBits) * kInvCodeMax;
  s.inv = reciprocal(s.scale);
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

// y = r / scale, at least the smallest code for a root r other than 0 and at most
// the largest: the middle one of y, 2^-9 and a number that is 0 for r = 0 and
// beyond 448 for every other root (the smallest is 2^-74.5).
__device__ __forceinline__ float lift_root(float r, float y) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_fmed3f(y, kCodeMin, std::fmin(r * 0x1p100f, kCodeMax));
#else
  return r == 0 ? 0.0f : y < kCodeMin ? kCodeMin : y > kCodeMax ? kCodeMax : y;
#endif
}

// sqrt of four numbers >= 0.  From 2^-102 on from the hardware's 1 / sqrt(x), good
// to one unit in the last place, and a correction by the exact residue, a third of
// the instructions of sqrtf: the rounded root for every such number (all were
// compared on MI355X).  Below that the residue underflows, and the root would be one
// unit off for up to 9 % of a binade; they, zeros, infinity and NaN go the long way.
constexpr uint32_t kRootFrom = 0x0c800000u;      // 2^-102
__device__ __forceinline__ void sqrt4(const float* x, float* root) {
#if defined(__HIP_DEVICE_COMPILE__)
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < kVec; ++e) {
    const uint32_t b = __float_as_uint(x[e]) - kRootFrom;      // wraps for those below
    top = b > top ? b : top;
  }
  if (top < 0x7f800000u - kRootFrom) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      const float r = __builtin_amdgcn_rsqf(x[e]);
      const float s = x[e] * r;
      root[e] = __builtin_fmaf(__builtin_fmaf(-s, s, x[e]), 0.5f * r, s);
    }
    return;
  }
#endif
#pragma unroll
  for (int e = 0; e < kVec; ++e) root[e] = sqrtf(x[e]);
}

template <bool NT, bool FULL> __device__ __forceinline__ void store_codes(gptr p, uint32_t i, Span s, uint32_t w) {
  if (FULL || whole4(i, s)) { store4b<NT>(p + i, w); return; }
  for (int e = 0; e < kVec; ++e) if (inside(i + e, s)) p[i + e] = (char)(w >> (8 * e));
}
template <bool NT, bool FULL> __device__ __forceinline__ uint32_t load_codes(cgptr p, uint32_t i, Span s) {
  if (FULL || whole4(i, s)) return load4b<NT>(p + i);
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < kVec; ++e) if (inside(i + e, s)) w |= (uint32_t)(uint8_t)p[i + e] << (8 * e);
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
  float scale_high, scale_low;   // grad_scale as max(1, |grad_scale|) times what is left: one of them is 1 or -1
  float norm_added;              // 1e-6 / scale_high
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

static_assert(sizeof(AdamTable) + sizeof(Hyper) + 16 <= 4096 && sizeof(Adam8Table) + sizeof(Hyper) + 16 <= 4096 &&
              sizeof(BlocksTable) + 16 <= 4096 && sizeof(NormTable) + 48 <= 4096, "kernel arguments");

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
    const float norm = *(const PCCL_GLOBAL float*)(uintptr_t)h.norm;
    if (h.skip_nonfinite && !(std::fabs(norm) <= 3.402823466e38f)) return false;
    if (h.max_norm > 0.0f) {
      // grad_scale * min(1, max_norm / (norm * |grad_scale| + 1e-6)), with a grad_scale above 1 taken into the
      // fraction: norm * grad_scale may overflow where the result does not.
      const float c = h.max_norm / (norm * std::fabs(h.scale_low) + h.norm_added);
      h.grad_scale = h.scale_low * (c >= h.scale_high ? h.scale_high : c);      // a NaN norm gives NaN gradients
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

// Four elements; v comes back as its root, too, which the 8-bit form stores.
// The moments are computed without fused multiply-adds: every operation rounds
// once by itself, so that a moment next to the border between two codes gets the
// same code as from elementary fp32 operations.
__device__ __forceinline__ void adamw4(const Hyper& h, float* p, const float* grad, float* m, float* v, float* root) {
  {
#pragma clang fp contract(off)
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      const float g = grad[e] * h.grad_scale;
      m[e] = h.beta1 * m[e] + h.one_minus_beta1 * g;
      v[e] = h.beta2 * v[e] + h.one_minus_beta2 * (g * g);
    }
  }
  sqrt4(v, root);
#pragma unroll
  for (int e = 0; e < kVec; ++e) {
    const float denom = root[e] * h.inv_root_bias + h.eps;    // never denormal: the host refuses such an eps
#if defined(__HIP_DEVICE_COMPILE__)
    const float update = m[e] * __builtin_amdgcn_rcpf(denom);  // one unit in the last place and one rounding
#else
    const float update = m[e] / denom;
#endif
    p[e] -= h.lr_decay * p[e] + h.step_size * update;   // the two small terms first: 1 - lr * decay would round them away
  }
}

// A tensor may start anywhere; the waves' shares are laid out so that their
// first moments start at multiples of 256 bytes.  Pieces of flat buffers that
// start at the same element of each have their other streams aligned with it.
// The first share then has this many elements before the tensor's start.
// Without it two waves share the cache lines at every border, and their
// non-temporal stores go to memory as partial lines: 300 tensors of odd sizes
// (43 Mi bf16 elements) 205 -> 172 us.
__host__ __device__ __forceinline__ uint32_t lead(const void* m) { return (uint32_t)((uintptr_t)m / 4 % 64); }

// Moments in 32 bits: one wave per 256 elements, 7-9 streams of which 4 are read
// and 3-4 written once.  Bound by HBM: 8 x 32 Mi elements, fp32 parameters, bf16
// gradients and copy, 7.52 GB in 1161-1184 us = 6.35-6.47 TB/s; all fp32 1145 us =
// 6.57; 300 ragged bf16 tensors, 0.94 GB in 149 us = 6.3.  Two or four times the
// elements a wave were slower (1286, 1310 us against 1254 before the occupancy
// was bounded, see adamw_lds): more bytes in flight spread over more DRAM pages.
template <class P, class G, class C, bool NT>
__global__ __launch_bounds__(kWave) void k_adamw(AdamTable args, const void* dev, int count, Hyper h) {
  const View<AdamEntry> t = view_of(args, dev, count);
  const int s = find_segment(t, count, blockIdx.x);
  if (!finish_hyper(h)) return;
  const uint32_t before = lead(t.e[s].m), item = blockIdx.x - t.start[s];
  const ptrdiff_t first = (ptrdiff_t)((size_t)item * kBlock) - before;
  const size_t end = t.e[s].n - (size_t)first;       // place of the tensor's end
  const Span span = {item ? 0 : before, at_most(end, kBlock)};
  const gptr pp = element(t.e[s].p, first, sizeof(typename P::elem));
  const cgptr gp = element(t.e[s].g, first, sizeof(typename G::elem));
  const gptr mp = element(t.e[s].m, first, 4);
  const gptr vp = element(t.e[s].v, first, 4);
  const gptr cp = C::kNone ? nullptr : element(t.e[s].c, first, 2);
  const uint32_t i = (threadIdx.x & (kWave - 1)) * kVec;
  with_bounds(span.lo == 0 && span.hi == kBlock, [&](auto full) {
    constexpr bool FULL = decltype(full)::value;
    const typename P::raw pw = load_upto4<P, NT, FULL>(pp, i, span);
    const typename G::raw gw = load_upto4<G, NT, FULL>(gp, i, span);
    const F32::raw mw = load_upto4<F32, NT, FULL>(mp, i, span), vw = load_upto4<F32, NT, FULL>(vp, i, span);
    float p[kVec], g[kVec], m[kVec], v[kVec], root[kVec];
    P::widen(pw, p);
    G::widen(gw, g);
    F32::widen(mw, m);
    F32::widen(vw, v);
    adamw4(h, p, g, m, v, root);
    store_upto4<P, NT, FULL>(pp, i, span, p);
    store_upto4<F32, NT, FULL>(mp, i, span, m);
    store_upto4<F32, NT, FULL>(vp, i, span, v);
    if constexpr (!C::kNone) store_upto4<C, NT, FULL>(cp, i, span, p);
  });
}

// Moments in 8 bits: one wave per U blocks, one after the other; the loads of a
// block are issued before the work on the one before it.  Eleven streams, and 193
// vector instructions a block (237 with random rounding), which keep the vector
// units 67-79 % busy: 8 x 32 Mi elements, fp32 parameters, bf16 gradients and
// copy, 4.31 GB in 695 us = 6.2 TB/s with either rounding (1, 2 or 4 blocks a
// wave with the best occupancy for each: 690-700).  With 16-bit parameters there
// is less memory time to hide the start of a wave behind, and two blocks share
// it: 2.7 GB in 512 us with one block a wave, 459 with two, 461 with four.
template <class P> constexpr int kAdam8Blocks = sizeof(typename P::elem) == 4 ? 1 : 2;
template <class P, class G, class C, int U, bool NT>
__global__ __launch_bounds__(kWave) void k_adamw8(Adam8Table args, const void* dev, int count, Hyper h) {
  if (kHostRun && threadIdx.x) return;
  const View<Adam8Entry> t = view_of(args, dev, count);
  const int s = find_segment(t, count, blockIdx.x);
  const size_t block = (size_t)(blockIdx.x - t.start[s]) * U, first = block * kBlock;
  const Span span = span_of(first, t.e[s].n, U * kBlock);
  const gptr pp = element(t.e[s].p, first, sizeof(typename P::elem));
  const cgptr gp = element(t.e[s].g, first, sizeof(typename G::elem));
  const gptr mp = element(t.e[s].m, first, 1);
  const gptr rp = element(t.e[s].r, first, 1);
  const gptr cp = C::kNone ? nullptr : element(t.e[s].c, first, 2);
  PCCL_GLOBAL float* const msp = (PCCL_GLOBAL float*)element(t.e[s].ms, block, 4);
  PCCL_GLOBAL float* const rsp = (PCCL_GLOBAL float*)element(t.e[s].rs, block, 4);
  with_bounds(span.hi == U * kBlock, [&](auto full) {
    constexpr bool FULL = decltype(full)::value;
    struct Loaded {
      typename P::raw p;
      typename G::raw g;
      uint32_t m, r;
      float ms, rs;
    } now[kLaneSlots], next[kLaneSlots];
    auto load = [&](int u, Loaded* l) {
      each_lane([&](int k, int lane) {
        const uint32_t i = u * kBlock + lane * kVec;
        l[k].p = load_upto4<P, NT, FULL>(pp, i, span);
        l[k].g = load_upto4<G, NT, FULL>(gp, i, span);
        l[k].m = load_codes<NT, FULL>(mp, i, span);
        l[k].r = load_codes<NT, FULL>(rp, i, span);
        l[k].ms = msp[u];
        l[k].rs = rsp[u];
      });
    };
    load(0, now);
    if (!finish_hyper(h)) return;      // behind the loads: it may wait for device memory itself
    const uint32_t key = noise_key(h.seed, h.step);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!FULL && u * kBlock >= span.hi) break;
      if (u + 1 < U && (FULL || (u + 1) * kBlock < span.hi)) load(u + 1, next);
      float m[kLaneSlots][kVec], r[kLaneSlots][kVec];
      uint32_t ma[kLaneSlots], ra[kLaneSlots];
      each_lane([&](int k, int lane) {
        const uint32_t i = u * kBlock + lane * kVec;
        float p[kVec], g[kVec], v[kVec];
        P::widen(now[k].p, p);
        G::widen(now[k].g, g);
        decode4(now[k].m, m[k]);
        decode4(now[k].r, r[k]);
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          m[k][e] *= now[k].ms;
          r[k][e] *= now[k].rs;
          v[e] = r[k][e] * r[k][e];
        }
        adamw4(h, p, g, m[k], v, r[k]);
        store_upto4<P, NT, FULL>(pp, i, span, p);
        if constexpr (!C::kNone) store_upto4<C, NT, FULL>(cp, i, span, p);
        ma[k] = amax4(m[k]);
        ra[k] = amax4(r[k]);
      });
      const BlockScale mb = block_scale(wave_max(ma)), rb = block_scale(wave_max(ra));
      each_lane([&](int k, int lane) {
        const uint32_t i = u * kBlock + lane * kVec;
        float y[kVec], z[kVec];
        uint32_t yc, zc;
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          y[e] = m[k][e] * mb.inv;
          z[e] = lift_root(r[k][e], r[k][e] * rb.inv);
        }
        if (h.stochastic) {
          uint32_t yb[kVec], zb[kVec];
#pragma unroll
          for (int e = 0; e < kVec; ++e) {
            const uint32_t bits = noise(key, first, i + e);
            yb[e] = bits << 16;
            zb[e] = bits & 0xffff0000u;
            y[e] = clamp_code(y[e]);
          }
          yc = encode4_stochastic(y, yb);
          zc = encode4_stochastic(z, zb);
        } else {
          yc = encode4(y);
          zc = encode4(z);
        }
        store_codes<NT, FULL>(mp, i, span, yc);
        store_codes<NT, FULL>(rp, i, span, zc);
        if (lane == 0) { msp[u] = mb.scale; rsp[u] = rb.scale; }
        now[k] = next[k];
      });
    }
  });
}

// ---------------------------------------------------------------------------
// 8-bit blocks
// ---------------------------------------------------------------------------
// One wave per U blocks, whose loads are all in flight before the first is used.
// Bound by HBM: 128 Mi elements bf16, 405 MB in 63.7 us = 6.35 TB/s; fp32, 671 MB
// in 101 us = 6.65, with roots 102; read back to bf16 63.5 us, to fp32 107 us =
// 6.3 TB/s.
template <class T, int U, bool NT>
__global__ __launch_bounds__(kWave) void k_quantize(BlocksTable args, int count, int root) {
  if (kHostRun && threadIdx.x) return;
  const View<BlocksEntry> t = view_of(args, nullptr, count);
  const uint32_t item0 = xcd_run(blockIdx.x, gridDim.x);
  const int s = find_segment(t, count, item0);
  const size_t block = (size_t)(item0 - t.start[s]) * U, first = block * kBlock;
  const Span span = span_of(first, t.e[s].n, U * kBlock);
  const gptr codes = element(t.e[s].codes, first, 1);
  const cgptr xp = element(t.e[s].x, first, sizeof(typename T::elem));
  PCCL_GLOBAL float* const scales = (PCCL_GLOBAL float*)element(t.e[s].scales, block, 4);
  with_bounds(span.hi == U * kBlock, [&](auto full) {
    constexpr bool FULL = decltype(full)::value;
    typename T::raw w[kLaneSlots][U];
    each_lane([&](int k, int lane) {
#pragma unroll
      for (int u = 0; u < U; ++u) w[k][u] = load_upto4<T, NT, FULL>(xp, u * kBlock + lane * kVec, span);
    });
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!FULL && u * kBlock >= span.hi) break;
      float x[kLaneSlots][kVec];
      uint32_t a[kLaneSlots];
      each_lane([&](int k, int) {
        T::widen(w[k][u], x[k]);
        if (root) sqrt4(x[k], x[k]);
        a[k] = amax4(x[k]);
      });
      const BlockScale b = block_scale(wave_max(a));
      each_lane([&](int k, int lane) {
        float y[kVec];
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          y[e] = x[k][e] * b.inv;
          if (root) y[e] = lift_root(x[k][e], y[e]);
        }
        store_codes<NT, FULL>(codes, u * kBlock + lane * kVec, span, encode4(y));
        if (lane == 0) scales[u] = b.scale;
      });
    }
  });
}

template <class T, int U, bool NT>
__global__ __launch_bounds__(kWave) void k_dequantize(BlocksTable args, int count, int root) {
  const View<BlocksEntry> t = view_of(args, nullptr, count);
  const uint32_t item0 = xcd_run(blockIdx.x, gridDim.x);
  const int s = find_segment(t, count, item0);
  const size_t block = (size_t)(item0 - t.start[s]) * U, first = block * kBlock;
  const Span span = span_of(first, t.e[s].n, U * kBlock);
  const cgptr codes = element(t.e[s].codes, first, 1);
  const gptr xp = element(t.e[s].x, first, sizeof(typename T::elem));
  const PCCL_GLOBAL float* const scales = (const PCCL_GLOBAL float*)element(t.e[s].scales, block, 4);
  const uint32_t lane4 = (threadIdx.x & (kWave - 1)) * kVec;
  with_bounds(span.hi == U * kBlock, [&](auto full) {
    constexpr bool FULL = decltype(full)::value;
    uint32_t w[U];
    float scale[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      w[u] = load_codes<NT, FULL>(codes, u * kBlock + lane4, span);
      scale[u] = FULL || u * kBlock < span.hi ? scales[u] : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[kVec];
      decode4(w[u], x);
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        x[e] *= scale[u];
        if (root) x[e] *= x[e];
      }
      store_upto4<T, NT, FULL>(xp, u * kBlock + lane4, span, x);
    }
  });
}

// ---------------------------------------------------------------------------
// gradient norm
// ---------------------------------------------------------------------------
constexpr int kNormUnroll = 8;                              // 16-byte vectors of a lane in one work item
constexpr size_t kNormBytes = (size_t)kWave * 16 * kNormUnroll;   // a work item: what one wave reads at once

// Sum over the threads of a workgroup, in a fixed order; valid in thread 0.
// `part`: the thread's own value on the device, all threads' on the host.
template <int T>
__device__ __forceinline__ double group_sum(const double* part) {
#if defined(__HIP_DEVICE_COMPILE__)
  __shared__ double waves[T / kWave];
  double x = part[0];
  for (int d = kWave / 2; d; d >>= 1) x += __shfl_xor(x, d);
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

// The elements of a 16-byte vector
template <class T> struct Vec16 {
  static constexpr int kCount = 16 / sizeof(typename T::elem);
  typedef typename T::elem elems __attribute__((ext_vector_type(kCount)));
  typedef float floats __attribute__((ext_vector_type(kCount)));
};

// Sum of the squares of a vector.  In fp32, as a tree of at most four roundings,
// where the result says that nothing overflowed and that what underflowed does
// not count; else (zeros, too) in 64 bits, where no square of an fp32 number is
// out of range.  All in 64 bits was bound by arithmetic (512 MiB of bf16: 186 us).
template <int N, class V> __device__ __forceinline__ double sum_squares(const V& x) {
  float t[N / 2];
#pragma unroll
  for (int e = 0; e < N / 2; ++e) t[e] = x[2 * e] * x[2 * e] + x[2 * e + 1] * x[2 * e + 1];
#pragma unroll
  for (int w = N / 4; w; w /= 2)
#pragma unroll
    for (int e = 0; e < w; ++e) t[e] += t[e + w];
  if (t[0] >= 0x1p-100f && t[0] <= 0x1p126f) return (double)t[0];
  double sum = 0;
#pragma unroll
  for (int e = 0; e < N; ++e) sum += (double)x[e] * (double)x[e];
  return sum;
}

// The partial sums, added up by the first wave of a workgroup in a fixed order;
// valid in thread 0.  They may have been written by other workgroups of the same
// launch on other dies, so they are read past the caches.
__device__ __forceinline__ double join_parts(const double* part, uint32_t count) {
  double sum[kLaneSlots];
  each_lane([&](int k, int lane) {
    double acc = 0;
#pragma unroll 4
    for (uint32_t i = lane; i < count; i += kWave) {
#if defined(__HIP_DEVICE_COMPILE__)
      acc += __hip_atomic_load(part + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#else
      acc += part[i];
#endif
    }
    sum[k] = acc;
  });
#if defined(__HIP_DEVICE_COMPILE__)
  for (int d = kWave / 2; d; d >>= 1) sum[0] += __shfl_xor(sum[0], d);
  return sum[0];
#else
  double total = 0;
  for (int l = 0; l < kWave; ++l) total += sum[l];
  return total;
#endif
}

// Writes a workgroup's partial sum and says to all its threads whether it was
// the last of the launch to do so.  The workgroups of a die count themselves at
// one place each, and the last ones of the dies at another: additions to one
// address take about 10 ns each, and 256 of them in a row were 2.5 us.  The
// counters, 64 bytes apart, are 0 before the launch and again after it.
constexpr uint32_t kTicketStep = 16;
static_assert(PCCL_OPTIM_TICKET_BYTES == (1 + kXcds) * kTicketStep * 4, "a counter per die, and one for the dies");

__device__ __forceinline__ bool last_to_write(double* part, double sum, uint32_t* ticket) {
  const uint32_t die = blockIdx.x % kXcds;
  const uint32_t of_die = (gridDim.x - die + kXcds - 1) / kXcds, dies = gridDim.x < kXcds ? gridDim.x : kXcds;
  uint32_t* const mine = ticket + (1 + die) * kTicketStep;
#if defined(__HIP_DEVICE_COMPILE__)
  __shared__ bool last;
  if (threadIdx.x == 0) {
    // All accesses are made where the dies meet, and the store is done when the counters say so.  (A release would
    // write the die's whole L2 back for it: 6 us on a norm of 1 GiB.)
    __hip_atomic_store(part, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    last = false;
    if (__hip_atomic_fetch_add(mine, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == of_die - 1) {
      __hip_atomic_store(mine, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (__hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == dies - 1) {
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
        __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = true;
      }
    }
  }
  __syncthreads();
  return last;
#else
  *part = sum;
  if (++*mine < of_die) return false;
  *mine = 0;
  if (++*ticket < dies) return false;
  *ticket = 0;
  return true;
#endif
}

// One partial sum per workgroup of T threads, to all[done + blockIdx.x]; every wave
// walks the work items that lie as many apart as the grid has waves.
// ALONE: the only workgroup of the whole norm; it writes the result itself.
// With a ticket the last workgroup to finish adds up the `parts` partial sums of
// this and the launches before it and writes the result; without one
// k_norm_join does, with the same bits, in a launch more (3 us: a norm of 8 x 1 Mi
// bf16 takes 7.0 us in one launch, 9.5 in two).
// Bound by HBM reads: 512 MiB of bf16 in 82.5 us = 6.5 TB/s, 1 GiB of fp32 in 160
// us = 6.7; a kernel that only reads 512 MiB takes 72 us.  Eight vectors a lane
// (8 KiB a wave) and 256 workgroups of 1024 were best (four: 87 us, two: 85).
template <class E, int T, bool NT, bool ALONE>
__global__ __launch_bounds__(T) void k_sum_squares(NormTable args, int count, uint32_t items, double* all, uint32_t parts,
                                                   uint32_t done, uint32_t* ticket, float* out) {
  if (kHostRun && threadIdx.x) return;
  typedef Vec16<E> V;
  typedef typename E::elem elem;
  constexpr uint32_t kElems = kNormBytes / sizeof(elem);
  constexpr int kSlots = kHostRun ? T : 1;
  const View<NormEntry> t = view_of(args, nullptr, count);
  double sum[kSlots];
  for (int k = 0; k < kSlots; ++k) {
    const uint32_t thread = kHostRun ? (uint32_t)k : threadIdx.x;
    const uint32_t lane = thread & (kWave - 1);
    double acc = 0;
    for (uint32_t item = blockIdx.x * (T / kWave) + wave_uniform(thread / kWave); item < items; item += gridDim.x * (T / kWave)) {
      const int s = find_segment(t, count, item);
      const size_t first = (size_t)(item - t.start[s]) * kElems;
      const uint32_t left = span_of(first, t.e[s].n, kElems).hi;
      const PCCL_GLOBAL elem* x = (const PCCL_GLOBAL elem*)element(t.e[s].x, first, sizeof(elem));
      if (left == kElems) {
        u32x4a w[kNormUnroll];
#pragma unroll
        for (int u = 0; u < kNormUnroll; ++u) w[u] = load16<NT>((cgptr)x + (u * kWave + lane) * 16u);
#pragma unroll
        for (int u = 0; u < kNormUnroll; ++u) {
          typename V::elems e;
          __builtin_memcpy(&e, &w[u], 16);
          acc += sum_squares<V::kCount>(__builtin_convertvector(e, typename V::floats));
        }
      } else {
        for (int u = 0; u < kNormUnroll; ++u) {
          const uint32_t i = (u * kWave + lane) * V::kCount;
          if (i + V::kCount <= left) {
            const u32x4a w = load16<false>((cgptr)x + i * (uint32_t)sizeof(elem));
            typename V::elems e;
            __builtin_memcpy(&e, &w, 16);
            acc += sum_squares<V::kCount>(__builtin_convertvector(e, typename V::floats));
          } else {
            for (uint32_t j = i; j < left && j < i + V::kCount; ++j) acc += (double)(float)x[j] * (double)(float)x[j];
          }
        }
      }
    }
    sum[k] = acc;
  }
  const double total = group_sum<T>(sum);
  if constexpr (ALONE) {
    if (threadIdx.x == 0) out[0] = (float)sqrt(total);
  } else if (!ticket) {
    if (threadIdx.x == 0) all[done + blockIdx.x] = total;
  } else if (last_to_write(all + done + blockIdx.x, total, ticket) && threadIdx.x < kWave) {
    const double norm2 = join_parts(all, parts);
    if (threadIdx.x == 0) out[0] = (float)sqrt(norm2);
  }
}

__global__ __launch_bounds__(kWave) void k_norm_join(const double* all, uint32_t parts, float* out) {
  if (kHostRun && threadIdx.x) return;
  const double norm2 = join_parts(all, parts);
  if (threadIdx.x == 0) out[0] = (float)sqrt(norm2);
}

}  // namespace pccl_optim_kernels

#endif  // PCCL_OPTIM_KERNELS_H
