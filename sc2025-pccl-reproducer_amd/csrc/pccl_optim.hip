// The optimizer-side operators of libpccl_hip.so behind the C ABI of
// include/pccl_optim.h: plans, checks and launches.  The kernels and what bounds
// them are in pccl_optim_kernels.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <exception>
#include <type_traits>
#include <vector>

#include "pccl_optim.h"
#include "pccl_optim_kernels.h"

using namespace pccl_optim_kernels;

namespace {

thread_local char g_err[512] = "";

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof g_err, fmt, ap);
  va_end(ap);
  return code;
}

// The status of a launch is what the launch call itself returns.
#ifndef PCCL_LAUNCH   // a host stand-in for the HIP runtime brings its own
thread_local hipError_t t_launch_error = hipSuccess;
template <class T> struct same_as { typedef T type; };
template <class... P>
void launch_kernel(void (*kernel)(P...), dim3 grid, dim3 block, unsigned lds, hipStream_t stream,
                   typename same_as<P>::type... args) {
  void* ptrs[] = {(void*)&args...};
  const hipError_t e = hipLaunchKernel((const void*)kernel, grid, block, ptrs, lds, stream);
  if (e != hipSuccess && t_launch_error == hipSuccess) t_launch_error = e;
}
#define PCCL_LAUNCH(kernel, grid, block, lds, stream, ...) launch_kernel(kernel, grid, block, lds, stream, __VA_ARGS__)
#else
hipError_t t_launch_error = hipSuccess;
#endif

int launch_status(const char* what) {
  const hipError_t e = t_launch_error;
  t_launch_error = hipSuccess;
  if (e != hipSuccess) return fail(PCCL_HIP_ELAUNCH, "%s: launch failed: %s", what, hipGetErrorString(e));
  return PCCL_HIP_OK;
}

// Plans whose tensors take this much memory together get the non-temporal hint on
// all accesses.  On data that has left the caches it is better at any size
// (AdamW over 29 / 117 / 235 MB: 9.8 / 25 / 43 us against 12.2 / 28 / 50; norm of
// 67 MB 17.5 against 29); on data that is still in the 256 MiB Infinity Cache it
// is worse (AdamW over 117 MB called on three such sets in turn 21.6 against
// 19.0).  A third of the cache is where calls in turn no longer find their data.
constexpr size_t kStreamFrom = (size_t)96 << 20;

// Work items of one launch.  The grid is counted in threads, in 32 bits.
constexpr size_t kMaxItems = ((size_t)1 << 26) - 1;

// Blocks of one wave: 4 KiB of what k_quantize reads (128 Mi elements, us at 1 / 2 / 4 / 8 blocks: bf16 135 101 72
// 67), 2 KiB of what k_dequantize writes (bf16 118 82 64 66; fp32 139 107 121 122).  Data that is still in the caches
// takes the same numbers, which were not measured apart for it.
template <class T> constexpr int kQuantizeBlocks = 4096 / (kBlock * sizeof(typename T::elem));
template <class T> constexpr int kDequantizeBlocks = 2048 / (kBlock * sizeof(typename T::elem));

constexpr int kNormThreads = 1024;        // threads of a workgroup of the norm
constexpr uint32_t kNormGroups = 256;     // workgroups, and partial sums, of one launch

size_t esize_of(int dtype) {
  return dtype == PCCL_HIP_F32 ? 4 : (dtype == PCCL_HIP_BF16 || dtype == PCCL_HIP_F16) ? 2 : 0;
}

enum Kind { kAdamW, kAdamW8, kNorm, kQuantize, kDequantize };

// Tensors that are alike in their types, for one launch or a few
struct Batch {
  int p, g, c;                 // element types; c = PCCL_OPTIM_NONE without a copy
  std::vector<int> tensor;     // their places in the plan
  std::vector<uint32_t> start;
  uint32_t items = 0;
};

struct Extent {
  uintptr_t lo, hi;   // [lo, hi)
  int index;
  const char* name;
  bool written;
};

}  // namespace

struct pccl_optim_plan {
  Kind kind;
  int count = 0, root = 0;
  bool stream = false;
  // by tensor; which of them are set depends on the kind
  std::vector<void*> a, b, c, d, e, f;   // AdamW: p, m, v, copy; AdamW8: p, m, r, copy, m scale, r scale; blocks: codes, scales, x
  std::vector<const void*> g;            // gradients, or the tensors of a norm
  std::vector<size_t> n;
  std::vector<int> gtype;
  std::vector<Batch> batches;
  std::vector<Extent> guarded;           // what a buffer that a run brings must not lie in, by address: what the plan
                                         // writes, and what a norm reads
};

namespace {

struct Checker {
  pccl_optim_plan& plan;
  const char* what;
  std::vector<Extent> all;

  int table(const void* tab, const char* name) const {
    if (plan.count && !tab) return fail(PCCL_HIP_EINVAL, "%s: %s is NULL", what, name);
    return PCCL_HIP_OK;
  }
  int type(int dtype, const char* name, int i) const {
    if (!esize_of(dtype))
      return fail(PCCL_HIP_EINVAL, "%s: unknown %s[%d] %d (0 = float32, 1 = bfloat16, 2 = float16)", what, name, i, dtype);
    return PCCL_HIP_OK;
  }
  // a tensor of the call: present, aligned to its elements, and noted for the overlap check
  int buffer(const void* p, size_t bytes, size_t align, const char* name, int i, bool written) {
    if (!bytes) return PCCL_HIP_OK;
    if (!p) return fail(PCCL_HIP_EINVAL, "%s: %s[%d] is NULL", what, name, i);
    if ((uintptr_t)p % align)
      return fail(PCCL_HIP_EINVAL, "%s: %s[%d] is not aligned to its element size (%zu bytes)", what, name, i, align);
    all.push_back(Extent{(uintptr_t)p, (uintptr_t)p + bytes, i, name, written});
    return PCCL_HIP_OK;
  }
  static int clash(const char* what, const Extent& x, const Extent& y) {
    return fail(PCCL_HIP_EINVAL, "%s: %s[%d] and %s[%d] overlap in memory (what an operator writes may share memory with nothing)",
                what, x.name, x.index, y.name, y.index);
  }
  // sweep by address: of what has started, the part that reaches farthest, and the written part that does
  int overlaps() {
    std::sort(all.begin(), all.end(), [](const Extent& x, const Extent& y) { return x.lo < y.lo; });
    const Extent *far = nullptr, *far_written = nullptr;
    for (const Extent& x : all) {
      if (x.written && far && far->hi > x.lo) return clash(what, *far, x);
      if (far_written && far_written->hi > x.lo) return clash(what, *far_written, x);
      if (!far || x.hi > far->hi) far = &x;
      if (x.written) far_written = &x;
      if (plan.kind == kNorm && !plan.guarded.empty() && plan.guarded.back().hi >= x.lo)
        plan.guarded.back().hi = std::max(plan.guarded.back().hi, x.hi);   // readers may overlap; kept apart and in order
      else if (x.written || plan.kind == kNorm) plan.guarded.push_back(x);
    }
    return PCCL_HIP_OK;
  }
};

// A buffer that a run brings along must not lie in what the plan guards.
int check_apart(const pccl_optim_plan& plan, const void* p, size_t bytes, const char* name, int i, const char* what) {
  if (!p || !bytes) return PCCL_HIP_OK;
  const Extent x{(uintptr_t)p, (uintptr_t)p + bytes, i, name, false};
  auto it = std::upper_bound(plan.guarded.begin(), plan.guarded.end(), x,
                             [](const Extent& u, const Extent& v) { return u.lo < v.lo; });
  if (it != plan.guarded.end() && it->lo < x.hi) return Checker::clash(what, *it, x);
  if (it != plan.guarded.begin() && (--it)->hi > x.lo) return Checker::clash(what, *it, x);
  return PCCL_HIP_OK;
}

// Puts the tensors that are not empty into batches: alike in type, in their
// order, at most `cap` of them.  items_of(i): the work items of tensor i.
template <class F>
int make_batches(pccl_optim_plan& plan, const int* p, const int* g, const int* c, F&& items_of, size_t cap, const char* what) {
  for (int i = 0; i < plan.count; ++i) {
    if (!plan.n[i]) continue;
    const int pt = p[i], gt = g ? g[i] : 0, ct = c ? c[i] : PCCL_OPTIM_NONE;
    const size_t items = items_of(i);
    if (items > kMaxItems)
      return fail(PCCL_HIP_EINVAL, "%s: tensor %d has %zu elements, more than one launch takes", what, i, plan.n[i]);
    Batch* to = nullptr;
    for (auto b = plan.batches.rbegin(); b != plan.batches.rend(); ++b)
      if (b->p == pt && b->g == gt && b->c == ct) {     // the last one of these types is the one that is open
        if (b->tensor.size() < cap && b->items + items <= kMaxItems) to = &*b;
        break;
      }
    if (!to) {
      plan.batches.push_back(Batch{pt, gt, ct, {}, {}, 0});
      to = &plan.batches.back();
    }
    to->tensor.push_back(i);
    to->start.push_back(to->items);
    to->items += (uint32_t)items;
  }
  return PCCL_HIP_OK;
}

// The entries of tensors in a table
void fill(AdamEntry& e, const pccl_optim_plan& plan, int i, const void* const* grads) {
  e = AdamEntry{plan.a[i], grads ? grads[i] : plan.g[i], plan.b[i], plan.c[i], plan.d[i], plan.n[i]};
}
void fill(Adam8Entry& e, const pccl_optim_plan& plan, int i, const void* const* grads) {
  e = Adam8Entry{plan.a[i], grads ? grads[i] : plan.g[i], plan.b[i], plan.c[i], (float*)plan.e[i], (float*)plan.f[i],
                 plan.d[i], plan.n[i]};
}
void fill(BlocksEntry& e, const pccl_optim_plan& plan, int i, const void* const*) {
  e = BlocksEntry{plan.a[i], (float*)plan.b[i], plan.c[i], plan.n[i]};
}
void fill(NormEntry& e, const pccl_optim_plan& plan, int i, const void* const*) { e = NormEntry{plan.g[i], plan.n[i]}; }

// A launch's share of a batch
struct Share {
  int count;
  uint32_t items;
  const void* dev;     // the table in device memory, or NULL
};

// launch(table, share) for a batch: once where its table lies in device memory,
// else as often as it takes to pass all tensors in kernel arguments.
template <class T, class F>
void each_launch(const pccl_optim_plan& plan, const Batch& b, const void* const* grads, const void* dev, F&& launch) {
  T t;
  const int total = (int)b.tensor.size();
  if (dev) {
    launch(t, Share{total, b.items, dev});
    return;
  }
  for (int k0 = 0; k0 < total; k0 += T::kInline) {
    const int count = std::min(total - k0, T::kInline);
    for (int k = 0; k < count; ++k) {
      fill(t.e[k], plan, b.tensor[k0 + k], grads);
      t.start[k] = b.start[k0 + k] - b.start[k0];
    }
    const uint32_t end = k0 + count < total ? b.start[k0 + count] : b.items;
    launch(t, Share{count, end - b.start[k0], nullptr});
  }
}

// Device tables: batch after batch, each its entries and then their first work items, from multiples of 64 bytes
template <class E> size_t table_size(const Batch& b) {
  return (b.tensor.size() * (sizeof(E) + sizeof(uint32_t)) + 63) / 64 * 64;
}
template <class T> size_t table_bytes(const pccl_optim_plan& plan) {
  size_t bytes = 0;
  bool more = false;         // than one launch takes in its arguments: only then is a table worth having
  for (const Batch& b : plan.batches) {
    bytes += table_size<typename T::entry>(b);
    more = more || b.tensor.size() > (size_t)T::kInline;
  }
  return more ? bytes : 0;
}
template <class T> void table_fill(const pccl_optim_plan& plan, char* to) {
  typedef typename T::entry E;
  for (const Batch& b : plan.batches) {
    for (size_t k = 0; k < b.tensor.size(); ++k) {
      E e;
      fill(e, plan, b.tensor[k], nullptr);
      memcpy(to + k * sizeof(E), &e, sizeof(E));
      memcpy(to + b.tensor.size() * sizeof(E) + k * sizeof(uint32_t), &b.start[k], sizeof(uint32_t));
    }
    to += table_size<E>(b);
  }
}

// Runs `make` on a new plan.  Nothing that the standard library throws leaves the library.
template <class F>
int new_plan(pccl_optim_plan** out, Kind kind, int count, const size_t* n, const char* what, F&& make) {
  if (!out) return fail(PCCL_HIP_EINVAL, "%s: plan is NULL", what);
  *out = nullptr;
  if (count < 0) return fail(PCCL_HIP_EINVAL, "%s: count %d is negative", what, count);
  if (count && !n) return fail(PCCL_HIP_EINVAL, "%s: n is NULL", what);
  pccl_optim_plan* plan = nullptr;
  int rc;
  try {
    plan = new pccl_optim_plan;
    plan->kind = kind;
    plan->count = count;
    plan->n.assign(n, n + count);
    Checker check{*plan, what, {}};
    rc = PCCL_HIP_OK;
    for (int i = 0; i < count && !rc; ++i)
      if (n[i] > PCCL_OPTIM_MAX_ELEMENTS)
        rc = fail(PCCL_HIP_EINVAL, "%s: tensor %d has %zu elements, more than %zu", what, i, n[i], (size_t)PCCL_OPTIM_MAX_ELEMENTS);
    if (!rc) rc = make(*plan, check);
    if (!rc) {
      rc = check.overlaps();
      size_t bytes = 0;
      for (const Extent& x : check.all) bytes += x.hi - x.lo;
      plan->stream = bytes >= kStreamFrom;
    }
  } catch (const std::exception& e) {
    rc = fail(PCCL_HIP_EINVAL, "%s: %s", what, e.what());
  }
  if (rc) { delete plan; return rc; }
  *out = plan;
  return PCCL_HIP_OK;
}

size_t items_for(size_t n, size_t per) { return (n + per - 1) / per; }
size_t blocks_of(size_t n) { return (n + kBlock - 1) / kBlock; }

// What AdamW with moments of either width checks and keeps.
int make_adamw(pccl_optim_plan& plan, Checker& check, void* const* params, const void* const* grads, void* const* m,
               void* const* v, float* const* ms, float* const* vs, void* const* copies, const int* pt, const int* gt,
               const int* ct) {
  const bool eight = plan.kind == kAdamW8;
  const char* vname = eight ? "exp_avg_rms" : "exp_avg_sq";
  int rc;
  if ((rc = check.table(params, "params")) || (rc = check.table(grads, "grads")) || (rc = check.table(m, "exp_avg")) ||
      (rc = check.table(v, vname)) || (rc = check.table(pt, "param_dtype")) || (rc = check.table(gt, "grad_dtype")))
    return rc;
  if (eight && ((rc = check.table(ms, "avg_scale")) || (rc = check.table(vs, "rms_scale")))) return rc;
  if (copies && (rc = check.table(ct, "copy_dtype"))) return rc;
  std::vector<int> ctype(plan.count, PCCL_OPTIM_NONE);
  for (int i = 0; i < plan.count; ++i) {
    const size_t n = plan.n[i], es = eight ? 1 : 4;
    if ((rc = check.type(pt[i], "param_dtype", i)) || (rc = check.type(gt[i], "grad_dtype", i))) return rc;
    if (copies && ct[i] != PCCL_OPTIM_NONE) {
      if (ct[i] != PCCL_HIP_BF16 && ct[i] != PCCL_HIP_F16)
        return fail(PCCL_HIP_EINVAL, "%s: copy_dtype[%d] is %d: a copy is bfloat16 or float16", check.what, i, ct[i]);
      if (pt[i] != PCCL_HIP_F32)
        return fail(PCCL_HIP_EINVAL, "%s: copies[%d]: only a float32 parameter has a copy", check.what, i);
      ctype[i] = ct[i];
    }
    if ((rc = check.buffer(params[i], n * esize_of(pt[i]), esize_of(pt[i]), "params", i, true)) ||
        (rc = check.buffer(grads[i], n * esize_of(gt[i]), esize_of(gt[i]), "grads", i, false)) ||
        (rc = check.buffer(m[i], n * es, es, "exp_avg", i, true)) || (rc = check.buffer(v[i], n * es, es, vname, i, true)))
      return rc;
    if (eight && ((rc = check.buffer(ms[i], blocks_of(n) * 4, 4, "avg_scale", i, true)) ||
                  (rc = check.buffer(vs[i], blocks_of(n) * 4, 4, "rms_scale", i, true))))
      return rc;
    if (ctype[i] != PCCL_OPTIM_NONE && (rc = check.buffer(copies[i], n * 2, 2, "copies", i, true))) return rc;
    plan.a.push_back(params[i]);
    plan.g.push_back(grads[i]);
    plan.b.push_back(m[i]);
    plan.c.push_back(v[i]);
    plan.d.push_back(ctype[i] != PCCL_OPTIM_NONE ? copies[i] : nullptr);
    plan.e.push_back(eight ? ms[i] : nullptr);
    plan.f.push_back(eight ? vs[i] : nullptr);
    plan.gtype.push_back(gt[i]);
  }
  auto items = [&](int i) {
    if (!eight) return blocks_of(plan.n[i] + lead(m[i]));
    return items_for(plan.n[i], kBlock * (esize_of(pt[i]) == 4 ? kAdam8Blocks<F32> : kAdam8Blocks<BF16>));
  };
  return make_batches(plan, pt, gt, ctype.data(), items, kTableMax, check.what);
}

int make_hyper(const pccl_optim_plan& plan, const pccl_optim_step& s, Hyper& h, const char* what) {
  auto bad = [&](const char* name, double x) { return fail(PCCL_HIP_EINVAL, "%s: %s = %g is not allowed", what, name, x); };
  // what the kernels hold in fp32 is checked as that: 0 there means something else, and infinity gives NaN
  auto fits = [](double x) { return std::isfinite((float)x); };
  if (!(s.lr >= 0) || !fits(s.lr)) return bad("lr", s.lr);
  if (!(s.beta1 >= 0 && s.beta1 < 1)) return bad("beta1", s.beta1);
  if (!(s.beta2 >= 0 && s.beta2 < 1)) return bad("beta2", s.beta2);
  if (!(s.eps >= 0) || !fits(s.eps) || (s.eps > 0 && s.eps < 0x1p-126)) return bad("eps", s.eps);
  if (!(s.weight_decay >= 0) || !std::isfinite(s.weight_decay)) return bad("weight_decay", s.weight_decay);
  if (!s.lr_dev && !fits(s.lr * s.weight_decay)) return bad("lr * weight_decay", s.lr * s.weight_decay);
  if (!fits(s.grad_scale) || (float)s.grad_scale == 0.0f) return bad("grad_scale", s.grad_scale);
  if (!(s.max_norm >= 0) || !fits(s.max_norm) || (s.max_norm > 0 && (float)s.max_norm == 0.0f)) return bad("max_norm", s.max_norm);
  if (s.max_norm > 0 && !s.norm) return fail(PCCL_HIP_EINVAL, "%s: max_norm without a norm", what);
  if (s.skip_nonfinite && !s.norm) return fail(PCCL_HIP_EINVAL, "%s: skip_nonfinite without a norm", what);
  if (!s.step_dev && s.step < 1) return fail(PCCL_HIP_EINVAL, "%s: step %lld: the first step is 1", what, (long long)s.step);
  if (s.stochastic && plan.kind != kAdamW8)
    return fail(PCCL_HIP_EINVAL, "%s: stochastic rounding is for moments in 8 bits", what);
  const struct { const void* p; size_t bytes; const char* name; } scalars[] = {
      {s.lr_dev, 4, "lr_dev"}, {s.step_dev, 8, "step_dev"}, {s.norm, 4, "norm"}};
  for (const auto& x : scalars) {
    if ((uintptr_t)x.p % x.bytes) return fail(PCCL_HIP_EINVAL, "%s: %s is not aligned to %zu bytes", what, x.name, x.bytes);
    if (int rc = check_apart(plan, x.p, x.bytes, x.name, 0, what)) return rc;
  }
  memset(&h, 0, sizeof h);
  h.beta1 = (float)s.beta1;
  h.one_minus_beta1 = (float)(1.0 - s.beta1);
  h.beta2 = (float)s.beta2;
  h.one_minus_beta2 = (float)(1.0 - s.beta2);
  h.eps = (float)s.eps;
  h.grad_scale = (float)s.grad_scale;
  h.max_norm = (float)s.max_norm;
  h.scale_high = std::max(1.0f, std::fabs(h.grad_scale));
  h.scale_low = h.grad_scale / h.scale_high;
  h.norm_added = 1e-6f / h.scale_high;
  h.skip_nonfinite = s.skip_nonfinite != 0;
  h.stochastic = s.stochastic != 0;
  h.seed = s.seed;
  h.step = s.step_dev ? 1 : (uint64_t)s.step;
  h.lr = s.lr;
  h.beta1_d = s.beta1;
  h.beta2_d = s.beta2;
  h.weight_decay = s.weight_decay;
  h.lr_dev = s.lr_dev;
  h.step_dev = s.step_dev;
  h.norm = s.norm;
  h.lr_decay = (float)(s.lr * s.weight_decay);
  const double step_size = s.lr / (1.0 - std::pow(s.beta1, (double)h.step));
  if (!s.lr_dev && !s.step_dev && !fits(step_size)) return bad("lr / (1 - beta1^step)", step_size);
  h.step_size = (float)step_size;
  h.inv_root_bias = (float)(1.0 / std::sqrt(1.0 - std::pow(s.beta2, (double)h.step)));
  return PCCL_HIP_OK;
}

// Calls f.template operator()<P, G, C>() for the types of a batch.
template <class P, class G, class F> void with_copy(int c, F&& f) {
  if constexpr (!std::is_same<P, F32>::value) f.template operator()<P, G, None>();
  else if (c == PCCL_HIP_BF16) f.template operator()<P, G, BF16>();
  else if (c == PCCL_HIP_F16) f.template operator()<P, G, F16>();
  else f.template operator()<P, G, None>();
}
template <class P, class F> void with_grad(int g, int c, F&& f) {
  if (g == PCCL_HIP_F32) with_copy<P, F32>(c, f);
  else if (g == PCCL_HIP_BF16) with_copy<P, BF16>(c, f);
  else with_copy<P, F16>(c, f);
}
template <class F> void with_types(const Batch& b, F&& f) {
  if (b.p == PCCL_HIP_F32) with_grad<F32>(b.g, b.c, f);
  else if (b.p == PCCL_HIP_BF16) with_grad<BF16>(b.g, b.c, f);
  else with_grad<F16>(b.g, b.c, f);
}

// Unused LDS of a workgroup of k_adamw when it streams from HBM: it takes the
// room of further waves on a CU (160 KiB of LDS), and fewer of them ask the
// memory for a narrower window of each of the 7-9 streams at any moment.
// Measured on MI355X, 8 tensors of 32 Mi elements, us at 0 / 6 / 8 / 9 / 10 / 11 / 13 KiB:
//   fp32 parameters, bf16 gradients, bf16 copy   1264 1244 1193 1179 1181 1167 1180
//   fp32 parameters, fp32 gradients              1219 1227 1183 1164 1163 1150 1144
//   bf16 parameters, bf16 gradients               942  923  905  905  905  914  969
// k_adamw8, which computes more per byte, loses by every limit that has an
// effect (688 without, 737 at 6 KiB).
unsigned adamw_lds(const pccl_optim_plan& plan, const Batch& b) {
  return !plan.stream ? 0 : b.p == PCCL_HIP_F32 ? 11264 : 8192;
}

struct AdamLaunch {
  const pccl_optim_plan& plan;
  const Batch& b;
  const Hyper& h;
  const void* const* grads;
  const void* dev;
  hipStream_t stream;
  template <class P, class G, class C> void operator()() const {
    if (plan.kind == kAdamW)
      each_launch<AdamTable>(plan, b, grads, dev, [&](const AdamTable& t, const Share& s) {
        const unsigned lds = adamw_lds(plan, b);
        if (plan.stream) PCCL_LAUNCH((k_adamw<P, G, C, true>), dim3(s.items), dim3(kWave), lds, stream, t, s.dev, s.count, h);
        else PCCL_LAUNCH((k_adamw<P, G, C, false>), dim3(s.items), dim3(kWave), lds, stream, t, s.dev, s.count, h);
      });
    else
      each_launch<Adam8Table>(plan, b, grads, dev, [&](const Adam8Table& t, const Share& s) {
        if (plan.stream) PCCL_LAUNCH((k_adamw8<P, G, C, kAdam8Blocks<P>, true>), dim3(s.items), dim3(kWave), 0, stream, t, s.dev, s.count, h);
        else PCCL_LAUNCH((k_adamw8<P, G, C, kAdam8Blocks<P>, false>), dim3(s.items), dim3(kWave), 0, stream, t, s.dev, s.count, h);
      });
  }
};

// f.template operator()<T>() for an element type
template <class F> void with_type(int dtype, F&& f) {
  if (dtype == PCCL_HIP_F32) f.template operator()<F32>();
  else if (dtype == PCCL_HIP_BF16) f.template operator()<BF16>();
  else f.template operator()<F16>();
}

struct BlocksLaunch {
  const pccl_optim_plan& plan;
  const Batch& b;
  hipStream_t stream;
  template <class T> void operator()() const {
    constexpr int Q = kQuantizeBlocks<T>, D = kDequantizeBlocks<T>;
    each_launch<BlocksTable>(plan, b, nullptr, nullptr, [&](const BlocksTable& t, const Share& s) {
      if (plan.kind == kQuantize) {
        if (plan.stream) PCCL_LAUNCH((k_quantize<T, Q, true>), dim3(s.items), dim3(kWave), 0, stream, t, s.count, plan.root);
        else PCCL_LAUNCH((k_quantize<T, Q, false>), dim3(s.items), dim3(kWave), 0, stream, t, s.count, plan.root);
      } else {
        if (plan.stream) PCCL_LAUNCH((k_dequantize<T, D, true>), dim3(s.items), dim3(kWave), 0, stream, t, s.count, plan.root);
        else PCCL_LAUNCH((k_dequantize<T, D, false>), dim3(s.items), dim3(kWave), 0, stream, t, s.count, plan.root);
      }
    });
  }
};

uint32_t norm_grid(uint32_t items) { return std::min<uint32_t>((items + kNormThreads / kWave - 1) / (kNormThreads / kWave), kNormGroups); }

// One workgroup does the whole norm where that takes less time than finding the
// last of several: 32 work items of 8 KiB, two a wave, 6.1 us against 6.8; 64 of
// them 8.0 against 6.8.
constexpr uint32_t kNormAlone = 32;
bool norm_alone(const pccl_optim_plan& plan) { return plan.batches.size() == 1 && plan.batches[0].items <= kNormAlone; }

uint32_t norm_parts(const pccl_optim_plan& plan) {
  if (norm_alone(plan)) return 0;
  uint32_t parts = 0;
  for (const Batch& b : plan.batches) parts += norm_grid(b.items);
  return parts;
}

struct NormLaunch {
  const pccl_optim_plan& plan;
  const Batch& b;
  double* all;
  uint32_t done;        // partial sums of the launches before this one
  uint32_t* ticket;     // of the last launch only
  float* out;
  hipStream_t stream;
  template <class T> void operator()() const {
    const uint32_t parts = norm_parts(plan);
    // a batch of a norm is never longer than a table in kernel arguments
    each_launch<NormTable>(plan, b, nullptr, nullptr, [&](const NormTable& t, const Share& s) {
      const dim3 grid(norm_alone(plan) ? 1 : norm_grid(s.items)), block(kNormThreads);
      if (norm_alone(plan))
        PCCL_LAUNCH((k_sum_squares<T, kNormThreads, false, true>), grid, block, 0, stream, t, s.count, s.items, all, parts, done, ticket, out);
      else if (plan.stream)
        PCCL_LAUNCH((k_sum_squares<T, kNormThreads, true, false>), grid, block, 0, stream, t, s.count, s.items, all, parts, done, ticket, out);
      else
        PCCL_LAUNCH((k_sum_squares<T, kNormThreads, false, false>), grid, block, 0, stream, t, s.count, s.items, all, parts, done, ticket, out);
    });
  }
};

int check_plan(const pccl_optim_plan* plan, const char* what, Kind a, Kind b) {
  if (!plan) return fail(PCCL_HIP_EINVAL, "%s: plan is NULL", what);
  if (plan->kind != a && plan->kind != b) return fail(PCCL_HIP_EINVAL, "%s: the plan is for another operator", what);
  return PCCL_HIP_OK;
}

int plan_blocks(pccl_optim_plan** out, Kind kind, const void* const* codes, const float* const* scales, const void* const* x,
                const size_t* n, const int* dtype, int count, int root, const char* what) {
  return new_plan(out, kind, count, n, what, [&](pccl_optim_plan& plan, Checker& check) {
    const bool q = kind == kQuantize;
    const char* xname = q ? "src" : "dst";
    int rc;
    if ((rc = check.table(codes, "codes")) || (rc = check.table(scales, "scales")) || (rc = check.table(x, xname)) ||
        (rc = check.table(dtype, "dtype")))
      return rc;
    plan.root = root != 0;
    for (int i = 0; i < count; ++i) {
      if ((rc = check.type(dtype[i], "dtype", i))) return rc;
      const size_t es = esize_of(dtype[i]);
      if ((rc = check.buffer(codes[i], n[i], 1, "codes", i, q)) ||
          (rc = check.buffer(scales[i], blocks_of(n[i]) * 4, 4, "scales", i, q)) ||
          (rc = check.buffer(x[i], n[i] * es, es, xname, i, !q)))
        return rc;
      plan.a.push_back((void*)codes[i]);
      plan.b.push_back((void*)scales[i]);
      plan.c.push_back((void*)x[i]);
    }
    auto items = [&](int i) { return items_for(n[i], (q ? 4096 : 2048) / esize_of(dtype[i])); };
    return make_batches(plan, dtype, nullptr, nullptr, items, BlocksTable::kInline, what);
  });
}

}  // namespace

extern "C" {

const char* pccl_optim_last_error(void) { return g_err; }

void pccl_optim_plan_free(pccl_optim_plan* plan) { delete plan; }

int pccl_optim_plan_adamw(pccl_optim_plan** plan, void* const* params, const void* const* grads, void* const* exp_avg,
                          void* const* exp_avg_sq, void* const* copies, const size_t* n, const int* param_dtype,
                          const int* grad_dtype, const int* copy_dtype, int count) {
  return new_plan(plan, kAdamW, count, n, "pccl_optim_plan_adamw", [&](pccl_optim_plan& p, Checker& check) {
    return make_adamw(p, check, params, grads, exp_avg, exp_avg_sq, nullptr, nullptr, copies, param_dtype, grad_dtype,
                      copy_dtype);
  });
}

int pccl_optim_plan_adamw8(pccl_optim_plan** plan, void* const* params, const void* const* grads, void* const* exp_avg,
                           void* const* exp_avg_rms, float* const* avg_scale, float* const* rms_scale,
                           void* const* copies, const size_t* n, const int* param_dtype, const int* grad_dtype,
                           const int* copy_dtype, int count) {
  return new_plan(plan, kAdamW8, count, n, "pccl_optim_plan_adamw8", [&](pccl_optim_plan& p, Checker& check) {
    return make_adamw(p, check, params, grads, exp_avg, exp_avg_rms, avg_scale, rms_scale, copies, param_dtype, grad_dtype,
                      copy_dtype);
  });
}

size_t pccl_optim_table_bytes(const pccl_optim_plan* plan) {
  if (!plan) return 0;
  return plan->kind == kAdamW ? table_bytes<AdamTable>(*plan) : plan->kind == kAdamW8 ? table_bytes<Adam8Table>(*plan) : 0;
}

int pccl_optim_table_fill(const pccl_optim_plan* plan, void* host, size_t bytes) {
  const char* what = "pccl_optim_table_fill";
  if (int rc = check_plan(plan, what, kAdamW, kAdamW8)) return rc;
  const size_t need = pccl_optim_table_bytes(plan);
  if (!need) return PCCL_HIP_OK;
  if (!host || bytes < need) return fail(PCCL_HIP_EINVAL, "%s: needs %zu bytes, got %zu", what, need, host ? bytes : (size_t)0);
  memset(host, 0, need);
  if (plan->kind == kAdamW) table_fill<AdamTable>(*plan, (char*)host);
  else table_fill<Adam8Table>(*plan, (char*)host);
  return PCCL_HIP_OK;
}

int pccl_optim_run_adamw(const pccl_optim_plan* plan, const void* const* grads, const void* table, const pccl_optim_step* step,
                         void* stream) {
  const char* what = "pccl_optim_run_adamw";
  if (int rc = check_plan(plan, what, kAdamW, kAdamW8)) return rc;
  if (!step) return fail(PCCL_HIP_EINVAL, "%s: step is NULL", what);
  if (table && !pccl_optim_table_bytes(plan)) return fail(PCCL_HIP_EINVAL, "%s: this plan has no table", what);
  if ((uintptr_t)table % 64) return fail(PCCL_HIP_EINVAL, "%s: table is not aligned to 64 bytes", what);
  Hyper h;
  if (int rc = make_hyper(*plan, *step, h, what)) return rc;
  if (grads)
    for (int i = 0; i < plan->count; ++i) {
      const size_t es = esize_of(plan->gtype[i]);
      if (!plan->n[i]) continue;
      if (!grads[i]) return fail(PCCL_HIP_EINVAL, "%s: grads[%d] is NULL", what, i);
      if ((uintptr_t)grads[i] % es)
        return fail(PCCL_HIP_EINVAL, "%s: grads[%d] is not aligned to its element size (%zu bytes)", what, i, es);
      if (int rc = check_apart(*plan, grads[i], plan->n[i] * es, "grads", i, what)) return rc;
    }
  const char* dev = grads ? nullptr : (const char*)table;
  for (const Batch& b : plan->batches) {
    with_types(b, AdamLaunch{*plan, b, h, grads, dev, (hipStream_t)stream});
    if (dev) dev += plan->kind == kAdamW ? table_size<AdamEntry>(b) : table_size<Adam8Entry>(b);
  }
  return launch_status(what);
}

int pccl_optim_plan_norm(pccl_optim_plan** plan, const void* const* tensors, const size_t* n, const int* dtype, int count) {
  const char* what = "pccl_optim_plan_norm";
  return new_plan(plan, kNorm, count, n, what, [&](pccl_optim_plan& p, Checker& check) {
    int rc;
    if ((rc = check.table(tensors, "tensors")) || (rc = check.table(dtype, "dtype"))) return rc;
    for (int i = 0; i < count; ++i) {
      if ((rc = check.type(dtype[i], "dtype", i))) return rc;
      if ((rc = check.buffer(tensors[i], n[i] * esize_of(dtype[i]), esize_of(dtype[i]), "tensors", i, false))) return rc;
      p.g.push_back(tensors[i]);
    }
    return make_batches(p, dtype, nullptr, nullptr, [&](int i) { return items_for(n[i] * esize_of(dtype[i]), kNormBytes); },
                        NormTable::kInline, what);
  });
}

size_t pccl_optim_norm_work(const pccl_optim_plan* plan) {
  return plan && plan->kind == kNorm ? (size_t)norm_parts(*plan) * sizeof(double) : 0;
}

int pccl_optim_run_norm(const pccl_optim_plan* plan, float* out, void* work, size_t work_bytes, uint32_t* ticket, void* stream) {
  const char* what = "pccl_optim_run_norm";
  if (int rc = check_plan(plan, what, kNorm, kNorm)) return rc;
  if (!out) return fail(PCCL_HIP_EINVAL, "%s: out is NULL", what);
  if ((uintptr_t)out % 4) return fail(PCCL_HIP_EINVAL, "%s: out is not aligned to 4 bytes", what);
  if ((uintptr_t)ticket % 4) return fail(PCCL_HIP_EINVAL, "%s: ticket is not aligned to 4 bytes", what);
  const size_t need = pccl_optim_norm_work(plan);
  if (need && (!work || work_bytes < need))
    return fail(PCCL_HIP_EINVAL, "%s: needs %zu bytes of work space, got %zu", what, need, work ? work_bytes : (size_t)0);
  if (need && (uintptr_t)work % sizeof(double)) return fail(PCCL_HIP_EINVAL, "%s: work is not aligned to 8 bytes", what);
  const struct { const void* p; size_t bytes; const char* name; } own[] = {
      {out, 4, "out"}, {need ? work : nullptr, need, "work"}, {ticket, PCCL_OPTIM_TICKET_BYTES, "ticket"}};
  for (const auto& x : own)
    if (int rc = check_apart(*plan, x.p, x.bytes, x.name, 0, what)) return rc;
  uint32_t done = 0;
  for (const Batch& b : plan->batches) {
    const bool last = &b == &plan->batches.back();
    with_type(b.p, NormLaunch{*plan, b, (double*)work, done, last ? ticket : nullptr, out, (hipStream_t)stream});
    done += norm_grid(b.items);
  }
  if (plan->batches.empty() || (!ticket && !norm_alone(*plan)))
    PCCL_LAUNCH(k_norm_join, dim3(1), dim3(kWave), 0, (hipStream_t)stream, (const double*)work, norm_parts(*plan), out);
  return launch_status(what);
}

int pccl_optim_plan_quantize(pccl_optim_plan** plan, void* const* codes, float* const* scales, const void* const* src,
                             const size_t* n, const int* dtype, int count, int root) {
  return plan_blocks(plan, kQuantize, codes, scales, src, n, dtype, count, root, "pccl_optim_plan_quantize");
}

int pccl_optim_plan_dequantize(pccl_optim_plan** plan, void* const* dst, const void* const* codes,
                               const float* const* scales, const size_t* n, const int* dtype, int count, int root) {
  return plan_blocks(plan, kDequantize, codes, scales, dst, n, dtype, count, root, "pccl_optim_plan_dequantize");
}

int pccl_optim_run_blocks(const pccl_optim_plan* plan, void* stream) {
  const char* what = "pccl_optim_run_blocks";
  if (int rc = check_plan(plan, what, kQuantize, kDequantize)) return rc;
  for (const Batch& b : plan->batches) with_type(b.p, BlocksLaunch{*plan, b, (hipStream_t)stream});
  return launch_status(what);
}

}  // extern "C"
