/*
 * pccl_optim.h -- C ABI of the optimizer-side kernels in libpccl_hip.so: what a
 * sharded training step runs between the reduce_scatter of its gradients and
 * the all_gather of its parameters, written for gfx950 (MI355X).
 *
 *   gradient norm     2-norm over many tensors
 *   AdamW             one step over many tensors, moments in 32 or in 8 bits
 *   8-bit blocks      tensors to e4m3 codes with one scale per 256 elements, and
 *                     back (the form the 8-bit moments are held in)
 *
 * The conventions are those of pccl_hip.h: 0 or a negative PCCL_HIP_E* code
 * with a message for the calling thread; pointer tables are HOST arrays of
 * DEVICE pointers; no device memory is allocated, freed or retained; work is
 * only enqueued on `stream`, nothing synchronises.
 *
 * Plans.  Checking a few hundred tensors and building their tables costs more
 * than the step of a small shard, so every operator is described once
 * (pccl_optim_plan_*) and run many times.  A plan is host memory only: it holds
 * the addresses it was given, never changes after it was made, and may be run
 * from several threads, on several streams and inside graph capture.  The
 * caller keeps the tensors alive; a plan does not notice that one was freed.
 *
 * Tensors are given by address and number of elements and need the alignment
 * of their element type, no more.  Empty tensors are allowed.  A tensor has at
 * most PCCL_OPTIM_MAX_ELEMENTS elements.  Memory that an operator writes may
 * share no byte with anything else in the same plan (PCCL_HIP_EINVAL).
 */
#ifndef PCCL_OPTIM_H
#define PCCL_OPTIM_H

#include <stddef.h>
#include <stdint.h>

#include "pccl_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Elements that share one scale in the 8-bit form. */
#define PCCL_OPTIM_BLOCK 256

/* Longest tensor: 2^26 - 1 workgroups of one launch, 256 elements each, the
 * first and the last of them possibly not whole. */
#define PCCL_OPTIM_MAX_ELEMENTS (((size_t)1 << 34) - 512)

/* In place of an element type: no copy for this tensor. */
#define PCCL_OPTIM_NONE (-1)

typedef struct pccl_optim_plan pccl_optim_plan;

/* Message of the last failure of a pccl_optim_* call on the calling thread. */
const char* pccl_optim_last_error(void);

/* Frees a plan; NULL is allowed.  Launches already enqueued are not affected. */
void pccl_optim_plan_free(pccl_optim_plan* plan);

/* ---- AdamW ---------------------------------------------------------------
 * For every element of every tensor, in fp32 whatever the types:
 *
 *   g' = g * grad_scale * c           c = min(1, max_norm / (norm * |grad_scale| + 1e-6)),
 *   m  = beta1 m + (1 - beta1) g'         1 without a norm or with max_norm = 0
 *   v  = beta2 v + (1 - beta2) g'^2
 *   p  = p - lr weight_decay p - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
 *   copy = p                          rounded to the copy's type
 *
 * params: fp32, bf16 or fp16 (updated in their own type, rounded to nearest);
 * grads: any of the three; exp_avg, exp_avg_sq: fp32; copies: NULL, or per
 * tensor a bf16 / fp16 tensor of the same length (the parameters in the type
 * that is gathered and computed with) where the parameter is fp32 and
 * copy_dtype[i] is not PCCL_OPTIM_NONE. */
int pccl_optim_plan_adamw(pccl_optim_plan** plan, void* const* params, const void* const* grads, void* const* exp_avg,
                          void* const* exp_avg_sq, void* const* copies, const size_t* n, const int* param_dtype,
                          const int* grad_dtype, const int* copy_dtype, int count);

/* The same with both moments in 8 bits (see the block form below): exp_avg and
 * exp_avg_rms hold e4m3 codes (one byte per element), avg_scale and rms_scale
 * one float per 256 elements of each tensor.  exp_avg_rms holds sqrt(v), whose
 * range in decades is half that of v.  A step reads the moments back, updates
 * them and the parameter in fp32, and writes the moments again. */
int pccl_optim_plan_adamw8(pccl_optim_plan** plan, void* const* params, const void* const* grads, void* const* exp_avg,
                           void* const* exp_avg_rms, float* const* avg_scale, float* const* rms_scale,
                           void* const* copies, const size_t* n, const int* param_dtype, const int* grad_dtype,
                           const int* copy_dtype, int count);

typedef struct {
  double lr, beta1, beta2, eps, weight_decay;   /* eps: 0, or a normal fp32 number; lr, lr weight_decay and
                                                   lr / (1 - beta1^step): finite as fp32 numbers */
  double grad_scale;        /* factor of every gradient, e.g. 1 / (loss scale * ranks); finite and not 0 as an fp32 number */
  double max_norm;          /* clip to this norm, which must not become 0 or infinite as an fp32 number; 0 = no clipping */
  int64_t step;             /* t, 1 for the first step */
  const float* lr_dev;      /* NULL, or the learning rate in device memory (replaces lr: a replayed graph reads it anew) */
  const int64_t* step_dev;  /* NULL, or t in device memory (replaces step); a value below 1 counts as 1 */
  const float* norm;        /* NULL, or the norm of the unscaled gradients in device memory (pccl_optim_run_norm) */
  int skip_nonfinite;       /* with norm: write nothing at all when it is infinite or NaN */
  int stochastic;           /* 8-bit moments: 1 = stochastic rounding, 0 = to nearest, ties to even */
  uint32_t seed;            /* of the stochastic rounding; the random bits depend on seed, step and element index */
} pccl_optim_step;

/* The addresses of a plan's tensors travel in kernel arguments, which hold 64
 * (AdamW) or 56 (8-bit) tensors of the same types a launch.  For a plan with
 * more, pccl_optim_table_bytes says how large a table of all of them is (0:
 * there is nothing to gain); pccl_optim_table_fill writes it into HOST memory,
 * and the caller copies it to the GPU, to a multiple of 64 bytes.  A run that is
 * given that copy takes one launch per 4096 tensors.  The copy has to be
 * complete before the run on its stream and to stay until the run is done; a
 * captured run reads it at every replay. */
size_t pccl_optim_table_bytes(const pccl_optim_plan* plan);
int pccl_optim_table_fill(const pccl_optim_plan* plan, void* host, size_t bytes);

/* One step.  grads: NULL for the gradients of the plan, or others of the same
 * lengths and types (a table of `count` pointers) that share no memory with
 * what the plan writes.  table: NULL, or the plan's table in device memory
 * (ignored with other gradients, whose addresses it does not have). */
int pccl_optim_run_adamw(const pccl_optim_plan* plan, const void* const* grads, const void* table,
                         const pccl_optim_step* step, void* stream);

/* ---- gradient norm -------------------------------------------------------
 * out[0] = sqrt(sum of x^2 over all elements of all tensors), fp32; 0 for no
 * elements.  Squares of huge and of tiny values neither overflow nor vanish;
 * the partial sums are kept in 64 bits and joined in a fixed order, so equal
 * inputs give equal bits.  Inf or NaN anywhere gives inf or NaN.
 * `work`: pccl_optim_norm_work(plan) bytes (may be 0) of device memory, 8-byte
 * aligned, that nothing else uses until the launch is done; its contents do not
 * matter.  `ticket`: NULL, or PCCL_OPTIM_TICKET_BYTES of device memory that are
 * all 0 and are 0 again afterwards; the norm then takes one launch where it
 * takes two without, with the same result.  Runs that share a ticket must not
 * overlap.  Neither out, work nor ticket may lie in the tensors. */
#define PCCL_OPTIM_TICKET_BYTES 576
int pccl_optim_plan_norm(pccl_optim_plan** plan, const void* const* tensors, const size_t* n, const int* dtype, int count);
size_t pccl_optim_norm_work(const pccl_optim_plan* plan);
int pccl_optim_run_norm(const pccl_optim_plan* plan, float* out, void* work, size_t work_bytes, uint32_t* ticket, void* stream);

/* ---- 8-bit blocks --------------------------------------------------------
 * Blocks of 256 consecutive elements from the start of each tensor, the last
 * one possibly shorter.  With a the largest |x| of a block, every operation in
 * fp32 and rounded by itself:
 *
 *   scale = max(a, 2^-100) * (1 / 448)      code = e4m3(x * (1 / scale)), to nearest, ties to even
 *
 * (what elementary operations that divide by a multiplication with the reciprocal
 * give, bit for bit).  The products are within 2^-22 of the quotients: of a value
 * that is so near to the middle between two codes either neighbour may be taken.
 * root = 1 (x >= 0, second moments) holds sqrt(x) in place of x and gives a
 * value other than 0 at least the smallest code, 2^-9, so that it is not read
 * back as 0.  Read back: code * scale, or its square.  Inf or NaN in a block
 * makes the whole block read back as inf or NaN.
 * codes: 1 byte per element; scales: (n + 255) / 256 floats. */
int pccl_optim_plan_quantize(pccl_optim_plan** plan, void* const* codes, float* const* scales, const void* const* src,
                             const size_t* n, const int* dtype, int count, int root);
int pccl_optim_plan_dequantize(pccl_optim_plan** plan, void* const* dst, const void* const* codes,
                               const float* const* scales, const size_t* n, const int* dtype, int count, int root);
int pccl_optim_run_blocks(const pccl_optim_plan* plan, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* PCCL_OPTIM_H */
