"""The optimizer side of a sharded training step, on the GPU.

A data-parallel program that shards its optimizer reduces and scatters its
gradients, takes their norm, runs the optimizer on the shard it owns and gathers
the parameters again.  `pccl.kernels` does the two collectives; this module does
what lies between them, over many tensors at once:

    grad_norm                             2-norm over all gradients, kept on the GPU
    adamw, adamw8                         AdamW with moments in 32 or in 8 bits
    quantize_blocks, dequantize_blocks    tensors to 8-bit codes and back

Each has a plan_* form that checks its tensors once and is called many times on
the same buffers, which is what a training loop wants: a call is then a few
microseconds of host time (and 0.1 for each tensor that is no view of a common
buffer, for its version counter).  A plan works on the memory that its tensors
had when it was made and keeps that memory alive; give a parameter new storage
(`.data = ...`) and it needs a new plan, and do not resize storage under a plan.

Like the rest of the package every call validates on the host, enqueues on the
current stream of the tensors' device and returns; nothing synchronises, nothing
runs on the CPU.  Tensors are contiguous; they may start anywhere.  Calls may be
captured into a graph, which may outlive the plan but not the tensors; the step
count and learning rate can live in device tensors so that a replay reads them
anew.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple, Union

import torch

from . import _optim_native, kernels
from ._optim_native import BLOCK, TICKET_BYTES, Step

CODE_DTYPE = torch.float8_e4m3fn      # of the 8-bit codes

_increment_version = torch.autograd.graph.increment_version
_current_device = kernels._current_device or torch.cuda.current_device


def block_count(numel: int) -> int:
    """Scales of a tensor of `numel` elements in the 8-bit form."""
    return (numel + BLOCK - 1) // BLOCK


def empty_blocks(tensor: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) for `tensor`, all zero: a fresh 8-bit moment, or the
    buffers that quantize_blocks fills."""
    codes = torch.zeros(tensor.numel(), dtype=torch.uint8, device=tensor.device).view(CODE_DTYPE).view(tensor.shape)
    return codes, torch.zeros(block_count(tensor.numel()), dtype=torch.float32, device=tensor.device)


# ---------------------------------------------------------------------------
# checks
# ---------------------------------------------------------------------------

def _check_list(what, name, tensors, like=None, dtype=None):
    """A list of tensors as long as `like`, on one GPU, each with the size of its partner."""
    tensors = list(tensors)
    if like is None:
        like = tensors
    if len(tensors) != len(like):
        raise ValueError(f"{what}: need one {name} tensor per entry of the first list ({len(like)}), got {len(tensors)}")
    gpu = like[0].get_device() if like else -1
    for i, (t, p) in enumerate(zip(tensors, like)):
        kernels.check_device_tensor(t, name)
        if dtype is not None and t.dtype != dtype:
            raise RuntimeError(f"{what}: {name}[{i}] must be of type {dtype}, got {t.dtype}")
        if t is not p and t.shape != p.shape and (t.numel() != p.numel() or (t.dim() > 1 and p.dim() > 1)):
            raise RuntimeError(f"{what}: {name}[{i}] has shape {tuple(t.shape)}, its partner {tuple(p.shape)}")
        if t.get_device() != gpu:
            _check_device(what, f"{name}[{i}]", t, like[0].device)
    return tensors


def _check_device(what, name, t, device):
    if t.device != device:
        raise RuntimeError(f"{what}: all tensors must be on one GPU ({name} is on {t.device}, others on {device})")


def _check_scales(what, name, scales, codes):
    scales = list(scales)
    if len(scales) != len(codes):
        raise ValueError(f"{what}: need one {name} tensor per entry of the first list ({len(codes)}), got {len(scales)}")
    for i, (s, c) in enumerate(zip(scales, codes)):
        kernels.check_device_tensor(s, f"{name}[{i}]")
        if s.dtype != torch.float32 or s.numel() != block_count(c.numel()):
            raise RuntimeError(f"{what}: {name}[{i}] must hold {block_count(c.numel())} float32 scales (one per {BLOCK} elements)")
        if s.get_device() != c.get_device():
            _check_device(what, f"{name}[{i}]", s, c.device)
    return scales


def _type_codes(what, name, tensors):
    codes = {}
    for i, t in enumerate(tensors):
        if t.dtype not in codes:
            try:
                codes[t.dtype] = kernels.dtype_code(t.dtype)
            except RuntimeError:
                raise RuntimeError(f"{what}: {name}[{i}] must be float32, bfloat16 or float16, got {t.dtype}") from None
    return [codes[t.dtype] for t in tensors]


def _scalar(what, name, t, dtype, device):
    """Address of a one-element tensor that the kernel reads."""
    kernels.check_device_tensor(t, name)
    if t.dtype != dtype or t.numel() != 1:
        raise RuntimeError(f"{what}: {name} must be a tensor of one {dtype} element")
    if device is not None:
        _check_device(what, name, t, device)
    return t.data_ptr()


def _capturing(index):
    return index is not None and torch.cuda.is_current_stream_capturing()


def _hold(*lists):
    """The memory of the tensors: it lives as long as the plan, also when a tensor
    object is given other storage."""
    return [t.untyped_storage() for ts in lists if ts is not None for t in ts if t is not None]


class _Plan:
    def __init__(self, lib, native, device, keep, written=()):
        self._lib, self._native, self._handle, self._device, self._keep = lib, native, native.handle, device, keep
        self._index = device.index if device is not None and device.type == "cuda" else None
        # what to raise the version counters of, as an in-place torch operation would: views share their base's
        self._written = list({id(b): b for b in (t if t._base is None else t._base for t in written)}.values())

    def _on_device(self, fn, *args):
        """fn(*args, stream) on the current stream of the tensors' device, whatever the current device is."""
        if self._index is None or self._index == _current_device():
            return fn(*args, kernels.stream_handle())
        with torch.cuda.device(self._index):
            return fn(*args, kernels.stream_handle())

    def _run(self, fn, *args):
        rc = self._on_device(fn, *args)
        if rc:
            self._lib.check(rc)
        if self._written:
            _increment_version(self._written)

    # Some plans keep device memory of their own.  It is written, read and freed on
    # ONE stream, the one the plan was made on; calls on other streams and captured
    # calls (a graph may outlive the plan) do without it.
    _own = _own_stream = None

    def _make_own(self, make):
        def put(stream):
            if not _capturing(self._index):
                self._own, self._own_stream = make(), stream
        self._on_device(put)

    def _usable(self, stream):
        return self._own is not None and stream == self._own_stream and not _capturing(self._index)


# ---------------------------------------------------------------------------
# AdamW
# ---------------------------------------------------------------------------

class AdamWPlan(_Plan):
    """One AdamW step over fixed tensors; made by plan_adamw and plan_adamw8."""

    def _prepare(self, what, grads, lr, betas, eps, weight_decay, table):
        self._what = what
        self._like = [(g.numel(), g.shape, g.dtype) for g in grads]      # for calls that bring other gradients
        self._base = Step(beta1=betas[0], beta2=betas[1], eps=eps, weight_decay=weight_decay, grad_scale=1.0)
        self._set_lr(self._base, lr)
        if isinstance(lr, torch.Tensor):
            self._keep += _hold([lr])
        if table:
            self._make_table()

    def _set_lr(self, s, lr):
        if isinstance(lr, torch.Tensor):
            s.lr_dev = _scalar(self._what, "lr", lr, torch.float32, self._device)
        else:
            s.lr_dev, s.lr = None, lr

    def _make_table(self):
        """The addresses of more tensors than one launch takes in its arguments, in device memory."""
        size = self._lib.table_bytes(self._native)
        if not size:
            return

        def make():
            pinned = self._index is not None
            host = torch.empty(size, dtype=torch.uint8, pin_memory=pinned)
            self._lib.table_fill(self._native, host.data_ptr(), size)
            return host.to(self._device, non_blocking=True) if pinned else host
        self._make_own(make)

    def _step(self, grads, s, stream):
        table = self._own.data_ptr() if grads is None and self._usable(stream) else None
        return self._lib.run_adamw_fn(self._handle, grads, table, s, stream)

    def __call__(self, step: Union[int, torch.Tensor], *, grads: Optional[Sequence[torch.Tensor]] = None,
                 lr: Union[None, float, torch.Tensor] = None, grad_scale: float = 1.0,
                 norm: Optional[torch.Tensor] = None, max_norm: Optional[float] = None, skip_nonfinite: bool = False,
                 seed: Optional[int] = None) -> None:
        s = Step.from_buffer_copy(self._base)
        if isinstance(step, torch.Tensor):
            s.step_dev = _scalar(self._what, "step", step, torch.int64, self._device)
        else:
            s.step = step
        if lr is not None:
            self._set_lr(s, lr)
        s.grad_scale = grad_scale
        if norm is not None:
            s.norm = _scalar(self._what, "norm", norm, torch.float32, self._device)
        if max_norm is not None:
            if not max_norm > 0:
                raise ValueError(f"{self._what}: max_norm must be positive, got {max_norm}")
            s.max_norm = max_norm
        if skip_nonfinite:
            s.skip_nonfinite = 1
        if seed is not None:
            if not 0 <= seed < 1 << 32:
                raise ValueError(f"{self._what}: seed must be in [0, 2**32), got {seed}")
            s.stochastic, s.seed = 1, seed
        self._run(self._step, None if grads is None else self._other(grads), s)

    def _other(self, grads):
        grads = list(grads)
        if len(grads) != len(self._like):
            raise ValueError(f"{self._what}: the plan has {len(self._like)} gradients, got {len(grads)}")
        for i, (g, (n, shape, dtype)) in enumerate(zip(grads, self._like)):
            kernels.check_device_tensor(g, f"grads[{i}]")
            if g.dtype != dtype or g.numel() != n or (g.shape != shape and g.dim() > 1 and len(shape) > 1):
                raise RuntimeError(f"{self._what}: grads[{i}] must have the type and shape of the plan's "
                                   f"({dtype}, {tuple(shape)}), got {g.dtype}, {tuple(g.shape)}")
            _check_device(self._what, f"grads[{i}]", g, self._device)
        return _optim_native._ptr_table([g.data_ptr() for g in grads])


def _plan_adamw(what, eight, params, grads, first, second, scales, copies, lr, betas, eps, weight_decay, table=True):
    params = _check_list(what, "params", params)
    device = params[0].device if params else None
    grads = _check_list(what, "grads", grads, params)
    names = ("exp_avg", "exp_avg_rms" if eight else "exp_avg_sq")
    dtype = CODE_DTYPE if eight else torch.float32
    first = _check_list(what, names[0], first, params, dtype)
    second = _check_list(what, names[1], second, params, dtype)
    if eight:
        scales = [_check_scales(what, nm, s, params) for nm, s in zip(("avg_scale", "rms_scale"), scales)]
    ptypes, gtypes = _type_codes(what, "params", params), _type_codes(what, "grads", grads)
    ctypes_, cptrs = None, None
    if copies is not None:
        copies = list(copies)
        if len(copies) != len(params):
            raise ValueError(f"{what}: need one entry of copies per parameter ({len(params)}), got {len(copies)}")
        some = [i for i, c in enumerate(copies) if c is not None]
        _check_list(what, "copies", [copies[i] for i in some], [params[i] for i in some])
        ctypes_, cptrs = [_optim_native.NONE] * len(params), [0] * len(params)
        for i in some:
            ctypes_[i] = _type_codes(what, "copies", [copies[i]])[0]
            cptrs[i] = copies[i].data_ptr()
    lib = _optim_native.load()
    ptrs = kernels._ptrs
    n = [p.numel() for p in params]
    if eight:
        native = lib.plan_adamw8(ptrs(params), ptrs(grads), ptrs(first), ptrs(second), ptrs(scales[0]), ptrs(scales[1]),
                                 cptrs, n, ptypes, gtypes, ctypes_)
    else:
        native = lib.plan_adamw(ptrs(params), ptrs(grads), ptrs(first), ptrs(second), cptrs, n, ptypes, gtypes, ctypes_)
    written = params + first + second + [t for s in scales or () for t in s] + [c for c in copies or () if c is not None]
    plan = AdamWPlan(lib, native, device, _hold(params, grads, first, second, copies, *(scales or ())), written)
    plan._prepare(what, grads, lr, betas, eps, weight_decay, table)
    return plan


def plan_adamw(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avg: Sequence[torch.Tensor],
               exp_avg_sq: Sequence[torch.Tensor], *, copies: Optional[Sequence[Optional[torch.Tensor]]] = None,
               lr: Union[float, torch.Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2) -> AdamWPlan:
    """AdamW over many tensors, moments in float32.

    A call is one launch for up to 4096 tensors of the same types if it uses the
    plan's own gradients, on the stream that was current when the plan was made,
    and is not captured; else one per 64 tensors (plan_adamw8: 56).

    params   float32, bfloat16 or float16, updated in place in their own type
    grads    of any of these types, read only
    exp_avg, exp_avg_sq    float32, updated in place
    copies   None, or per float32 parameter a bfloat16 / float16 tensor (or
             None) that receives the updated parameter: the one to gather

    Call the plan once per step, `plan(step, ...)`:

    step        1 for the first step; or a one-element int64 tensor on the GPU
    grads       other gradients than the plan's, of the same types and shapes
                (a loop whose gradients are new tensors at every step passes them here)
    lr          another learning rate; or a one-element float32 tensor on the GPU
    grad_scale  factor of all gradients (1 / loss scale, 1 / ranks)
    norm, max_norm    the result of grad_norm over the gradients as they are
                (before grad_scale) and the norm to clip to: the gradients are
                scaled by min(1, max_norm / (norm * |grad_scale| + 1e-6))
    skip_nonfinite    with norm: write nothing at all when it is inf or NaN

    The update is p -= lr * weight_decay * p + lr * mhat / (sqrt(vhat) + eps),
    computed in float32.  Sixteen-bit parameters are rounded to nearest once per
    step, which loses updates below half a unit in their last place; keep float32
    parameters with 16-bit `copies` where that matters."""
    return _plan_adamw("adamw", False, params, grads, exp_avg, exp_avg_sq, None, copies, lr, betas, eps, weight_decay)


def plan_adamw8(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avg: Sequence[torch.Tensor],
                exp_avg_rms: Sequence[torch.Tensor], avg_scale: Sequence[torch.Tensor], rms_scale: Sequence[torch.Tensor],
                *, copies: Optional[Sequence[Optional[torch.Tensor]]] = None, lr: Union[float, torch.Tensor] = 1e-3,
                betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2) -> AdamWPlan:
    """plan_adamw with the moments in 8 bits: 2.03 bytes per element in place of 8.

    exp_avg, exp_avg_rms are float8_e4m3fn codes, avg_scale and rms_scale one
    float32 per 256 elements of each tensor (empty_blocks makes both, all zero).
    exp_avg_rms holds the square root of the second moment.

    The plan takes one argument more, `seed`: an int in [0, 2**32) rounds the
    moments stochastically, with random bits made from (seed, step, index of the
    element in its tensor); None rounds to nearest.  With beta2 = 0.999 a second
    moment moves by 0.05 % of its root a step while neighbouring codes are 6-12 %
    apart, so to nearest an element never moves against the others of its block;
    stochastically it follows on average.  Use a seed for training."""
    return _plan_adamw("adamw8", True, params, grads, exp_avg, exp_avg_rms, (avg_scale, rms_scale), copies, lr, betas, eps,
                       weight_decay)


def adamw(params, grads, exp_avg, exp_avg_sq, step, *, copies=None, lr=1e-3, betas=(0.9, 0.999), eps=1e-8,
          weight_decay=1e-2, grad_scale=1.0, norm=None, max_norm=None, skip_nonfinite=False) -> None:
    """One AdamW step; see plan_adamw."""
    plan = _plan_adamw("adamw", False, params, grads, exp_avg, exp_avg_sq, None, copies, lr, betas, eps, weight_decay,
                       table=False)
    plan(step, grad_scale=grad_scale, norm=norm, max_norm=max_norm, skip_nonfinite=skip_nonfinite)


def adamw8(params, grads, exp_avg, exp_avg_rms, avg_scale, rms_scale, step, *, seed=None, copies=None, lr=1e-3,
           betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, grad_scale=1.0, norm=None, max_norm=None,
           skip_nonfinite=False) -> None:
    """One AdamW step with moments in 8 bits; see plan_adamw8."""
    plan = _plan_adamw("adamw8", True, params, grads, exp_avg, exp_avg_rms, (avg_scale, rms_scale), copies, lr, betas, eps,
                       weight_decay, table=False)
    plan(step, grad_scale=grad_scale, norm=norm, max_norm=max_norm, skip_nonfinite=skip_nonfinite, seed=seed)


# ---------------------------------------------------------------------------
# gradient norm
# ---------------------------------------------------------------------------

class GradNormPlan(_Plan):
    """The norm of fixed tensors; made by plan_grad_norm."""

    def _prepare(self, keep_work):
        self._size = self._lib.norm_work(self._native)
        if self._size and keep_work:       # the partial sums and, behind them, the ticket
            self._make_own(lambda: torch.zeros(self._size + TICKET_BYTES, dtype=torch.uint8, device=self._device))

    def _norm(self, out, stream):
        if not self._size:
            return self._lib.run_norm_fn(self._handle, out, None, 0, None, stream)
        if self._usable(stream):
            at = self._own.data_ptr()
            return self._lib.run_norm_fn(self._handle, out, at, self._size, at + self._size, stream)
        # partial sums of this call alone: two streams or two graphs do not share them
        work = torch.empty(self._size // 8, dtype=torch.float64, device=self._device)
        return self._lib.run_norm_fn(self._handle, out, work.data_ptr(), self._size, None, stream)

    def __call__(self, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        if out is None:
            out = torch.empty(1, dtype=torch.float32, device=self._device)
            self._run(self._norm, out.data_ptr())
        else:
            self._run(self._norm, _scalar("grad_norm", "out", out, torch.float32, self._device))
            _increment_version(out)
        return out


def plan_grad_norm(tensors: Sequence[torch.Tensor]) -> GradNormPlan:
    """The 2-norm over all elements of all tensors (float32, bfloat16, float16,
    mixed as they come).  Calling the plan returns it as a one-element float32
    tensor on the GPU, or writes it into the one given.  No sum over- or
    underflows; inf or NaN among the elements gives inf or NaN; equal inputs give
    equal bits.  The norm over several ranks is the norm of their norms."""
    return _plan_grad_norm(tensors, True)


def _plan_grad_norm(tensors, keep_work):
    tensors = _check_list("grad_norm", "tensors", tensors)
    if not tensors:
        raise ValueError("grad_norm: need at least one tensor (it names the GPU)")
    device = tensors[0].device
    lib = _optim_native.load()
    native = lib.plan_norm(kernels._ptrs(tensors), [t.numel() for t in tensors], _type_codes("grad_norm", "tensors", tensors))
    plan = GradNormPlan(lib, native, device, _hold(tensors))
    plan._prepare(keep_work)
    return plan


def grad_norm(tensors: Sequence[torch.Tensor], out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The 2-norm over all elements of all tensors; see plan_grad_norm."""
    return _plan_grad_norm(tensors, False)(out)


# ---------------------------------------------------------------------------
# 8-bit blocks
# ---------------------------------------------------------------------------

class BlocksPlan(_Plan):
    """A conversion of fixed tensors; made by plan_quantize_blocks and plan_dequantize_blocks."""

    def __call__(self) -> None:
        self._run(self._lib.run_blocks_fn, self._handle)


def _plan_blocks(what, codes, scales, tensors, root):
    quantize = what == "quantize_blocks"
    tensors = _check_list(what, "tensors", tensors)
    device = tensors[0].device if tensors else None
    codes = _check_list(what, "codes", codes, tensors, CODE_DTYPE)
    scales = _check_scales(what, "scales", scales, tensors)
    types = _type_codes(what, "tensors", tensors)
    lib, ptrs, n = _optim_native.load(), kernels._ptrs, [t.numel() for t in tensors]
    if quantize:
        native = lib.plan_quantize(ptrs(codes), ptrs(scales), ptrs(tensors), n, types, root)
    else:
        native = lib.plan_dequantize(ptrs(tensors), ptrs(codes), ptrs(scales), n, types, root)
    return BlocksPlan(lib, native, device, _hold(codes, scales, tensors), codes + scales if quantize else tensors)


def plan_quantize_blocks(codes: Sequence[torch.Tensor], scales: Sequence[torch.Tensor], tensors: Sequence[torch.Tensor], *,
                         root: bool = False) -> BlocksPlan:
    """Tensors to float8_e4m3fn codes with one float32 scale per 256 elements.

    With a the largest magnitude of a block: scale = max(a, 2**-100) * (1 / 448),
    code = the e4m3 value nearest to x * (1 / scale), each operation rounded to
    float32, so x is off by at most 2**-4 of itself or 2**-10 of the scale (and by
    the roundings, 2**-22).  root=True is for second moments (x >= 0): the codes
    hold sqrt(x), and no x but 0 gets the code 0.  An inf or NaN spoils its whole
    block.  Codes and scales of the ranks' shards can be gathered like any other
    tensors (for that, let shards be multiples of 256)."""
    return _plan_blocks("quantize_blocks", codes, scales, tensors, root)


def plan_dequantize_blocks(tensors: Sequence[torch.Tensor], codes: Sequence[torch.Tensor], scales: Sequence[torch.Tensor], *,
                           root: bool = False) -> BlocksPlan:
    """The values that codes and scales stand for, code * scale (its square with
    root=True), into float32, bfloat16 or float16 tensors."""
    return _plan_blocks("dequantize_blocks", codes, scales, tensors, root)


def quantize_blocks(codes, scales, tensors, *, root: bool = False) -> None:
    """See plan_quantize_blocks."""
    plan_quantize_blocks(codes, scales, tensors, root=root)()


def dequantize_blocks(tensors, codes, scales, *, root: bool = False) -> None:
    """See plan_dequantize_blocks."""
    plan_dequantize_blocks(tensors, codes, scales, root=root)()
