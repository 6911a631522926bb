"""ctypes binding of the optimizer-side part of libpccl_hip.so (C ABI: include/pccl_optim.h).

Like `_native`, everything here works on plain integers; torch never appears.
"""
from __future__ import annotations

import ctypes
import os
import threading
from typing import Optional, Sequence

from ._native import LIB_PATH, NativeError, _ptr_table, _size_table

BLOCK = 256                       # elements that share one scale
MAX_ELEMENTS = (1 << 34) - 512    # of one tensor
TICKET_BYTES = 576                # counters of a norm in one launch
NONE = -1                         # in place of an element type: no copy

_vp = ctypes.c_void_p
_sz = ctypes.c_size_t
_int = ctypes.c_int
_vpp = ctypes.POINTER(ctypes.c_void_p)
_szp = ctypes.POINTER(ctypes.c_size_t)
_intp = ctypes.POINTER(ctypes.c_int)


class Step(ctypes.Structure):
    """pccl_optim_step"""
    _fields_ = [("lr", ctypes.c_double), ("beta1", ctypes.c_double), ("beta2", ctypes.c_double),
                ("eps", ctypes.c_double), ("weight_decay", ctypes.c_double), ("grad_scale", ctypes.c_double),
                ("max_norm", ctypes.c_double), ("step", ctypes.c_int64), ("lr_dev", _vp), ("step_dev", _vp),
                ("norm", _vp), ("skip_nonfinite", _int), ("stochastic", _int), ("seed", ctypes.c_uint32)]


# name -> (restype, argtypes); must list every symbol include/pccl_optim.h declares
SIGNATURES = {
    "pccl_optim_last_error": (ctypes.c_char_p, []),
    "pccl_optim_plan_free": (None, [_vp]),
    "pccl_optim_plan_adamw": (_int, [_vpp, _vpp, _vpp, _vpp, _vpp, _vpp, _szp, _intp, _intp, _intp, _int]),
    "pccl_optim_plan_adamw8": (_int, [_vpp, _vpp, _vpp, _vpp, _vpp, _vpp, _vpp, _vpp, _szp, _intp, _intp, _intp, _int]),
    "pccl_optim_table_bytes": (_sz, [_vp]),
    "pccl_optim_table_fill": (_int, [_vp, _vp, _sz]),
    "pccl_optim_run_adamw": (_int, [_vp, _vpp, _vp, ctypes.POINTER(Step), _vp]),
    "pccl_optim_plan_norm": (_int, [_vpp, _vpp, _szp, _intp, _int]),
    "pccl_optim_norm_work": (_sz, [_vp]),
    "pccl_optim_run_norm": (_int, [_vp, _vp, _vp, _sz, _vp, _vp]),
    "pccl_optim_plan_quantize": (_int, [_vpp, _vpp, _vpp, _vpp, _szp, _intp, _int, _int]),
    "pccl_optim_plan_dequantize": (_int, [_vpp, _vpp, _vpp, _vpp, _szp, _intp, _int, _int]),
    "pccl_optim_run_blocks": (_int, [_vp, _vp]),
}


def _int_table(vals: Optional[Sequence[int]]):
    return None if vals is None else (ctypes.c_int * len(vals))(*vals)


class Plan:
    """A native plan; freed with the object."""

    def __init__(self, lib: "OptimLib", handle):
        self.lib, self.handle = lib, handle

    def __del__(self):
        handle, self.handle = getattr(self, "handle", None), None
        if handle:
            self.lib._lib.pccl_optim_plan_free(handle)


class OptimLib:
    """One loaded build of the library."""

    def __init__(self, path: str = LIB_PATH):
        if not os.path.exists(path):
            raise RuntimeError(
                f"{path} not found: the HIP library has not been built. "
                "Run `make -C sc2025-pccl-reproducer_amd/csrc` (or pccl.build_kernels.build()) first; "
                "there is no fallback implementation.")
        self.path = path
        self._lib = ctypes.CDLL(path)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(self._lib, name)   # AttributeError if the symbol is missing
            fn.restype = res
            fn.argtypes = args
        self.run_adamw_fn = self._lib.pccl_optim_run_adamw
        self.run_norm_fn = self._lib.pccl_optim_run_norm
        self.run_blocks_fn = self._lib.pccl_optim_run_blocks

    def last_error(self) -> str:
        return self._lib.pccl_optim_last_error().decode("utf-8", "replace")

    def check(self, rc: int):
        if rc:
            raise NativeError(self.last_error() or f"libpccl_hip error {rc}")

    def _plan(self, fn, *args) -> Plan:
        handle = ctypes.c_void_p()
        self.check(fn(ctypes.byref(handle), *args))
        return Plan(self, handle)

    # -- plans (addresses are ints) ----------------------------------------
    def plan_adamw(self, params, grads, exp_avg, exp_avg_sq, copies, n, param_dtype, grad_dtype, copy_dtype) -> Plan:
        return self._plan(self._lib.pccl_optim_plan_adamw, _ptr_table(params), _ptr_table(grads), _ptr_table(exp_avg),
                          _ptr_table(exp_avg_sq), _ptr_table(copies), _size_table(n), _int_table(param_dtype),
                          _int_table(grad_dtype), _int_table(copy_dtype), len(n))

    def plan_adamw8(self, params, grads, exp_avg, exp_avg_rms, avg_scale, rms_scale, copies, n, param_dtype, grad_dtype,
                    copy_dtype) -> Plan:
        return self._plan(self._lib.pccl_optim_plan_adamw8, _ptr_table(params), _ptr_table(grads), _ptr_table(exp_avg),
                          _ptr_table(exp_avg_rms), _ptr_table(avg_scale), _ptr_table(rms_scale), _ptr_table(copies),
                          _size_table(n), _int_table(param_dtype), _int_table(grad_dtype), _int_table(copy_dtype), len(n))

    def plan_norm(self, tensors, n, dtype) -> Plan:
        return self._plan(self._lib.pccl_optim_plan_norm, _ptr_table(tensors), _size_table(n), _int_table(dtype), len(n))

    def plan_quantize(self, codes, scales, src, n, dtype, root=False) -> Plan:
        return self._plan(self._lib.pccl_optim_plan_quantize, _ptr_table(codes), _ptr_table(scales), _ptr_table(src),
                          _size_table(n), _int_table(dtype), len(n), 1 if root else 0)

    def plan_dequantize(self, dst, codes, scales, n, dtype, root=False) -> Plan:
        return self._plan(self._lib.pccl_optim_plan_dequantize, _ptr_table(dst), _ptr_table(codes), _ptr_table(scales),
                          _size_table(n), _int_table(dtype), len(n), 1 if root else 0)

    # -- runs ----------------------------------------------------------------
    def table_bytes(self, plan: Plan) -> int:
        return self._lib.pccl_optim_table_bytes(plan.handle)

    def table_fill(self, plan: Plan, host: int, nbytes: int):
        self.check(self._lib.pccl_optim_table_fill(plan.handle, host, nbytes))

    def run_adamw(self, plan: Plan, step: Step, grads=None, table=None, stream=0):
        self.check(self.run_adamw_fn(plan.handle, _ptr_table(grads), table, ctypes.byref(step), stream))

    def norm_work(self, plan: Plan) -> int:
        return self._lib.pccl_optim_norm_work(plan.handle)

    def run_norm(self, plan: Plan, out, work=0, work_bytes=0, ticket=0, stream=0):
        self.check(self.run_norm_fn(plan.handle, out, work, work_bytes, ticket, stream))

    def run_blocks(self, plan: Plan, stream=0):
        self.check(self.run_blocks_fn(plan.handle, stream))


_lock = threading.Lock()
_loaded: Optional[OptimLib] = None


def load() -> OptimLib:
    """The process-wide library instance; raises if it has not been built."""
    global _loaded
    with _lock:
        if _loaded is None:
            _loaded = OptimLib(LIB_PATH)
        return _loaded
