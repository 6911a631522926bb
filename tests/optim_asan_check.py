"""Run by tests/test_optim_sanitizer.py in a child process with the
AddressSanitizer runtime preloaded: drives the instrumented CPU build of the
optimizer-side operators over numpy buffers without slack, so that any access
out of bounds ends the process.  Ragged, empty and misaligned tensors."""
import importlib.util
import os
import sys

import numpy as np

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sc2025-pccl-reproducer_amd", "pccl")
sys.path.insert(0, os.path.dirname(PKG))


def module(name):
    """A torch-free module of the package, without importing the package."""
    spec = importlib.util.spec_from_file_location("pccl_bare." + name, os.path.join(PKG, name + ".py"))
    mod = importlib.util.module_from_spec(spec)
    sys.modules["pccl_bare." + name] = mod
    spec.loader.exec_module(mod)
    return mod


import types  # noqa: E402

sys.modules["pccl_bare"] = types.ModuleType("pccl_bare")
sys.modules["pccl_bare"].__path__ = [PKG]
module("_native")
nat = module("_optim_native")
lib = nat.OptimLib(sys.argv[1])
rng = np.random.default_rng(0)
SIZE = {0: 4, 1: 2, 2: 2}
LENGTHS = [0, 1, 2, 3, 4, 5, 63, 64, 65, 127, 255, 256, 257, 1023, 1025, 2047, 4100]


def buffer(n, size, shift):
    """n elements of `size` bytes that start `shift` elements into an allocation and end with it."""
    a = np.zeros((n + shift) * size, np.uint8)
    return a, (a.ctypes.data + shift * size if n else 0)


def tensors(lengths, sizes, shift):
    both = [buffer(n, s, shift) for n, s in zip(lengths, sizes)]
    return [b[0] for b in both], [b[1] for b in both]


def fill(arrays, code):
    for a in arrays:
        x = rng.standard_normal(a.size // SIZE[code]).astype(np.float32)
        a[:] = (x if code == 0 else (x.view(np.uint32) >> 16).astype(np.uint16) if code == 1 else x.astype(np.float16)).view(np.uint8)


checked = 0
step = nat.Step(lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.1, grad_scale=1.0, step=3)
scalars = np.array([2.0], np.float32), np.array([5], np.int64), np.array([1e-3], np.float32)
for lengths in (LENGTHS, [7] * 150, [300]):
    count = len(lengths)
    blocks = [(n + 255) // 256 for n in lengths]
    for shift in (0, 1, 3):
        for pt, gt, ct in ((0, 0, -1), (0, 1, 1), (0, 2, 2), (1, 1, -1), (2, 0, -1)):
            keep, p = tensors(lengths, [SIZE[pt]] * count, shift)
            fill(keep, pt)
            kg, g = tensors(lengths, [SIZE[gt]] * count, shift)
            fill(kg, gt)
            kc, c = tensors(lengths, [2] * count, shift) if ct >= 0 else (None, None)
            for eight in (False, True):
                km, m = tensors(lengths, [1 if eight else 4] * count, shift)
                kv, v = tensors(lengths, [1 if eight else 4] * count, shift)
                types_ = ([pt] * count, [gt] * count, None if c is None else [ct] * count)
                if eight:
                    ks, s = tensors(blocks, [4] * count, 0)
                    kr, r = tensors(blocks, [4] * count, 0)
                    plan = lib.plan_adamw8(p, g, m, v, s, r, c, lengths, *types_)
                else:
                    plan = lib.plan_adamw(p, g, m, v, c, lengths, *types_)
                for mode in range(4):
                    if mode & 1:
                        step.norm, step.max_norm, step.step_dev, step.lr_dev = (
                            scalars[0].ctypes.data, 0.5, scalars[1].ctypes.data, scalars[2].ctypes.data)
                    else:
                        step.norm, step.max_norm, step.step_dev, step.lr_dev = None, 0.0, None, None
                    step.stochastic, step.seed = (1, 7) if eight and mode & 2 else (0, 0)
                    table, size = None, lib.table_bytes(plan)
                    if mode & 2 and size:
                        raw = np.zeros(size + 64, np.uint8)
                        table = (raw.ctypes.data + 63) // 64 * 64
                        lib.table_fill(plan, table, size)
                    lib.run_adamw(plan, step, g if mode == 1 else None, table)
                    checked += 1
        for code in (0, 1, 2):
            kx, x = tensors(lengths, [SIZE[code]] * count, shift)
            fill(kx, code)
            kq, q = tensors(lengths, [1] * count, shift)
            ks, s = tensors(blocks, [4] * count, 0)
            for root in (0, 1):
                if root:
                    for a in kx:      # second moments are not negative
                        a.view(np.uint32 if code == 0 else np.uint16)[:] &= 0x7fffffff if code == 0 else 0x7fff
                lib.run_blocks(lib.plan_quantize(q, s, x, lengths, [code] * count, root))
                lib.run_blocks(lib.plan_dequantize(x, q, s, lengths, [code] * count, root))
                checked += 2
            plan = lib.plan_norm(x, lengths, [code] * count)
            out = np.zeros(1, np.float32)
            work = np.zeros(lib.norm_work(plan), np.uint8)
            ticket = np.zeros(nat.TICKET_BYTES, np.uint8)
            both = []
            for counter in (0, ticket.ctypes.data):
                lib.run_norm(plan, out.ctypes.data, work.ctypes.data if work.size else 0, work.size, counter)
                both.append(out.tobytes())
            assert both[0] == both[1] and not ticket.any()
            checked += 2
print("ASAN CHECK OK", checked)
