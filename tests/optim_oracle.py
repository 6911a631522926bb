"""The optimizer-side operators from their definitions, in 64 bits, with the
error that fp32 arithmetic may add to each result, and the targets they run on."""
import os
import subprocess

import numpy as np
import pytest
import torch

from conftest import CSRC, HOST_CLANG, ROOT

U = 2.0 ** -24            # half a unit in the last place of fp32, relative
TINY = 2.0 ** -149        # smallest fp32 number: what an underflow loses at most
BLOCK = 256
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SMALLEST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def cpu_library(out=os.path.join(ROOT, "tests", "build", "libpccl_optim_cpu.so"), flags=("-O1",)):
    """The unchanged source of the operators, compiled for the host."""
    srcs = [os.path.join(CSRC, "pccl_optim.hip"), os.path.join(CSRC, "pccl_optim_kernels.h"),
            os.path.join(ROOT, "include", "pccl_hip.h"), os.path.join(ROOT, "include", "pccl_optim.h"),
            os.path.join(ROOT, "tests", "hip_cpu_shim", "hip", "hip_runtime.h")]
    if os.path.exists(out) and all(os.path.getmtime(out) >= os.path.getmtime(s) for s in srcs):
        return out
    if not os.path.exists(HOST_CLANG):
        pytest.skip("host clang++ of the ROCm toolchain not found")
    os.makedirs(os.path.dirname(out), exist_ok=True)
    part = f"{out}.{os.getpid()}"          # put in place whole: test processes may build it side by side
    subprocess.run([HOST_CLANG, "-x", "c++", "-std=c++17", "-g", "-fPIC", "-shared", "-ffp-contract=off", *flags,
                    "-I", os.path.join(ROOT, "tests", "hip_cpu_shim"), "-I", os.path.join(ROOT, "include"), "-I", CSRC,
                    "-o", part, srcs[0]], check=True, capture_output=True)
    os.replace(part, out)
    return out


def half_step(dtype):
    """Relative rounding error of a type."""
    return torch.finfo(dtype).eps / 2


def f64(t):
    return t.detach().double().cpu().numpy().reshape(-1)


def rounded(x, err, dtype):
    """Largest distance from x of a value within err of it that is then rounded to dtype."""
    return err + half_step(dtype) * (np.abs(x) + err) + SMALLEST[dtype] / 2


# ---------------------------------------------------------------------------
# AdamW
# ---------------------------------------------------------------------------

def adamw(p, g, m, v, step, *, lr, betas, eps, weight_decay, grad_scale=1.0, norm=None, max_norm=None, m_err=0.0, v_err=0.0):
    """{name: (value, error bound)} for p, m, v and sqrt(v), from 64-bit arrays.
    m_err, v_err: relative errors that the moments already carry when they are
    read (the 8-bit form multiplies a code by its scale, and squares)."""
    b1, b2 = betas
    c = 1.0
    if max_norm is not None:
        ratio = max_norm / (norm * abs(grad_scale) + 1e-6)
        c = ratio if not ratio >= 1 else 1.0
    g = g * (grad_scale * c)
    # grad_scale and max_norm rounded, norm * grad_scale, + 1e-6 (rounded), /, * grad_scale, * g
    eg = 8 * U * np.abs(g) + TINY
    a, b = b1 * m, (1 - b1) * g
    mn = a + b                         # factor and product rounded for each term, and the sum
    em = 3 * U * (np.abs(a) + np.abs(b)) + (1 - b1) * eg + np.abs(a) * m_err + 3 * TINY
    a, b = b2 * v, (1 - b2) * g * g
    vn = a + b                         # g^2 is one product more
    ev = 4 * U * (a + b) + (1 - b2) * (2 * np.abs(g) * eg + eg * eg) + a * v_err + 4 * TINY
    root = np.sqrt(vn)
    er = np.sqrt(vn + ev) - np.sqrt(np.maximum(vn - ev, 0)) + U * root + TINY
    bias1, bias2 = 1 - b1 ** step, np.sqrt(1 - b2 ** step)
    den = root / bias2 + eps           # 1 / bias2 and eps rounded, product, sum
    ed = er / bias2 + 3 * U * den + TINY
    with np.errstate(divide="ignore", invalid="ignore"):
        upd = mn / den
        # m * (1 / den): the reciprocal instruction is good to one unit in the last place (2 U), and one rounding
        eu = np.where(den > ed, (em + np.abs(upd) * ed) / np.maximum(den - ed, TINY) + 3.1 * U * np.abs(upd) + TINY, np.inf)
        size = lr / bias1
        change = lr * weight_decay * p + size * upd
        ec = 3 * U * (np.abs(lr * weight_decay * p) + np.abs(size * upd)) + size * eu + 3 * TINY
        pn = p - change
        ep = ec + U * (np.abs(pn) + ec)
    return {"p": (pn, ep), "m": (mn, em), "v": (vn, ev), "root": (root, er)}


# ---------------------------------------------------------------------------
# e4m3 blocks
# ---------------------------------------------------------------------------

def _mix(x):
    x = x & 0xffffffff
    x = x ^ (x >> 16)
    x = (x * 0x7feb352d) & 0xffffffff
    x = x ^ (x >> 15)
    x = (x * 0x846ca68b) & 0xffffffff
    return x ^ (x >> 16)


def noise(seed, step, n):
    """The 32 random bits of each of n elements."""
    return noise_at(seed, step, np.arange(n, dtype=np.uint64))


def noise_at(seed, step, i):
    """... of the elements with these indices (uint64)."""
    key, mask = _mix(_mix(seed) + step), np.uint64(0xffffffff)
    x = ((i & mask) + np.uint64(key) + (i >> np.uint64(32)) * np.uint64(0x9e3779b1)) & mask
    x ^= x >> np.uint64(16)
    x = (x * np.uint64(0x7feb352d)) & mask
    x ^= x >> np.uint64(15)
    x = (x * np.uint64(0x846ca68b)) & mask
    return x ^ (x >> np.uint64(16))


def spacing(y):
    """Distance of the e4m3 codes around |y|."""
    y = np.abs(y)
    e = np.where(y > 0, np.frexp(np.where(y > 0, y, 1))[1] - 1, -6)
    return 2.0 ** (np.maximum(e, -6) - 3)


def check_blocks(codes, scales, x, err, root, bits=None, what=""):
    """Codes (as values) and scales of one tensor against its values x, known to
    err.  bits: 16 random bits per element, or None for rounding to nearest.
    Every code has to be one that the definition gives for some value in reach."""
    n = x.size
    assert codes.size == n and scales.size == (n + BLOCK - 1) // BLOCK
    pad = scales.size * BLOCK - n
    x, err, codes = (np.pad(a, (0, pad)).reshape(-1, BLOCK) for a in (x, np.broadcast_to(err, x.shape), codes))
    bits = None if bits is None else np.pad(bits.astype(np.float64), (0, pad)).reshape(-1, BLOCK) / 65536
    top = np.abs(x).max(1)
    want = np.maximum(top, 2.0 ** -100) / 448
    reach = (np.abs(x) + err).max(1) - top + np.where(top > 0, 0, err.max(1))
    assert (np.abs(scales - want) <= (reach + U * top) / 448 + U * want).all(), f"{what}: scales"
    y = np.abs(x) / want[:, None]
    # the value's own error, the error of the scale, and the roundings of scale, 1 / scale and their product
    ey = err / want[:, None] + y * ((reach / want / 448)[:, None] + 5 * U)
    if root:
        lifted = np.where((x > 0) & (y < 2.0 ** -9), 2.0 ** -9, y)
        ey = np.where(lifted == y, ey, np.maximum(ey - (lifted - y), 0))
        # within reach of 0 both 0 and the smallest code are right
        maybe_zero = (x <= err) & (codes == 0)
        y = lifted
    else:
        maybe_zero = np.zeros_like(codes, bool)
    mag = np.abs(codes)
    low, high = np.maximum(y - ey, 0), y + ey
    if bits is None:
        def code_of(t):
            return np.minimum(np.round(t / spacing(t)) * spacing(t), 448)
    else:
        def code_of(t):      # below 2^-6 an fp32 sum rounds the value to a 2^-20 of the spacing: counted in the reach
            return np.minimum(np.floor(t / spacing(t) + bits) * spacing(t), 448)
        low, high = np.maximum(low - 2.0 ** -29, 0), high + 2.0 ** -29
    ok = ((mag >= code_of(low)) & (mag <= code_of(high))) | maybe_zero
    assert ok.all(), (what, np.argwhere(~ok)[:5], mag[~ok][:5], y[~ok][:5])
    flips = (codes != 0) & (np.abs(x) > err) & (np.sign(codes) != np.sign(x))
    assert not flips.any(), f"{what}: sign"
