"""Edges of pccl.optim: scales and codes next to a border, scalars next to the
ends of fp32, what a call marks as modified, how many tensors a launch and a
table hold, plans used from several threads."""
import math
import threading

import numpy as np
import pytest
import torch

import optim_oracle as Q
from optim_oracle import BLOCK, TYPES, f64
from test_optim import (HYPER, Flat, check_adamw, check_adamw8, cpu, make, values, values8, where)  # noqa: F401 - fixtures


def fp32(x):
    return np.asarray(x, np.float32)


# ---------------------------------------------------------------------------
# scales and codes: scale = a / 448 and code = e4m3(x / scale), each rounded once
# ---------------------------------------------------------------------------

def maxima(dtype, where):
    """Largest values of blocks: every mantissa of a 16-bit type, random ones of fp32, at exponents over the whole range."""
    if dtype == "bf16":
        bits = (np.arange(128, dtype=np.uint32) << 16) | (np.array([27, 40, 100, 127, 200, 254], np.uint32) << 23)[:, None]
        return bits.reshape(-1).view(np.float32)
    if dtype == "f16":
        return np.arange(0x0400, 0x7c00, 7 if where.name == "hip" else 31, dtype=np.uint16).view(np.float16).astype(np.float32)
    rng = np.random.default_rng(101)
    mantissa = rng.integers(0, 1 << 23, 4000 if where.name == "hip" else 1000).astype(np.uint32)
    exponent = rng.integers(27, 255, mantissa.size).astype(np.uint32)        # from 2^-100, below which the scale is that of 2^-100
    ends = fp32([2.0 ** -100, 1e-45, 0.0, np.finfo(np.float32).max, 1.0, 448.0, 1568.0])
    return np.concatenate([(exponent << 23 | mantissa).view(np.float32), ends])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_a_scale_is_the_rounded_quotient(where, dtype):
    from pccl import optim
    a = maxima(dtype, where)
    x = np.zeros((a.size, BLOCK), np.float32)
    x[np.arange(a.size), np.arange(a.size) * 37 % BLOCK] = a * np.where(np.arange(a.size) % 2, -1, 1)
    x = torch.from_numpy(x.reshape(-1)).to(TYPES[dtype]).to(where.device)
    codes, scales = optim.empty_blocks(x)
    optim.quantize_blocks([codes], [scales], [x])
    where.sync()
    want = np.maximum(fp32(a), fp32(2.0 ** -100)) / fp32(448)
    assert np.array_equal(scales.cpu().numpy(), want)


def test_a_scale_of_roots_is_the_rounded_quotient(where):
    from pccl import optim
    r = fp32(np.arange(1, 2000, 2))                    # exact roots
    x = np.zeros((r.size, BLOCK), np.float32)
    x[:, 5] = r * r
    x = torch.from_numpy(x.reshape(-1)).to(where.device)
    codes, scales = optim.empty_blocks(x)
    optim.quantize_blocks([codes], [scales], [x], root=True)
    where.sync()
    assert np.array_equal(scales.cpu().numpy(), r / fp32(448))


def test_codes_of_a_block_whose_scale_is_exact(where):
    """1568 / 448 is 3.5, and 4.15625 / 3.5, 5.03125 / 3.5 lie half way between two codes."""
    from pccl import optim
    x = torch.tensor([1568.0, 4.15625, 5.03125, -4.15625]).to(where.device)
    codes, scales = optim.empty_blocks(x)
    optim.quantize_blocks([codes], [scales], [x])
    where.sync()
    assert float(scales) == 3.5 and codes.float().cpu().tolist() == [448.0, 1.25, 1.5, -1.25]


# ---------------------------------------------------------------------------
# scalars
# ---------------------------------------------------------------------------

def test_scalars_that_leave_fp32_are_refused(cpu):
    """What the kernels hold in fp32 is checked there: 0 would turn clipping off, infinity the parameters into NaN."""
    from pccl import _native, optim
    norm, step_dev, lr_dev = torch.tensor([10.0]), torch.tensor([5]), torch.tensor([1e-3])

    def lists():
        return [torch.full((8,), x) for x in (1.0, 5.0, 0.0, 0.0)]
    for bad in (dict(max_norm=1e-46, norm=norm), dict(max_norm=7e-46, norm=norm), dict(max_norm=1e39, norm=norm), dict(eps=1e39),
                dict(lr=1e39), dict(lr=1e30, weight_decay=1e30), dict(lr=1e38)):
        ts = lists()
        with pytest.raises(_native.NativeError, match="is not allowed"):
            optim.adamw(*[[t] for t in ts], 1, **bad)
        assert all(torch.equal(a, b) for a, b in zip(ts, lists()))
    with pytest.raises(_native.NativeError, match="is not allowed"):
        optim.adamw(*[[t] for t in lists()], step_dev, lr=1e39)
    # 1e38 / (1 - beta1^t) fits once t is large, and the device's own lr replaces the host's
    optim.adamw(*[[t] for t in lists()], 1000, lr=1e38, weight_decay=0.0)
    optim.adamw(*[[t] for t in lists()], step_dev, lr=1e38, weight_decay=0.0)
    optim.adamw(*[[t] for t in lists()], 1, lr=lr_dev, weight_decay=1e39)


@pytest.mark.parametrize("max_norm", [2.0 ** -149, 1e-40, 1e38])
def test_the_smallest_and_largest_norm_to_clip_to(where, max_norm):
    from pccl import optim
    s = make([40], where.device, seed=71)
    old = values(s, "pgmv")
    norm = torch.tensor([10.0], device=where.device)
    optim.adamw(*(s[k].list for k in "pgmv"), 3, norm=norm, max_norm=max_norm, **HYPER)
    where.sync()
    # the clip factor is a denormal of one bit and its neighbours: off by half of 2^-149, a gradient below 1e-2 with it
    check_adamw(s, old, 3, "clip", norm=10.0, max_norm=max_norm, **HYPER)
