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
