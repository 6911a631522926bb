"""AdamW with 32- and 8-bit moments, the gradient norm and the 8-bit blocks
(pccl.optim) against their definitions in 64 bits (optim_oracle), on the GPU and
on the CPU build of the same source."""
import math
import threading

import numpy as np
import pytest
import torch

import optim_oracle as Q
from conftest import Target
from optim_oracle import BLOCK, SMALLEST, TYPES, U, f64

HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05)
# around the 4 elements of a lane and the 256 of a wave and block
EDGES = [0, 1, 2, 3, 4, 5, 63, 64, 65, 255, 256, 257, 511, 513, 1000, 4099]


def _cpu(monkeypatch):
    from pccl import _optim_native, kernels
    lib = _optim_native.OptimLib(Q.cpu_library())

    def check_host_tensor(t, name):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if not t.is_contiguous():
            raise RuntimeError(f"{name} tensor must be contiguous.")

    monkeypatch.setattr(_optim_native, "_loaded", lib)
    monkeypatch.setattr(kernels, "check_device_tensor", check_host_tensor)
    monkeypatch.setattr(kernels, "stream_handle", lambda: 0)
    return Target("cpu-build", "cpu", lib)


@pytest.fixture(params=[pytest.param("hip", marks=pytest.mark.gpu), "cpu-build"])
def where(request, monkeypatch):
    if request.param == "hip":
        from pccl import _optim_native
        return Target("hip", "cuda:0", _optim_native.load())
    return _cpu(monkeypatch)


@pytest.fixture
def cpu(monkeypatch):
    return _cpu(monkeypatch)


class Flat:
    """Tensors of given sizes at given distances in one buffer, so that they start
    at any multiple of their element; what lies between them must not change."""

    def __init__(self, sizes, dtype, device, gap, fill=lambda n: torch.zeros(n), gen=None):
        total = sum(sizes) + gap * (len(sizes) + 1)
        host = torch.full((total,), 7.0).to(dtype) if dtype != torch.float8_e4m3fn else \
            torch.full((total,), 0x5b, dtype=torch.uint8).view(dtype)
        self.spans, at = [], gap
        for n in sizes:
            self.spans.append((at, n))
            host[at:at + n] = fill(n).to(dtype)
            at += n + gap
        self.flat = host.to(device)
        self.before = self.raw(host)
        self.list = [self.flat[a:a + n] for a, n in self.spans]

    @staticmethod
    def raw(t):
        t = t.detach().cpu().contiguous()
        return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()]).numpy().copy()

    def check_between(self, what):
        now, keep = self.raw(self.flat), np.ones(self.flat.numel(), bool)
        for a, n in self.spans:
            keep[a:a + n] = False
        assert np.array_equal(now[keep], self.before[keep]), f"{what}: wrote outside its tensors"

    def check_same(self, what):
        assert np.array_equal(self.raw(self.flat), self.before), f"{what}: changed"


def make(sizes, device, *, p="f32", g="f32", c=None, gap=3, seed=0, eight=False, scale=1e-3):
    """The tensors of a step in earnest: gradients of 1e-6 to 1e-2, some zero."""
    gen = torch.Generator().manual_seed(seed)

    def normal(n):
        return torch.randn(n, generator=gen)

    def grads(n):
        x = normal(n) * scale * 10 ** (torch.rand(n, generator=gen) * 4 - 3)
        x[torch.rand(n, generator=gen) < 0.05] = 0
        return x

    s = {"p": Flat(sizes, TYPES[p], device, gap, lambda n: normal(n) * 0.1),
         "g": Flat(sizes, TYPES[g], device, gap, grads),
         "c": None if c is None else Flat(sizes, TYPES[c], device, gap)}
    if not eight:
        s["m"] = Flat(sizes, torch.float32, device, gap, lambda n: grads(n) * 0.3)
        s["v"] = Flat(sizes, torch.float32, device, gap, lambda n: grads(n) ** 2)
    else:
        blocks = [(n + BLOCK - 1) // BLOCK for n in sizes]

        def codes(n, signed):
            x = torch.rand(n, generator=gen) * 448 * torch.rand(n, generator=gen) ** 4
            return x * torch.sign(normal(n)) if signed else x
        s["m"] = Flat(sizes, torch.float8_e4m3fn, device, gap, lambda n: codes(n, True))
        s["r"] = Flat(sizes, torch.float8_e4m3fn, device, gap, lambda n: codes(n, False))
        s["ms"] = Flat(blocks, torch.float32, device, gap, lambda n: scale / 448 * torch.rand(n, generator=gen))
        s["rs"] = Flat(blocks, torch.float32, device, gap, lambda n: scale / 448 * torch.rand(n, generator=gen))
    return s


def close(got, want, err, what):
    got = f64(got)
    bad = ~(np.abs(got - want) <= err)
    assert not bad.any(), (what, np.flatnonzero(bad)[:5], got[bad][:5], want[bad][:5], err[bad][:5])


def check_adamw(s, old, step, what, **hyper):
    for i in range(len(s["p"].list)):
        r = Q.adamw(*(old[k][i] for k in "pgmv"), step, **hyper)
        pt = s["p"].list[i].dtype
        close(s["p"].list[i], r["p"][0], Q.rounded(*r["p"], pt) if pt != torch.float32 else r["p"][1], f"{what}: p[{i}]")
        close(s["m"].list[i], *r["m"], f"{what}: m[{i}]")
        close(s["v"].list[i], *r["v"], f"{what}: v[{i}]")
        if s["c"] is not None:
            close(s["c"].list[i], r["p"][0], Q.rounded(*r["p"], s["c"].list[i].dtype), f"{what}: copy[{i}]")
    for k in ("p", "m", "v", "c"):
        if s[k] is not None:
            s[k].check_between(f"{what}: {k}")
    s["g"].check_same(f"{what}: gradients")


def values(s, keys):
    return {k: [f64(t) for t in s[k].list] for k in keys}


COMBOS = [("f32", "f32", None), ("f32", "f32", "bf16"), ("f32", "f32", "f16"), ("f32", "bf16", None),
          ("f32", "bf16", "bf16"), ("f32", "bf16", "f16"), ("f32", "f16", None), ("f32", "f16", "bf16"),
          ("f32", "f16", "f16"), ("bf16", "f32", None), ("bf16", "bf16", None), ("bf16", "f16", None),
          ("f16", "f32", None), ("f16", "bf16", None), ("f16", "f16", None)]


# ---------------------------------------------------------------------------
# AdamW, 32-bit moments
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("gap", [0, 1, 4])
@pytest.mark.parametrize("p,g,c", COMBOS)
def test_adamw_every_type_and_edge(where, p, g, c, gap):
    from pccl import optim
    print(f"adamw {p} {g} {c} gap {gap} on {where.name}", flush=True)
    s = make(EDGES, where.device, p=p, g=g, c=c, gap=gap, seed=1)
    old = values(s, "pgmv")
    optim.adamw(s["p"].list, s["g"].list, s["m"].list, s["v"].list, 7, copies=s["c"] and s["c"].list, **HYPER)
    where.sync()
    check_adamw(s, old, 7, "adamw", **HYPER)


@pytest.mark.parametrize("hyper", [dict(lr=0.0), dict(weight_decay=0.0), dict(betas=(0.0, 0.0)), dict(eps=0.0, betas=(0.9, 0.999)),
                                   dict(eps=1.0), dict(betas=(0.5, 0.9999)), dict(lr=10.0, weight_decay=0.5)])
@pytest.mark.parametrize("step", [1, 2, 1000, 10 ** 7])
def test_adamw_hyperparameters(where, hyper, step):
    from pccl import optim
    h = dict(HYPER, **hyper)
    s = make([777], where.device, seed=2)
    if h["eps"] == 0:                      # 0 / 0 is nobody's business: no element without a second moment
        s["v"].list[0] += 1e-12
    old = values(s, "pgmv")
    optim.adamw(s["p"].list, s["g"].list, s["m"].list, s["v"].list, step, **h)
    where.sync()
    check_adamw(s, old, step, f"adamw {hyper} step {step}", **h)


@pytest.mark.parametrize("norm,max_norm,scale", [(4.0, 1.0, 1.0), (0.5, 1.0, 1.0), (0.0, 1.0, 1.0), (1e30, 1e-3, 1.0),
                                                 (800.0, 0.25, 1 / 256), (800.0, 0.25, -1 / 256), (3.0, 5.0, 2.0)])
@pytest.mark.parametrize("skip", [False, True])
def test_adamw_clips_by_a_norm_on_the_device(where, norm, max_norm, scale, skip):
    from pccl import optim
    s = make([5, 600], where.device, g="bf16", c="bf16", seed=3)
    old = values(s, "pgmv")
    t = torch.tensor([norm], dtype=torch.float32, device=where.device)
    optim.adamw(s["p"].list, s["g"].list, s["m"].list, s["v"].list, 3, copies=s["c"].list, norm=t, max_norm=max_norm,
                grad_scale=scale, skip_nonfinite=skip, **HYPER)
    where.sync()
    check_adamw(s, old, 3, "clip", norm=float(t), max_norm=max_norm, grad_scale=scale, **HYPER)


@pytest.mark.parametrize("norm", [math.inf, math.nan])
@pytest.mark.parametrize("eight", [False, True])
def test_a_step_without_a_finite_norm_is_skipped_whole(where, norm, eight):
    from pccl import optim
    s = make([5, 600], where.device, c="f16", seed=4, eight=eight)
    s["g"].list[0][2] = norm
    t = torch.tensor([norm], device=where.device)
    lists = [s[k].list for k in (("p", "g", "m", "r", "ms", "rs") if eight else ("p", "g", "m", "v"))]
    (optim.adamw8 if eight else optim.adamw)(*lists, 3, copies=s["c"].list, norm=t, max_norm=1.0, skip_nonfinite=True, **HYPER)
    where.sync()
    for k in s:
        if k != "g":
            s[k].check_same(f"skipped step: {k}")


def test_a_norm_that_is_not_finite_reaches_the_parameters_unless_skipped(where):
    from pccl import optim
    s = make([70], where.device, seed=5)
    optim.adamw(s["p"].list, s["g"].list, s["m"].list, s["v"].list, 3, norm=torch.tensor([math.nan], device=where.device),
                max_norm=1.0, **HYPER)
    where.sync()
    assert np.isnan(f64(s["p"].list[0])).all()


def test_adamw_an_infinite_or_nan_gradient_stays_in_its_element(where):
    from pccl import optim
    s = make([300], where.device, seed=6)
    g = s["g"].list[0]
    g[7], g[150] = math.nan, math.inf
    old = values(s, "pgmv")
    optim.adamw(s["p"].list, [g], s["m"].list, s["v"].list, 3, **HYPER)
    where.sync()
    bad = [7, 150]
    assert np.isnan(f64(s["p"].list[0])[bad]).all()
    good = np.delete(np.arange(300), bad)
    with np.errstate(invalid="ignore"):
        r = Q.adamw(*(old[k][0] for k in "pgmv"), 3, **HYPER)
    close(s["p"].list[0][torch.from_numpy(good).to(where.device)], r["p"][0][good], r["p"][1][good], "others")


def test_adamw_first_steps_from_zero(where):
    """m = v = 0: the first update is lr * sign(g), up to eps."""
    from pccl import optim
    s = make([500], where.device, seed=7)
    for k in "mv":
        s[k].list[0].zero_()
    plan = optim.plan_adamw(s["p"].list, s["g"].list, s["m"].list, s["v"].list, **HYPER)
    for step in (1, 2, 3):
        old = values(s, "pgmv")
        plan(step)
        where.sync()
        check_adamw(s, old, step, f"step {step}", **HYPER)


def test_adamw_tiny_and_huge_gradients(where):
    """Squares that underflow give v = 0 and no division by zero; the largest that do not overflow stay finite."""
    from pccl import optim
    g = torch.tensor([0.0, 1e-45, 1e-30, 1e-22, 1e-18, 1.0, 1e10, 1e18, -1e18, -1e-30], device=where.device)
    s = make([10], where.device, seed=8)
    for k in "mv":
        s[k].list[0].zero_()
    old = dict(values(s, "pmv"), g=[f64(g)])
    optim.adamw(s["p"].list, [g], s["m"].list, s["v"].list, 1, **HYPER)
    where.sync()
    r = Q.adamw(*(old[k][0] for k in "pgmv"), 1, **HYPER)
    for k in "pmv":
        close(s[k].list[0], *r[k], f"extreme gradients: {k}")


@pytest.mark.parametrize("eight", [False, True])
def test_more_tensors_than_one_launch_holds_and_mixed_types(where, eight):
    from pccl import optim
    n = 150
    gen = np.random.default_rng(9)
    parts = []
    for i in range(n):
        p, g, c = COMBOS[int(gen.integers(len(COMBOS)))]
        size = int(gen.choice([0, 1, 5, 255, 256, 300, 700]))
        parts.append(make([size], where.device, p=p, g=g, c=c, gap=1, seed=100 + i, eight=eight))
    keys = ("p", "g", "m", "r", "ms", "rs") if eight else ("p", "g", "m", "v")
    old = [values(s, keys) for s in parts]
    copies = [None if s["c"] is None else s["c"].list[0] for s in parts]
    lists = [[s[k].list[0] for s in parts] for k in keys]
    (optim.adamw8 if eight else optim.adamw)(*lists, 4, copies=copies, **HYPER)
    where.sync()
    for i, s in enumerate(parts):
        if eight:
            check_adamw8(s, old[i], 4, f"tensor {i}", **HYPER)
        else:
            check_adamw(s, old[i], 4, f"tensor {i}", **HYPER)


@pytest.mark.parametrize("count", [57, 64, 65, 300, 4200])
@pytest.mark.parametrize("eight", [False, True])
def test_many_tensors_of_one_type(where, count, eight):
    """Addresses in kernel arguments, in a table in device memory (once for up to 4096), and with other gradients."""
    from pccl import optim
    gen = np.random.default_rng(count)
    sizes = [int(x) for x in gen.choice([0, 1, 3, 255, 256, 257, 300] if count < 1000 else [0, 1, 2, 5], count)]
    s = make(sizes, where.device, g="bf16", c="f16", gap=1, seed=15, eight=eight)
    other = make(sizes, where.device, g="bf16", gap=2, seed=16)
    keys = ("p", "g", "m", "r", "ms", "rs") if eight else ("p", "g", "m", "v")
    plan = (optim.plan_adamw8 if eight else optim.plan_adamw)(*(s[k].list for k in keys), copies=s["c"].list, **HYPER)
    assert (plan._own is not None) == (sum(n > 0 for n in sizes) > (56 if eight else 64))
    check, read = (check_adamw8, values8) if eight else (check_adamw, lambda s: values(s, "pgmv"))
    old = read(s)
    plan(3)
    where.sync()
    check(s, old, 3, "own gradients", **HYPER)
    old = dict(read(s), g=values(other, "g")["g"])
    plan(4, grads=other["g"].list)
    where.sync()
    check(s, old, 4, "other gradients", **HYPER)


def test_plan_takes_other_gradients(where):
    from pccl import optim
    s = make([3, 900], where.device, g="bf16", seed=10)
    other = make([3, 900], where.device, g="bf16", seed=11, gap=5)
    plan = optim.plan_adamw(s["p"].list, s["g"].list, s["m"].list, s["v"].list, **HYPER)
    old = dict(values(s, "pmv"), g=values(other, "g")["g"])
    plan(2, grads=other["g"].list)
    where.sync()
    check_adamw(s, old, 2, "other gradients", **HYPER)
    old = values(s, "pgmv")
    plan(3)                                # and its own again
    where.sync()
    check_adamw(s, old, 3, "own gradients", **HYPER)


@pytest.mark.parametrize("step", [1, 2, 3, 255, 4097, 10 ** 6])
def test_step_and_lr_in_device_memory(where, step):
    from pccl import optim
    s = make([3, 900], where.device, seed=12)
    plan = optim.plan_adamw(s["p"].list, s["g"].list, s["m"].list, s["v"].list, **HYPER)
    old = values(s, "pgmv")
    lr = torch.tensor([2e-2], device=where.device)
    plan(torch.tensor([step], device=where.device), lr=lr)
    where.sync()
    check_adamw(s, old, step, "device scalars", **dict(HYPER, lr=float(lr)))


def test_a_step_below_one_in_device_memory_counts_as_one(where):
    from pccl import optim
    out = []
    for step in (torch.tensor([0], device=where.device), torch.tensor([-5], device=where.device), 1):
        s = make([40], where.device, seed=13)
        optim.adamw(s["p"].list, s["g"].list, s["m"].list, s["v"].list, step, **HYPER)
        where.sync()
        out.append(f64(s["p"].list[0]))
    assert np.array_equal(out[0], out[1])
    assert np.allclose(out[0], out[2], rtol=1e-6, atol=0)


def test_written_tensors_are_marked_as_modified(where):
    from pccl import optim
    s = make([40], where.device, c="bf16", seed=14)
    p, c = s["p"].list[0].clone().requires_grad_(), s["c"].list[0].clone()
    before = p._version, c._version
    optim.adamw([p], s["g"].list, s["m"].list, s["v"].list, 1, copies=[c])
    assert p._version > before[0] and c._version > before[1]


# ---------------------------------------------------------------------------
# AdamW, 8-bit moments
# ---------------------------------------------------------------------------

def check_adamw8(s, old, step, what, seed=None, **hyper):
    for i in range(len(s["p"].list)):
        n = old["p"][i].size
        if not n:
            continue

        def read(codes, scales):
            return old[codes][i] * np.repeat(old[scales][i], BLOCK)[:n]
        m, r = read("m", "ms"), read("r", "rs")
        # code * scale is one rounding; its square another, and doubles the first
        res = Q.adamw(old["p"][i], old["g"][i], m, r * r, step, m_err=U, v_err=3.1 * U, **hyper)
        pt = s["p"].list[i].dtype
        close(s["p"].list[i], res["p"][0], Q.rounded(*res["p"], pt) if pt != torch.float32 else res["p"][1], f"{what}: p[{i}]")
        if s["c"] is not None:
            close(s["c"].list[i], res["p"][0], Q.rounded(*res["p"], s["c"].list[i].dtype), f"{what}: copy[{i}]")
        bits = None if seed is None else Q.noise(seed, step, n)
        Q.check_blocks(f64(s["m"].list[i].float()), f64(s["ms"].list[i]), *res["m"], False,
                       None if bits is None else bits & np.uint64(0xffff), f"{what}: m[{i}]")
        Q.check_blocks(f64(s["r"].list[i].float()), f64(s["rs"].list[i]), *res["root"], True,
                       None if bits is None else bits >> np.uint64(16), f"{what}: r[{i}]")
    for k in ("p", "m", "r", "ms", "rs", "c"):
        if s[k] is not None:
            s[k].check_between(f"{what}: {k}")
    s["g"].check_same(f"{what}: gradients")


def values8(s):
    out = values(s, ("p", "g", "ms", "rs"))
    out.update({k: [f64(t.float()) for t in s[k].list] for k in ("m", "r")})
    return out


@pytest.mark.parametrize("gap", [0, 1])
@pytest.mark.parametrize("seed", [None, 0, 123456789, 2 ** 32 - 1])
@pytest.mark.parametrize("p,g,c", COMBOS)
def test_adamw8_every_type_and_edge(where, p, g, c, seed, gap):
    from pccl import optim
    print(f"adamw8 {p} {g} {c} seed {seed} gap {gap} on {where.name}", flush=True)
    s = make(EDGES, where.device, p=p, g=g, c=c, gap=gap, seed=21, eight=True)
    old = values8(s)
    optim.adamw8(*(s[k].list for k in ("p", "g", "m", "r", "ms", "rs")), 7, seed=seed, copies=s["c"] and s["c"].list, **HYPER)
    where.sync()
    check_adamw8(s, old, 7, "adamw8", seed=seed, **HYPER)


@pytest.mark.parametrize("seed", [None, 5])
def test_adamw8_from_empty_blocks_over_several_steps(where, seed):
    from pccl import optim
    s = make([1, 700], where.device, g="bf16", c="bf16", seed=22, eight=True)
    for k in ("m", "r"):
        s[k] = Flat([1, 700], torch.float8_e4m3fn, where.device, 3)
    for k in ("ms", "rs"):
        s[k] = Flat([1, 3], torch.float32, where.device, 3)
    plan = optim.plan_adamw8(*(s[k].list for k in ("p", "g", "m", "r", "ms", "rs")), copies=s["c"].list, **HYPER)
    norm = torch.tensor([2.0], device=where.device)
    for step in range(1, 6):
        old = values8(s)
        t = torch.tensor([step], device=where.device) if step % 2 else step
        plan(t, seed=seed, norm=norm, max_norm=0.5, grad_scale=0.5)
        where.sync()
        check_adamw8(s, old, step, f"step {step}", seed=seed, norm=2.0, max_norm=0.5, grad_scale=0.5, **HYPER)


def test_adamw8_zero_gradients_of_a_fresh_state_change_nothing_but_decay(where):
    from pccl import optim
    p = torch.randn(600).to(where.device)
    m, ms = optim.empty_blocks(p)
    r, rs = optim.empty_blocks(p)
    want = f64(p) * (1 - 0.01 * 0.5)
    optim.adamw8([p], [torch.zeros_like(p)], [m], [r], [ms], [rs], 1, lr=0.01, weight_decay=0.5, seed=3)
    where.sync()
    close(p, want, 3 * U * np.abs(want), "decay")
    assert not m.float().any() and not r.float().any()
    assert torch.isfinite(ms).all() and torch.isfinite(rs).all()


@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_adamw8_a_bad_gradient_shows_in_its_block_only(where, value):
    from pccl import optim
    s = make([1024], where.device, seed=23, eight=True)
    g = s["g"].list[0]
    g[300] = value
    optim.adamw8(s["p"].list, [g], *(s[k].list for k in ("m", "r", "ms", "rs")), 3, seed=1, **HYPER)
    where.sync()
    p, ms, rs = f64(s["p"].list[0]), f64(s["ms"].list[0]), f64(s["rs"].list[0])
    assert np.isnan(p[300]) and np.isfinite(np.delete(p, 300)).all()
    assert not np.isfinite(ms[1]) and not np.isfinite(rs[1])
    assert np.isfinite(np.delete(ms, 1)).all() and np.isfinite(np.delete(rs, 1)).all()
    out = [torch.empty(1024, device=where.device) for _ in range(2)]
    optim.dequantize_blocks(out[:1], s["m"].list, s["ms"].list)
    optim.dequantize_blocks(out[1:], s["r"].list, s["rs"].list, root=True)
    where.sync()
    for x in out:
        bad = ~np.isfinite(f64(x))
        assert bad[300] and not bad[:256].any() and not bad[512:].any()


def test_adamw8_follows_a_slow_second_moment_only_with_random_rounding(where):
    """Why the moments are rounded stochastically: gradients of one half of a block
    drop to a tenth.  With beta2 = 0.99 a root moves by at most 0.5 % a step, a
    twelfth of the half step to the next code, so nearest rounding never lets the
    half move against the other.  The expected value after T steps is known."""
    from pccl import optim
    n, steps, b2 = 256, 100, 0.99
    small = torch.arange(n) % 2 == 1
    g = torch.where(small, 0.1, 1.0).to(where.device)
    want = math.sqrt(b2 ** steps + (1 - b2 ** steps) * 0.01)        # of the half whose gradients fell, from 1
    got = {}
    for seed in (None, 17):
        p = torch.zeros(n, device=where.device)
        m, ms = optim.empty_blocks(p)
        r, rs = optim.empty_blocks(p)
        optim.quantize_blocks([r], [rs], [torch.ones(n, device=where.device)], root=True)
        plan = optim.plan_adamw8([p], [g], [m], [r], [ms], [rs], betas=(0.9, b2), weight_decay=0.0)
        for step in range(1, steps + 1):
            plan(step, seed=seed)
        v = torch.empty(n, device=where.device)
        optim.dequantize_blocks([v], [r], [rs], root=True)
        where.sync()
        got[seed] = float(v.cpu()[small].sqrt().mean())
    assert got[None] == pytest.approx(1.0, abs=1e-3)
    # a root of one element scatters by the spacing of the codes around it, 1/16 at 0.6, over sqrt(steps in memory);
    # 128 elements bring a scatter of 0.2 (far above it) below 0.02; five of those
    assert abs(got[17] - want) < 0.1


# ---------------------------------------------------------------------------
# gradient norm
# ---------------------------------------------------------------------------

def check_norm(got, tensors, what):
    """fp32 partial products may be off by 2^-23 of themselves each; the root halves it, rounding adds 2^-24."""
    x = np.concatenate([f64(t) for t in tensors]) if tensors else np.zeros(0)
    big = np.abs(x).max() if x.size else 0
    want = 0.0 if big == 0 else big * math.sqrt(float(np.sum(np.square(x / big))))
    assert abs(float(got) - want) <= 4 * U * want + TINY_OUT, (what, float(got), want)


TINY_OUT = 2.0 ** -149


@pytest.mark.parametrize("sizes", [[0], [1], [5], EDGES, [4096] * 3, [70001], [3, 100003, 0, 17], [1] * 130, [20000] * 70])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("gap", [0, 1])
def test_norm(where, sizes, dtype, gap):
    from pccl import optim
    print(f"norm {len(sizes)} tensors of {dtype} gap {gap} on {where.name}", flush=True)
    gen = torch.Generator().manual_seed(31)
    s = Flat(sizes, TYPES[dtype], where.device, gap, lambda n: torch.randn(n, generator=gen) * 0.01)
    plan = optim.plan_grad_norm(s.list)
    got = plan()
    again = torch.full((1,), 9.0, device=where.device)
    assert plan(again) is again
    where.sync()
    check_norm(got, s.list, "norm")
    once = optim.grad_norm(s.list)          # without memory of a plan's own
    where.sync()
    assert torch.equal(got, again) and torch.equal(got, once) and got.shape == (1,) and got.dtype == torch.float32


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_norm_of_more_than_every_wave_takes_at_once(where, dtype):
    from pccl import optim
    gen = torch.Generator().manual_seed(35)
    ts = [torch.randn(n, generator=gen).to(TYPES[dtype]).to(where.device) for n in (9000001, 13, 9500000)]
    got = optim.grad_norm(ts)
    where.sync()
    check_norm(got, ts, "large")


def test_norm_of_mixed_types(where):
    from pccl import optim
    gen = torch.Generator().manual_seed(32)
    ts = [torch.randn(n, generator=gen).to(TYPES[t]).to(where.device) for n, t in
          ((7, "f32"), (4000, "bf16"), (0, "f16"), (333, "f16"), (9000, "f32"), (1, "bf16"))]
    got = optim.grad_norm(ts)
    where.sync()
    check_norm(got, ts, "mixed")


@pytest.mark.parametrize("dtype,magnitude", [("f32", 1e30), ("f32", 1e-30), ("f32", 1e-44), ("f32", 1e19), ("bf16", 1e30),
                                             ("bf16", 1e-38), ("f16", 6e4), ("f16", 6e-8), ("f32", 1e-19), ("f32", 3e-23)])
@pytest.mark.parametrize("n", [1, 300, 40000])
def test_norm_neither_overflows_nor_underflows(where, dtype, magnitude, n):
    from pccl import optim
    gen = torch.Generator().manual_seed(33)
    x = (torch.sign(torch.randn(n, generator=gen)) * magnitude).to(TYPES[dtype]).to(where.device)
    got = optim.grad_norm([x])
    where.sync()
    check_norm(got, [x], f"{dtype} {magnitude}")


def test_norm_of_values_of_all_magnitudes(where):
    from pccl import optim
    gen = torch.Generator().manual_seed(34)
    x = torch.randn(50000, generator=gen) * 10 ** (torch.rand(50000, generator=gen) * 70 - 35)
    x = x.to(where.device)
    for part in (x, x[x.abs() < 1e-20], x[x.abs() < 1e-5], x[x.abs() < 1e15]):
        part = part.contiguous()
        got = optim.grad_norm([part])
        where.sync()
        check_norm(got, [part], "all magnitudes")


@pytest.mark.parametrize("n", [10, 50000])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_norm_shows_what_is_not_finite(where, n, dtype, value):
    from pccl import optim
    for at in (0, n // 2, n - 1):
        x = torch.ones(n, dtype=TYPES[dtype])
        x[at] = value
        got = optim.grad_norm([x.to(where.device)])
        where.sync()
        assert not math.isfinite(float(got))
        assert math.isnan(float(got)) == math.isnan(value)


# ---------------------------------------------------------------------------
# 8-bit blocks
# ---------------------------------------------------------------------------

def block_buffers(sizes, device, gap):
    return (Flat(sizes, torch.float8_e4m3fn, device, gap),
            Flat([(n + BLOCK - 1) // BLOCK for n in sizes], torch.float32, device, gap))


@pytest.mark.parametrize("gap", [0, 1, 3])
@pytest.mark.parametrize("root", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("sizes", [EDGES, [256] * 130, [70001], [3, 1700003, 500]])     # the last: several runs per die
def test_blocks_there_and_back(where, sizes, dtype, root, gap):
    from pccl import optim
    gen = torch.Generator().manual_seed(41)

    def fill(n):
        x = torch.randn(n, generator=gen) * 10 ** (torch.rand(n, generator=gen) * 3 - 3)
        x[torch.rand(n, generator=gen) < 0.1] = 0
        return x * x if root else x
    src = Flat(sizes, TYPES[dtype], where.device, gap, fill)
    codes, scales = block_buffers(sizes, where.device, gap)
    optim.quantize_blocks(codes.list, scales.list, src.list, root=root)
    where.sync()
    src.check_same("source")
    codes.check_between("codes"); scales.check_between("scales")
    for i, t in enumerate(src.list):
        x = f64(t)
        if x.size:
            x = np.sqrt(x) if root else x
            Q.check_blocks(f64(codes.list[i].float()), f64(scales.list[i]), x, U * np.abs(x) if root else 0 * x, root,
                           what=f"tensor {i}")
    for back in ("f32", "bf16", "f16"):
        dst = Flat(sizes, TYPES[back], where.device, gap)
        keep = Flat.raw(codes.flat), Flat.raw(scales.flat)
        optim.dequantize_blocks(dst.list, codes.list, scales.list, root=root)
        where.sync()
        dst.check_between("read back")
        assert np.array_equal(keep[0], Flat.raw(codes.flat)) and np.array_equal(keep[1], Flat.raw(scales.flat))
        for i, t in enumerate(dst.list):
            n = t.numel()
            want = f64(codes.list[i].float()) * np.repeat(f64(scales.list[i]), BLOCK)[:n]
            want = want * want if root else want
            err = 4 * U * np.abs(want) + Q.TINY
            close(t, want, Q.rounded(want, err, t.dtype) if back != "f32" else err, f"read back {i}")


def test_blocks_every_code_comes_back(where):
    """All 254 finite codes: a block whose largest value is 448 keeps them exactly, and reads them back exactly."""
    from pccl import optim
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    every = torch.where(torch.isnan(every), torch.tensor(448.0), every).to(where.device)
    codes, scales = optim.empty_blocks(every)
    optim.quantize_blocks([codes], [scales], [every])
    out = torch.empty_like(every)
    optim.dequantize_blocks([out], [codes], [scales])
    where.sync()
    assert float(scales) == 1.0 and torch.equal(out, every)


def test_blocks_round_ties_to_even(where):
    from pccl import optim
    x = torch.tensor([448.0, 17.0, 19.0, 21.0, -17.0, 2.0 ** -10, 3 * 2.0 ** -10, 5 * 2.0 ** -10, 2.0 ** -6 * 1.0625, 440.0, 432.0])
    want = torch.tensor([448.0, 16.0, 20.0, 20.0, -16.0, 0.0, 2.0 ** -8, 2.0 ** -8, 2.0 ** -6, 448.0, 448.0])
    x = x.to(where.device)
    codes, scales = optim.empty_blocks(x)
    optim.quantize_blocks([codes], [scales], [x])
    where.sync()
    assert float(scales) == 1.0
    # 440 lies between 416 and 448, nearer to 448; 432 is their tie, and 448 has the even mantissa
    assert codes.float().cpu().tolist() == want.tolist()


@pytest.mark.parametrize("root", [False, True])
def test_blocks_of_zeros_denormals_and_the_largest(where, root):
    from pccl import optim
    big = torch.finfo(torch.float32).max
    rows = [torch.zeros(256), torch.full((256,), 1e-45), torch.full((256,), 1e-38), torch.full((256,), big),
            torch.cat([torch.tensor([big]), torch.full((255,), 1e-45)])]
    x = torch.cat(rows).to(where.device)
    codes, scales = optim.empty_blocks(x)
    optim.quantize_blocks([codes], [scales], [x], root=root)
    out = torch.empty_like(x)
    optim.dequantize_blocks([out], [codes], [scales], root=root)
    where.sync()
    v = np.sqrt(f64(x)) if root else f64(x)
    Q.check_blocks(f64(codes.float()), f64(scales), v, 2 * U * v, root, what="extremes")
    got, c = f64(out).reshape(5, 256), f64(codes.float()).reshape(5, 256)
    assert (got[0] == 0).all() and np.isfinite(f64(scales)).all()
    if root:                               # no second moment but 0 is held as 0
        assert (c[1:] > 0).all()


def test_a_root_never_vanishes_beside_a_large_one(where):
    from pccl import optim
    x = torch.full((512,), 1e-30)
    x[0] = 1.0
    x[256:] = 0
    x = x.to(where.device)
    codes, scales = optim.empty_blocks(x)
    optim.quantize_blocks([codes], [scales], [x], root=True)
    where.sync()
    c = codes.float().cpu()
    assert c[0] == 448 and (c[1:256] == 2.0 ** -9).all() and (c[256:] == 0).all()


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_blocks_what_is_not_finite_spoils_its_block_only(where, value):
    from pccl import optim
    x = torch.ones(768)
    x[400] = value
    x = x.to(where.device)
    codes, scales = optim.empty_blocks(x)
    optim.quantize_blocks([codes], [scales], [x])
    out = torch.empty_like(x)
    optim.dequantize_blocks([out], [codes], [scales])
    where.sync()
    bad = ~np.isfinite(f64(out))
    assert bad[256:512].all() and not bad[:256].any() and not bad[512:].any()


# ---------------------------------------------------------------------------
# together, as they are used
# ---------------------------------------------------------------------------

def test_a_sharded_step_over_virtual_ranks(where, monkeypatch):
    """reduce_scatter of the gradients, their norm, AdamW on every rank's shard with
    the copy to gather, all_gather of the parameters; three steps of it."""
    from pccl import _native, kernels, optim
    if where.device == "cpu":
        import conftest
        monkeypatch.setattr(_native, "_loaded", _native.NativeLib(conftest.build_cpu_library()))
    P, B = 4, 515
    gen = torch.Generator().manual_seed(51)
    master = [torch.randn(B, generator=gen).to(where.device) for _ in range(P)]
    m = [torch.zeros(B, device=where.device) for _ in range(P)]
    v = [torch.zeros(B, device=where.device) for _ in range(P)]
    shard = [torch.empty(B, dtype=torch.bfloat16, device=where.device) for _ in range(P)]
    copy = [torch.empty(B, dtype=torch.bfloat16, device=where.device) for _ in range(P)]
    full = [torch.empty(P * B, dtype=torch.bfloat16, device=where.device) for _ in range(P)]
    step_plan = optim.plan_adamw(master, shard, m, v, copies=copy, **HYPER)
    norm_plan = optim.plan_grad_norm(shard)
    for step in (1, 2, 3):
        grads = [(torch.randn(P * B, generator=gen) * 0.1).to(torch.bfloat16).to(where.device) for _ in range(P)]
        kernels.reduce_scatter_ranks(shard, grads, "ring")
        norm = norm_plan()
        where.sync()
        old = {"p": [f64(t) for t in master], "g": [f64(t) for t in shard], "m": [f64(t) for t in m], "v": [f64(t) for t in v]}
        step_plan(step, grad_scale=1 / P, norm=norm, max_norm=0.5, skip_nonfinite=True)
        kernels.all_gather_ranks(full, copy, "recursive")
        where.sync()
        # the ring adds in rank order, rounding every hop: the oracle of the collective is pinned elsewhere
        total = np.stack([f64(g) for g in grads]).sum(0)
        got = np.concatenate(old["g"])
        assert np.abs(got - total).max() <= 3 * 2.0 ** -8 * np.stack([np.abs(f64(g)) for g in grads]).sum(0).max()
        check_norm(norm, shard, "norm")
        for r in range(P):
            res = Q.adamw(*(old[k][r] for k in "pgmv"), step, norm=float(norm), max_norm=0.5, grad_scale=1 / P, **HYPER)
            close(master[r], *res["p"], f"rank {r} step {step}")
            close(copy[r], res["p"][0], Q.rounded(*res["p"], torch.bfloat16), f"copy {r} step {step}")
            assert torch.equal(full[r], torch.cat(copy))


def test_a_sharded_step_as_a_rank_program(where, monkeypatch):
    """The same as every rank of a data-parallel program would write it: the norm of
    all shards is the norm of the ranks' norms, gathered."""
    import pccl
    from pccl import _native, optim
    if where.device == "cpu":
        import conftest
        monkeypatch.setattr(_native, "_loaded", _native.NativeLib(conftest.build_cpu_library()))
    P, B, device = 4, 260, where.device
    gen = torch.Generator().manual_seed(55)
    grads = [torch.randn(P * B, generator=gen).to(torch.bfloat16).to(device) for _ in range(P)]
    start = torch.randn(P * B, generator=gen).to(device)
    full = [torch.zeros(P * B, dtype=torch.bfloat16, device=device) for _ in range(P)]
    norms = [torch.zeros(P, device=device) for _ in range(P)]
    kept = [None] * P

    def rank_main(comm):
        r = comm.Get_rank()
        shard = torch.empty(B, dtype=torch.bfloat16, device=device)
        pccl.reduce_scatter_mpi(shard, grads[r], comm, "ring")
        mine = optim.grad_norm([shard])
        pccl.all_gather_mpi(norms[r], mine, comm, "ring")
        norm = optim.grad_norm([norms[r]])
        master = start[r * B:(r + 1) * B].clone()
        m, ms = optim.empty_blocks(master)
        v, vs = optim.empty_blocks(master)
        copy = torch.empty(B, dtype=torch.bfloat16, device=device)
        optim.adamw8([master], [shard], [m], [v], [ms], [vs], 1, seed=r, copies=[copy], grad_scale=1 / P, norm=norm, max_norm=1.0,
                     **HYPER)
        pccl.all_gather_mpi(full[r], copy, comm, "ring")
        kept[r] = (shard, norm, copy)
    pccl.VirtualWorld(P, device).run(rank_main)
    where.sync()
    shards = [k[0] for k in kept]
    whole = np.concatenate([f64(t) for t in shards])
    for r in range(P):
        assert abs(float(kept[r][1]) - np.linalg.norm(whole)) <= 8 * U * np.linalg.norm(whole)
        zero = np.zeros(B)
        res = Q.adamw(f64(start[r * B:(r + 1) * B]), f64(shards[r]), zero, zero, 1, norm=float(kept[r][1]), max_norm=1.0,
                      grad_scale=1 / P, **HYPER)
        close(kept[r][2], res["p"][0], Q.rounded(*res["p"], torch.bfloat16), f"rank {r}")
        assert torch.equal(full[r], torch.cat([k[2] for k in kept]))


def test_the_norm_of_norms_is_the_norm(where):
    from pccl import optim
    gen = torch.Generator().manual_seed(52)
    shards = [(torch.randn(n, generator=gen)).to(torch.bfloat16).to(where.device) for n in (900, 1, 5000, 40000)]
    parts = torch.zeros(len(shards), device=where.device)
    for i, t in enumerate(shards):
        optim.grad_norm([t], out=parts[i:i + 1])
    got = optim.grad_norm([parts])
    where.sync()
    x = np.concatenate([f64(t) for t in shards])
    assert abs(float(got) - np.linalg.norm(x)) <= 8 * U * np.linalg.norm(x)      # two levels of the bound above


def test_weights_gathered_as_codes(where, monkeypatch):
    from pccl import _native, kernels, optim
    if where.device == "cpu":
        import conftest
        monkeypatch.setattr(_native, "_loaded", _native.NativeLib(conftest.build_cpu_library()))
    P, B = 4, 768
    gen = torch.Generator().manual_seed(53)
    shards = [torch.randn(B, generator=gen).to(torch.bfloat16).to(where.device) for _ in range(P)]
    codes, scales = zip(*(optim.empty_blocks(t) for t in shards))
    optim.quantize_blocks(codes, scales, shards)
    all_codes = [torch.empty(P * B, dtype=torch.float8_e4m3fn, device=where.device) for _ in range(P)]
    all_scales = [torch.empty(P * B // BLOCK, device=where.device) for _ in range(P)]
    kernels.all_gather_ranks(all_codes, codes, "ring")
    kernels.all_gather_ranks(all_scales, scales, "ring")
    out = [torch.empty(P * B, dtype=torch.bfloat16, device=where.device) for _ in range(P)]
    optim.dequantize_blocks(out, all_codes, all_scales)
    where.sync()
    want = np.concatenate([f64(t) for t in shards])
    scale = np.repeat(np.concatenate([f64(s) for s in scales]), BLOCK)
    for t in out:      # half a spacing of the codes, then bfloat16
        err = np.maximum(2.0 ** -4 * np.abs(want), 2.0 ** -10 * scale) * (1 + 1e-5)
        close(t, want, Q.rounded(want, err, torch.bfloat16), "gathered weights")


def test_resume_from_32_bit_moments(where):
    """A 32-bit checkpoint goes to 8 bits, steps there, and is read back."""
    from pccl import optim
    s = make([1000], where.device, seed=54)
    p, g, m, v = (s[k].list[0] for k in "pgmv")
    mc, ms = optim.empty_blocks(m)
    rc, rs = optim.empty_blocks(v)
    optim.quantize_blocks([mc], [ms], [m])
    optim.quantize_blocks([rc], [rs], [v], root=True)
    where.sync()
    old = {"p": [f64(p)], "g": [f64(g)], "m": [f64(mc.float())], "r": [f64(rc.float())], "ms": [f64(ms)], "rs": [f64(rs)]}
    optim.adamw8([p], [g], [mc], [rc], [ms], [rs], 5, seed=8, **HYPER)
    m2, v2 = torch.empty_like(m), torch.empty_like(v)
    optim.dequantize_blocks([m2], [mc], [ms])
    optim.dequantize_blocks([v2], [rc], [rs], root=True)
    where.sync()
    md = old["m"][0] * np.repeat(old["ms"][0], BLOCK)[:1000]
    rd = old["r"][0] * np.repeat(old["rs"][0], BLOCK)[:1000]
    res = Q.adamw(old["p"][0], old["g"][0], md, rd * rd, 5, m_err=U, v_err=3.1 * U, **HYPER)
    close(p, *res["p"], "p")
    # a whole spacing with random rounding: 2^-3 of the value, or 2^-9 of the scale
    close(m2, res["m"][0], 2.0 ** -3 * np.abs(res["m"][0]) * 1.001 + 2.0 ** -9 * np.repeat(f64(ms), BLOCK)[:1000] * 1.001, "m")


# ---------------------------------------------------------------------------
# refusals: on the host, before anything is launched
# ---------------------------------------------------------------------------

def test_refusals_of_tensors(cpu):
    from pccl import _native, optim
    f = torch.zeros
    p, g, m, v = f(8), f(8), f(8), f(8)
    E = _native.NativeError

    def step(**k):
        a = dict(p=[p], g=[g], m=[m], v=[v], copies=None)
        a.update(k)
        optim.adamw(a["p"], a["g"], a["m"], a["v"], 1, copies=a["copies"])
    step()
    with pytest.raises(ValueError, match="one grads tensor per entry"):
        step(g=[])
    with pytest.raises(RuntimeError, match="exp_avg_sq.*shape"):
        step(v=[f(9)])
    with pytest.raises(RuntimeError, match="shape"):
        step(p=[f(2, 4)], g=[f(4, 2)])
    with pytest.raises(RuntimeError, match="exp_avg.* must be of type torch.float32"):
        step(m=[f(8, dtype=torch.bfloat16)])
    with pytest.raises(RuntimeError, match="must be float32, bfloat16 or float16"):
        step(g=[f(8, dtype=torch.float64)])
    with pytest.raises(RuntimeError, match="contiguous"):
        step(g=[f(16)[::2]])
    with pytest.raises(TypeError, match="must be a torch.Tensor"):
        step(g=[None])
    with pytest.raises(E, match="overlap in memory"):
        step(p=[p, p], g=[g, g], m=[m, f(8)], v=[v, f(8)])
    with pytest.raises(E, match="overlap in memory"):
        step(g=[p])
    with pytest.raises(E, match="overlap in memory"):
        step(m=[v])
    big = f(15)
    with pytest.raises(E, match="overlap in memory"):
        step(p=[big[:8]], g=[big[7:]])
    with pytest.raises(E, match="only a float32 parameter has a copy"):
        step(p=[f(8, dtype=torch.bfloat16)], copies=[f(8, dtype=torch.float16)])
    with pytest.raises(E, match="a copy is bfloat16 or float16"):
        step(copies=[f(8)])
    with pytest.raises(ValueError, match="one entry of copies"):
        step(copies=[])
    step(p=[p, f(8)], g=[g, g], m=[m, f(8)], v=[v, f(8)])      # gradients may share memory: they are only read


def test_refusals_of_scalars(cpu):
    from pccl import _native, optim
    f = torch.zeros
    lists = [[f(8)] for _ in range(4)]
    plan = optim.plan_adamw(*lists)
    E = _native.NativeError
    one = torch.ones(1)
    for bad in (dict(lr=-1.0), dict(lr=math.nan), dict(lr=math.inf), dict(grad_scale=0.0), dict(grad_scale=math.nan),
                dict(grad_scale=1e300), dict(max_norm=math.inf, norm=one), dict(max_norm=1.0), dict(skip_nonfinite=True),
                dict(seed=3)):
        with pytest.raises(E):
            plan(1, **bad)
    for bad in (dict(max_norm=0.0, norm=one), dict(max_norm=-1.0, norm=one), dict(seed=-1), dict(seed=2 ** 32)):
        with pytest.raises(ValueError):
            plan(1, **bad)
    for step in (0, -3):
        with pytest.raises(E, match="the first step is 1"):
            plan(step)
    for bad in (dict(norm=torch.ones(2)), dict(norm=torch.ones(1, dtype=torch.float64)), dict(lr=torch.ones(3)),
                dict(grads=[f(8, dtype=torch.float16)]), dict(grads=[f(9)])):
        with pytest.raises(RuntimeError):
            plan(1, **bad)
    with pytest.raises(RuntimeError, match="int64"):
        plan(torch.ones(1))
    with pytest.raises(ValueError):
        plan(1, grads=[])
    with pytest.raises(E, match="overlap"):
        plan(1, grads=lists[0])
    with pytest.raises(E, match="overlap"):
        plan(1, norm=lists[2][0][3:4], max_norm=1.0)
    for bad in (dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(betas=(math.nan, 0.9)), dict(eps=-1e-8), dict(weight_decay=-1.0)):
        with pytest.raises(E):
            optim.adamw(*lists, 1, **bad)


def test_refusals_of_blocks_and_norm(cpu):
    from pccl import _native, optim
    x = torch.zeros(300)
    codes, scales = optim.empty_blocks(x)
    assert codes.dtype == torch.float8_e4m3fn and scales.numel() == 2
    optim.quantize_blocks([codes], [scales], [x])
    with pytest.raises(RuntimeError, match="float8_e4m3fn"):
        optim.quantize_blocks([torch.zeros(300, dtype=torch.uint8)], [scales], [x])
    with pytest.raises(RuntimeError, match="2 float32 scales"):
        optim.quantize_blocks([codes], [torch.zeros(3)], [x])
    with pytest.raises(ValueError):
        optim.quantize_blocks([codes], [], [x])
    with pytest.raises(RuntimeError, match="must be float32, bfloat16 or float16"):
        optim.dequantize_blocks([x.double()], [codes], [scales])
    with pytest.raises(_native.NativeError, match="overlap"):
        optim.dequantize_blocks([x, x], [codes, codes], [scales, scales])
    with pytest.raises(RuntimeError, match="avg_scale"):
        optim.adamw8([x], [x.clone()], [codes], [codes], [torch.zeros(1)], [scales], 1)
    with pytest.raises(ValueError, match="at least one tensor"):
        optim.grad_norm([])
    with pytest.raises(RuntimeError):
        optim.grad_norm([x], out=torch.zeros(2))
    with pytest.raises(RuntimeError, match="contiguous"):
        optim.grad_norm([torch.zeros(4, 4).t()])
    for i in (0, 150, 299):
        with pytest.raises(_native.NativeError, match="overlap"):
            optim.grad_norm([x[:200], x, x[10:20]], out=x[i:i + 1])


def test_tensors_on_the_cpu_are_refused():
    """The product library has no CPU path."""
    from pccl import optim
    x = torch.zeros(8)
    with pytest.raises(RuntimeError, match="must reside on the GPU"):
        optim.grad_norm([x])
    with pytest.raises(RuntimeError, match="must reside on the GPU"):
        optim.adamw([x], [x], [x], [x], 1)


def test_c_entries_refuse_with_a_code_and_a_message():
    """The product library itself, without a GPU: every refusal comes before a launch."""
    import ctypes
    from pccl import _native, _optim_native
    lib = _optim_native.load()
    E = _native.NativeError
    with pytest.raises(E, match=r"params\[0\] is NULL"):
        lib.plan_adamw([0], [64], [128], [192], None, [4], [0], [0], None)
    with pytest.raises(E, match=r"unknown grad_dtype\[0\] 7"):
        lib.plan_adamw([64], [128], [192], [256], None, [4], [0], [7], None)
    with pytest.raises(E, match="not aligned to its element size"):
        lib.plan_adamw([66], [128], [192], [256], None, [4], [0], [0], None)
    with pytest.raises(E, match="more than"):
        lib.plan_norm([64], [_optim_native.MAX_ELEMENTS + 1], [0])
    with pytest.raises(E, match="more than"):
        lib.plan_norm([64], [2 ** 63], [0])
    with pytest.raises(E, match="overlap"):
        lib.plan_quantize([64], [64 + 252], [4096], [256], [0])
    raw = lib._lib
    h = ctypes.c_void_p()
    assert raw.pccl_optim_plan_norm(None, None, None, None, 0) == -1
    assert raw.pccl_optim_plan_norm(ctypes.byref(h), None, None, None, -1) == -1 and not h
    assert raw.pccl_optim_plan_norm(ctypes.byref(h), None, None, None, 1) == -1 and not h
    assert raw.pccl_optim_run_norm(None, None, None, 0, None, None) == -1
    assert raw.pccl_optim_run_blocks(None, None) == -1
    assert raw.pccl_optim_run_adamw(None, None, None, None, None) == -1
    assert raw.pccl_optim_table_fill(None, None, 0) == -1 and raw.pccl_optim_table_bytes(None) == 0
    assert raw.pccl_optim_norm_work(None) == 0
    raw.pccl_optim_plan_free(None)
    norm = lib.plan_norm([64], [1 << 20], [0])
    with pytest.raises(E, match="another operator"):
        lib.run_blocks(norm)
    with pytest.raises(E, match="bytes of work space"):
        lib.run_norm(norm, 1 << 30, 0, 0)
    with pytest.raises(E, match="out is NULL"):
        lib.run_norm(norm, 0, 1 << 30, 1 << 20)
    for out, work, ticket in ((64, 1 << 30, 0), (1 << 30, 64 + (1 << 22) - 8, 0), (1 << 30, 1 << 31, 128)):
        with pytest.raises(E, match="overlap"):
            lib.run_norm(norm, out, work, 1 << 20, ticket)
    step = lib.plan_adamw([64], [128], [192], [256], None, [4], [0], [0], None)
    s = _optim_native.Step(lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, grad_scale=1.0, step=1)
    with pytest.raises(E, match=r"grads\[0\] is NULL"):
        lib.run_adamw(step, s, [0])
    with pytest.raises(E, match="not aligned"):
        lib.run_adamw(step, s, [66])
    with pytest.raises(E, match="has no table"):
        lib.run_adamw(step, s, None, 64)
    many = lib.plan_adamw(*[[(1 + k) << 20 | i << 6 for i in range(65)] for k in range(4)], None, [4] * 65, [0] * 65, [0] * 65, None)
    assert lib.table_bytes(many) >= 65 * 52
    with pytest.raises(E, match="bytes, got"):
        lib.table_fill(many, 64, 65 * 52 - 1)
    with pytest.raises(E, match="not aligned to 64"):
        lib.run_adamw(many, s, None, 32)
    with pytest.raises(E, match="another operator"):
        lib.table_fill(norm, 64, 1 << 20)


def test_header_lists_what_the_binding_and_the_library_have():
    import ctypes
    import os
    import re
    import subprocess
    from conftest import ROOT
    from pccl import _native, _optim_native
    path = os.path.join(ROOT, "include", "pccl_optim.h")
    text = re.sub(r"/\*.*?\*/", "", open(path).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(pccl_optim_\w+)\s*\(", text)))
    assert names == sorted(_optim_native.SIGNATURES)
    lib = ctypes.CDLL(_native.LIB_PATH)
    for name in names:
        assert hasattr(lib, name)
    src = ('#include "pccl_optim.h"\n#include <stdio.h>\n'
           'int main(void){printf("%d %zu", PCCL_OPTIM_BLOCK, sizeof(pccl_optim_step)); return 0;}\n')
    exe = os.path.join(ROOT, "tests", "build", "optim_header")
    os.makedirs(os.path.dirname(exe), exist_ok=True)
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-pedantic", "-I", os.path.join(ROOT, "include"), "-x", "c", "-",
                    "-o", exe], input=src, text=True, check=True)
    out = subprocess.run([exe], capture_output=True, text=True, check=True).stdout
    assert out == f"{_optim_native.BLOCK} {ctypes.sizeof(_optim_native.Step)}"


# ---------------------------------------------------------------------------
# streams, graphs, threads
# ---------------------------------------------------------------------------

@pytest.mark.gpu
def test_graph_replays_with_step_and_lr_on_the_device():
    """norm -> AdamW captured once and replayed: every replay gives what the same eager calls give."""
    from pccl import optim
    dev = "cuda:0"
    def fresh():
        s = make([5, 100003], dev, g="bf16", c="bf16", seed=61)
        plan = optim.plan_adamw(s["p"].list, s["g"].list, s["m"].list, s["v"].list, copies=s["c"].list, **HYPER)
        norm = optim.plan_grad_norm(s["g"].list)
        step, lr = torch.zeros(1, dtype=torch.int64, device=dev), torch.full((1,), 1e-2, device=dev)

        def body():
            step.add_(1)
            plan(step, lr=lr, norm=norm(), max_norm=0.5, skip_nonfinite=True)
            lr.mul_(0.5)
        return s, body
    a, eager = fresh()
    b, body = fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body()                              # warm-up, counted as the first step
    torch.cuda.current_stream().wait_stream(side)
    eager()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        body()
    for k in range(4):
        gen = torch.Generator().manual_seed(70 + k)
        for i, n in enumerate((5, 100003)):
            g = (torch.randn(n, generator=gen) * 0.01).to(torch.bfloat16).to(dev)
            a["g"].list[i].copy_(g); b["g"].list[i].copy_(g)
        eager()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for key in ("p", "m", "v", "c"):
            assert torch.equal(a[key].flat, b[key].flat), f"replay {k}: {key}"


@pytest.mark.gpu
def test_two_captured_graphs_do_not_share_work_space():
    from pccl import optim
    dev = "cuda:0"
    xs = [torch.randn(300000, device=dev), torch.randn(300000, device=dev) * 3]
    graphs, outs = [], []
    for x in xs:
        plan = optim.plan_grad_norm([x])
        plan()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(plan())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, x in zip(outs, xs):
            check_norm(o, [x], "replayed norm")


@pytest.mark.gpu
def test_calls_follow_the_current_stream():
    from pccl import optim
    dev = "cuda:0"
    s = make([200003], dev, seed=62)
    plan = optim.plan_adamw(s["p"].list, s["g"].list, s["m"].list, s["v"].list, **HYPER)
    norm = optim.plan_grad_norm(s["g"].list)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    old = values(s, "pmv")
    with torch.cuda.stream(side):
        big = torch.randn(1 << 25, device=dev)
        for _ in range(20):
            big = big * 1.0001
        s["g"].list[0].copy_(torch.randn(200003, device=dev) * 0.01)      # behind slow work on the same stream
        n = norm()
        plan(4, norm=n, max_norm=1.0)
    torch.cuda.synchronize()
    old["g"] = [f64(s["g"].list[0])]
    check_norm(n, s["g"].list, "norm on a stream")
    r = Q.adamw(*(old[k][0] for k in "pgmv"), 4, norm=float(n), max_norm=1.0, **HYPER)
    close(s["p"].list[0], *r["p"], "step on a stream")


@pytest.mark.gpu
def test_one_plan_from_several_threads():
    """A plan is not changed by a run: threads with streams of their own and other scalars do not disturb each other."""
    from pccl import optim
    dev = "cuda:0"
    s = make([1000], dev, seed=63)
    gs = [torch.randn(1000, device=dev) * 0.01 for _ in range(4)]
    norms = [optim.plan_grad_norm([torch.full((70000,), float(k + 1), device=dev)]) for k in range(4)]
    plan = optim.plan_grad_norm([torch.randn(500000, device=dev)])
    want = plan().clone()
    torch.cuda.synchronize()
    errors = []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(50):
                    a, b = plan(), norms[k]()
                    torch.cuda.current_stream().synchronize()
                    assert torch.equal(a, want)
                    assert abs(float(b) - (k + 1) * math.sqrt(70000)) <= 4 * U * (k + 1) * math.sqrt(70000)
        except BaseException as e:            # noqa: BLE001 - reported by the main thread
            errors.append(e)
    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    del s, gs


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [False, True])
def test_a_plan_of_many_tensors_on_other_streams_and_in_a_graph_that_outlives_it(eight):
    """The table in device memory is used on the plan's own stream alone; elsewhere the results are the same."""
    from pccl import optim
    dev, sizes = "cuda:0", [300 + k for k in range(150)]
    keys = ("p", "g", "m", "r", "ms", "rs") if eight else ("p", "g", "m", "v")
    def fresh():
        s = make(sizes, dev, seed=64, eight=eight)
        return s, (optim.plan_adamw8 if eight else optim.plan_adamw)(*(s[k].list for k in keys), **HYPER)
    a, plan_a = fresh()
    b, plan_b = fresh()
    assert plan_a._own is not None
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    plan_a(1)
    with torch.cuda.stream(side):
        plan_b(1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan_b(2)
    del plan_b
    for _ in range(3):
        junk = [torch.full((1 << 20,), 255, dtype=torch.uint8, device=dev) for _ in range(8)]     # where the plan's table was
        plan_a(2)
        graph.replay()
        torch.cuda.synchronize()
        del junk
    for k in keys:
        assert np.array_equal(Flat.raw(a[k].flat), Flat.raw(b[k].flat)), k


@pytest.mark.gpu
def test_plans_made_and_single_calls_made_during_capture():
    """Neither allocates host memory, copies or clears anything while a graph is captured."""
    from pccl import optim
    dev, sizes = "cuda:0", [2000 + k for k in range(70)]
    a, b = (make(sizes, dev, seed=65, c="bf16") for _ in range(2))
    norm = torch.zeros(1, device=dev)

    def body(s):
        optim.plan_grad_norm(s["g"].list)(norm)
        optim.plan_adamw(s["p"].list, s["g"].list, s["m"].list, s["v"].list, copies=s["c"].list, **HYPER)(
            2, norm=norm, max_norm=0.1)
        optim.adamw(s["p"].list, s["g"].list, s["m"].list, s["v"].list, 3, copies=s["c"].list, norm=optim.grad_norm(s["g"].list),
                    max_norm=0.1, **HYPER)
    body(a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        body(b)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for k in ("p", "m", "v", "c"):
            assert np.array_equal(Flat.raw(a[k].flat), Flat.raw(b[k].flat)), k
        body(a)
        torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [False, True])
def test_adamw_offsets_beyond_32_bits(eight):
    """A tensor of more than 2^32 elements, zero but for a few: they are stepped, and nothing else is."""
    from pccl import optim
    dev, n = "cuda:0", (1 << 32) + 1000
    if torch.cuda.mem_get_info()[0] < 120 << 30:
        pytest.skip("needs 120 GiB of free GPU memory")
    at = torch.tensor([0, 5, (1 << 31) + 7, (1 << 32) - 1, 1 << 32, n - 2, n - 1], device=dev)
    p, g = torch.zeros(n, dtype=torch.bfloat16, device=dev), torch.zeros(n, dtype=torch.bfloat16, device=dev)
    p[at], g[at] = 0.5, torch.tensor([1.0, 0.25, -2.0, 3.0, 0.75, -0.3, 1.0], device=dev).to(torch.bfloat16)
    old = f64(p[at]), f64(g[at])
    if eight:
        m, ms = optim.empty_blocks(p)
        v, vs = optim.empty_blocks(p)
        optim.adamw8([p], [g], [m], [v], [ms], [vs], 1, seed=9, **HYPER)
    else:
        m, v = (torch.zeros(n, device=dev) for _ in range(2))
        optim.adamw([p], [g], [m], [v], 1, **HYPER)
    torch.cuda.synchronize()
    zero = np.zeros(at.numel())
    r = Q.adamw(*old, zero, zero, 1, **HYPER)
    close(p[at], r["p"][0], Q.rounded(*r["p"], torch.bfloat16), "parameters")
    assert int((p != 0).sum()) == at.numel()
    if not eight:
        close(m[at], *r["m"], "first moments")
        assert int((m != 0).sum()) == at.numel() and int((v != 0).sum()) == at.numel()
        return
    # of the last two elements of the tensor the smaller one is rounded by the random bits of its own index
    i = np.array([n - 2, n - 1], dtype=np.uint64)
    bits = Q.noise_at(9, 1, i)
    y = np.abs(r["m"][0][5:]) / (np.abs(r["m"][0][5:]).max() / 448)
    want = np.floor(y / Q.spacing(y) + (bits & np.uint64(0xffff)).astype(float) / 65536) * Q.spacing(y)
    assert np.abs(f64(m[at[5:]].float())).tolist() == want.tolist()
    assert int((m.view(torch.uint8) & 0x7f != 0).sum()) == at.numel() and int((v.view(torch.uint8) != 0).sum()) == at.numel()


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """A tensor of more than 2^32 elements: its last blocks are computed and lie where they should."""
    from pccl import optim
    dev, n = "cuda:0", (1 << 32) + 1000
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GiB of free GPU memory")
    x = torch.zeros(n, dtype=torch.bfloat16, device=dev)
    x[-3], x[5], x[1 << 31] = 3.0, 4.0, 12.0
    got = optim.grad_norm([x])
    codes, scales = optim.empty_blocks(x)
    optim.quantize_blocks([codes], [scales], [x])
    torch.cuda.synchronize()
    assert float(got) == 13.0
    last = (n - 3) // BLOCK
    assert float(scales[last]) == pytest.approx(3 / 448, rel=1e-6) and float(scales[0]) == pytest.approx(4 / 448, rel=1e-6)
    assert float(codes[-3].float()) == 448.0 and float(codes[5].float()) == 448.0 and float(codes[1 << 31].float()) == 448.0
    assert int((scales > 1e-20).sum()) == 3
    x.zero_()
    optim.dequantize_blocks([x], [codes], [scales])
    torch.cuda.synchronize()
    assert float(x[-3]) == 3.0 and float(x[1 << 31]) == 12.0 and int((x != 0).sum()) == 3
