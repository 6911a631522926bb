"""Edges of pccl.optim: scalars next to the ends of fp32, the 8-bit form bit for
bit, what a call marks as modified, how many tensors a launch and a table hold,
plans used from several threads."""
import math
import threading

import numpy as np
import pytest
import torch

import optim_oracle as Q
from optim_oracle import BLOCK, TYPES
from test_optim import (HYPER, Flat, check_adamw, check_adamw8, cpu, make, values, values8, where)  # noqa: F401 - fixtures


def fp32(x):
    return np.asarray(x, np.float32)


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


# ---------------------------------------------------------------------------
# the 8-bit form, bit for bit
# ---------------------------------------------------------------------------

def plain_codes(x, root=False, u16=None):
    """(codes, scales) of fp32 values in elementary fp32 operations, each rounded by itself: scale = max(a, 2^-100) * (1/448),
    code = e4m3(x * (1 / scale)).  u16: 16 random bits per value, added below the mantissa bits that e4m3 keeps."""
    one, n = fp32(1), x.size
    x = np.pad(x, (0, -n % BLOCK)).reshape(-1, BLOCK)
    scale = np.maximum(np.abs(x).max(1), fp32(2.0 ** -100)) * (one / fp32(448))
    y = x * (one / scale)[:, None]
    if root:
        y = np.where((x != 0) & (y < fp32(2.0 ** -9)), fp32(2.0 ** -9), y)
    if u16 is not None:
        u16 = np.pad(u16.astype(np.uint32), (0, -n % BLOCK)).reshape(-1, BLOCK)
        a = np.minimum(np.abs(y), fp32(448))
        shift = np.where(a < fp32(2.0 ** -6), fp32(2.0 ** -6), fp32(0))        # subnormal codes are as far apart as those from 2^-6 on
        cut = (((a + shift).view(np.uint32) + (u16 << 4)) & np.uint32(0xfff00000)).view(np.float32) - shift
        y = np.copysign(cut, y)
    assert y.dtype == np.float32 and scale.dtype == np.float32
    y = torch.from_numpy(np.clip(y, -448, 448).reshape(-1)[:n].copy()).to(torch.float8_e4m3fn)
    return y.view(torch.uint8).numpy(), scale


def read(codes, scales):
    """code * scale, rounded to fp32."""
    return codes.float().cpu().numpy() * np.repeat(scales.cpu().numpy(), BLOCK)[:codes.numel()]


def block_values(dtype, where, root):
    """Values of all magnitudes and, in every second block, ones that lie on codes and half way between them."""
    blocks = 4000 if where.name == "hip" else 400
    rng = np.random.default_rng(101)
    x = rng.standard_normal((blocks, BLOCK)) * 10.0 ** rng.uniform(-4, 0, (blocks, BLOCK))
    step = rng.integers(1, 32, (blocks, 1)) * 2.0 ** rng.integers(-6, 3, (blocks, 1))
    x[::2] = (step * rng.integers(-255, 256, (blocks, BLOCK)) / 8)[::2]
    x[::2, 0] = (step * 56)[::2, 0]
    if dtype == "f32":
        x *= 2.0 ** rng.integers(-95, 110, (blocks, 1)) if not root else 2.0 ** rng.integers(-40, 50, (blocks, 1))
        x[1], x[3], x[5, 0] = 0, 1e-45, np.finfo(np.float32).max if not root else 2.0 ** 60
    x = torch.from_numpy(x.reshape(-1)[:-100]).to(TYPES[dtype])
    return (x.float() * x.float()).to(TYPES[dtype]) if root else x


@pytest.mark.parametrize("root", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_blocks_are_those_of_elementary_fp32_operations(where, dtype, root):
    from pccl import optim
    x = block_values(dtype, where, root).to(where.device)
    codes, scales = optim.empty_blocks(x)
    optim.quantize_blocks([codes], [scales], [x], root=root)
    back = torch.empty(x.shape, device=where.device)
    optim.dequantize_blocks([back], [codes], [scales], root=root)
    where.sync()
    v = x.float().cpu().numpy()
    with np.errstate(invalid="ignore"):
        want_codes, want_scales = plain_codes(np.sqrt(v) if root else v, root)
        r = read(codes, scales)
    assert np.array_equal(scales.cpu().numpy(), want_scales)
    got, back = codes.view(torch.uint8).cpu().numpy(), back.cpu().numpy()
    fine = np.repeat(np.isfinite(want_scales), BLOCK)[:got.size]      # squares beyond float16: the codes of such a block are open
    assert np.array_equal(got[fine], want_codes[fine]), np.flatnonzero((got != want_codes) & fine)[:5]
    assert np.array_equal(back[fine], (r * r if root else r)[fine]) and not np.isfinite(back[~fine]).any()


@pytest.mark.parametrize("seed", [None, 0, 4000000000])
@pytest.mark.parametrize("g", ["f32", "bf16", "f16"])
def test_moments_are_those_of_elementary_fp32_operations(where, g, seed):
    """Both moments of two steps, to nearest and with random bits, clipped by a norm, at a grad_scale that is a power of two."""
    from pccl import optim
    b1, b2 = 0.9, 0.99
    grad = (block_values(g, where, False).float() * 2.0 ** -4).to(TYPES[g])
    grad = torch.where(grad.float().abs() < 1e15, grad, torch.zeros_like(grad)).to(where.device)
    p = torch.zeros(grad.numel(), device=where.device)
    m, ms = optim.empty_blocks(p)
    r, rs = optim.empty_blocks(p)
    norm = torch.tensor([2.5 * 1024], device=where.device)
    plan = optim.plan_adamw8([p], [grad], [m], [r], [ms], [rs], betas=(b1, b2))
    # max_norm / (norm * grad_scale + 1e-6), then times grad_scale, then times the gradient
    factor = fp32(1) / (fp32(2.5) + fp32(1e-6)) * fp32(2.0 ** -10)
    gs = grad.float().cpu().numpy() * factor
    for step in (1, 2):
        old_m, old_r = read(m, ms), read(r, rs)
        plan(step, seed=seed, norm=norm, max_norm=1.0, grad_scale=2.0 ** -10)
        where.sync()
        new_m = fp32(b1) * old_m + fp32(1 - b1) * gs
        new_r = np.sqrt(fp32(b2) * (old_r * old_r) + fp32(1 - b2) * (gs * gs))
        assert new_m.dtype == new_r.dtype == np.float32
        bits = None if seed is None else Q.noise(seed, step, p.numel())
        for name, codes, scales, x, root, u in (("m", m, ms, new_m, False, None if bits is None else bits & np.uint64(0xffff)),
                                                ("r", r, rs, new_r, True, None if bits is None else bits >> np.uint64(16))):
            want_codes, want_scales = plain_codes(x, root, u)
            assert np.array_equal(scales.cpu().numpy(), want_scales), (name, step)
            got = codes.view(torch.uint8).cpu().numpy()
            assert np.array_equal(got, want_codes), (name, step, np.flatnonzero(got != want_codes)[:5])


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("norm,grad_scale,max_norm", [(1e38, 1e3, 1.0), (3e38, -2.0 ** 20, 0.5), (1e30, 2.0 ** 60, 1e-3), (3e38, 2.0 ** -20, 1.0),
                                                      (1e-30, 2.0 ** 100, 1.0), (1e-30, 2.0 ** -100, 1.0), (1e-30, 2.0 ** -149, 1.0),
                                                      (2.0, 1 / 3, 0.1), (2.0, -7.0, 20.0)])
def test_clipping_where_norm_times_grad_scale_leaves_fp32(where, norm, grad_scale, max_norm, eight):
    """The clipped gradients have the norm that was asked for, also where norm * grad_scale or the factor alone overflow
    or underflow."""
    from pccl import optim
    s = make([600], where.device, seed=72, eight=eight)
    g = s["g"].list[0]
    g.copy_(torch.randn(600, generator=torch.Generator().manual_seed(72)).to(where.device) * (norm / 600 ** 0.5))
    s["g"].before = Flat.raw(s["g"].flat)
    if not eight:
        s["m"].list[0].zero_()
    old = values8(s) if eight else values(s, "pgmv")
    t = torch.tensor([norm], dtype=torch.float32, device=where.device)
    keys = ("p", "g", "m", "r", "ms", "rs") if eight else ("p", "g", "m", "v")
    (optim.adamw8 if eight else optim.adamw)(*(s[k].list for k in keys), 3, norm=t, max_norm=max_norm, grad_scale=grad_scale, **HYPER)
    where.sync()
    (check_adamw8 if eight else check_adamw)(s, old, 3, "clip", norm=float(t), max_norm=max_norm, grad_scale=grad_scale, **HYPER)


# ---------------------------------------------------------------------------
# what a call marks as modified
# ---------------------------------------------------------------------------

def test_everything_that_is_written_is_marked_as_modified(where):
    from pccl import optim
    n = 300

    def f(x=0.0, dtype=torch.float32):
        return torch.full((n,), x, dtype=dtype).to(where.device)
    for eight in (False, True):
        p, g, c, other = f(1.0), f(0.1), f(dtype=torch.bfloat16), f(0.2)
        if eight:
            (m, ms), (v, vs) = optim.empty_blocks(p), optim.empty_blocks(p)
            written, lists = [p, m, v, ms, vs, c], [[p], [g], [m], [v], [ms], [vs]]
        else:
            m, v = f(), f()
            written, lists = [p, m, v, c], [[p], [g], [m], [v]]
        plan = (optim.plan_adamw8 if eight else optim.plan_adamw)(*lists, copies=[c])
        norm = torch.ones(1).to(where.device)
        for call in (lambda: plan(1), lambda: plan(2, grads=[other], norm=norm, max_norm=1.0),
                     lambda: (optim.adamw8 if eight else optim.adamw)(*lists, 3, copies=[c])):
            before, same = [t._version for t in written], [t._version for t in (g, other, norm)]
            call()
            assert all(t._version > b for t, b in zip(written, before)), [t._version - b for t, b in zip(written, before)]
            assert [t._version for t in (g, other, norm)] == same
    out, x = torch.empty(1).to(where.device), f(3.0)
    for call in (optim.plan_grad_norm([x]), lambda o: optim.grad_norm([x], o)):
        before = out._version, x._version
        assert call(out) is out
        assert out._version > before[0] and x._version == before[1]
    codes, scales = optim.empty_blocks(x)
    before = codes._version, scales._version, x._version
    optim.quantize_blocks([codes], [scales], [x])
    assert codes._version > before[0] and scales._version > before[1] and x._version == before[2]
    before = codes._version, scales._version, x._version
    optim.dequantize_blocks([x], [codes], [scales])
    assert (codes._version, scales._version) == before[:2] and x._version > before[2]
    where.sync()


def test_a_saved_value_that_a_call_overwrites_is_noticed(where):
    """What autograd kept of a moment, a scale or a norm raises torch's error once a call has written over it."""
    from pccl import optim
    p, g, m, v = (torch.full((300,), x).to(where.device) for x in (1.0, 0.1, 0.2, 0.3))
    norm = torch.ones(1).to(where.device)
    for saved, call in ((m, lambda: optim.adamw([p], [g], [m], [v], 1)), (v, lambda: optim.adamw([p], [g], [m], [v], 1)),
                        (norm, lambda: optim.grad_norm([g], norm))):
        w = torch.ones(1, requires_grad=True, device=where.device)
        y = (w * saved).sum()
        call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    where.sync()


def test_views_and_tensors_of_inference_mode_are_written(where):
    """Pieces of one buffer share its counter; a tensor made in inference mode has none and is written all the same."""
    from pccl import optim
    flat = torch.zeros(600).to(where.device)
    m, v = torch.zeros(600).to(where.device), torch.zeros(600).to(where.device)
    before = flat._version, m._version
    optim.adamw([flat[:300], flat[300:]], [torch.ones(300).to(where.device)] * 2, [m[:300], m[300:]], [v[:300], v[300:]], 1)
    where.sync()
    assert flat._version > before[0] and m._version > before[1] and (flat != 0).all()
    with torch.inference_mode():
        x = torch.full((300,), 2.0).to(where.device)
        codes, scales = optim.empty_blocks(x)
        out = torch.empty(1).to(where.device)
        optim.quantize_blocks([codes], [scales], [x])
        optim.grad_norm([x], out)
        where.sync()
        assert (codes.float() == 448).all() and abs(float(out) - 2 * math.sqrt(300)) < 1e-4
    optim.dequantize_blocks([x], [codes], [scales])
    where.sync()


# ---------------------------------------------------------------------------
# how many tensors a launch and a table hold
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("count", [55, 56, 57, 63, 64, 65, 112, 113, 128, 129, 4095, 4096, 4097, 4200])
@pytest.mark.parametrize("eight", [False, True])
def test_exactly_so_many_tensors(where, count, eight):
    """Tensors with elements in numbers around those that a launch (64; 56 with 8-bit moments) and a table (4096) hold, and
    empty ones between them, which take no place: own gradients through the table, others without."""
    from pccl import optim
    gen = np.random.default_rng(count)
    full = [int(x) for x in gen.choice([1, 3, 255, 256, 257, 300] if count < 1000 else [1, 2, 5, 300], count, p=None if count < 1000 else [0.5, 0.3, 0.19, 0.01])]
    sizes = sorted(full[: count // 2]) + [0, 0, 0] + full[count // 2:] + [0]
    keys = ("p", "g", "m", "r", "ms", "rs") if eight else ("p", "g", "m", "v")
    s = make(sizes, where.device, g="bf16", c="f16", gap=1, seed=81, eight=eight)
    other = make(sizes, where.device, g="bf16", gap=2, seed=82)
    plan = (optim.plan_adamw8 if eight else optim.plan_adamw)(*(s[k].list for k in keys), copies=s["c"].list, **HYPER)
    assert (plan._own is not None) == (count > (56 if eight else 64))
    check, state = (check_adamw8, values8) if eight else (check_adamw, lambda s: values(s, "pgmv"))
    old = state(s)
    plan(3)
    where.sync()
    check(s, old, 3, "own gradients", **HYPER)
    old = dict(state(s), g=values(other, "g")["g"])
    plan(4, grads=other["g"].list)
    where.sync()
    check(s, old, 4, "other gradients", **HYPER)


@pytest.mark.parametrize("counts", [[70, 70, 70], [1, 65, 3], [4100, 5, 60], [57, 0, 57]])
@pytest.mark.parametrize("eight", [False, True])
def test_a_table_of_several_batches(where, counts, eight):
    """Tensors of three kinds of types, mixed: each kind has its part of the table, and one of them more than a launch serves."""
    from pccl import optim
    kinds = [("f32", "bf16", "bf16"), ("bf16", "bf16", None), ("f32", "f32", None)]
    keys = ("p", "g", "m", "r", "ms", "rs") if eight else ("p", "g", "m", "v")
    gen = np.random.default_rng(len(counts) + counts[0])
    sets = []
    for k, (n, (p, g, c)) in enumerate(zip(counts, kinds)):
        sizes = [int(x) for x in gen.choice([1, 2, 5, 256, 300], n)]
        sets.append(make(sizes, where.device, p=p, g=g, c=c, gap=1, seed=90 + k, eight=eight))
    places = gen.permutation([(k, i) for k, n in enumerate(counts) for i in range(n)])
    lists = [[sets[k][key].list[i] for k, i in places] for key in keys]
    copies = [None if sets[k]["c"] is None else sets[k]["c"].list[i] for k, i in places]
    plan = (optim.plan_adamw8 if eight else optim.plan_adamw)(*lists, copies=copies, **HYPER)
    assert (plan._own is not None) == (max(counts) > (56 if eight else 64))
    check, state = (check_adamw8, values8) if eight else (check_adamw, lambda s: values(s, "pgmv"))
    for step in (3, 4):
        old = [state(s) for s in sets]
        plan(step)
        where.sync()
        for s, o in zip(sets, old):
            check(s, o, step, f"step {step}", **HYPER)


# ---------------------------------------------------------------------------
# threads
# ---------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("eight", [False, True])
def test_a_plan_of_adamw_from_several_threads(eight):
    """Threads on streams of their own run steps with lr, step, gradients, seed and clipping of their own, each through its
    own plan, all at once; the results are those of the same steps one after the other."""
    from pccl import optim
    dev, threads, steps = "cuda:0", 4, 25
    sizes = [300 + k for k in range(70)]
    keys = ("p", "g", "m", "r", "ms", "rs") if eight else ("p", "g", "m", "v")

    def fresh():
        out = []
        for k in range(threads):
            s = make(sizes, dev, g="bf16", c="bf16", seed=100 + k, eight=eight)
            other = make(sizes, dev, g="bf16", seed=200 + k)["g"].list
            plan = (optim.plan_adamw8 if eight else optim.plan_adamw)(*(s[x].list for x in keys), copies=s["c"].list, **HYPER)
            out.append((s, other, plan, torch.tensor([1.0 + k], device=dev)))
        return out

    def run(k, job):
        s, other, plan, norm = job
        more = dict(seed=k) if eight else {}
        for t in range(1, steps + 1):
            plan(t + 10 * k, lr=1e-3 * (k + 1), grad_scale=1 / (k + 1), norm=norm, max_norm=0.5 + k, grads=other if t % 3 == 0 else None, **more)
    a, b = fresh(), fresh()
    torch.cuda.synchronize()
    for k in range(threads):
        run(k, a[k])
    errors = []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                run(k, b[k])
                torch.cuda.current_stream().synchronize()
        except BaseException as e:            # noqa: BLE001 - reported by the main thread
            errors.append(e)
    ts = [threading.Thread(target=work, args=(k,)) for k in range(threads)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for k in range(threads):
        for x in keys + ("c",):
            assert np.array_equal(Flat.raw(a[k][0][x].flat), Flat.raw(b[k][0][x].flat)), (k, x)


@pytest.mark.gpu
def test_one_plan_with_other_scalars_from_several_threads():
    """One plan, one thread after the other on streams of their own: what a call brings (lr, step, gradients) is that call's."""
    from pccl import optim
    dev, n = "cuda:0", 5000
    s, t = (make([n], dev, seed=300) for _ in range(2))
    gs = [torch.randn(n, generator=torch.Generator().manual_seed(k)).to(dev) * 0.01 for k in range(8)]
    plan, plain = (optim.plan_adamw(*(x[k].list for k in "pgmv"), **HYPER) for x in (s, t))
    torch.cuda.synchronize()
    turn, errors = threading.Condition(), []
    done = [0]

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                with turn:
                    turn.wait_for(lambda: done[0] == k or errors, timeout=60)
                    plan(k + 1, lr=1e-3 * (k + 1), grads=[gs[k]])
                    torch.cuda.current_stream().synchronize()
                    done[0] += 1
                    turn.notify_all()
        except BaseException as e:            # noqa: BLE001 - reported by the main thread
            with turn:
                errors.append(e)
                turn.notify_all()
    ts = [threading.Thread(target=work, args=(k,)) for k in range(8)]
    for x in ts:
        x.start()
    for x in ts:
        x.join()
    assert not errors, errors
    for k in range(8):
        plain(k + 1, lr=1e-3 * (k + 1), grads=[gs[k]])
    torch.cuda.synchronize()
    for key in "pmv":
        assert np.array_equal(Flat.raw(s[key].flat), Flat.raw(t[key].flat)), key
