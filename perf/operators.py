"""The optimizer-side operators of a sharded training step, as cases to measure.

Between the reduce_scatter of the gradients and the all_gather of the parameters
a data-parallel program takes the norm of its gradients and runs the optimizer on
its shard.  Each case is one call of one operator on inputs made from a seed:

  adamw       AdamW over many tensors, moments in 32 bits
  adamw8      the same, moments in 8 bits with a scale per block of 256
  norm        2-norm over many gradient tensors
  quantize    tensors to 8-bit codes with a scale per block of 256
  dequantize  and back

The tensors of a case are pieces of flat buffers, as a sharded optimizer keeps
them, so the plain form can work on the flat buffers without a loop.
"""
import math
import os
import random
import sys

import torch

own = False

BLOCK = 256                       # elements per scale
LARGEST = 448.0                   # largest finite e4m3 value
FLOOR = 2.0 ** -100               # smallest block maximum a scale is made from
CHUNK = 4096                      # elements that share a gradient magnitude in the inputs

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2, "none": 0}
LR, BETA1, BETA2, EPS, DECAY = 3e-4, 0.9, 0.95, 1e-8, 0.1


def _optim():
    path = os.path.join(os.getcwd(), "sc2025-pccl-reproducer_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from pccl import optim
    return optim


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def _case(name, op, tensors, smallest, largest, p="f32", g="f32", c="none", clip=False, scale=1.0, seed=-1, root=False,
          sizes=1):
    return {"name": name, "op": op, "tensors": tensors, "smallest": smallest, "largest": largest, "sizes": sizes,
            "p": p, "g": g, "c": c, "clip": clip, "scale": scale, "seed": seed, "root": root}


def listed():
    Mi = 1 << 20
    return [
        # a single tensor of the smallest message of the latency sweep (4 KiB of a 16-bit type): launch cost only
        _case("adamw-one-small", "adamw", 1, 2048, 2048),
        # a model trained in bfloat16 throughout: 300 weights, biases and norm gains of odd sizes, packed end to end
        _case("adamw-many-bf16", "adamw", 300, 509, 1048583, p="bf16", g="bf16"),
        # the shards of 8 ranks (64 MiB of bfloat16 gradients each, the blocks of the 8-rank reduce_scatter) with fp32
        # master weights and the bfloat16 copy that the all_gather sends out, clipped by the global norm
        _case("adamw-ranks-mixed", "adamw", 8, 32 * Mi, 32 * Mi, g="bf16", c="bf16", clip=True),
        # the shards of 4 ranks of a small model: launch cost
        _case("adamw8-small", "adamw8", 4, 8192, 8192, g="bf16", c="bf16"),
        # odd sizes in float16 with a loss scale, clipped, rounded stochastically
        _case("adamw8-ragged-f16", "adamw8", 64, 1, 1500007, g="f16", c="f16", clip=True, scale=1.0 / 1024, seed=77),
        # the 8-rank shards again, states in 8 bits
        _case("adamw8-ranks-mixed", "adamw8", 8, 32 * Mi, 32 * Mi, g="bf16", c="bf16", clip=True, seed=5),
        # the gradient shards of 8 ranks, smallest message: launch cost
        _case("norm-small", "norm", 8, 2048, 2048, g="bf16"),
        # the gradient shards of 8 ranks at the size of the reduce_scatter benchmark
        _case("norm-ranks", "norm", 8, 32 * Mi, 32 * Mi, g="bf16"),
        # second moments of a 32-bit checkpoint going to 8 bits, tensors of odd sizes
        _case("quantize-state", "quantize", 40, 1, 6000011, g="f32", root=True),
        # weight shards of 16 ranks before an all_gather of their codes
        _case("quantize-weights", "quantize", 16, 8 * Mi, 8 * Mi, g="bf16"),
        # a few small second moments read back to 32 bits
        _case("dequantize-small", "dequantize", 4, 4099, 4099, g="f32", root=True),
        # the gathered codes of 16 ranks read back to weights
        _case("dequantize-weights", "dequantize", 16, 8 * Mi, 8 * Mi, g="bf16"),
    ]


def draw(rng):
    op = rng.choice(["adamw", "adamw", "adamw8", "adamw8", "norm", "quantize", "dequantize"])
    tensors = rng.choice([1, 2, 3, 4, 8, 16]) if rng.random() < 0.5 else int(math.exp(rng.uniform(0, math.log(300))))
    most = (1 << 27) // tensors                      # of one tensor, so that no case is larger than the listed ones
    largest = max(1, min(most, int(2.0 ** rng.uniform(6, 26)) + rng.randrange(64)))
    smallest = largest if rng.random() < 0.4 else max(1, int(largest ** rng.uniform(0.0, 1.0)))
    kinds = ["f32", "bf16", "f16"]
    case = _case("", op, tensors, smallest, largest, g=rng.choice(kinds), sizes=rng.randrange(1 << 20))
    del case["name"]
    if op in ("adamw", "adamw8"):
        case["p"] = rng.choice(["f32", "f32", "bf16", "f16"])
        case["c"] = rng.choice(["none", "bf16", "f16"]) if case["p"] == "f32" else "none"
        case["clip"] = rng.random() < 0.5
        case["scale"] = rng.choice([1.0, 0.125, 1.0 / 1024])
        if op == "adamw8":
            case["seed"] = rng.choice([-1, rng.randrange(1 << 31)])
    elif op != "norm":
        case["root"] = case["g"] == "f32" and rng.random() < 0.5
    return case


def _sizes(case):
    """The lengths of a case's tensors: all alike, or spread over the logarithm of the range."""
    a, b = case["smallest"], case["largest"]
    if a == b:
        return [a] * case["tensors"]
    r = random.Random(case["sizes"])
    return [min(b, max(a, round(math.exp(r.uniform(math.log(a), math.log(b)))))) for _ in range(case["tensors"])]


def _padded(n):
    return (n + BLOCK - 1) // BLOCK * BLOCK


def work(case):
    n = sum(_sizes(case))
    blocks = sum(_padded(k) // BLOCK for k in _sizes(case))
    g = BYTES[case["g"]]
    if case["op"] == "adamw":
        return {"bytes": n * (2 * BYTES[case["p"]] + g + BYTES[case["c"]] + 16), "flops": 15 * n}
    if case["op"] == "adamw8":
        return {"bytes": n * (2 * BYTES[case["p"]] + g + BYTES[case["c"]] + 4) + 16 * blocks, "flops": 25 * n}
    if case["op"] == "norm":
        return {"bytes": n * g, "flops": 2 * n}
    return {"bytes": n * (g + 1) + 4 * blocks, "flops": 3 * n}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    sizes = _sizes(case)
    blocked = case["op"] not in ("adamw", "norm")    # blocks restart at every tensor: there the pieces start at whole blocks
    starts, end = [], 0
    for n in sizes:
        starts.append(end)
        end += _padded(n) if blocked else n

    def pieces(flat):
        return [flat[s:s + n] for s, n in zip(starts, sizes)]

    def clear(flat):                                 # what lies between the pieces
        if blocked:
            for s, n in zip(starts, sizes):
                flat[s + n:s + _padded(n)] = 0
        return flat

    def normal():
        return torch.randn(end, device=dev, generator=gen)

    # gradient magnitudes from 1e-6 to 1e-2, alike over stretches; one stretch in 64 has not been reached by any token
    chunks = (end + CHUNK - 1) // CHUNK
    size = 10.0 ** (torch.rand(chunks, device=dev, generator=gen) * 4 - 6)
    size[torch.rand(chunks, device=dev, generator=gen) < 1 / 64] = 0
    size = size.repeat_interleave(CHUNK)[:end]
    s = {"case": dict(case), "step": 100}
    op = case["op"]
    if op in ("adamw", "adamw8"):
        s["p"] = clear((normal() * 0.02).to(TYPES[case["p"]]))
        s["g"] = clear((normal() * size / case["scale"]).to(TYPES[case["g"]]))
        m = clear(normal() * size * 0.3)
        v = clear(size * size * (0.25 + torch.rand(end, device=dev, generator=gen)))
        s["c"] = None if case["c"] == "none" else torch.zeros(end, dtype=TYPES[case["c"]], device=dev)
        s["norm"] = torch.full((1,), 2.5 / case["scale"], device=dev) if case["clip"] else None
        if op == "adamw":
            s["m"], s["v"] = m, v
        else:
            s["m"], s["m_scale"] = _encode(m, False, None)
            s["r"], s["r_scale"] = _encode(v.sqrt(), True, None)
    elif op == "norm":
        s["g"] = (normal() * size).to(TYPES[case["g"]])
    else:
        x = normal() * size
        x = clear((x * x if case["root"] else x).to(TYPES[case["g"]]))
        s["m"] = torch.zeros(end, dtype=torch.float8_e4m3fn, device=dev)
        s["m_scale"] = torch.zeros(end // BLOCK, device=dev)
        if op == "dequantize":
            s["m"], s["m_scale"] = _encode(x.float().sqrt() if case["root"] else x.float(), case["root"], None)
            x = torch.zeros_like(x)
        s["x"] = x
    if own:
        # what a program keeps: the tensors, and the plan over them
        optim = _optim()
        t = {k: pieces(v) for k, v in s.items() if k in ("p", "g", "m", "v", "r", "c", "x") and v is not None}
        for k in ("m_scale", "r_scale"):
            if k in s:
                t[k] = [s[k][a // BLOCK:a // BLOCK + _padded(n) // BLOCK] for a, n in zip(starts, sizes)]
        hyper = {"lr": LR, "betas": (BETA1, BETA2), "eps": EPS, "weight_decay": DECAY}
        if op == "adamw":
            s["plan"] = optim.plan_adamw(t["p"], t["g"], t["m"], t["v"], copies=t.get("c"), **hyper)
        elif op == "adamw8":
            s["plan"] = optim.plan_adamw8(t["p"], t["g"], t["m"], t["r"], t["m_scale"], t["r_scale"], copies=t.get("c"),
                                          **hyper)
        elif op == "norm":
            s["plan"] = optim.plan_grad_norm(t["g"])
        elif op == "quantize":
            s["plan"] = optim.plan_quantize_blocks(t["m"], t["m_scale"], t["x"], root=case["root"])
        else:
            s["plan"] = optim.plan_dequantize_blocks(t["x"], t["m"], t["m_scale"], root=case["root"])
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    case, op = s["case"], s["case"]["op"]
    if op == "norm":
        return s["plan"]()
    if op in ("quantize", "dequantize"):
        s["plan"]()
    elif op == "adamw":
        s["plan"](s["step"], grad_scale=case["scale"], norm=s["norm"], max_norm=1.0 if case["clip"] else None)
    else:
        s["plan"](s["step"], grad_scale=case["scale"], norm=s["norm"], max_norm=1.0 if case["clip"] else None,
                  seed=case["seed"] if case["seed"] >= 0 else None)
    return _outputs(s)


def _outputs(s):
    names = {"adamw": ("p", "m", "v", "c"), "adamw8": ("p", "m", "m_scale", "r", "r_scale", "c"),
             "quantize": ("m", "m_scale"), "dequantize": ("x",)}[s["case"]["op"]]
    return {k: s[k] for k in names if s[k] is not None}


def _run_plain(s):
    case, op = s["case"], s["case"]["op"]
    if op == "norm":
        x = s["g"].double()
        return torch.sqrt(torch.sum(x * x)).float().reshape(1)
    if op == "quantize":
        x = s["x"].float()
        codes, scales = _encode(torch.sqrt(x) if case["root"] else x, case["root"], None)
        s["m"].copy_(codes)
        s["m_scale"].copy_(scales)
        return _outputs(s)
    if op == "dequantize":
        x = _decode(s["m"], s["m_scale"])
        s["x"].copy_(x * x if case["root"] else x)
        return _outputs(s)
    g = s["g"].float() * case["scale"]
    if case["clip"]:
        g = g * torch.clamp(1.0 / (s["norm"] * case["scale"] + 1e-6), max=1.0)
    if op == "adamw":
        m, v = s["m"], s["v"]
    else:
        m, v = _decode(s["m"], s["m_scale"]), _decode(s["r"], s["r_scale"])
        v = v * v
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * (g * g)
    root = torch.sqrt(v)
    t = s["step"]
    denom = root / math.sqrt(1 - BETA2 ** t) + EPS
    p = s["p"].float() * (1 - LR * DECAY) - (LR / (1 - BETA1 ** t)) * (m / denom)
    s["p"].copy_(p)
    if s["c"] is not None:
        s["c"].copy_(p)
    if op == "adamw":
        s["m"].copy_(m)
        s["v"].copy_(v)
    else:
        low = high = None
        if case["seed"] >= 0:
            bits = _noise(case["seed"], t, s["place"] if "place" in s else _place(s), m.device)
            low, high = bits & 0xffff, bits >> 16
        codes, scales = _encode(m, False, low)
        s["m"].copy_(codes)
        s["m_scale"].copy_(scales)
        codes, scales = _encode(root, True, high)
        s["r"].copy_(codes)
        s["r_scale"].copy_(scales)
    return _outputs(s)


def _place(s):
    """Index of every element within its tensor (the pieces start at whole blocks); kept, it does not depend on the data."""
    sizes = _sizes(s["case"])
    lens = torch.tensor([_padded(n) for n in sizes], device="cuda")
    first = torch.repeat_interleave(torch.cumsum(lens, 0) - lens, lens)
    s["place"] = torch.arange(first.numel(), device="cuda") - first
    return s["place"]


def _mix(x):
    """A 32-bit multiply-xorshift mix on values held in 64 bits."""
    x = x & 0xffffffff
    x = x ^ (x >> 16)
    x = (x * 0x7feb352d) & 0xffffffff
    x = x ^ (x >> 15)
    x = (x * 0x846ca68b) & 0xffffffff
    return x ^ (x >> 16)


def _noise(seed, step, place, device):
    """32 random bits for every element: a function of the seed, the step and the element's index."""
    key = _mix(_mix(seed) + step)
    return _mix((place & 0xffffffff) + key + (place >> 32) * 0x9e3779b1)


def _encode(x, root, u16):
    """fp32 values (blocks of 256) as e4m3 codes and a scale per block; u16: 16 random bits for each value, or None."""
    x = x.reshape(-1, BLOCK)
    top = torch.amax(torch.abs(x), dim=1, keepdim=True)
    scale = torch.where(top < FLOOR, torch.full_like(top, FLOOR), top) / LARGEST
    y = x * (1.0 / scale)
    if root:                                          # a value that is not 0 is not written as 0
        y = torch.where((x > 0) & (y < 2.0 ** -9), torch.full_like(y, 2.0 ** -9), y)
    if u16 is not None:                               # the 20 mantissa bits that e4m3 drops, plus random ones, cut off
        a = torch.abs(y)
        shift = torch.where(a < 2.0 ** -6, 2.0 ** -6, 0.0)          # subnormal codes have one spacing, that of 2^-6
        cut = ((a + shift).view(torch.int32) + (u16.reshape(-1, BLOCK) << 4).int()) & ~0xfffff
        y = torch.sign(y) * torch.clamp(cut.view(torch.float32) - shift, max=LARGEST)
    return y.to(torch.float8_e4m3fn).reshape(-1), scale.reshape(-1)


def _decode(codes, scale):
    return (codes.float().reshape(-1, BLOCK) * scale.reshape(-1, 1)).reshape(-1)


# ---------------------------------------------------------------------------
# the same from the definition in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        return torch.linalg.vector_norm(s["g"].double()).reshape(1)
    if op == "quantize":
        x = s["x"].double()
        codes, scales = _exact_block_codes(x.sqrt() if case["root"] else x, case["root"], None)
        return {"m": codes, "m_scale": scales}
    if op == "dequantize":
        x = s["m"].double().view(-1, BLOCK).mul(s["m_scale"].double().unsqueeze(1)).view(-1)
        return {"x": x.square() if case["root"] else x}
    t, out = s["step"], {}
    factor = case["scale"]
    if case["clip"]:
        factor *= min(1.0, 1.0 / (float(s["norm"]) * case["scale"] + 1e-6))
    g = s["g"].double().mul_(factor)
    if op == "adamw":
        m, v = s["m"].double(), s["v"].double()
    else:
        m = s["m"].double().view(-1, BLOCK).mul(s["m_scale"].double().unsqueeze(1)).view(-1)
        v = s["r"].double().view(-1, BLOCK).mul(s["r_scale"].double().unsqueeze(1)).view(-1).square_()
    m.lerp_(g, 1 - BETA1)
    v.mul_(BETA2).addcmul_(g, g, value=1 - BETA2)
    del g
    step = m / (1 - BETA1 ** t) / ((v / (1 - BETA2 ** t)).sqrt_().add_(EPS))
    p = s["p"].double()
    out["p"] = p - LR * (step + DECAY * p)
    del step, p
    if s["c"] is not None:
        out["c"] = out["p"]
    if op == "adamw":
        out["m"], out["v"] = m, v
        return out
    low = high = None
    if case["seed"] >= 0:
        bits = _noise(case["seed"], t, _place(s), m.device)
        low, high = bits % 65536, bits // 65536
    out["m"], out["m_scale"] = _exact_block_codes(m, False, low)
    out["r"], out["r_scale"] = _exact_block_codes(v.sqrt_(), True, high)
    return out


def _exact_block_codes(x, root, u16):
    """The nearest e4m3 value (ties to even), or by random bits its lower or upper neighbour, in 64 bits throughout."""
    x = x.view(-1, BLOCK)
    scale = x.abs().amax(1).clamp_(min=FLOOR) / LARGEST
    y = x / scale.unsqueeze(1)
    if root:
        y = y.clamp(min=2.0 ** -9) * (x != 0)
    _, e = torch.frexp(y)                             # |y| = f * 2^e with f in [1/2, 1)
    y = torch.ldexp(y, 4 - e.clamp(min=-5))           # in units of the last place
    if u16 is None:
        y = y.round()
    else:
        y = (y.abs() + u16.view(-1, BLOCK) / 65536.0).floor() * y.sign()
    y = torch.ldexp(y, e.clamp(min=-5) - 4)
    return y.clamp(-LARGEST, LARGEST).view(-1), scale
