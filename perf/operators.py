"""Operators that hold the expert layer's numbers in few bits, and the cases they are measured on.

The numbers are held in microscaled blocks: 32 neighbours along the axis that is summed over
share one power of two, 2^e with e = floor(log2(largest magnitude)) - emax, stored as a byte
e + 127 (a block of zeros has byte 0).  Every value divided by it is rounded to nearest, ties
to the even code, and what lies beyond the largest code becomes that code:

  4 bits  e2m1, magnitudes 0 0.5 1 1.5 2 3 4 6, emax = 2, two codes a byte (the earlier in the low half)
  8 bits  e4m3, largest magnitude 448, subnormals of 2^-9, emax = 8

  rows      quantise the rows of a matrix and read them back
  weights   quantise expert weights [E][K][N] along K and read them back
  linear    y[T][N] = q4(x)[T][K] . W[N][K]^T, W held in 4 bits
  experts   o = q4(silu(g) * u) . Wd[e]^T with g, u = q4(x) . Wg[e]^T, q4(x) . Wu[e]^T over the
            rows of each expert; all three weights held in 4 bits
  train     the expert feed-forward's training step: o = (silu(g) * u) . Wd[e] in bf16, g and u
            kept in 8 bits, and from them the gradients of x and of the three weights

`own` false: the plain form in elementary operations; true: the framework's kernels.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

BLOCK = 32


def _microscale():
    """The framework's module; its package's folder is not named like a Python module."""
    name = "project_axiom_ai_llm_b200"
    if name not in sys.modules:
        folder = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "project-axiom-ai-llm_b200")
        spec = importlib.util.spec_from_file_location(name, os.path.join(folder, "__init__.py"),
                                                      submodule_search_locations=[folder])
        module = importlib.util.module_from_spec(spec)
        sys.modules[name] = module
        spec.loader.exec_module(module)
    return importlib.import_module(name + ".microscale")


# ---- cases ------------------------------------------------------------------------------------

def listed():
    return [
        # one token's activations before a product in 4 bits: latency
        dict(name="rows 4 bits, 1 x 4096", op="rows", bits=4, rows=1, k=4096, dtype="bf16"),
        # a prompt's activations, fp32 as a residual stream may be held; odd number of rows
        dict(name="rows 4 bits, 8191 x 5632 fp32", op="rows", bits=4, rows=8191, k=5632, dtype="fp32"),
        # activations of one training batch laid aside in 8 bits
        dict(name="rows 8 bits, 16384 x 4096", op="rows", bits=8, rows=16384, k=4096, dtype="bf16"),
        # a small layer's experts quantised after loading
        dict(name="weights 8 x 256 x 512", op="weights", experts=8, k=256, n=512, dtype="bf16"),
        # a large layer's experts, from their fp32 master copy
        dict(name="weights 8 x 2048 x 5632 fp32", op="weights", experts=8, k=2048, n=5632, dtype="fp32"),
        # a projection of one token while text is generated
        dict(name="linear 1 token 4096 -> 14336", op="linear", tokens=1, k=4096, n=14336),
        # a projection of a long prompt
        dict(name="linear 8192 tokens 4096 -> 14336", op="linear", tokens=8192, k=4096, n=14336),
        # the experts of a wide layer for one token
        dict(name="experts 1 token, 8 x 4096 x 14336", op="experts", tokens=1, d=4096, f=14336, experts=8, top_k=2, skew=0.0),
        # many narrow experts, a short odd batch, a few experts far more popular than the rest
        dict(name="experts 515 tokens, 64 x 2048 x 1408", op="experts", tokens=515, d=2048, f=1408, experts=64, top_k=6, skew=3.0),
        # the wide layer's experts on a long prompt
        dict(name="experts 8192 tokens, 8 x 4096 x 14336", op="experts", tokens=8192, d=4096, f=14336, experts=8, top_k=2, skew=0.0),
        # a training step of a small layer
        dict(name="train 64 tokens, 8 x 256 x 512", op="train", tokens=64, d=256, f=512, experts=8, top_k=2, skew=0.0),
        # a training step of a full layer
        dict(name="train 8192 tokens, 16 x 2048 x 4096", op="train", tokens=8192, d=2048, f=4096, experts=16, top_k=2, skew=0.0),
    ]


def _spread(rng, low, high, step=1):
    """A multiple of `step` from low to high, even over the logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return min(high, max(low, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(("rows", "weights", "linear", "experts", "train"))
    if op == "rows":
        k = _spread(rng, 64, 14336, 32)
        most = 16384 * 4096 // k
        return dict(op=op, bits=rng.choice((4, 8)), rows=_spread(rng, 1, min(most, 65536)), k=k, dtype=rng.choice(("bf16", "fp32")))
    if op == "weights":
        k, n = _spread(rng, 64, 4096, 32), _spread(rng, 64, 6144, 8)
        most = max(1, 8 * 2048 * 5632 // (k * n))
        return dict(op=op, experts=rng.randint(1, min(most, 64)), k=k, n=n, dtype=rng.choice(("bf16", "fp32")))
    if op == "linear":
        return dict(op=op, tokens=_spread(rng, 1, 8192), k=_spread(rng, 64, 4096, 32), n=_spread(rng, 64, 14336, 8))
    skew = rng.choice((0.0, 3.0))
    top_k = rng.choice((1, 2, 4, 6))
    experts = rng.choice((8, 12, 16, 64))
    if op == "experts":
        d, f = _spread(rng, 128, 4096, 32), _spread(rng, 128, 8192, 32)
        while experts * d * f > 8 * 4096 * 14336 // 2:
            f = max(128, f // 64 * 32)
        most = 8192 * 2 * 4096 * 14336 // (top_k * d * f)
        return dict(op=op, tokens=_spread(rng, 1, max(1, min(most, 8192))), d=d, f=f, experts=experts, top_k=top_k, skew=skew)
    d, f = _spread(rng, 128, 2048, 8), _spread(rng, 128, 4096, 32)
    while experts * d * f > 16 * 2048 * 4096:
        f = max(128, f // 64 * 32)
    most = 8192 * 2 * 2048 * 4096 // (top_k * d * f)
    return dict(op=op, tokens=_spread(rng, 1, max(1, min(most, 8192))), d=d, f=f, experts=experts, top_k=top_k, skew=skew)


def work(case):
    """Each input once, each output once, and the products' multiplications and additions."""
    op = case["op"]
    if op == "rows":
        n = case["rows"] * case["k"]
        return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + n * 2, "flops": 0}
    if op == "weights":
        n = case["experts"] * case["k"] * case["n"]
        return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + n * 2, "flops": 0}
    held = 0.5 + 1 / BLOCK  # bytes of one weight in 4 bits
    if op == "linear":
        t, k, n = case["tokens"], case["k"], case["n"]
        return {"bytes": 2 * t * k + held * n * k + 2 * t * n, "flops": 2 * t * k * n}
    rows, d, f, e = case["tokens"] * case["top_k"], case["d"], case["f"], case["experts"]
    touched = e * (1 - (1 - case["top_k"] / e) ** case["tokens"])  # experts that get a row, on average
    if op == "experts":
        return {"bytes": 4 * rows * d + held * 3 * touched * d * f, "flops": 6 * rows * d * f}
    return {"bytes": 8 * rows * d + 6 * touched * d * f + 6 * e * d * f, "flops": 18 * rows * d * f}


# ---- inputs -----------------------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, std, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, std, generator=g).to(dtype)


def _held_weights(g, experts, k, n):
    """Weights as a checkpoint in 4 bits holds them: codes [E][N][K/2], scale bytes [E][N][K/32]."""
    codes, scales = [], []
    for _ in range(experts):
        c, s = _quantise(_normal(g, (n, k), 0.02).float(), 4)
        codes.append((c[:, 0::2] | (c[:, 1::2] << 4)).to(torch.uint8))
        scales.append(s)
    return torch.stack(codes), torch.stack(scales)


def _row_counts(g, case):
    """Rows of each expert when every token picks its top_k of noisy scores."""
    scores = torch.rand(case["tokens"], case["experts"], generator=g, device="cuda")
    rank = torch.randperm(case["experts"], generator=g, device="cuda").float() + 1
    scores = scores + case["skew"] * rank.pow(-1.2)
    picked = scores.topk(case["top_k"], dim=1).indices.reshape(-1)
    return torch.bincount(picked, minlength=case["experts"]).tolist()


def _segments(counts, align):
    """The layer's table of row ranges {first row in, first row out, rows, expert}, each range
    padded to a multiple of `align` rows, and the number of rows."""
    table, at = [], 0
    for e, c in enumerate(counts):
        rows = -(-c // align) * align
        table.append((at, at, rows, e))
        at += rows
    return table, at


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    dtype = torch.float32 if case.get("dtype") == "fp32" else torch.bfloat16
    if op == "rows":
        s = {"op": op, "bits": case["bits"], "x": _normal(g, (case["rows"], case["k"]), 1.0, dtype)}
    elif op == "weights":
        s = {"op": op, "w": _normal(g, (case["experts"], case["k"], case["n"]), 0.02, dtype)}
    elif op == "linear":
        s = {"op": op, "x": _normal(g, (case["tokens"], case["k"]), 1.0), "w": _held_weights(g, 1, case["k"], case["n"])}
    else:
        d, f, e = case["d"], case["f"], case["experts"]
        counts = _row_counts(g, case)
        table, rows = _segments(counts, 64 if op == "train" else 1)
        s = {"op": op, "table": table, "segments": torch.tensor(table, dtype=torch.int32, device="cuda")}
        s["x"] = _normal(g, (rows, d), 1.0)
        if op == "experts":
            s["gate"], s["up"], s["down"] = (_held_weights(g, e, *kn) for kn in ((d, f), (d, f), (f, d)))
        else:
            s["d_o"] = _normal(g, (rows, d), 1.0)
            for (at, _, n, _), c in zip(table, counts):  # rows that only fill a range up hold zeros
                s["x"][at + c:at + n] = 0
                s["d_o"][at + c:at + n] = 0
            s["gate"], s["up"] = _normal(g, (e, d, f), 0.02), _normal(g, (e, d, f), 0.02)
            s["down"] = _normal(g, (e, f, d), 0.02)
    if own:  # what a program keeps from call to call: laid-out weights and workspaces
        ms = s["microscale"] = _microscale()
        if op == "linear":
            s["plan"] = ms.Mx4Linear(ms.Mx4Weights.from_checkpoint(*s["w"]), case["tokens"])
        elif op == "experts":
            s["plan"] = ms.Mx4ExpertFfn(*(ms.Mx4Weights.from_checkpoint(*s[n]) for n in ("gate", "up", "down")),
                                        rows=s["x"].shape[0], tokens=case["tokens"])
        elif op == "train":
            s["plan"] = ms.Mx8TrainFfn(s["gate"], s["up"], s["down"], rows=s["x"].shape[0])
    return s


# ---- the plain form ---------------------------------------------------------------------------

def _scale_exponent(amax, emax):
    _, e = torch.frexp(amax)
    return torch.where(amax > 0, e - 1 - emax, torch.full_like(e, -127)).clamp(-127, 127)


def _round_magnitude(a, bits):
    if bits == 4:
        a = a.clamp(max=6.0)
        step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    else:
        a = a.clamp(max=448.0)
        step = torch.ldexp(torch.ones_like(a), (torch.frexp(a)[1] - 1).clamp(min=-6) - 3)
    return torch.round(a / step) * step


def _split(x, bits):
    """Rounded values relative to their block's scale, [..., K/32, 32], and the scale's exponent."""
    b = x.reshape(*x.shape[:-1], -1, BLOCK)
    e = _scale_exponent(b.abs().amax(-1), 2 if bits == 4 else 8)
    a = torch.ldexp(b, -e.unsqueeze(-1))
    return torch.copysign(_round_magnitude(a.abs(), bits), a), e


def _held(x, bits):
    """x as its blocks hold it."""
    v, e = _split(x.float(), bits)
    return torch.ldexp(v, e.unsqueeze(-1)).reshape(x.shape)


def _quantise(x, bits):
    """4-bit codes (one a byte) and scale bytes."""
    v, e = _split(x, bits)
    a = v.abs()
    code = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = code | (torch.signbit(v).to(torch.uint8) << 3)
    return code.reshape(x.shape), (e + 127).to(torch.uint8)


def _values(codes, scales, dtype=torch.float32):
    """[N][K] of codes [N][K/2] and scale bytes [N][K/32]."""
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], dtype=dtype, device=codes.device)
    v = torch.stack((table[(codes & 15).long()], table[(codes >> 4).long()]), -1)
    v = torch.ldexp(v.reshape(codes.shape[0], -1, BLOCK), (scales.int() - 127).unsqueeze(-1))
    return v.reshape(codes.shape[0], -1)


def _plain(s):
    op = s["op"]
    if op == "rows":
        return {"values": _held(s["x"], s["bits"]).bfloat16()}
    if op == "weights":
        return {"values": _held(s["w"].transpose(1, 2), 4).transpose(1, 2).bfloat16()}
    if op == "linear":
        return {"y": (_held(s["x"], 4) @ _values(s["w"][0][0], s["w"][1][0]).T).bfloat16()}
    x = s["x"]
    if op == "experts":
        o = torch.empty_like(x)
        held = _held(x, 4)
        for at, _, n, e in s["table"]:
            if n == 0:
                continue
            a = held[at:at + n]
            g = a @ _values(s["gate"][0][e], s["gate"][1][e]).T
            u = a @ _values(s["up"][0][e], s["up"][1][e]).T
            h = _held(g / (1 + torch.exp(-g)) * u, 4)
            o[at:at + n] = (h @ _values(s["down"][0][e], s["down"][1][e]).T).bfloat16()
        return {"o": o}
    o, d_x = torch.empty_like(x), torch.empty_like(x)
    d_gate, d_up, d_down = (torch.zeros_like(s[n]) for n in ("gate", "up", "down"))
    for at, _, n, e in s["table"]:
        if n == 0:
            continue
        a, d_o = x[at:at + n].float(), s["d_o"][at:at + n].float()
        wg, wu, wd = s["gate"][e].float(), s["up"][e].float(), s["down"][e].float()
        g, u = a @ wg, a @ wu
        o[at:at + n] = ((g / (1 + torch.exp(-g)) * u) @ wd).bfloat16()
        g, u = _held(g, 8), _held(u, 8)
        sig = 1 / (1 + torch.exp(-g))
        d_h = d_o @ wd.T
        d_g, d_u = d_h * u * sig * (1 + g * (1 - sig)), d_h * g * sig
        d_x[at:at + n] = (d_g @ wg.T + d_u @ wu.T).bfloat16()
        d_gate[e], d_up[e] = (a.T @ d_g).bfloat16(), (a.T @ d_u).bfloat16()
        d_down[e] = ((g * sig * u).T @ d_o).bfloat16()
    return {"o": o, "d_x": d_x, "d_gate": d_gate, "d_up": d_up, "d_down": d_down}


def run(state):
    if not own:
        return _plain(state)
    op, ms = state["op"], state["microscale"]
    if op == "rows":
        if state["bits"] == 4:
            return {"values": ms.dequantize_rows(ms.quantize_rows(state["x"]))}
        return {"values": ms.dequantize_rows8(*ms.quantize_rows8(state["x"]))}
    if op == "weights":
        return {"values": ms.dequantize_weights(ms.quantize_weights(state["w"]))}
    plan = state["plan"]
    if op == "linear":
        return {"y": plan.forward(state["x"])}
    if op == "experts":
        return {"o": plan.forward(state["x"], state["segments"])}
    o = plan.forward(state["x"], state["segments"])
    return {"o": o, **plan.backward(state["d_o"])}


# ---- the definition in 64 bits ----------------------------------------------------------------

def _exact_held(x, bits):
    """Blocks along the last axis, by comparison with the midpoints between codes (4 bits) or by
    adding and taking away a number whose last bit is the step (8 bits)."""
    x = x.double()
    b = x.unflatten(-1, (-1, BLOCK))
    top = b.abs().amax(-1, keepdim=True)
    power = torch.floor(torch.log2(top))
    power = torch.where(torch.exp2(power) > top, power - 1, power)  # log2 may round up to a whole number
    power = torch.where(torch.exp2(power + 1) <= top, power + 1, power)
    scale = torch.exp2((power - (2 if bits == 4 else 8)).clamp(min=-127))
    scale = torch.where(top > 0, scale, torch.ones_like(scale))
    a = b.abs() / scale
    if bits == 4:
        value = torch.zeros_like(a)
        low = 0.0
        for i, high in enumerate((.5, 1., 1.5, 2., 3., 4., 6.)):
            middle = (low + high) / 2  # the tie goes to the even one of codes i and i + 1
            value = torch.where(a > middle if i % 2 == 0 else a >= middle, torch.full_like(a, high), value)
            low = high
    else:
        a = a.clamp(max=448.0)
        step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
        step = torch.where(step * 16 <= a, step * 2, step)
        step = torch.where((step * 8 > a) & (step > 2.0 ** -9), step / 2, step)
        big = step * 1.5 * 2.0 ** 52
        value = (a + big) - big
    return (torch.sign(b) * value * scale).flatten(-2)


def _exact_weights(codes, scales):
    """[N][K] of one expert's codes and scale bytes, from the bits of the codes."""
    c = torch.stack((codes.bitwise_and(15), codes.bitwise_right_shift(4)), -1).flatten(-2)
    exponent, fraction = (c >> 1 & 3).double(), (c & 1).double()
    v = torch.where(exponent > 0, (1 + fraction / 2) * torch.exp2(exponent - 1), fraction / 2)
    v = v * (1 - 2 * (c >> 3).double())
    return v * torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, -1)


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "rows":
        return {"values": _exact_held(s["x"], s["bits"])}
    if op == "weights":
        return {"values": torch.stack([_exact_held(w.T, 4).T for w in s["w"]])}
    if op == "linear":
        return {"y": torch.einsum("tk,nk->tn", _exact_held(s["x"], 4), _exact_weights(s["w"][0][0], s["w"][1][0]))}
    x = s["x"].double()
    if op == "experts":
        o = torch.zeros_like(x)
        for first, _, count, e in s["table"]:
            a = _exact_held(x[first:first + count], 4)
            g, u = (torch.einsum("tk,nk->tn", a, _exact_weights(s[n][0][e], s[n][1][e])) for n in ("gate", "up"))
            h = _exact_held(g * torch.sigmoid(g) * u, 4)
            o[first:first + count] = torch.einsum("tk,nk->tn", h, _exact_weights(s["down"][0][e], s["down"][1][e]))
        return {"o": o}
    o, d_x = torch.zeros_like(x), torch.zeros_like(x)
    d_gate, d_up, d_down = (torch.zeros(s[n].shape, dtype=torch.float64, device=x.device) for n in ("gate", "up", "down"))
    for first, _, count, e in s["table"]:
        rows = slice(first, first + count)
        d_o = s["d_o"][rows].double()
        wg, wu, wd = (s[n][e].double() for n in ("gate", "up", "down"))
        g, u = x[rows] @ wg, x[rows] @ wu
        o[rows] = (torch.nn.functional.silu(g) * u) @ wd
        g, u = _exact_held(g, 8), _exact_held(u, 8)
        sig = torch.sigmoid(g)
        h = g * sig
        d_h = torch.einsum("td,fd->tf", d_o, wd)
        d_u = d_h * h
        d_g = d_h * u * (sig + h * (1 - sig))
        d_x[rows] = torch.einsum("tf,df->td", d_g, wg) + torch.einsum("tf,df->td", d_u, wu)
        d_gate[e], d_up[e] = torch.einsum("td,tf->df", x[rows], d_g), torch.einsum("td,tf->df", x[rows], d_u)
        d_down[e] = torch.einsum("tf,td->fd", h * u, d_o)
    return {"o": o, "d_x": d_x, "d_gate": d_gate, "d_up": d_up, "d_down": d_down}
