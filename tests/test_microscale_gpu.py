"""Microscaled operands on the GPU against 64-bit references: codes and scale bytes exactly, products
exactly where their sums provably fit 24 bits, else within the error of a sum in 32 bits."""
import importlib

import pytest
import torch

import microscale_ref as ref

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ms(axm):
    return importlib.import_module("project_axiom_ai_llm_b200.microscale")


def generator(dev, seed):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def awkward(rows, k, dtype, dev, seed):
    """Normal rows with every block of another size, zeros, ties, subnormals, the largest values,
    infinities and NaNs among them."""
    g = generator(dev, seed)
    x = torch.empty(rows, k, device=dev).normal_(generator=g)
    power = torch.randint(-40, 40, (rows, k // 32), generator=g, device=dev).float()
    x = x * torch.exp2(power).repeat_interleave(32, 1)
    b = x.view(rows, -1, 32)
    ties = torch.tensor([0.25, -.75, 1.25, -1.75, 2.5, -3.5, 5.0, 4.0], device=dev).repeat(4)
    n = b.shape[0] * b.shape[1]
    flat = b.view(n, 32)
    flat[0::11] = ties * torch.exp2(torch.randint(-100, 100, (flat[0::11].shape[0], 1), generator=g, device=dev).float())
    flat[1::13] = 0.0
    flat[2::17] = torch.finfo(dtype).max
    flat[3::19] = 1e-39
    flat[4::23, 5] = float("nan")
    flat[5::29, 31] = -float("inf")
    flat[6::31] = 2.0 ** -126
    return x.to(dtype)


def table(counts, dev, align=1):
    rows, at = [], 0
    for e, c in enumerate(counts):
        n = -(-c // align) * align
        rows.append((at, at, n, e))
        at += n
    return torch.tensor(rows, dtype=torch.int32, device=dev), at


def same(a, b):
    """Equal, NaN in the same places."""
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))


def held_float(x, bits, dtype):
    """Blocks as held, rounded to dtype (exact but for the smallest subnormals)."""
    return (ref.held4(x) if bits == 4 else ref.held8(x)).to(dtype)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("rows,k", [(1, 32), (1, 4096), (7, 96), (129, 288), (300, 544), (1031, 2048), (77, 128), (1001, 64), (515, 256), (3, 224)])
def test_rows_4_bits(ms, cuda_device, rows, k, dtype):
    x = awkward(rows, k, dtype, cuda_device, rows + k)
    q = ms.quantize_rows(x)
    code, s = ref.quantize4(x)
    got = ref.unpack4(q.codes)
    fine = (s != 255).repeat_interleave(32, 1)
    assert torch.equal(got[fine], code[fine])
    tiles = ref.tile_order(s)
    there = ref.tile_order(torch.ones_like(s)) != 0
    packed = q.scales.view(-1, tiles.shape[1], 512)[:tiles.shape[0]]
    assert torch.equal(packed[there], tiles[there])
    # bytes of blocks behind K are 0 in every row that exists
    if k % 256:
        rows_of = ref.tile_order(torch.ones(rows, (k + 255) // 256 * 8, dtype=torch.uint8, device=cuda_device)) != 0
        assert (packed[rows_of & ~there] == 0).all()
    for out in (BF16, FP32):
        assert same(ms.dequantize_rows(q, out), held_float(x, 4, out))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("rows,k", [(1, 32), (3, 4096), (129, 288), (1031, 416), (77, 128), (1001, 64), (515, 256), (3, 224)])
def test_rows_8_bits(ms, cuda_device, rows, k, dtype):
    x = awkward(rows, k, dtype, cuda_device, rows * k)
    codes, s = ms.quantize_rows8(x)
    assert torch.equal(s, ref.scale_bytes(x, 8))
    for out in (BF16, FP32):
        assert same(ms.dequantize_rows8(codes, s, out), held_float(x, 8, out))


def test_rows_with_strides_and_sources(ms, cuda_device):
    wide = awkward(40, 640, BF16, cuda_device, 4)
    x = wide[:, 64:64 + 288]  # row stride 640, 16-byte aligned
    assert same(ms.dequantize_rows(ms.quantize_rows(x)), held_float(x, 4, BF16))
    out = torch.full((40, 640), 3.0, dtype=BF16, device=cuda_device)
    ms.dequantize_rows(ms.quantize_rows(x), out=out[:, 64:64 + 288])
    assert same(out[:, 64:64 + 288], held_float(x, 4, BF16))
    assert (out[:, :64] == 3).all() and (out[:, 352:] == 3).all()
    # rows gathered on the way, two slots a source row, one of them empty
    src = torch.tensor([3, 79, -1, 0, 3, 42], dtype=torch.int32, device=cuda_device)
    want = held_float(x, 4, BF16)[(src.long() // 2).clamp(min=0)]
    want[2] = 0
    assert same(ms.dequantize_rows(ms.quantize_rows(x, row_src=src, row_div=2)), want)
    with pytest.raises(Exception):
        ms.quantize_rows(wide[:, 4:4 + 288])  # not 16-byte aligned


@pytest.mark.parametrize("k", [96, 160, 544])
@pytest.mark.parametrize("counts", [[5], [0, 3, 0, 0, 200, 1, 0], [128, 128, 127, 129, 0], [1] * 70, [300, 0, 0]])
def test_rows_by_segments(ms, cuda_device, counts, k):
    segs, rows = table(counts, cuda_device)
    x = awkward(rows + 9, k, FP32, cuda_device, sum(counts))  # nine rows behind the last segment
    q = ms.quantize_rows(x, segments=segs)
    s = ref.scale_bytes(x, 2)
    got = q.scales.view(-1, (k + 255) // 256 * 2, 512)
    at = 0
    for e, c in enumerate(counts):
        if c:
            tiles = ref.tile_order(s[at:at + c])
            there = ref.tile_order(torch.ones_like(s[at:at + c])) != 0
            first = at // 128 + e
            assert torch.equal(got[first:first + tiles.shape[0]][there], tiles[there])
        at += c
    out = torch.full((rows + 9, k), 7.0, device=cuda_device)
    ms.dequantize_rows(q, out=out)
    assert same(out[:rows], held_float(x, 4, FP32)[:rows])
    assert (out[rows:] == 7).all()


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("e,k,n", [(1, 32, 8), (3, 96, 72), (2, 288, 136), (1, 544, 1000), (2, 2048, 64)])
def test_weights(ms, cuda_device, e, k, n, dtype):
    w = awkward(e * n, k, dtype, cuda_device, e + k + n).view(e, n, k).transpose(1, 2).contiguous()
    q = ms.quantize_weights(w)
    wt = w.transpose(1, 2).contiguous()
    code, s = ref.quantize4(wt)
    fine = (s != 255).repeat_interleave(32, -1)
    assert torch.equal(ref.unpack4(q.codes)[fine], code[fine])
    want = torch.stack([ref.tile_order(s[i]) for i in range(e)])
    there = torch.stack([ref.tile_order(torch.ones_like(s[i])) for i in range(e)]) != 0
    assert torch.equal(q.scales.view(want.shape)[there], want[there])
    for out in (BF16, FP32):
        assert same(ms.dequantize_weights(q, out), ref.held4(wt).to(out).transpose(1, 2))
    p = ms.Mx4Weights.from_checkpoint(ref.pack4(code), s)
    assert torch.equal(p.scales.view(want.shape)[there], want[there])


def held_operand(rows, k, dev, seed, spread):
    """Random 4-bit rows: packed codes, scale bytes and values; scales of 2^0 .. 2^spread.  Every
    block begins with the largest code, so that its values quantise to themselves."""
    g = generator(dev, seed)
    code = torch.randint(0, 16, (rows, k), generator=g, device=dev, dtype=torch.uint8)
    code[:, ::32] = 7
    s = torch.randint(127, 128 + spread, (rows, k // 32), generator=g, device=dev, dtype=torch.uint8)
    return ref.pack4(code), s, ref.values4(code, s)


LINEAR = [(1, 32, 8), (1, 4096, 264), (2, 256, 136), (3, 64, 256), (16, 544, 1000), (17, 288, 512), (33, 96, 40),
          (64, 1024, 384), (100, 512, 248), (127, 256, 128), (128, 320, 264), (129, 64, 520), (257, 736, 1288),
          (700, 128, 2048)]


@pytest.mark.parametrize("t,k,n", LINEAR)
def test_linear_exact(ms, cuda_device, t, k, n):
    """x is made of values that quantise to themselves; every sum of magnitudes fits 24 bits of the
    smallest product, so whatever the order of additions the result is the exact one."""
    _, _, x = held_operand(t, k, cuda_device, t + k, 1)
    assert torch.equal(ref.held4(x), x)
    codes, s, w = held_operand(n, k, cuda_device, n, 1)
    want = x @ w.T
    assert float((x.abs() @ w.abs().T).max()) < 2 ** 24 * 0.25 and float((want * 4 - torch.round(want * 4)).abs().max()) == 0
    plan = ms.Mx4Linear(ms.Mx4Weights.from_checkpoint(codes.unsqueeze(0), s.unsqueeze(0)), t + 3)
    for dt in (FP32, BF16):
        for x_dt in (FP32, BF16):
            out = torch.full((t + 1, n), float("nan"), dtype=dt, device=cuda_device)
            plan.forward(x.to(x_dt), out=out[:t])
            assert torch.equal(out[:t], want.to(dt)), (dt, x_dt)
            assert torch.isnan(out[t]).all()
    assert plan.status() == 0


@pytest.mark.parametrize("t,k,n", [(1, 4096, 1024), (5, 2048, 392), (40, 1056, 640), (200, 4096, 512), (513, 1408, 1032)])
def test_linear_wide_scales(ms, cuda_device, t, k, n):
    g = generator(cuda_device, t)
    x = torch.empty(t, k, device=cuda_device).normal_(generator=g) * torch.exp2(
        torch.randint(-20, 20, (t, k // 32), generator=g, device=cuda_device).float()).repeat_interleave(32, 1)
    codes, s, w = held_operand(n, k, cuda_device, n, 20)
    plan = ms.Mx4Linear(ms.Mx4Weights.from_checkpoint(codes.unsqueeze(0), s.unsqueeze(0)), t)
    y = plan.forward(x, dtype=FP32)
    a = ref.held4(x)
    # each of k additions rounds (or cuts) at 2^-23 of a partial sum of at most sum |a w|
    bound = k * 2.0 ** -23 * (a.abs() @ w.abs().T)
    assert ((y.double() - a @ w.T).abs() <= bound).all()
    assert plan.status() == 0


def test_nothing_to_do(ms, cuda_device):
    """No rows: nothing happens, and nothing fails."""
    empty = torch.empty(0, 64, dtype=BF16, device=cuda_device)
    assert ms.dequantize_rows(ms.quantize_rows(empty)).shape == (0, 64)
    assert ms.dequantize_rows8(*ms.quantize_rows8(empty)).shape == (0, 64)
    w = ms.quantize_weights(torch.ones(1, 64, 24, device=cuda_device))
    assert ms.Mx4Linear(w, 4).forward(empty).shape == (0, 24)
    v = ms.quantize_weights(torch.ones(1, 24 * 4, 64, device=cuda_device))
    w = ms.quantize_weights(torch.ones(1, 64, 24 * 4, device=cuda_device))
    segs, _ = table([0], cuda_device)
    assert ms.Mx4ExpertFfn(w, w, v, rows=4, tokens=4).forward(empty, segs).shape == (0, 64)
    out = torch.full((3, 64), 2.0, dtype=BF16, device=cuda_device)  # rows, but none in the table
    ms.Mx4ExpertFfn(w, w, v, rows=4, tokens=4).forward(torch.ones(3, 64, dtype=BF16, device=cuda_device), segs, out=out)
    assert (out == 2).all()


def test_linear_not_finite(ms, cuda_device):
    x = torch.ones(4, 64, device=cuda_device)
    x[1, 3], x[2, 40] = float("nan"), float("inf")
    codes, s, w = held_operand(16, 64, cuda_device, 2, 1)
    s[5, 1] = 255
    y = ms.Mx4Linear(ms.Mx4Weights.from_checkpoint(codes.unsqueeze(0), s.unsqueeze(0)), 4).forward(x)
    bad = torch.isnan(y)
    assert bad[1].all() and bad[2].all() and bad[:, 5].all()
    assert not bad[[0, 3]][:, [c for c in range(16) if c != 5]].any()


FFN = [([1], 64, 32), ([0, 1, 0, 1], 256, 512), ([3, 0, 2, 0, 0, 11], 96, 160), ([16, 1, 0, 15], 288, 416),
       ([40, 17, 0, 64], 544, 224), ([129, 0, 1, 300, 128], 160, 352), ([1] * 40 + [0] * 24 + [90], 128, 96),
       ([260, 255], 1024, 1408), ([0] * 9 + [33, 70], 96, 64), ([50, 3, 45, 64, 65, 0, 40], 160, 288), ([1] * 60 + [200, 130], 64, 96),
       ([12, 16, 17, 0, 1, 9], 320, 160), ([3] * 512, 64, 64)]


def exact_expert_weights(ms, e, k, n, dev, seed, shift):
    """[E][N][K] 4-bit weights of two neighbouring scales around 2^-shift, and their values."""
    code, s, v = held_operand(e * n, k, dev, seed, 1)
    s = s - shift
    return ms.Mx4Weights.from_checkpoint(code.view(e, n, -1), s.view(e, n, -1)), (v * 2.0 ** -shift).view(e, n, k)


def ffn_reference(x, segs, gate, up, down):
    """(o, bound on its error).  x, gate and up are such that g and u are exact in 32 bits; silu(g) u
    then carries the errors of e^-g (2 + 1.173 |g| ulp), a division (2 ulp), a sum and a product."""
    o, slack = torch.zeros_like(x, dtype=torch.float64), torch.zeros_like(x, dtype=torch.float64)
    for _, at, n, e in segs.tolist():
        if n == 0:
            continue
        a = ref.held4(x[at:at + n])
        for w in (gate[e], up[e]):
            unit = 0.25 * float(2.0 ** (torch.frexp(w.abs().max())[1] - 4))  # scales of two neighbouring powers
            assert float((a.abs() @ w.abs().T).max()) < 2 ** 24 * unit
        g, u = a @ gate[e].T, a @ up[e].T
        h = g * torch.sigmoid(g) * u
        rel = (6 + 1.2 * float(g.abs().max())) * 2.0 ** -23
        lo, hi = ref.candidates(h, rel, ref.held4, 2)
        held = ref.held4(h)
        o[at:at + n] = held @ down[e].T
        slack[at:at + n] = (torch.maximum(hi - held, held - lo) @ down[e].abs().T +
                            h.shape[1] * 2.0 ** -23 * (torch.maximum(lo.abs(), hi.abs()) @ down[e].abs().T))
    return o, slack


@pytest.mark.parametrize("counts,d,f", FFN)
def test_expert_ffn(ms, cuda_device, counts, d, f):
    segs, rows = table(counts, cuda_device)
    e = len(counts)
    _, _, x = held_operand(rows + 5, d, cuda_device, rows, 1)
    x = x.to(BF16)
    assert torch.equal(ref.held4(x), x.double())
    shift = (d.bit_length() + 7) // 2  # g of a few units
    qg, gate = exact_expert_weights(ms, e, d, f, cuda_device, 1, shift)
    qu, up = exact_expert_weights(ms, e, d, f, cuda_device, 2, shift)
    qd, down = exact_expert_weights(ms, e, f, d, cuda_device, 3, shift)
    plan = ms.Mx4ExpertFfn(qg, qu, qd, rows=rows + 5, tokens=max(counts))
    o, slack = ffn_reference(x, segs, gate, up, down)
    for dt in (FP32, BF16):
        out = torch.full((rows + 5, d), float("nan"), dtype=dt, device=cuda_device)
        plan.forward(x, segs, out=out)
        assert plan.status() == 0
        half = 0.0 if dt == FP32 else 2.0 ** -8
        err = (out[:rows].double() - o[:rows]).abs()
        assert (err <= slack[:rows] + half * (o[:rows].abs() + slack[:rows])).all(), float((err - slack[:rows]).max())
        assert torch.isnan(out[rows:].float()).all()  # rows behind the last segment are left as they were
    assert float(slack[:rows].norm()) < 0.02 * float(o.norm())  # the bound says something


@pytest.mark.parametrize("rows", [40, 600, 3000])
def test_tables_that_do_not_fit(ms, cuda_device, rows):
    """Rows behind the matrices' end, segments that start outside and experts that do not exist are left
    out; the rest is computed as without them (few rows, one-CTA and pair kernels)."""
    d, f, e = 64, 96, 4
    q = [ms.quantize_weights(torch.randn(e, k, n, device=cuda_device) * 0.2) for k, n in ((d, f), (d, f), (f, d))]
    x = torch.randn(rows, d, device=cuda_device).to(BF16)
    n = rows // 4
    good = [(0, 0, n, 1), (n, n, n, 0), (2 * n, 2 * n, rows - 2 * n, 3)]
    odd = [(0, 0, n, 1), (n, n, n, 0), (2 * n, 2 * n, 5 * rows, 3), (rows, rows, 7, 2), (1 << 30, 1 << 30, 9, 2)]
    wrong = [(0, 0, n, 1), (n, n, n, 9), (2 * n, 2 * n, rows - 2 * n, 3)]
    plan = ms.Mx4ExpertFfn(*q, rows=rows, tokens=rows, segments=5)
    out = []
    for t in (good, odd, wrong):
        o = torch.full((rows, d), 5.0, dtype=BF16, device=cuda_device)
        plan.forward(x, torch.tensor(t, dtype=torch.int32, device=cuda_device), out=o)
        assert plan.status() == 0
        out.append(o)
    # another table may choose another kernel: compare as sums in another order, but for single roundings
    # of h that fall the other way (one step of e2m1 of one product)
    same_rows = (out[0].float() - out[1].float()).norm() <= 0.01 * out[0].float().norm()
    assert bool(same_rows)
    assert (out[2][n:2 * n] == 5).all()
    keep = torch.cat((torch.arange(n), torch.arange(2 * n, rows))).to(cuda_device)
    assert torch.equal(out[2][keep], out[0][keep])


def layer_weights(ms, axm, cfg, dev, seed=0):
    """4-bit weights of a layer, and the same layer's values in the engine's layout in bf16."""
    D, F, E, S = cfg["d"], cfg["f"], cfg["e"], cfg.get("shared", 0)
    g = generator(dev, seed)
    q, v = {}, {}

    def draw(*shape):
        return torch.empty(*shape, device=dev).normal_(0, 0.05, generator=g)

    q["router_w"] = v["router_w"] = draw(D, E)
    for name, n, (k, m) in [("gate", E, (D, F)), ("up", E, (D, F)), ("down", E, (F, D)), ("shared_gate", S, (D, F)),
                            ("shared_up", S, (D, F)), ("shared_down", S, (F, D))]:
        if n:
            q[name] = ms.quantize_weights(draw(n, k, m))
            v[name] = ms.dequantize_weights(q[name], FP32).double()
    return q, v


LAYER = [dict(t=1, d=64, f=96, e=4, k=2), dict(t=5, d=256, f=512, e=8, k=2, shared=1), dict(t=64, d=256, f=512, e=8, k=2),
         dict(t=130, d=96, f=160, e=12, k=4, shared=2), dict(t=700, d=256, f=352, e=64, k=6, shared=2)]


@pytest.mark.parametrize("cfg", LAYER, ids=lambda c: "-".join(str(v) for v in c.values()))
def test_layer(ms, axm, cuda_device, cfg):
    """The layer's output from its own routing (whose exactness the layer's other tests show): the
    chosen experts' feed-forwards by the stage's own call, combined in 64 bits."""
    q, _ = layer_weights(ms, axm, cfg, cuda_device)
    T, D, E, k, S = cfg["t"], cfg["d"], cfg["e"], cfg["k"], cfg.get("shared", 0)
    x = torch.empty(T, D, device=cuda_device).normal_(generator=generator(cuda_device, 9)).to(BF16)
    layer = ms.Mx4MoeLayer(q, T, k)
    out, hist = layer.forward(x)
    assert layer.status() == 0
    idx, gate = layer.topk_idx.long(), layer.topk_gate.double()
    assert torch.equal(hist.long(), torch.bincount(idx.reshape(-1), minlength=E))
    logits = x.double() @ q["router_w"].double()
    assert torch.equal(logits.gather(1, idx).sum(1) >= logits.topk(k).values.sum(1) - 1e-3, torch.ones(T, dtype=torch.bool, device=cuda_device))

    def stage(w, counts, rows):
        segs, n = table(counts, cuda_device)
        plan = ms.Mx4ExpertFfn(*w, rows=n, tokens=T)
        return plan.forward(rows, segs, dtype=FP32).double()

    order = torch.argsort(idx.reshape(-1), stable=True)
    o = torch.empty(T * k, D, dtype=torch.float64, device=cuda_device)
    o[order] = stage((q["gate"], q["up"], q["down"]), hist.tolist(), x[order // k].contiguous())
    y = (o.view(T, k, D) * gate.unsqueeze(-1)).sum(1)
    size = (o.view(T, k, D) * gate.unsqueeze(-1)).abs().sum(1)
    for i in range(S):
        one = [ms.Mx4Weights.from_checkpoint(q[n].codes[i:i + 1].contiguous(), ref.scale_bytes(
            ms.dequantize_weights(q[n], FP32)[i].T, 2).unsqueeze(0)) for n in ("shared_gate", "shared_up", "shared_down")]
        add = stage(one, [T], x)
        y, size = y + add, size + add.abs()
    # y in 32 bits (k + S products and sums), rounded to bf16, then x + y rounded again
    bound = (k + S + 1) * 2.0 ** -23 * size + 2.0 ** -8 * (y.abs() + size * 2.0 ** -20) + 2.0 ** -8 * ((x.double() + y).abs() + 2.0 ** -8 * y.abs()) + 1e-30
    assert ((out.double() - (x.double() + y)).abs() <= bound).all()
    # in place, without the residual, and accumulating the histogram
    z = x.clone()
    layer.forward(z, out=z)
    assert torch.equal(z, out)


def test_captured_calls_and_streams(ms, axm, cuda_device):
    """A captured call replays with new inputs; another stream gives the same bits; two objects'
    workspaces do not meet."""
    cfg = dict(t=33, d=256, f=160, e=8, k=2)
    q, _ = layer_weights(ms, axm, cfg, cuda_device)
    x = [torch.empty(33, 256, device=cuda_device).normal_(generator=generator(cuda_device, i)).to(BF16) for i in range(2)]
    a, b = ms.Mx4MoeLayer(q, 33, 2), ms.Mx4MoeLayer(q, 33, 2)
    want = [a.forward(v)[0].clone() for v in x]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [b.forward(v)[0] for v in x]
    torch.cuda.synchronize()
    assert all(torch.equal(p, r) for p, r in zip(want, got))
    held, out = x[0].clone(), torch.empty_like(x[0])
    lin = ms.Mx4Linear(ms.quantize_weights(torch.randn(1, 256, 72, device=cuda_device)), 33)
    y = torch.empty(33, 72, dtype=BF16, device=cuda_device)
    want_y = [lin.forward(v).clone() for v in x]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.forward(held, out=out)
        lin.forward(held, out=y)
    for v, w, wy in list(zip(x, want, want_y)) * 2:
        held.copy_(v)
        out.zero_()
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w) and torch.equal(y, wy)


def test_same_bits_again(ms, cuda_device):
    """A call gives the same bits every time."""
    w = ms.quantize_weights(torch.randn(1, 1056, 520, device=cuda_device))
    for t in (1, 7, 300):
        x = torch.randn(t, 1056, device=cuda_device).to(BF16)
        plan = ms.Mx4Linear(w, t)
        first = plan.forward(x, dtype=FP32).clone()
        assert all(torch.equal(first, plan.forward(x, dtype=FP32)) for _ in range(5))


TRAIN = [([1], 8, 32), ([64], 64, 64), ([0, 1, 0, 70], 72, 160), ([3, 0, 2, 0, 0, 11], 256, 512),
         ([129, 0, 1, 300, 128], 520, 352), ([1] * 30 + [0] * 5 + [65], 136, 96), ([260, 255], 1032, 1408)]


def whole_values(g, shape, top, dev, scale):
    """Whole numbers -top..top times a power of two, in bf16 exactly."""
    return (torch.randint(-top, top + 1, shape, generator=g, device=dev).double() * scale)


@pytest.mark.parametrize("counts,d,f", TRAIN)
def test_train_step(ms, cuda_device, counts, d, f):
    """Inputs are small whole numbers times powers of two: g, u and dH are exact in 32 bits, so the
    kept codes must be the reference's, and every other output is off by its roundings alone."""
    dev = cuda_device
    e = len(counts)
    segs, rows = table(counts, dev, 64)
    gen = generator(dev, sum(counts) + d)
    shift = 2.0 ** -((d.bit_length() + 4) // 2)
    x = whole_values(gen, (rows + 3, d), 4, dev, 0.5)
    d_o = whole_values(gen, (rows + 3, d), 4, dev, 0.25)
    for (at, _, n, i), c in zip(segs.tolist(), counts):
        x[at + c:at + n] = 0
        d_o[at + c:at + n] = 0
    gate, up = (whole_values(gen, (e, d, f), 4, dev, shift) for _ in range(2))
    down = whole_values(gen, (e, f, d), 4, dev, shift)
    assert d * 16 < 2 ** 24
    for dt, half in ((FP32, 0.0), (BF16, 2.0 ** -8)):
        plan = ms.Mx8TrainFfn(gate.to(BF16), up.to(BF16), down.to(BF16), rows=rows + 3, dtype=dt)
        o = torch.full((rows + 3, d), float("nan"), dtype=dt, device=dev)
        plan.forward(x.to(BF16), segs, out=o)
        got = plan.backward(d_o.to(BF16))
        assert plan.status() == 0
        gc, gs, uc, us = plan.checkpoint
        tiny = 2.0 ** -23
        for _, at, n, i in segs.tolist():
            r = slice(at, at + n)
            if n == 0:
                assert all((got[k][i] == 0).all() for k in ("d_gate", "d_up", "d_down"))
                continue
            g, u = x[r] @ gate[i], x[r] @ up[i]
            for codes, scales, v in ((gc, gs, g), (uc, us, u)):
                assert torch.equal(scales[r], ref.scale_bytes(v, 8))
                assert same(ms.dequantize_rows8(codes[r].contiguous(), scales[r].contiguous(), FP32).double(), ref.held8(v))

            def check(name, value, want, slack):
                err = (value.double() - want).abs()
                bound = slack + half * (want.abs() + slack) + 1e-30
                assert (err <= bound).all(), (name, float((err / bound.clamp(min=1e-30)).max()))

            # o: h rounded to bf16 after a sigmoid of a few ulp, then a sum of f products
            fast = (8 + 1.2 * float(g.abs().max())) * tiny
            h = g * torch.sigmoid(g) * u
            check("o", o[r], h @ down[i], (2.0 ** -8 + fast + f * tiny) * 1.01 * (h.abs() @ down[i].abs()))
            g, u = ref.held8(g), ref.held8(u)
            (d_x, d_wg, d_wu, d_wd), (d_h, s, d_g, d_u, hh) = ref.ffn_backward(x[r], g, u, d_o[r], gate[i], up[i], down[i])
            # the slope's two terms may cancel: its error is that of their magnitudes
            e_g = (d_h * u).abs() * (s + (g * s * (1 - s)).abs()) * fast + 2.0 ** -8 * 1.01 * d_g.abs()
            e_u = (2.0 ** -8 * 1.01 + fast) * d_u.abs()
            e_h = (2.0 ** -8 * 1.01 + fast) * hh.abs()
            a_g, a_u, a_h = d_g.abs() + e_g, d_u.abs() + e_u, hh.abs() + e_h
            check("d_x", got["d_x"][r], d_x, e_g @ gate[i].abs().T + e_u @ up[i].abs().T +
                  2 * f * tiny * (a_g @ gate[i].abs().T + a_u @ up[i].abs().T))
            xa, da = x[r].abs(), d_o[r].abs()
            check("d_gate", got["d_gate"][i], d_wg, xa.T @ e_g + n * tiny * (xa.T @ a_g))
            check("d_up", got["d_up"][i], d_wu, xa.T @ e_u + n * tiny * (xa.T @ a_u))
            check("d_down", got["d_down"][i], d_wd, e_h.T @ da + n * tiny * (a_h.T @ da))
        assert torch.isnan(o[rows:].float()).all()  # rows behind the last segment are left as they were
        alone = plan.backward(d_o.to(BF16), weight_grads=False)
        assert set(alone) == {"d_x"} and torch.equal(alone["d_x"][:rows], got["d_x"][:rows])


def test_train_step_again_captured_and_shared_scratch(ms, cuda_device):
    """The same bits again, from a captured pair of passes and with another object using the same
    scratch between forward and backward: what is kept is the checkpoint alone."""
    dev = cuda_device
    segs, rows = table([70, 0, 64, 9], dev, 64)
    gen = generator(dev, 1)
    w = [torch.empty(4, a, b, device=dev).normal_(0, .05, generator=gen).to(BF16) for a, b in ((128, 160), (128, 160), (160, 128))]
    xs, ds = ([torch.empty(rows, 128, device=dev).normal_(generator=gen).to(BF16) for _ in range(2)] for _ in range(2))
    a = ms.Mx8TrainFfn(*w, rows=rows)
    b = ms.Mx8TrainFfn(*w, rows=rows, scratch=a.scratch)
    want = []
    for x, d in zip(xs, ds):
        o = a.forward(x, segs)
        want.append((o, a.backward(d)))
    oa, ob = a.forward(xs[0], segs), b.forward(xs[1], segs)
    gb, ga = b.backward(ds[1]), a.backward(ds[0])
    for (o, g), (o2, g2) in zip(want, ((oa, ga), (ob, gb))):
        assert torch.equal(o, o2) and all(torch.equal(g[k], g2[k]) for k in g)
    x, d = xs[0].clone(), ds[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = a.forward(x, segs)
        g = a.backward(d)
    for i in (1, 0, 1):
        x.copy_(xs[i])
        d.copy_(ds[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want[i][0]) and all(torch.equal(g[k], want[i][1][k]) for k in g)
    with pytest.raises(RuntimeError):
        ms.Mx8TrainFfn(*w, rows=rows).backward(d)


def test_train_step_without_rows(ms, cuda_device):
    w = [torch.ones(2, a, b, dtype=BF16, device=cuda_device) for a, b in ((64, 32), (64, 32), (32, 64))]
    segs, rows = table([0, 0], cuda_device)
    plan = ms.Mx8TrainFfn(*w, rows=0)
    x = torch.empty(0, 64, dtype=BF16, device=cuda_device)
    plan.forward(x, segs)
    g = plan.backward(x)
    assert all((g[k] == 0).all() for k in ("d_gate", "d_up", "d_down"))


def test_train_step_not_finite(ms, cuda_device):
    """A NaN in one row of x: that row's outputs and, as sums over rows, the weights' gradients are NaN;
    the other rows' outputs are untouched."""
    dev = cuda_device
    gen = generator(dev, 2)
    w = [torch.empty(1, a, b, device=dev).normal_(0, .05, generator=gen).to(BF16) for a, b in ((64, 96), (64, 96), (96, 64))]
    x, d = (torch.empty(64, 64, device=dev).normal_(generator=gen).to(BF16) for _ in range(2))
    segs, _ = table([64], dev, 64)
    plan = ms.Mx8TrainFfn(*w, rows=64)
    o, g = plan.forward(x, segs), plan.backward(d)
    y = x.clone()
    y[5, 3] = float("nan")
    o2, g2 = plan.forward(y, segs), plan.backward(d)
    keep = torch.arange(64, device=dev) != 5
    assert torch.equal(o[keep], o2[keep]) and torch.equal(g["d_x"][keep], g2["d_x"][keep])
    assert torch.isnan(o2[5]).all() and torch.isnan(g2["d_x"][5]).all() and torch.isnan(g2["d_gate"]).any()


def train_weights(gen, dev, d, f, e, shared, shift):
    w = {"router_w": torch.empty(d, e, device=dev).normal_(0, 0.1, generator=gen)}
    for n, k, shape in (("w_gate", e, (d, f)), ("w_up", e, (d, f)), ("w_down", e, (f, d)), ("shared_gate", shared, (d, f)),
                        ("shared_up", shared, (d, f)), ("shared_down", shared, (f, d))):
        if k:
            w[n] = whole_values(gen, (k, *shape), 4, dev, shift).to(BF16)
    return w


@pytest.mark.parametrize("t,d,f,e,k,shared", [(1, 32, 64, 2, 1, 0), (70, 96, 160, 5, 2, 0), (130, 256, 512, 8, 2, 2),
                                              (515, 160, 96, 16, 4, 1), (1000, 512, 704, 8, 2, 0)])
def test_training_step_of_the_layer(ms, axm, cuda_device, t, d, f, e, k, shared):
    """AXM_FLAG_SAVE_8BIT against the same step without it.  The forward pass is the same bit for bit.
    Of the backward pass the weights' gradients are compared with the formula at the kept values
    (whole numbers, so that g, u and dH are exact); the router's gradient with what the error of the
    kept expert rows, half a step of e4m3, can make of it."""
    dev = cuda_device
    gen = generator(dev, t + d)
    w = train_weights(gen, dev, d, f, e, shared, 2.0 ** -((d.bit_length() + 4) // 2))
    x = whole_values(gen, (t, d), 4, dev, 0.5).to(BF16)
    d_out = whole_values(gen, (t, d), 4, dev, 0.25).float()
    plain = axm.MoeTrainLayer(w, t, k)
    in8 = axm.MoeTrainLayer(w, t, k, save_8bit=True)
    out, aux, want = plain.step(x, d_out)
    out8, aux8, got = in8.step(x, d_out)
    torch.cuda.synchronize()
    for layer in (plain, in8):
        assert int(layer.workspace[:4].view(torch.int32).item()) == 0
    assert torch.equal(out, out8) and torch.equal(aux, aux8) and torch.equal(plain.histogram, in8.histogram)

    # routing and gates as the layer's router gives them
    lib = axm.load()
    import helpers
    desc = axm.make_desc(t, d, f, e, k, 0, axm.ROUTER_FP32, axm.FLAG_RESIDUAL)
    logits, idx, gate, _ = helpers.run_router(axm, desc, x, w["router_w"])
    X, dO = x.double(), d_out.double()
    tiny = 2.0 ** -23
    slack_o = torch.zeros(t, k, dtype=torch.float64, device=dev)  # on the gates' gradients

    def compare(name, value, ref_value, slack):
        err = (value.double() - ref_value).abs()
        assert (err <= slack + 1e-30).all(), (name, float((err / (slack + 1e-30)).max()))

    def expert(rows, d_o, wg, wu, wd, names, i):
        if rows.numel() == 0:
            assert all((got[n][i] == 0).all() for n in names)
            return None
        g, u = X[rows] @ wg, X[rows] @ wu
        o = (g * torch.sigmoid(g) * u) @ wd
        fast = (8 + 1.2 * float(g.abs().max())) * tiny
        g, u = ref.held8(g), ref.held8(u)
        (_, d_wg, d_wu, d_wd), (d_h, s, d_g, d_u, h) = ref.ffn_backward(X[rows], g, u, d_o, wg, wu, wd)
        # d_o = bf16(gate dOut) is not a whole number: dH is a sum in 32 bits
        e_dh = d * tiny * (d_o.abs() @ wd.abs().T)
        slope = s + (g * s * (1 - s)).abs()
        e_g = (d_h * u).abs() * slope * fast + e_dh * u.abs() * slope + 2.0 ** -8 * 1.01 * d_g.abs()
        e_u = (2.0 ** -8 * 1.01 + fast) * d_u.abs() + e_dh * (g * s).abs()
        e_h = (2.0 ** -8 * 1.01 + fast) * h.abs()
        n, xa, da = int(rows.numel()), X[rows].abs(), d_o.abs()
        for nm, v, e1, mag in ((names[0], d_wg, e_g, d_g), (names[1], d_wu, e_u, d_u)):
            compare(nm, got[nm][i], v, xa.T @ e1 + n * tiny * (xa.T @ (mag.abs() + e1)))
        compare(names[2], got[names[2]][i], d_wd, e_h.T @ da + n * tiny * ((h.abs() + e_h).T @ da))
        return o

    for i in range(e):
        tok, slot = (idx == i).nonzero(as_tuple=True)
        d_o = (gate[tok, slot].unsqueeze(1) * d_out[tok]).to(BF16).double()
        o = expert(tok, d_o, *(w[n][i].double() for n in ("w_gate", "w_up", "w_down")), ("d_w_gate", "d_w_up", "d_w_down"), i)
        if tok.numel():
            b = o.unflatten(1, (-1, 32)).abs()
            step = torch.maximum(2.0 ** -4 * b, 2.0 ** -4 * 2.0 ** -6 * b.amax(-1, keepdim=True))  # half a step; subnormals
            step = torch.maximum(step, torch.where(b > 448 / 512 * b.amax(-1, keepdim=True), b / 8, step))  # 448 .. 512 saturate
            slack_o[tok, slot] = (dO[tok].abs() * (1.02 * step.flatten(1) + 2.0 ** -7 * b.flatten(1))).sum(1)
    for i in range(shared):
        expert(torch.arange(t, device=dev), d_out.to(BF16).double(),
               *(w[n][i].double() for n in ("shared_gate", "shared_up", "shared_down")),
               ("d_shared_gate", "d_shared_up", "d_shared_down"), i)

    # d gate / d logits, slot by slot, magnitudes
    z = logits.double().requires_grad_(True)
    p = torch.softmax(z, 1).gather(1, idx.long())
    gates = p / p.sum(1, keepdim=True)
    reach = torch.zeros(t, e, dtype=torch.float64, device=dev)
    for j in range(k):
        grad, = torch.autograd.grad(gates[:, j].sum(), z, retain_graph=True)
        reach += grad.abs() * slack_o[:, j:j + 1]
    slack = X.abs().T @ reach
    compare("d_router_w", got["d_router_w"], want["d_router_w"].double(), slack + 1e-4 * want["d_router_w"].abs().max().double())

    # d_x: the router's share, and 8 bits against 16 in the experts' (held8 is off by 2^-4 of a value
    # at most, its slope included: see the bound on the weights' gradients above for the exact part)
    far = (got["d_x"] - want["d_x"]).double()
    through = (want["d_x"].double() - dO)
    assert float(far.norm()) <= 0.08 * float(through.norm()) + float((reach @ w["router_w"].double().abs().T).norm())

    # one scratch for two layers, the second running between the first one's passes
    size = axm.train_split_bytes(in8.desc)[1]
    scratch = torch.empty(size, dtype=torch.uint8, device=dev)
    a, b = (axm.MoeTrainLayer(w, t, k, save_8bit=True, scratch=scratch) for _ in range(2))
    assert a.workspace.numel() + size == in8.workspace.numel()
    y = torch.flip(x, (0,)).contiguous()
    a.forward(x)
    b.forward(y)
    b.backward(y, d_out)
    a.backward(x, d_out)
    assert torch.equal(a.out, out8) and torch.equal(a.d_x, got["d_x"]) and torch.equal(a.d_w_down, got["d_w_down"])


def test_rows_of_a_segment_that_starts_before_the_first(ms, axm, cuda_device):
    """Such a segment has no tiles: its rows get codes and no scale bytes, nothing is written behind the
    scale buffer (one tile, 1024 bytes; row 1 of this one would be in its second tile), and reading leaves them as they are."""
    x = torch.randn(2, 64, device=cuda_device).to(BF16)
    segs = torch.tensor([(-127, -127, 129, 0)], dtype=torch.int32, device=cuda_device)
    scales = torch.full((4 * 1024,), 77, dtype=torch.uint8, device=cuda_device)
    codes = torch.empty(2, 32, dtype=torch.uint8, device=cuda_device)
    lib, stream = axm.load(), axm.current_stream()
    axm.check(lib.axm_mx4_quantize_rows(x.data_ptr(), axm.DTYPE_BF16, 64, None, 1, 2, 64, segs.data_ptr(), 1,
                                        codes.data_ptr(), scales.data_ptr(), stream))
    assert (scales == 77).all()
    out = torch.full((2, 64), 3.0, dtype=BF16, device=cuda_device)
    axm.check(lib.axm_mx4_dequantize_rows(codes.data_ptr(), scales.data_ptr(), 2, 64, segs.data_ptr(), 1, out.data_ptr(),
                                          axm.DTYPE_BF16, 64, stream))
    assert (out == 3).all()


@pytest.mark.parametrize("counts", [[50, 3, 0, 17], [200, 1, 2, 5, 0, 9, 3, 4], [130, 140, 150, 160]])
def test_expert_ffn_with_more_rows_than_expected(ms, cuda_device, counts):
    """tokens only guides the choice of kernel: 0 and 1 give what the true number gives, but for sums in
    another order and the single roundings of h that fall the other way (as in the test above)."""
    e, d, f = len(counts), 64, 96
    q = [ms.quantize_weights(torch.randn(e, k, n, device=cuda_device) * 0.2) for k, n in ((d, f), (d, f), (f, d))]
    segs, rows = table(counts, cuda_device)
    x = torch.randn(rows, d, device=cuda_device).to(BF16)
    out = []
    for tokens in (rows, 1, 0):
        plan = ms.Mx4ExpertFfn(*q, rows=rows, tokens=tokens)
        out.append(plan.forward(x, segs, out=torch.full((rows, d), float("nan"), device=cuda_device)))
        assert plan.status() == 0
    for o in out[1:]:
        assert (o - out[0]).norm() <= 0.01 * out[0].norm()


def test_train_step_with_experts_left_out(ms, cuda_device):
    """Weight gradients of experts that the table does not name are zero, with a table of no segments all."""
    w = [torch.randn(3, a, b, device=cuda_device).to(BF16) for a, b in ((64, 32), (64, 32), (32, 64))]
    x = torch.randn(64, 64, device=cuda_device).to(BF16)
    plan = ms.Mx8TrainFfn(*w, rows=64)
    for table_rows, left in (([(0, 0, 64, 1)], [0, 2]), ([], [0, 1, 2])):
        for _ in range(3):  # the allocator hands out used memory
            torch.full((1 << 20,), float("nan"), device=cuda_device)
        segs = torch.tensor(table_rows, dtype=torch.int32, device=cuda_device).reshape(-1, 4)
        plan.forward(x, segs)
        g = plan.backward(x)
        assert all((g[k][left] == 0).all() for k in ("d_gate", "d_up", "d_down"))
        assert all(torch.isfinite(g[k].float()).all() for k in ("d_gate", "d_up", "d_down"))


def test_status_before_the_first_call(ms, cuda_device):
    junk = [torch.full((1 << 22,), 0x5a, dtype=torch.uint8, device=cuda_device) for _ in range(4)]
    del junk
    w = ms.quantize_weights(torch.ones(1, 64, 64, device=cuda_device))
    plan = ms.Mx4Linear(w, 4)
    assert plan.status() == 0
    plan.forward(torch.empty(0, 64, dtype=BF16, device=cuda_device))
    assert plan.status() == 0


def test_calls_with_wrong_indexes_are_refused(ms, cuda_device):
    """On the host, before a launch."""
    x = torch.zeros(4, 64, dtype=BF16, device=cuda_device)
    with pytest.raises(ValueError):
        ms.quantize_rows(x, row_src=torch.zeros(4, dtype=torch.int64, device=cuda_device))
    with pytest.raises(ValueError):
        ms.quantize_rows(x, row_src=torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError):
        ms.quantize_rows(x, segments=torch.zeros(1, 4, dtype=torch.int64, device=cuda_device))
    w = ms.quantize_weights(torch.ones(1, 64, 64, device=cuda_device))
    with pytest.raises(ValueError):
        ms.Mx4Linear(w, 4).forward(x, out=torch.zeros(64, 4, dtype=BF16, device=cuda_device).t())
    with pytest.raises(ValueError):
        ms.quantize_rows(x, segments=torch.zeros(0, 4, dtype=torch.int32, device=cuda_device))


def room(bytes_needed):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < bytes_needed:
        pytest.skip(f"{bytes_needed >> 30} GB of free memory are needed")


@pytest.fixture
def give_back():
    yield
    torch.cuda.empty_cache()


def test_rows_past_32_bits(ms, cuda_device, give_back):
    """More than 2^32 values: the last rows are what they are alone."""
    room(45 << 30)
    rows, k = (1 << 20) + 4099, 4096
    x = torch.empty(rows, k, dtype=BF16, device=cuda_device).normal_(generator=generator(cuda_device, 1))
    tail = x[-700:].contiguous()
    back = ms.dequantize_rows(ms.quantize_rows(x))
    assert torch.equal(back[-700:], ms.dequantize_rows(ms.quantize_rows(tail)))
    del back
    codes, scales = ms.quantize_rows8(x)
    alone = ms.quantize_rows8(tail)
    assert torch.equal(codes[-700:], alone[0]) and torch.equal(scales[-700:], alone[1])
    assert torch.equal(ms.dequantize_rows8(codes, scales)[-700:], ms.dequantize_rows8(*alone))


def test_weights_past_32_bits(ms, cuda_device, give_back):
    room(30 << 30)
    w = torch.empty(17, 16384, 16384, dtype=BF16, device=cuda_device).normal_(generator=generator(cuda_device, 2))
    back, alone = ms.dequantize_weights(ms.quantize_weights(w)), ms.dequantize_weights(ms.quantize_weights(w[16:].contiguous()))
    assert torch.equal(back[16], alone[0])


def test_linear_past_32_bits(ms, cuda_device, give_back):
    """An output of more than 2^32 values; one stage of the reduction, so rows alone give the same bits."""
    room(25 << 30)
    rows, k, n = 300007, 64, 14400
    w = ms.quantize_weights(torch.randn(1, k, n, device=cuda_device))
    x = torch.empty(rows, k, dtype=BF16, device=cuda_device).normal_(generator=generator(cuda_device, 3))
    plan = ms.Mx4Linear(w, rows)
    out = plan.forward(x)
    assert plan.status() == 0
    assert torch.equal(out[-1031:], plan.forward(x[-1031:].contiguous()))


def test_train_step_past_32_bits(ms, cuda_device, give_back):
    """Checkpoints of more than 2^32 codes: the last expert's rows and gradients are what they are alone."""
    room(75 << 30)
    d, f, first, last = 64, 4096, 1 << 20, 4096
    g = generator(cuda_device, 4)
    w = [torch.empty(2, a, b, device=cuda_device).normal_(0, 0.1, generator=g).to(BF16) for a, b in ((d, f), (d, f), (f, d))]
    x, d_o = (torch.empty(first + last, d, dtype=BF16, device=cuda_device).normal_(generator=g) for _ in range(2))

    def run(w, x, d_o, counts):
        segs, rows = table(counts, cuda_device)
        plan = ms.Mx8TrainFfn(*w, rows=rows)
        o, grads = plan.forward(x, segs), plan.backward(d_o)
        assert plan.status() == 0
        return o, grads

    o, grads = run(w, x, d_o, [first, last])
    o = o[-last:].clone()
    grads = {"d_x": grads["d_x"][-last:].clone(), **{n: grads[n][1].clone() for n in ("d_gate", "d_up", "d_down")}}
    alone, want = run([t[1:].contiguous() for t in w], x[-last:].contiguous(), d_o[-last:].contiguous(), [last])
    assert torch.equal(o, alone) and torch.equal(grads["d_x"], want["d_x"])
    assert all(torch.equal(grads[n], want[n][0]) for n in ("d_gate", "d_up", "d_down"))


def test_two_streams_at_once(ms, cuda_device):
    """Calls with workspaces of their own run side by side without touching one another's results."""
    w = ms.quantize_weights(torch.randn(1, 512, 1024, device=cuda_device))
    xs = [torch.randn(t, 512, device=cuda_device).to(BF16) for t in (1, 300)]
    plans = [ms.Mx4Linear(w, 300) for _ in xs]
    want = [p.forward(x) for p, x in zip(plans, xs)]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(50):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(plans[i].forward(xs[i]))
    torch.cuda.synchronize()
    for i, p in enumerate(plans):
        assert p.status() == 0 and all(torch.equal(g, want[i]) for g in got[i])
