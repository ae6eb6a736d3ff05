"""Microscaled operands: the reference's own rules, sizes, and refusals.  Every refusal comes
before anything is enqueued, so none of this needs a GPU."""
import ctypes
import importlib

import pytest
import torch

import microscale_ref as ref

FAKE = ctypes.c_void_p(1 << 20)  # never dereferenced: the calls below are refused first
ODD = ctypes.c_void_p((1 << 20) + 8)


@pytest.fixture(scope="module")
def lib(axm):
    return axm.load()


def two(call, *args):
    a, b = ctypes.c_size_t(0), ctypes.c_size_t(0)
    assert call(*args, ctypes.byref(a), ctypes.byref(b)) == 0
    return a.value, b.value


def test_reference_blocks():
    x = torch.tensor([[0.25, .75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0] * 4])  # ties, largest magnitude 5 -> scale 1
    assert int(ref.scale_bytes(x, 2)) == 127
    assert ref.held4(x).reshape(-1, 8)[0].tolist() == [0, 1, 1, 2, 2, 4, 4, 4]
    assert ref.held4(-x).reshape(-1, 8)[0].tolist() == [0, -1, -1, -2, -2, -4, -4, -4]
    y = torch.full((1, 32), 7.5)  # 4 <= 7.5 < 8: scale 1, beyond the largest code
    assert (ref.held4(y) == 6).all()
    z = torch.zeros(1, 32)
    assert int(ref.scale_bytes(z, 2)) == 0 and (ref.held4(z) == 0).all()
    z[0, 3] = float("nan")
    assert int(ref.scale_bytes(z, 2)) == 255 and torch.isnan(ref.held4(z)).all() and torch.isnan(ref.held8(z)).all()
    assert (ref.held8(torch.full((1, 32), 511.0)) == 448).all()


def test_reference_8_bits_agrees_with_the_type():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(64, 256, generator=g) * torch.exp2(torch.randint(-30, 30, (64, 1), generator=g).float())
    s = ref.scale_bytes(x, 8)
    scale = torch.exp2(s.double() - 127).repeat_interleave(32, -1)
    v = (x.double() / scale).clamp(-448, 448).float().to(torch.float8_e4m3fn).double() * scale
    assert torch.equal(v, ref.held8(x))


def test_sizes(lib):
    assert two(lib.axm_mx4_rows_bytes, 1, 0, 32) == (16, 2 * 512)
    assert two(lib.axm_mx4_rows_bytes, 300, 5, 544) == (300 * 272, (300 // 128 + 5) * 6 * 512)
    assert two(lib.axm_mx4_weights_bytes, 3, 256, 136) == (3 * 136 * 128, 3 * 2 * 2 * 512)
    assert two(lib.axm_mx4_rows_bytes, 0, 0, 32)[0] == 0


@pytest.mark.parametrize("args", [(-1, 0, 32), (4, 0, 0), (4, 0, 48), (4, -1, 32)])
def test_row_sizes_refused(lib, args):
    a, b = ctypes.c_size_t(0), ctypes.c_size_t(0)
    assert lib.axm_mx4_rows_bytes(*args, ctypes.byref(a), ctypes.byref(b)) == -1


@pytest.mark.parametrize("args", [(0, 32, 8), (1, 33, 8), (1, 32, 12), (1, 0, 8), (70000, 32, 8), (1, 32, 0)])
def test_weight_sizes_refused(lib, args):
    a, b = ctypes.c_size_t(0), ctypes.c_size_t(0)
    assert lib.axm_mx4_weights_bytes(*args, ctypes.byref(a), ctypes.byref(b)) == -1


def test_row_calls_refuse(lib, axm):
    def q(x=FAKE, dt=0, ld=64, src=None, div=1, rows=4, k=64, seg=None, nseg=0, c=FAKE, s=FAKE):
        return lib.axm_mx4_quantize_rows(x, dt, ld, src, div, rows, k, seg, nseg, c, s, None)

    bad = [dict(x=None), dict(c=None), dict(s=None), dict(dt=2), dict(ld=60), dict(ld=68), dict(ld=32), dict(k=48),
           dict(rows=-1), dict(src=FAKE, div=0), dict(seg=FAKE, nseg=0), dict(nseg=-1), dict(x=ODD), dict(c=ODD),
           dict(s=ODD), dict(dt=1, ld=66)]
    for kw in bad:
        assert q(**kw) == axm.AXM_ERR_ARGUMENT, kw
    assert q(rows=0) == axm.AXM_OK

    def d(c=FAKE, s=FAKE, rows=4, k=64, seg=None, nseg=0, out=FAKE, dt=0, ld=64):
        return lib.axm_mx4_dequantize_rows(c, s, rows, k, seg, nseg, out, dt, ld, None)

    for kw in [dict(c=None), dict(s=None), dict(out=None), dict(dt=5), dict(ld=63), dict(out=ODD), dict(k=40),
               dict(seg=FAKE, nseg=0), dict(c=ODD)]:
        assert d(**kw) == axm.AXM_ERR_ARGUMENT, kw
    assert d(rows=0) == axm.AXM_OK
    assert lib.axm_mx8_quantize_rows(FAKE, 0, 64, 4, 48, FAKE, FAKE, None) == axm.AXM_ERR_ARGUMENT
    assert lib.axm_mx8_quantize_rows(FAKE, 0, 64, 4, 64, ODD, FAKE, None) == axm.AXM_ERR_ARGUMENT
    assert lib.axm_mx8_dequantize_rows(FAKE, None, 4, 64, FAKE, 0, 64, None) == axm.AXM_ERR_ARGUMENT
    assert lib.axm_mx8_dequantize_rows(FAKE, FAKE, 0, 64, FAKE, 0, 64, None) == axm.AXM_OK


def test_weight_calls_refuse(lib, axm):
    for args in [(None, 0, 1, 32, 8, FAKE, FAKE), (FAKE, 0, 1, 32, 8, None, FAKE), (FAKE, 3, 1, 32, 8, FAKE, FAKE),
                 (FAKE, 0, 1, 40, 8, FAKE, FAKE), (FAKE, 0, 1, 32, 9, FAKE, FAKE), (ODD, 0, 1, 32, 8, FAKE, FAKE)]:
        assert lib.axm_mx4_quantize_weights(*args, None) == axm.AXM_ERR_ARGUMENT, args
    for args in [(None, FAKE, 1, 32, 8, FAKE, 0), (FAKE, FAKE, 1, 32, 8, ODD, 0), (FAKE, FAKE, 1, 32, 8, FAKE, 9)]:
        assert lib.axm_mx4_dequantize_weights(*args, None) == axm.AXM_ERR_ARGUMENT, args
    assert lib.axm_mx4_pack_scales(None, 1, 32, 8, FAKE, None) == axm.AXM_ERR_ARGUMENT
    assert lib.axm_mx4_pack_scales(FAKE, 1, 32, 8, ODD, None) == axm.AXM_ERR_ARGUMENT


def test_linear_refuses(lib, axm):
    n = ctypes.c_size_t(0)
    assert lib.axm_mx4_linear_workspace_bytes(5, 64, 24, ctypes.byref(n)) == 0 and n.value > 0
    assert lib.axm_mx4_linear_workspace_bytes(5, 64, 20, ctypes.byref(n)) == axm.AXM_ERR_ARGUMENT

    def call(x=FAKE, dt=0, ld=64, t=5, k=64, nn=24, wc=FAKE, ws=FAKE, out=FAKE, odt=0, work=FAKE, size=1 << 26):
        return lib.axm_mx4_linear(x, dt, ld, t, k, nn, wc, ws, out, odt, work, size, None)

    for kw in [dict(x=None), dict(wc=None), dict(ws=None), dict(out=None), dict(dt=7), dict(odt=7), dict(ld=62),
               dict(t=-1), dict(k=65), dict(nn=12), dict(out=ODD), dict(wc=ODD)]:
        assert call(**kw) == axm.AXM_ERR_ARGUMENT, kw
    for kw in [dict(work=None), dict(work=ODD), dict(size=16)]:
        assert call(**kw) == axm.AXM_ERR_WORKSPACE, kw
    assert call(t=0) == axm.AXM_OK
    if not torch.cuda.is_available():
        assert call() == axm.AXM_ERR_DEVICE


def experts(axm, p=FAKE):
    return axm.Mx4ExpertWeights(*[p] * 6)


def test_expert_ffn_refuses(lib, axm):
    n = ctypes.c_size_t(0)
    for d, rows, segs in [(axm.make_desc(4, 40, 64, 2, 1), 4, 2), (axm.make_desc(4, 64, 40, 2, 1), 4, 2),
                          (axm.make_desc(-1, 64, 64, 2, 1), 4, 2), (axm.make_desc(4, 64, 64, 2, 1), -1, 2),
                          (axm.make_desc(4, 64, 64, 2, 1), 4, 513), (axm.make_desc(4, 64, 64, 0, 1), 4, 2)]:
        assert lib.axm_mx4_expert_ffn_workspace_bytes(ctypes.byref(d), rows, segs, ctypes.byref(n)) == axm.AXM_ERR_ARGUMENT
    d = axm.make_desc(4, 64, 64, 2, 1)
    w = experts(axm)

    def call(x=FAKE, rows=4, seg=FAKE, nseg=2, e=w, o=FAKE, dt=0, work=FAKE, size=1 << 26):
        return lib.axm_mx4_expert_ffn(ctypes.byref(d), x, rows, seg, nseg, None if e is None else ctypes.byref(e), o, dt,
                                      work, size, None)

    half = experts(axm)
    half.up_scales = None
    for kw in [dict(x=None), dict(seg=None), dict(o=None), dict(e=None), dict(e=half), dict(e=experts(axm, ODD)),
               dict(dt=4), dict(x=ODD), dict(o=ODD), dict(rows=-2), dict(nseg=-1)]:
        assert call(**kw) == axm.AXM_ERR_ARGUMENT, kw
    assert call(size=8) == axm.AXM_ERR_WORKSPACE and call(work=None) == axm.AXM_ERR_WORKSPACE
    assert call(rows=0) == axm.AXM_OK and call(nseg=0) == axm.AXM_OK


def test_layer_refuses(lib, axm):
    n = ctypes.c_size_t(0)
    for d in [axm.make_desc(4, 40, 64, 2, 1), axm.make_desc(4, 64, 64, 2, 3), axm.make_desc(4, 64, 64, 300, 2),
              axm.make_desc(4, 64, 64, 2, 1, 9)]:
        assert lib.axm_moe_mx4_workspace_bytes(ctypes.byref(d), ctypes.byref(n)) == axm.AXM_ERR_ARGUMENT
    d = axm.make_desc(4, 64, 64, 4, 2, 1)
    assert lib.axm_moe_mx4_workspace_bytes(ctypes.byref(d), ctypes.byref(n)) == 0
    w = experts(axm)
    t = axm.MoeTensors()
    t.x = t.router_w = t.out = FAKE.value

    def call(tensors=t, e=w, s=w, work=FAKE, size=n.value):
        return lib.axm_moe_forward_mx4(ctypes.byref(d), ctypes.byref(tensors), None if e is None else ctypes.byref(e),
                                       None if s is None else ctypes.byref(s), work, size, None)

    bare = axm.MoeTensors()
    assert call(tensors=bare) == axm.AXM_ERR_ARGUMENT
    assert call(e=None) == axm.AXM_ERR_ARGUMENT
    assert call(s=None) == axm.AXM_ERR_ARGUMENT  # num_shared 1
    assert call(size=n.value - 1) == axm.AXM_ERR_WORKSPACE
    if not torch.cuda.is_available():
        assert call() == axm.AXM_ERR_DEVICE


def test_python_refuses():
    ms = importlib.import_module("project_axiom_ai_llm_b200.microscale")
    with pytest.raises(ValueError):
        ms.quantize_rows(torch.zeros(4, 64))  # host memory
    with pytest.raises(ValueError):
        ms.quantize_weights(torch.zeros(1, 64, 8))
    with pytest.raises(ValueError):
        ms.Mx4Weights.from_checkpoint(torch.zeros(1, 8, 16, dtype=torch.uint8), torch.zeros(1, 8, 1, dtype=torch.uint8))


def test_train8_refuses(lib, axm):
    a, b = ctypes.c_size_t(0), ctypes.c_size_t(0)
    assert two(lib.axm_mx8_checkpoint_bytes, 128, 96) == (128 * 96, 128 * 3)
    for args in [(-1, 32), (4, 0), (4, 40)]:
        assert lib.axm_mx8_checkpoint_bytes(*args, ctypes.byref(a), ctypes.byref(b)) == axm.AXM_ERR_ARGUMENT
    keep = axm.Mx8Checkpoint(*[FAKE] * 4)

    def forward(d=(64, 64), e=2, x=FAKE, rows=64, seg=FAKE, nseg=2, w=FAKE, k=keep, h=FAKE, o=FAKE, dt=0):
        desc = axm.make_desc(64, *d, e, 1)
        return lib.axm_mx8_expert_ffn_train(ctypes.byref(desc), x, rows, seg, nseg, w, FAKE, FAKE,
                                            None if k is None else ctypes.byref(k), h, o, dt, None, None)

    half, odd = axm.Mx8Checkpoint(*[FAKE] * 4), axm.Mx8Checkpoint(*[FAKE] * 4)
    half.up_scales, odd.gate_codes = None, ODD
    common = [dict(d=(60, 64)), dict(d=(64, 40)), dict(e=0), dict(x=None), dict(x=ODD), dict(rows=-1), dict(seg=None),
              dict(nseg=513), dict(nseg=-1), dict(w=None), dict(k=None), dict(k=half), dict(k=odd), dict(h=None), dict(dt=2)]
    for kw in common + [dict(o=None), dict(o=ODD)]:
        assert forward(**kw) == axm.AXM_ERR_ARGUMENT, kw
    assert forward(rows=0) == axm.AXM_OK and forward(nseg=0) == axm.AXM_OK

    def backward(d=(64, 64), e=2, x=FAKE, rows=64, seg=FAKE, nseg=2, w=FAKE, k=keep, h=FAKE, dt=0, d_o=FAKE, d_x=FAKE,
                 dw=(FAKE, FAKE, FAKE)):
        desc = axm.make_desc(64, *d, e, 1)
        return lib.axm_mx8_expert_ffn_backward(ctypes.byref(desc), x, rows, seg, nseg, None if k is None else ctypes.byref(k),
                                               d_o, w, FAKE, FAKE, h, FAKE, FAKE, d_x, *dw, dt, None, None)

    for kw in common + [dict(d_o=None), dict(d_x=None), dict(d_x=ODD), dict(dw=(FAKE, None, FAKE)), dict(dw=(FAKE, ODD, FAKE))]:
        assert backward(**kw) == axm.AXM_ERR_ARGUMENT, kw
    assert backward(nseg=0) == axm.AXM_OK


def test_backward_reference_against_differences():
    """The reference's gradients are the derivatives of sum(d_o * ((silu(g) u) Wd)) where g and u are
    held exactly (64-bit central differences: truncation about 1e-4 ** 2, rounding about 1e-16 / 1e-4)."""
    gen = torch.Generator().manual_seed(5)
    x, d_o = (torch.randn(6, 8, generator=gen, dtype=torch.float64) for _ in range(2))
    wg, wu = (torch.randn(8, 4, generator=gen, dtype=torch.float64) for _ in range(2))
    wd = torch.randn(4, 8, generator=gen, dtype=torch.float64)

    def loss(x, wg, wu, wd):
        g, u = x @ wg, x @ wu
        return float((d_o * ((g * torch.sigmoid(g) * u) @ wd)).sum())

    grads, _ = ref.ffn_backward(x, x @ wg, x @ wu, d_o, wg, wu, wd)
    args = [x, wg, wu, wd]
    for i, grad in enumerate(grads):
        for at in range(args[i].numel()):
            both = []
            for h in (1e-4, -1e-4):
                moved = [a.clone() for a in args]
                moved[i].view(-1)[at] += h
                both.append(loss(*moved))
            assert abs((both[0] - both[1]) / 2e-4 - float(grad.reshape(-1)[at])) < 1e-5


def test_training_step_workspaces(lib, axm):
    """The two pieces add up to the one workspace; 8 bits keep less than a third of what bf16 keeps of a
    large layer; sizes and flags that do not fit are refused."""
    for flags in (0, axm.FLAG_SAVE_8BIT):
        for shared in (0, 2):
            d = axm.make_desc(300, 256, 512, 8, 2, shared, flags=axm.FLAG_RESIDUAL | flags)
            n = ctypes.c_size_t(0)
            assert lib.axm_moe_train_workspace_bytes(ctypes.byref(d), ctypes.byref(n)) == 0
            assert sum(axm.train_split_bytes(d)) == n.value
    plain = axm.train_split_bytes(axm.make_desc(8192, 2048, 4096, 16, 2))
    in8 = axm.train_split_bytes(axm.make_desc(8192, 2048, 4096, 16, 2, flags=axm.FLAG_RESIDUAL | axm.FLAG_SAVE_8BIT))
    assert 3 * in8[0] < plain[0]
    t = axm.MoeTrain()
    for f in ("x", "router_w", "w_gate", "w_up", "w_down", "out", "d_out", "d_x"):
        setattr(t, f, FAKE.value)
    for d in (axm.make_desc(4, 40, 64, 4, 2, flags=axm.FLAG_SAVE_8BIT), axm.make_desc(4, 64, 40, 4, 2, flags=axm.FLAG_SAVE_8BIT)):
        a, b = ctypes.c_size_t(0), ctypes.c_size_t(0)
        assert lib.axm_moe_train_split_bytes(ctypes.byref(d), ctypes.byref(a), ctypes.byref(b)) == axm.AXM_ERR_ARGUMENT
        assert lib.axm_moe_forward_train(ctypes.byref(d), ctypes.byref(t), FAKE, 1 << 30, None) == axm.AXM_ERR_ARGUMENT
        assert lib.axm_moe_backward(ctypes.byref(d), ctypes.byref(t), FAKE, 1 << 30, None) == axm.AXM_ERR_ARGUMENT
    d = axm.make_desc(4, 64, 64, 4, 2, flags=axm.FLAG_SAVE_8BIT)
    kept, scratch = axm.train_split_bytes(d)
    for call in (lib.axm_moe_forward_train_split, lib.axm_moe_backward_split):
        for k, kb, sc, sb in ((FAKE, kept - 1, FAKE, scratch), (FAKE, kept, FAKE, scratch - 1), (None, kept, FAKE, scratch),
                              (FAKE, kept, None, scratch), (ODD, kept, FAKE, scratch), (FAKE, kept, ODD, scratch)):
            assert call(ctypes.byref(d), ctypes.byref(t), k, kb, sc, sb, None) == axm.AXM_ERR_WORKSPACE
        if not torch.cuda.is_available():
            assert call(ctypes.byref(d), ctypes.byref(t), FAKE, kept, FAKE, scratch, None) == axm.AXM_ERR_DEVICE


def test_index_and_out_checks():
    """What the calls of the Python layer refuse before they hand an address to the library."""
    ms = importlib.import_module("project_axiom_ai_llm_b200.microscale")
    dev = torch.device("cpu")
    ms._check_index(None, 4, dev, "segments")
    ms._check_index(torch.zeros(3, 4, dtype=torch.int32), 4, dev, "segments")
    ms._check_index(torch.zeros(3, dtype=torch.int32), None, dev, "row_src")
    for t, width in [(torch.zeros(3, 4), 4), (torch.zeros(3, 4, dtype=torch.int64), 4), (torch.zeros(3, 5, dtype=torch.int32), 4),
                     (torch.zeros(12, dtype=torch.int32), 4), (torch.zeros(4, 3, dtype=torch.int32).t(), 4),
                     (torch.zeros(3, dtype=torch.int64), None), (torch.zeros(6, dtype=torch.int32)[::2], None),
                     (torch.zeros(3, 1, dtype=torch.int32), None), (torch.zeros(3, 4, dtype=torch.int32, device="meta"), 4)]:
        with pytest.raises(ValueError):
            ms._check_index(t, width, dev, "table")
    bf16 = torch.bfloat16
    ms._check_out(torch.zeros(3, 8, dtype=bf16), (3, 8), dev, bf16)
    for t in [torch.zeros(3, 8), torch.zeros(2, 8, dtype=bf16), torch.zeros(3, 16, dtype=bf16)[:, ::2],
              torch.zeros(3, 8, dtype=bf16, device="meta")]:
        with pytest.raises(ValueError):
            ms._check_out(t, (3, 8), dev, bf16)


def test_weights_of_other_sizes_or_devices():
    ms = importlib.import_module("project_axiom_ai_llm_b200.microscale")

    def weights(e, k, n, device="cpu"):
        return ms.Mx4Weights(torch.empty(e, n, k // 2, dtype=torch.uint8, device=device),
                             torch.empty(16, dtype=torch.uint8, device=device), e, k, n)

    a, d = weights(4, 64, 96), weights(4, 96, 64)
    with pytest.raises(ValueError):
        ms._expert_table(a, a, a)
    with pytest.raises(ValueError):
        ms._expert_table(a, a, weights(4, 96, 64, "meta"))
    base = dict(router_w=torch.zeros(64, 4), gate=a, up=a, down=d)
    small, small_d = weights(1, 64, 32), weights(1, 32, 64)
    for change in [dict(shared_gate=small, shared_up=small, shared_down=small_d), dict(router_w=torch.zeros(4, 64).t()),
                   dict(router_w=torch.zeros(64, 4, dtype=torch.float64)), dict(router_w=torch.zeros(64, 4, device="meta")),
                   dict(router_bias=torch.zeros(3)), dict(router_bias=torch.zeros(4, dtype=torch.bfloat16)),
                   dict(router_w=torch.zeros(64, 5))]:
        with pytest.raises(ValueError):
            ms.Mx4MoeLayer({**base, **change}, tokens=4, top_k=2)


def test_training_scratch_refused(axm):
    w = dict(router_w=torch.zeros(64, 4), w_gate=torch.zeros(4, 64, 96, dtype=torch.bfloat16))
    need = axm.train_split_bytes(axm.make_desc(8, 64, 96, 4, 2, flags=axm.FLAG_RESIDUAL | axm.FLAG_SAVE_8BIT))[1]
    for scratch in [torch.empty(need - 1, dtype=torch.uint8), torch.empty(need, dtype=torch.float32),
                    torch.empty(2 * need, dtype=torch.uint8)[::2], torch.empty(need, dtype=torch.uint8, device="meta")]:
        with pytest.raises(ValueError):
            axm.MoeTrainLayer(w, 8, 2, device="cpu", save_8bit=True, scratch=scratch)


def test_sharded_training_refuses_8_bits(lib, axm):
    """On the host, with a layout that the same call accepts without the flag."""
    world, e, d, f, t, k = 2, 8, 256, 512, 64, 2
    lo, n, zero = axm.EpLayout(), ctypes.c_size_t(0), ctypes.c_size_t(0)
    cap = t * k * world + 63 * (e // world)
    assert lib.axm_ep_region_bytes(world, e, d, t * k, cap, ctypes.byref(lo), ctypes.byref(n)) == axm.AXM_OK
    lo.rank, lo.row_align = 0, 64

    def call(flags):
        desc = axm.make_desc(t, d, f, e, k, flags=flags)
        return lib.axm_moe_ep_train_workspace_bytes(ctypes.byref(lo), ctypes.byref(desc), ctypes.byref(n), ctypes.byref(zero))

    assert call(axm.FLAG_RESIDUAL) == axm.AXM_OK
    assert call(axm.FLAG_RESIDUAL | axm.FLAG_SAVE_8BIT) == axm.AXM_ERR_ARGUMENT
    assert b"AXM_FLAG_SAVE_8BIT" in lib.axm_last_error()


def test_train8_empty_table_without_an_address(lib, axm):
    """Zero segments: nothing to do, with rows and with a table that has no address (an empty tensor's)."""
    desc, keep = axm.make_desc(64, 64, 64, 2, 1), axm.Mx8Checkpoint(*[FAKE] * 4)
    assert lib.axm_mx8_expert_ffn_train(ctypes.byref(desc), FAKE, 64, None, 0, FAKE, FAKE, FAKE, ctypes.byref(keep), FAKE, FAKE,
                                        0, None, None) == axm.AXM_OK
    assert lib.axm_mx8_expert_ffn_backward(ctypes.byref(desc), FAKE, 64, None, 0, ctypes.byref(keep), FAKE, FAKE, FAKE, FAKE,
                                           FAKE, FAKE, FAKE, FAKE, None, None, None, 0, None, None) == axm.AXM_OK
