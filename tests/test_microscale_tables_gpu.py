"""Segment tables at the edge of what the microscaled calls document."""
import importlib

import pytest
import torch

import microscale_ref as ref
from test_microscale_gpu import awkward, exact_expert_weights, ffn_reference, generator, held_float, held_operand, same, table

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ms(axm):
    return importlib.import_module("project_axiom_ai_llm_b200.microscale")


def entries(rows, dev):
    return torch.tensor([(at, at, n, e) for at, n, e in rows], dtype=torch.int32, device=dev)


# (first row, rows, expert), ordered by the first row; the number of rows in all
EMPTY_ENTRIES = {
    "at a segment's first row": ([(0, 5, 0), (0, 0, 1), (5, 3, 2)], 8),
    "inside a segment": ([(0, 5, 0), (3, 0, 1), (5, 3, 2)], 8),
    "before the first, and at the end": ([(0, 0, 1), (0, 20, 0), (7, 0, 2), (20, 22, 3), (42, 0, 1)], 42),
    "more than 32 inside a segment": ([(0, 20, 0)] + [(7, 0, i % 4) for i in range(70)] + [(20, 9, 3)], 29),
    "32 to a round's end": ([(0, 20, 2)] + [(11, 0, 1)] * 31 + [(20, 9, 3), (29, 5, 0)], 34),
    "one-CTA kernel": ([(0, 130, 0), (0, 0, 1), (77, 0, 3), (130, 120, 2)], 250),
    "pair kernel": ([(0, 300, 0), (0, 0, 1), (100, 0, 2), (300, 400, 3)], 700),
}


@pytest.mark.parametrize("name", EMPTY_ENTRIES)
def test_entries_without_rows(ms, cuda_device, name):
    """They may start anywhere: the rows around them are quantised, multiplied and read back as without
    them.  The workspace begins as scale bytes of 255: a row without its own would be NaN."""
    rows_of, rows = EMPTY_ENTRIES[name]
    segs = entries(rows_of, cuda_device)
    x = awkward(rows, 96, FP32, cuda_device, rows)
    q = ms.quantize_rows(x, segments=segs)
    assert same(ms.dequantize_rows(q, out=torch.full((rows, 96), 7.0, device=cuda_device)), held_float(x, 4, FP32))
    d, f = 96, 160
    _, _, x = held_operand(rows, d, cuda_device, rows, 1)
    x = x.to(BF16)
    shift = (d.bit_length() + 7) // 2
    (qg, gate), (qu, up), (qd, down) = (exact_expert_weights(ms, 4, k, n, cuda_device, i, shift)
                                        for i, (k, n) in enumerate(((d, f), (d, f), (f, d))))
    plan = ms.Mx4ExpertFfn(qg, qu, qd, rows=rows, tokens=rows, segments=len(rows_of))
    o, slack = ffn_reference(x, segs, gate, up, down)
    plan.workspace.fill_(255)
    got = plan.forward(x, segs, out=torch.full((rows, d), float("nan"), device=cuda_device))
    assert plan.status() == 0
    assert ((got.double() - o).abs() <= slack).all()


@pytest.mark.parametrize("counts", [[5, 0, 3], [60, 70], [300, 0, 290]])
@pytest.mark.parametrize("offset", [1, 2, 3])
def test_tables_at_any_address(ms, cuda_device, counts, offset):
    """A table is an array of int32: it may be a slice that starts anywhere in another tensor (few-rows,
    one-CTA and pair kernels; the 8-bit training calls)."""
    segs, rows = table(counts, cuda_device, 64)
    moved = torch.full((segs.numel() + 8,), -7, dtype=torch.int32, device=cuda_device)[offset:offset + segs.numel()].view(-1, 4)
    moved.copy_(segs)
    assert moved.data_ptr() % 16 == 4 * offset and moved.is_contiguous()
    x = torch.randn(rows, 64, device=cuda_device).to(BF16)
    assert torch.equal(ms.dequantize_rows(ms.quantize_rows(x, segments=moved)), ms.dequantize_rows(ms.quantize_rows(x, segments=segs)))
    w = [torch.randn(3, *kn, device=cuda_device).to(BF16) for kn in ((64, 96), (64, 96), (96, 64))]
    plan = ms.Mx4ExpertFfn(*(ms.quantize_weights(t) for t in w), rows=rows, tokens=rows)
    assert torch.equal(plan.forward(x, moved), plan.forward(x, segs)) and plan.status() == 0
    plan = ms.Mx8TrainFfn(*w, rows=rows)
    want = [plan.forward(x, segs), *plan.backward(x).values()]
    got = [plan.forward(x, moved), *plan.backward(x).values()]
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and plan.status() == 0


def test_training_tables_that_do_not_fit(ms, axm, cuda_device):
    """The 8-bit training calls keep a table's entries inside `rows`: rows behind the matrices' end are cut
    off, entries that start outside or name no expert are left out, everything else is as with the table
    that fits.  Every buffer is a slice of one allocation, with 8 KiB around each that nothing may touch."""
    dev, rows, d, f, e = cuda_device, 198, 64, 96, 4
    fits = [(0, 0, 64, 0), (64, 64, 128, 2), (192, 192, 6, 1), (0, 0, 0, 3)]
    padded = [(0, 0, 64, 0), (64, 64, 128, 2), (192, 192, 64, 1), (0, 0, 0, 3)]  # as if x were padded too
    far = [(0, 0, 64, 0), (64, 64, 128, 2), (192, 192, 1 << 30, 1), (1 << 30, 1 << 30, 64, 3)]
    before = [(0, 0, 64, 0), (64, 64, 128, 2), (192, 192, 70, 1), (-64, -64, 128, 3)]
    unknown = fits + [(0, 0, 64, e), (64, 64, 64, 0xffff), (0, 0, 128, -1), (rows, rows, 64, 3), (64, 64, -64, 7)]
    g = generator(dev, 1)
    whole = dict(x=(rows, d, BF16), d_o=(rows, d, BF16), wg=(e * d, f, BF16), wu=(e * d, f, BF16), wd=(e * f, d, BF16),
                 gc=(rows, f, torch.uint8), gs=(rows, f // 32, torch.uint8), uc=(rows, f, torch.uint8), us=(rows, f // 32, torch.uint8),
                 h=(rows, f, BF16), dg=(rows, f, BF16), du=(rows, f, BF16))
    lib, stream, desc = axm.load(), axm.current_stream(), axm.make_desc(rows, d, f, e, 1)
    gap = 8192
    for dtype, code in ((BF16, axm.DTYPE_BF16), (FP32, axm.DTYPE_FP32)):
        shapes = {**whole, "o": (rows, d, dtype), "d_x": (rows, d, dtype), "dwg": (e * d, f, dtype), "dwu": (e * d, f, dtype), "dwd": (e * f, d, dtype)}
        inputs = {n: torch.empty(shapes[n][:2], device=dev).normal_(0, 0.3, generator=g).to(BF16) for n in ("x", "d_o", "wg", "wu", "wd")}
        want = None
        for name, entries_ in (("fits", fits), ("padded", padded), ("far", far), ("before", before), ("unknown", unknown)):
            at, places = gap, {}
            for n, (r, c, t) in shapes.items():
                size = r * c * t.itemsize
                places[n] = (at, size)
                at = (at + size + 255 & -256) + gap
            pool = torch.full((at,), 0x5a, dtype=torch.uint8, device=dev)
            v = {n: pool[a:a + s].view(shapes[n][2]).view(shapes[n][:2]) for n, (a, s) in places.items()}
            for n in inputs:
                v[n].copy_(inputs[n])
            free = torch.ones(at, dtype=torch.bool, device=dev)
            for a, s in places.values():
                free[a:a + s] = False
            segs = torch.tensor(entries_, dtype=torch.int32, device=dev)
            keep = axm.Mx8Checkpoint(*(v[n].data_ptr() for n in ("gc", "gs", "uc", "us")))
            status = torch.zeros(1, dtype=torch.int32, device=dev)
            p = {n: t.data_ptr() for n, t in v.items()}
            axm.check(lib.axm_mx8_expert_ffn_train(desc, p["x"], rows, segs.data_ptr(), len(entries_), p["wg"], p["wu"], p["wd"], keep,
                                                   p["h"], p["o"], code, status.data_ptr(), stream))
            axm.check(lib.axm_mx8_expert_ffn_backward(desc, p["x"], rows, segs.data_ptr(), len(entries_), keep, p["d_o"], p["wg"], p["wu"],
                                                      p["wd"], p["h"], p["dg"], p["du"], p["d_x"], p["dwg"], p["dwu"], p["dwd"], code,
                                                      status.data_ptr(), stream))
            assert int(status.item()) == 0 and (pool[free] == 0x5a).all(), name
            got = {n: pool[a:a + s].clone() for n, (a, s) in places.items()}
            want = got if want is None else want
            assert all(torch.equal(got[n], want[n]) for n in got), (name, [n for n in got if not torch.equal(got[n], want[n])])
            assert torch.isfinite(v["d_x"].float()).all() and (v["dwg"].view(e, d, f)[3] == 0).all()


@pytest.mark.parametrize("rows", [40, 250, 700])  # few-rows, one-CTA and pair kernels
@pytest.mark.parametrize("expert", [1 << 16, (1 << 20) + 1, 1 << 29, -(1 << 31), -65536])
def test_experts_whose_low_bits_look_right(ms, cuda_device, rows, expert):
    """An id is compared as a whole: such an entry's rows are left as they are and no other expert's gradient is
    touched."""
    d, f, n = 64, 96, rows // 2
    w = [torch.randn(2, *kn, device=cuda_device).to(BF16) for kn in ((d, f), (d, f), (f, d))]
    x = torch.randn(rows, d, device=cuda_device).to(BF16)
    good, odd = entries([(0, n, 1), (n, 0, 0)], cuda_device), entries([(0, n, 1), (n, rows - n, expert)], cuda_device)
    plan = ms.Mx4ExpertFfn(*(ms.quantize_weights(t) for t in w), rows=rows, tokens=rows)
    want, got = (plan.forward(x, t, out=torch.full((rows, d), 5.0, dtype=BF16, device=cuda_device)) for t in (good, odd))
    assert plan.status() == 0 and torch.equal(want, got) and (got[n:] == 5).all()
    rows, n = -(-rows // 64) * 64, -(-n // 64) * 64  # the training layout
    x = torch.randn(rows, d, device=cuda_device).to(BF16)
    good = entries([(0, n, 1), (n, 0, 0)], cuda_device)
    odd = entries([(0, n, 1), (n, rows - n, expert), (n, 0, 0)], cuda_device)
    plan = ms.Mx8TrainFfn(*w, rows=rows)
    outs = []
    for t in (good, odd):
        o = plan.forward(x, t, out=torch.full((rows, d), 5.0, dtype=BF16, device=cuda_device))
        g = plan.backward(x)
        outs.append([o, g["d_x"][:n], g["d_gate"], g["d_up"], g["d_down"]])
    assert plan.status() == 0 and all(torch.equal(a, b) for a, b in zip(*outs)) and (outs[1][0][n:] == 5).all()
    assert (outs[1][2][0] == 0).all() and bool((outs[1][2][1] != 0).any())
