"""Segment tables at the edge of what the microscaled calls document."""
import importlib

import pytest
import torch

import microscale_ref as ref
from test_microscale_gpu import awkward, exact_expert_weights, ffn_reference, held_float, held_operand, same, table

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
