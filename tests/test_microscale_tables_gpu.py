"""Segment tables at the edge of what the microscaled calls document."""
import importlib

import pytest
import torch

import microscale_ref as ref
from test_microscale_gpu import awkward, exact_expert_weights, ffn_reference, held_float, held_operand, same

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
