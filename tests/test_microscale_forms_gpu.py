"""Forms of the 4-bit kernels that a call reaches by few sizes or options only, against 64-bit references."""
import importlib

import pytest
import torch

from test_microscale_gpu import exact_expert_weights, ffn_reference, held_operand, table

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ms(axm):
    return importlib.import_module("project_axiom_ai_llm_b200.microscale")


# one segment of 65 to 128 rows (128-row tiles, one accumulator): few column tiles, whose reduction is cut, and more
# column tiles than SMs, so that a CTA takes the accumulator up again; segments of 17 to 32 rows (32-row tiles)
FEW = [([97], 320, 224), ([128], 1024, 96), ([65], 64, 19232), ([20, 24, 0, 22, 23], 288, 416), ([32, 17, 30, 25], 64, 2080),
       ([90, 3, 2, 1], 96, 160), ([70, 0, 2, 30, 11], 160, 96)]


@pytest.mark.parametrize("counts,d,f", FEW)
def test_few_rows_instances(ms, cuda_device, counts, d, f):
    segs, rows = table(counts, cuda_device)
    _, _, x = held_operand(rows + 3, d, cuda_device, rows, 1)
    x = x.to(BF16)
    shift = (d.bit_length() + 7) // 2
    (qg, gate), (qu, up), (qd, down) = (exact_expert_weights(ms, len(counts), k, n, cuda_device, i, shift)
                                        for i, (k, n) in enumerate(((d, f), (d, f), (f, d))))
    plan = ms.Mx4ExpertFfn(qg, qu, qd, rows=rows + 3, tokens=max(counts))
    o, slack = ffn_reference(x, segs, gate, up, down)
    first = None
    for _ in range(3):
        plan.workspace[256:].fill_(255)
        got = plan.forward(x, segs, out=torch.full((rows + 3, d), float("nan"), device=cuda_device))
        assert plan.status() == 0
        assert ((got[:rows].double() - o[:rows]).abs() <= slack[:rows]).all()
        assert torch.isnan(got[rows:]).all()
        assert first is None or torch.equal(first[:rows], got[:rows])
        first = got
    # the bound says something: f products whose errors are counted as if they all pointed one way
    assert float(slack[:rows].norm()) < (0.02 if f < 4096 else 0.5) * float(o[:rows].norm())
