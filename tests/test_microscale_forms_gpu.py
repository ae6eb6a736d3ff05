"""Forms of the 4-bit kernels that a call reaches by few sizes or options only, against 64-bit references."""
import importlib

import pytest
import torch

import helpers
from test_microscale_gpu import exact_expert_weights, ffn_reference, generator, held_operand, table

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


@pytest.mark.parametrize("t", [1, 23, 300, 1100])  # few-rows, one-CTA and pair kernels
@pytest.mark.parametrize("residual,accumulate,biased,router,shared", [
    (False, False, False, FP32, 0), (True, True, False, FP32, 1), (True, False, True, FP32, 0), (True, False, False, BF16, 2),
    (False, True, True, BF16, 1)])
def test_layer_options(ms, axm, cuda_device, t, residual, accumulate, biased, router, shared):
    """Without the residual, with the histogram added up, with a router bias, with bf16 router weights: the
    routing is that of the layer's router on the same inputs, the output the chosen experts' sum in 64 bits."""
    d, f, e, k = 160, 96, 12, 3
    g = generator(cuda_device, t)
    _, _, x = held_operand(t, d, cuda_device, t, 1)
    x = x.to(BF16)
    shift = (d.bit_length() + 7) // 2
    q, v = {}, {}
    for i, (name, n, (a, b)) in enumerate([("gate", e, (d, f)), ("up", e, (d, f)), ("down", e, (f, d)), ("shared_gate", shared, (d, f)),
                                           ("shared_up", shared, (d, f)), ("shared_down", shared, (f, d))]):
        if n:
            q[name], v[name] = exact_expert_weights(ms, n, a, b, cuda_device, i, shift)
    q["router_w"] = torch.empty(d, e, device=cuda_device).normal_(0, 0.02, generator=g).to(router)
    q["router_bias"] = torch.empty(e, device=cuda_device).normal_(0, 2, generator=g) if biased else None
    layer = ms.Mx4MoeLayer(q, t, k, residual=residual, hist_accumulate=accumulate)
    layer.histogram.fill_(1000)
    layer.workspace[256:].fill_(255)
    out, hist = layer.forward(x)
    desc = axm.make_desc(t, d, f, e, k, 0, axm.ROUTER_FP32 if router is FP32 else axm.ROUTER_BF16, axm.FLAG_RESIDUAL)
    _, idx, gate, _ = helpers.run_router(axm, desc, x, q["router_w"], q["router_bias"])
    assert torch.equal(layer.topk_idx, idx) and torch.equal(layer.topk_gate, gate)
    counts = torch.bincount(idx.reshape(-1).long(), minlength=e)
    assert torch.equal(hist.long(), counts + (1000 if accumulate else 0))
    again, hist = layer.forward(x)
    assert torch.equal(again, out) and torch.equal(hist.long(), 2 * counts + 1000 if accumulate else counts)
    assert layer.status() == 0

    order = torch.argsort(idx.reshape(-1).long(), stable=True)
    o, slack = (torch.empty(t * k, d, dtype=torch.float64, device=cuda_device) for _ in range(2))
    o[order], slack[order] = ffn_reference(x[order // k].contiguous(), table(counts.tolist(), cuda_device)[0], v["gate"], v["up"], v["down"])
    w = gate.double().unsqueeze(-1)
    y, err, size = ((p.view(t, k, d) * w).sum(1) for p in (o, slack, o.abs()))
    for i in range(shared):
        add, more = ffn_reference(x, table([t], cuda_device)[0], v["shared_gate"][i:], v["shared_up"][i:], v["shared_down"][i:])
        y, err, size = y + add, err + more, size + add.abs()
    # k products and k + shared sums in 32 bits, rounded to bf16, and with the residual added and rounded again
    err = err + (k + shared + 2) * 2.0 ** -23 * (size + err)
    err = err + 2.0 ** -8 * (y.abs() + err)
    want = y
    if residual:
        want = x.double() + y
        err = err + 2.0 ** -8 * (want.abs() + err)
    assert ((out.double() - want).abs() <= err + 1e-30).all()
    assert float(err.norm()) < 0.05 * float(want.norm())
