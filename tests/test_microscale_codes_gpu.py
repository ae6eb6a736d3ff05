"""Every code under the smallest, middle and largest scale bytes, as another program may have written them; rows
with any stride."""
import importlib

import pytest
import torch

import microscale_ref as ref
from test_microscale_gpu import same

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ms(axm):
    return importlib.import_module("project_axiom_ai_llm_b200.microscale")


def all_8_bit_codes(k, dev):
    """Codes [256][k], scale bytes, and what they stand for in 64 bits."""
    rows = 256
    codes = (torch.arange(rows * k, device=dev) * 37 % 256).to(torch.uint8).view(rows, k)
    scales = torch.tensor([0, 1, 2, 3, 9, 127, 200, 240, 252, 253, 254, 255], dtype=torch.uint8, device=dev)
    scales = scales[torch.arange(rows * (k // 32), device=dev) % 12].view(rows, -1)
    value = codes.view(torch.float8_e4m3fn).double()
    assert torch.isnan(value[codes & 127 == 127]).all() and (value[codes == 126] == 448).all() and len(torch.unique(codes)) == 256
    want = value * torch.exp2(scales.double() - 127).repeat_interleave(32, 1)
    want[scales.repeat_interleave(32, 1) == 255] = float("nan")
    return codes, scales, want


@pytest.mark.parametrize("k", [32, 96, 544])
def test_8_bit_codes_in_fp32(ms, cuda_device, k):
    """Exactly what the block holds, down to 2^-136 (beyond the largest of fp32: infinities)."""
    codes, scales, want = all_8_bit_codes(k, cuda_device)
    finite = (codes & 127 != 127)  # the code that stands for NaN apart
    got = ms.dequantize_rows8(codes, scales, FP32)
    assert float(want[finite & (want > 0)].min()) < 2.0 ** -133  # below the smallest of bf16
    assert same(got[finite], want[finite].float())


def test_4_bit_codes(ms, cuda_device):
    """e2m1 as rows and as weights, in either type (2^-128, the smallest, is exact in both)."""
    e, n, k = 2, 24, 384
    code = (torch.arange(e * n * k, device=cuda_device) * 5 % 16).to(torch.uint8).view(e, n, k)
    scales = torch.tensor([0, 1, 2, 127, 240, 251, 252, 255], dtype=torch.uint8, device=cuda_device)
    scales = scales[torch.arange(e * n * (k // 32), device=cuda_device) % 8].view(e, n, -1)
    want = ref.values4(code, scales)
    q = ms.Mx4Weights.from_checkpoint(ref.pack4(code), scales)
    buffer = torch.cat((ref.pack4(code[0]).flatten(), ref.tile_order(scales[0]).flatten()))
    rows = ms.Mx4Rows(buffer, n * k // 2, n, k)
    for out in (FP32, BF16):
        assert same(ms.dequantize_weights(q, out), want.to(out).transpose(1, 2))
        assert same(ms.dequantize_rows(rows, out), want[0].to(out))


@pytest.mark.parametrize("k", [32, 96, 544])
def test_8_bit_codes_that_stand_for_nan(ms, cuda_device, k):
    """0x7f and 0xff read as NaN in either type; in bf16 every other code is rounded once."""
    codes, scales, want = all_8_bit_codes(k, cuda_device)
    assert torch.isnan(want).any()
    assert same(ms.dequantize_rows8(codes, scales, FP32), want.float())
    assert same(ms.dequantize_rows8(codes, scales, BF16), want.float().to(BF16))  # 64 to 32 bits is exact here


@pytest.mark.parametrize("stride", [5, 4097])
def test_one_row_with_any_stride(ms, cuda_device, stride):
    """The stride of a single row is never used: a row cut out of a matrix of odd width is taken as it is."""
    pool = torch.randn(2 * 4096, device=cuda_device).to(BF16)
    x = torch.as_strided(pool, (1, 288), (stride, 1))
    want = ms.dequantize_rows(ms.quantize_rows(x.clone()))
    assert torch.equal(ms.dequantize_rows(ms.quantize_rows(x)), want)
    assert torch.equal(ms.dequantize_rows8(*ms.quantize_rows8(x)), ms.dequantize_rows8(*ms.quantize_rows8(x.clone())))
    out = torch.as_strided(torch.zeros_like(pool), (1, 288), (stride, 1))
    assert torch.equal(ms.dequantize_rows(ms.quantize_rows(x), out=out), want)
    plan = ms.Mx4Linear(ms.quantize_weights(torch.randn(1, 288, 72, device=cuda_device)), 4)
    assert torch.equal(plan.forward(x), plan.forward(x.clone()))
