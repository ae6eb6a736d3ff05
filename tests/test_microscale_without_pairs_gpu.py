"""The 4-bit products where CTA pairs are not wanted (AXM_GEMM_2SM=0, read once per process): the one-CTA
kernel does the same tiles.  The tests of the products are run again in a child process with the switch set."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))

NAMES = """
import sys
sys.path.insert(0, {here!r})
import importlib, torch
from conftest import load_package
load_package()
ms = importlib.import_module("project_axiom_ai_llm_b200.microscale")
plan = ms.Mx4Linear(ms.quantize_weights(torch.randn(1, 256, 512, device="cuda")), 600)
x = torch.randn(600, 256, device="cuda").bfloat16()
plan.forward(x)
torch.cuda.synchronize()
with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as p:
    plan.forward(x)
    torch.cuda.synchronize()
print(" ".join(e.key for e in p.key_averages()))
"""


def child(switch, *args):
    r = subprocess.run([sys.executable, *args], env=dict(os.environ, AXM_GEMM_2SM=switch), capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    return r.stdout


def test_the_switch_chooses_the_kernel(cuda_device):
    names = [child(switch, "-c", NAMES.format(here=HERE)) for switch in ("1", "0")]
    assert "mx4_gemm_pair_kernel" in names[0] and "mx4_gemm_single_kernel" not in names[0]
    assert "mx4_gemm_single_kernel" in names[1] and "mx4_gemm_pair_kernel" not in names[1]


def test_products_pass_without_pairs(cuda_device):
    out = child("0", "-m", "pytest", "-q", "-x", "-m", "gpu", "-p", "no:cacheprovider", os.path.join(HERE, "test_microscale_gpu.py"),
                os.path.join(HERE, "test_microscale_tables_gpu.py"), "-k",
                "linear_exact or linear_wide or expert_ffn or tables_that or test_layer or without_rows or captured")
    assert " passed" in out
