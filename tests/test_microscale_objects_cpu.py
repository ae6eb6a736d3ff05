"""What the Python objects of the microscaled calls refuse before anything reaches the library."""
import ctypes
import importlib

import pytest
import torch


class Elsewhere:
    """A tensor of a second device, as far as a check of arguments sees it."""

    dtype = torch.uint8

    def __init__(self, size):
        self.size, self.device = size, torch.device("cpu", 1)

    def numel(self):
        return self.size

    def is_contiguous(self):
        return True


def test_training_scratch_of_another_device_of_the_same_kind(axm):
    w = dict(router_w=torch.zeros(64, 4), w_gate=torch.zeros(4, 64, 96, dtype=torch.bfloat16))
    need = axm.train_split_bytes(axm.make_desc(8, 64, 96, 4, 2, flags=axm.FLAG_RESIDUAL | axm.FLAG_SAVE_8BIT))[1]
    axm.MoeTrainLayer(w, 8, 2, device="cpu", save_8bit=True, weight_grads=False, scratch=torch.empty(need, dtype=torch.uint8))
    with pytest.raises(ValueError, match="scratch"):
        axm.MoeTrainLayer(w, 8, 2, device="cpu", save_8bit=True, weight_grads=False, scratch=Elsewhere(need))


def test_layer_refuses_matrices_off_16_bytes(axm):
    """x, the router's weights and both outputs are read and written in 16-byte pieces."""
    lib, fake = axm.load(), 1 << 20  # never dereferenced
    desc = axm.make_desc(4, 64, 64, 4, 2)
    size = ctypes.c_size_t(0)
    assert lib.axm_moe_mx4_workspace_bytes(ctypes.byref(desc), ctypes.byref(size)) == axm.AXM_OK
    weights = axm.Mx4ExpertWeights(*[fake] * 6)
    for field in ("x", "router_w", "out", "y"):
        for off in (2, 8):
            t = axm.MoeTensors()
            t.x = t.router_w = t.out = t.y = fake
            setattr(t, field, fake + off)
            assert lib.axm_moe_forward_mx4(ctypes.byref(desc), ctypes.byref(t), ctypes.byref(weights), None, fake, size.value,
                                           None) == axm.AXM_ERR_ARGUMENT, (field, off)
            assert b"aligned" in lib.axm_last_error()


def test_calls_by_keyword(axm):
    """The documented names of the first arguments: host tensors come as far as the call's own refusal."""
    ms = importlib.import_module("project_axiom_ai_llm_b200.microscale")
    x, codes, scales = torch.zeros(4, 64), torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    for call, kw in [(ms.quantize_rows, dict(x=x)), (ms.quantize_rows8, dict(x=x)), (ms.quantize_weights, dict(w=x.view(1, 4, 64))),
                     (ms.dequantize_rows8, dict(codes=codes, scales=scales)), (ms.dequantize_rows8, dict(scales=scales, codes=codes))]:
        with pytest.raises(ValueError, match="CUDA"):
            call(**kw)
    with pytest.raises(TypeError):
        ms.quantize_rows()


def test_more_experts_than_a_table_can_name(axm):
    """A segment's expert is read from 16 bits."""
    lib, fake, size = axm.load(), 1 << 20, ctypes.c_size_t(0)
    keep = axm.Mx8Checkpoint(*[fake] * 4)
    for experts, status in ((65535, axm.AXM_OK), (65536, axm.AXM_ERR_ARGUMENT), (70000, axm.AXM_ERR_ARGUMENT)):
        desc = axm.make_desc(4, 64, 64, experts, 1)
        assert lib.axm_mx4_expert_ffn_workspace_bytes(ctypes.byref(desc), 4, 2, ctypes.byref(size)) == status
        assert lib.axm_mx8_expert_ffn_train(ctypes.byref(desc), None, 0, None, 0, None, None, None, ctypes.byref(keep), None, None, 0,
                                            None, None) == status
