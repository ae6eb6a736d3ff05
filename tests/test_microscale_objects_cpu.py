"""What the Python objects of the microscaled calls refuse before anything reaches the library."""
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
