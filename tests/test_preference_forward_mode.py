"""Forward-mode derivatives, which the operators do not have, are refused and not dropped."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from reversability_amd.preference import tied_head_logprobs

LABELS = torch.zeros(2, dtype=torch.int64)


@pytest.mark.parametrize("operand", [0, 1])
@pytest.mark.parametrize("grad", [True, False])
def test_dual_operands_are_refused(operand, grad):
    """Also where neither requires a gradient and no autograd node is made (on the CPU:
    the refusal comes before the device's)."""
    operands = [torch.zeros(2, 64).half(), torch.zeros(64, 64).half()]
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        operands[operand] = forward_ad.make_dual(operands[operand],
                                                 torch.ones_like(operands[operand]))
        with pytest.raises(NotImplementedError, match="forward"):
            tied_head_logprobs(*operands, 64, LABELS)


def test_a_level_without_dual_operands_is_no_refusal():
    with forward_ad.dual_level(), pytest.raises(ValueError, match="CUDA"):
        tied_head_logprobs(torch.zeros(2, 64).half(), torch.zeros(64, 64).half(), 64, LABELS)


@pytest.mark.gpu
def test_dual_operands_on_the_gpu(cuda_device):
    x, head = (torch.zeros(n, 64, device=cuda_device).half() for n in (2, 64))
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward"):
        tied_head_logprobs(forward_ad.make_dual(x, x), head, 64, LABELS.to(cuda_device))
