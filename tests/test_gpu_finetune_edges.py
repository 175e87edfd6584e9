"""Updates that cannot be made are refused before any gradient is touched."""
from __future__ import annotations

import pytest
import torch

from reversability_amd import build_model
from reversability_amd.preference import policy_backward, preference_backward

MODEL = {"vocab_size": 203, "max_sequence_length": 32, "n_layers": 2, "n_heads": 2,
         "d_model": 32, "d_ff": 64}


def made(device):
    torch.manual_seed(7)
    model = build_model({"model": MODEL, "method": "baseline"}).to(device)
    ids = torch.randint(203, (4, 16), device=device)
    return model, ids, ids.roll(-1, 1), torch.full((4, 16), -5.0, device=device)


def updates(model, ids, labels, logp):
    yield lambda: preference_backward(model, ids, labels, logp)
    yield lambda: policy_backward(model, ids, labels, logp, logp[:, 0].contiguous())


def test_without_gradients_on_the_cpu():
    model, *batch = made("cpu")
    for update in updates(model, *batch):
        with torch.no_grad(), pytest.raises(ValueError, match="gradients"):
            update()


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["no_grad", "frozen"])
def test_without_gradients(cuda_device, how):
    """The head's gradient used to be added before the hidden states' backward failed."""
    model, *batch = made(cuda_device)
    model.requires_grad_(how == "no_grad")
    for update in updates(model, *batch):
        with torch.set_grad_enabled(how == "frozen"), pytest.raises(ValueError, match="gradients"):
            update()
    assert all(p.grad is None for p in model.parameters())
    model.requires_grad_(True)
    for update in updates(model, *batch):
        update()
    assert all(p.grad is not None for p in model.parameters())
