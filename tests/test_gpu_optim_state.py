"""Resuming FusedAdamW and FusedAdamW8bit on the GPU from checkpoints of several kinds: the
resumed run takes the steps that the first one would have taken, bit for bit."""
from __future__ import annotations

import io

import pytest
import torch

from reversability_amd.optim import FusedAdamW, FusedAdamW8bit

pytestmark = pytest.mark.gpu

SHAPES = [(33,), (64, 96), (1031, 7)]


def made(kind, device, start=None):
    g = torch.Generator().manual_seed(5)
    base = [0.02 * torch.randn(s, generator=g) for s in SHAPES] if start is None else start
    params = [t.detach().to(device).clone().requires_grad_(True) for t in base]
    return params, kind(params, lr=1e-2)


def steps(params, opt, seeds):
    for seed in seeds:
        g = torch.Generator().manual_seed(seed)
        for p in params:
            p.grad = 0.01 * torch.randn(p.shape, generator=g).to(p.device)
        opt.step()


@pytest.mark.parametrize("kind", [FusedAdamW, FusedAdamW8bit])
def test_resumed_from_a_checkpoint_on_the_cpu(cuda_device, kind):
    params, opt = made(kind, cuda_device)
    steps(params, opt, range(3))
    file = io.BytesIO()
    torch.save(opt.state_dict(), file)
    file.seek(0)
    twins, other = made(kind, cuda_device, params)
    other.load_state_dict(torch.load(file, map_location="cpu", weights_only=True))
    steps(params, opt, range(3, 5))
    steps(twins, other, range(3, 5))
    for p, q in zip(params, twins):
        assert torch.equal(p, q)
        assert float(other.state[q]["step"]) == 5.0


def test_8_bit_moments_made_after_a_plain_checkpoint(cuda_device):
    """A run that was saved before one of its large parameters had moments: the
    parameter gets 8-bit ones, as in a run that never stopped."""
    params, opt = made(FusedAdamW, cuda_device)
    params[2].requires_grad_(False)  # frozen so far
    for p in params[:2]:
        p.grad = torch.ones_like(p)
    opt.step()
    twins, other = made(FusedAdamW8bit, cuda_device, params)
    other.load_state_dict(opt.state_dict())
    steps(twins, other, [1])
    assert "exp_avg_scale" not in other.state[twins[1]]
    assert other.state[twins[2]]["exp_avg_scale"].dtype == torch.uint8
    assert float(other.state[twins[2]]["step"]) == 2.0
    assert not torch.equal(twins[2], params[2])


@pytest.mark.parametrize("kind", [FusedAdamW, FusedAdamW8bit])
def test_a_refused_step_can_be_taken_again(cuda_device, kind):
    """A gradient of the second group that is refused after unscale_clip_: nothing has
    changed, and the step that follows still unscales and clips."""
    params, opt = made(kind, cuda_device)
    twins, other = made(kind, cuda_device)
    for o, (a, b, c) in ((opt, params), (other, twins)):
        del o.param_groups[0]["params"][1:]
        o.add_param_group({"params": [b, c]})
    before = [p.detach().clone() for p in params]
    for p, q in zip(params, twins):
        p.grad = q.grad = torch.full_like(p, 3.0) * 1024
    scalers = [torch.amp.GradScaler("cuda", init_scale=1024.0) for _ in range(2)]
    for o, s in zip((opt, other), scalers):
        s.scale(torch.ones((), device=cuda_device))
        o.unscale_clip_(s, 0.5)
    right = params[1].grad
    params[1].grad = right.t().contiguous().t()
    with pytest.raises(ValueError, match="contiguous"):
        scalers[0].step(opt)
    assert all(torch.equal(p, b) for p, b in zip(params, before)) and not opt.state
    params[1].grad = right
    opt.step()
    scalers[1].step(other)
    for p, q, b in zip(params, twins, before):
        assert torch.equal(p, q) and not torch.equal(p, b)
        assert torch.equal(opt.state[p]["exp_avg"].float(), other.state[q]["exp_avg"].float())


@pytest.mark.parametrize("kind", [FusedAdamW, FusedAdamW8bit])
def test_empty_parameters_are_passed_over(cuda_device, kind):
    """A parameter without elements beside others, in a group of its own, and alone."""
    params, opt = made(kind, cuda_device)
    twins, other = made(kind, cuda_device)
    empty = [torch.empty(0, 7, device=cuda_device, requires_grad=True) for _ in range(2)]
    other.param_groups[0]["params"].insert(1, empty[0])
    other.add_param_group({"params": [empty[1]]})
    for p, q in zip(params, twins):
        p.grad = torch.full_like(p, 3.0)
        q.grad = p.grad.clone()
    for e in empty:
        e.grad = torch.empty_like(e)
    for o in (opt, other):
        o.unscale_clip_(None, 0.5)
        o.step()
    assert float(other.state[twins[0]]["step"]) == 1.0
    # the random bits follow a parameter's place: only the moments' codes may differ
    assert all(torch.equal(p, q) for p, q in zip(params, twins))
    alone = kind([empty[0]])
    assert float(alone.unscale_clip_(None, 1.0)) == 0.0
    alone.step()
