"""State of FusedAdamW and FusedAdamW8bit on the CPU: what a checkpoint leaves, and what a
step refuses before it launches anything (fake CUDA tensors: no kernel is launched)."""
from __future__ import annotations

import copy
import pickle

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from reversability_amd import optim
from reversability_amd.optim import FusedAdamW, FusedAdamW8bit

KINDS = [FusedAdamW, FusedAdamW8bit]
SHAPES = [(128, 64), (16,)]


def checkpoint(kind, step, shapes=SHAPES):
    """A state dict on the CPU after one step of ``kind``."""
    opt = kind([torch.zeros(s, requires_grad=True) for s in shapes])
    for p in opt.param_groups[0]["params"]:
        opt.state[p].update(opt._new_moments(p), step=step)
    return opt.state_dict()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("step", [torch.tensor(3.0), torch.tensor(3), torch.tensor([3.0]), 3])
def test_checkpoint_lands_on_the_parameters_device(kind, step):
    params = [torch.zeros(s, device="meta", requires_grad=True) for s in SHAPES]
    opt = kind(params)
    opt.load_state_dict(checkpoint(kind, step))
    for p in params:
        assert all(t.device == p.device for t in opt.state[p].values())
        assert opt.state[p]["step"].dtype == torch.float32 and opt.state[p]["step"].shape == ()
    assert opt.state[params[0]]["step"] is opt.state[params[1]]["step"]


@pytest.mark.parametrize("kind", KINDS)
def test_a_loaded_step_count_is_the_optimizers_own(kind):
    state = checkpoint(kind, torch.tensor(3.0))
    opt = kind([torch.zeros(s, requires_grad=True) for s in SHAPES])
    opt.load_state_dict(state)
    p = opt.param_groups[0]["params"][0]
    opt.state[p]["step"].add_(1)
    assert float(state["state"][0]["step"]) == 3.0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("key", ["step", "exp_avg", "exp_avg_sq", "dtype"])
def test_state_elsewhere_is_refused(kind, key):
    """Moments or a step count that the kernels would read on another device."""
    with FakeTensorMode():
        params = [torch.zeros(s, device="cuda:0", requires_grad=True) for s in SHAPES]
        opt = kind(params)
        for p in params:
            p.grad = torch.ones_like(p)
            moments = {k: torch.zeros_like(p) for k in ("exp_avg", "exp_avg_sq")}
            opt.state[p].update(moments, step=torch.zeros((), device="cuda:0"))
        assert len(opt._group_params(opt.param_groups[0])) == 2
        for p in params:
            if key == "dtype":
                opt.state[p]["step"] = opt.state[p]["step"].double()
            else:
                opt.state[p][key] = opt.state[p][key].cpu()
        with pytest.raises(ValueError, match="state"):
            opt.step()


@pytest.mark.parametrize("source", [FusedAdamW, torch.optim.AdamW])
def test_plain_checkpoint_keeps_the_seed(source):
    """A checkpoint without 8-bit moments has no seed in its groups; parameters that it
    holds no moments for get 8-bit ones later."""
    params = [torch.zeros(s, requires_grad=True) for s in SHAPES]
    opt = FusedAdamW8bit(params, seed=7)
    opt.add_param_group({"params": [torch.zeros(3, requires_grad=True)], "lr": 2.0})
    other = source([torch.zeros(s, requires_grad=True) for s in SHAPES])
    other.add_param_group({"params": [torch.zeros(3, requires_grad=True)], "lr": 3.0})
    opt.load_state_dict(other.state_dict())
    assert [g["seed"] for g in opt.param_groups] == [7, 7]
    assert opt.param_groups[1]["lr"] == 3.0
    saved = FusedAdamW8bit([torch.zeros(s, requires_grad=True) for s in SHAPES], seed=9)
    opt = FusedAdamW8bit(params, seed=7)
    opt.load_state_dict(saved.state_dict())
    assert opt.param_groups[0]["seed"] == 9


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bad", ["gradient", "parameter", "device", "type", "step"])
def test_a_refusal_in_the_second_group_comes_first(kind, bad, monkeypatch):
    """Nothing is launched, no state is made and unscale_clip_'s factors wait for the
    step that is taken."""
    with FakeTensorMode():
        devices = ["cuda:0", {"device": "cuda:1", "type": "cpu"}.get(bad, "cuda:0")]
        first = [torch.zeros(s, device="cuda:0", requires_grad=True) for s in SHAPES]
        p, q = (torch.zeros(s, device=d, requires_grad=True) for s, d in zip(SHAPES, devices))
        for t in (*first, p, q):
            t.grad = torch.ones_like(t)
        opt = kind([{"params": first}, {"params": [p, q]}])
        if bad == "gradient":
            p.grad = torch.ones(64, 128, device="cuda:0").t()
        elif bad == "parameter":
            p.data = torch.zeros(64, 128, device="cuda:0").t()
        elif bad == "step":
            opt.state[p]["step"] = torch.zeros(())
        waiting = opt._pending = (torch.ones(1), torch.ones(1))
        monkeypatch.setattr(kind, "_update", lambda *_: pytest.fail("launched"))
        with pytest.raises(ValueError, match="FusedAdamW"):
            opt.step()
        assert opt._pending is waiting
        assert not any("exp_avg" in st for st in opt.state.values())


@pytest.mark.parametrize("kind", KINDS)
def test_empty_parameters_are_no_work(kind):
    with FakeTensorMode():
        full, empty = (torch.zeros(s, device="cuda:0", requires_grad=True) for s in ((5,), (0, 7)))
        full.grad, empty.grad = torch.ones_like(full), torch.ones_like(empty)
        opt = kind([full, empty])
        assert opt._group_params(opt.param_groups[0]) == [full]


def test_unscale_clip_launches_on_the_gradients_device(monkeypatch):
    """Every launch is made with the gradients' device current."""
    inside, launches = [], []

    class Guard:
        def __init__(self, t):
            self.device = t.device

        def __enter__(self):
            inside.append(self.device)

        def __exit__(self, *exc):
            inside.pop()

    class Library:
        rv_adamw_max_tensors = staticmethod(lambda: 1)
        rv_grad_chunks = staticmethod(lambda *_: 1)

        def __getattr__(self, name):
            return lambda *_: launches.append((name, list(inside))) or 0

    p = [torch.zeros(5, requires_grad=True) for _ in range(2)]
    for t in p:
        t.grad = torch.ones_like(t)
    monkeypatch.setattr(optim, "library", Library)
    monkeypatch.setattr(optim, "_DeviceGuard", Guard)
    monkeypatch.setattr(optim, "_stream", lambda t: 0)
    FusedAdamW(p).unscale_clip_(None, 1.0)
    assert [name for name, _ in launches] == ["rv_grad_sq_partials"] * 2 + ["rv_grad_clip_coef"]
    assert all(devices == [p[0].device] for _, devices in launches)


@pytest.mark.parametrize("copied", [copy.deepcopy, lambda o: pickle.loads(pickle.dumps(o))])
def test_copies_keep_their_options(copied):
    params = [torch.zeros(s, requires_grad=True) for s in SHAPES]
    twin = copied(FusedAdamW8bit(params, lr=0.5, min_8bit_numel=10, seed=3))
    assert (twin.min_8bit_numel, twin.defaults["seed"]) == (10, 3)
    assert twin.param_groups[0]["seed"] == 3 and twin.param_groups[0]["lr"] == 0.5
    small = twin.param_groups[0]["params"][1]
    assert twin._new_moments(small)["exp_avg"].dtype == torch.float8_e4m3fn
    twin.load_state_dict(FusedAdamW8bit(params, min_8bit_numel=99).state_dict())
    assert twin.min_8bit_numel == 10


@pytest.mark.parametrize("kind", KINDS)
def test_moments_of_another_shape_are_refused(kind):
    """The kernels would read past them; nothing is loaded."""
    opt = kind([torch.zeros(s, requires_grad=True) for s in [(128, 65), (16,)]])
    for state in (checkpoint(kind, torch.tensor(1.0)), checkpoint(FusedAdamW, torch.tensor(1.0))):
        with pytest.raises(ValueError, match="shape"):
            opt.load_state_dict(state)
        assert not opt.state


@pytest.mark.parametrize("kind", KINDS)
def test_transposed_moments_keep_their_elements(kind):
    """Moments saved with other strides (of a transposed parameter): the kernels pair
    them with the parameter's elements by their place in memory."""
    state = checkpoint(FusedAdamW, torch.tensor(1.0))
    moment = torch.randn(64, 128).t()
    state["state"][0]["exp_avg"] = moment
    opt = kind([torch.zeros(s, requires_grad=True) for s in SHAPES])
    opt.load_state_dict(state)
    loaded = opt.state[opt.param_groups[0]["params"][0]]["exp_avg"]
    assert torch.equal(loaded, moment) and loaded.is_contiguous()
