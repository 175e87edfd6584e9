"""Models with a window, sinks and a rotation on the fused training path: their gradients, and
whole updates captured in a graph."""
from __future__ import annotations

import copy

import pytest
import torch
import torch.nn.functional as F

from reversability_amd import build_model, paths
from reversability_amd.attention import Rotary, enable_attention
from reversability_amd.linear import enable_linear
from reversability_amd.optimized_v3 import install_v3

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("method", ["baseline", "midpoint", "euler"])
@pytest.mark.parametrize("window,sinks,rotated", [(24, 2, False), (24, 2, True), (None, 0, True)])
def test_fused_models_train_with_a_window(cuda_device, method, window, sinks, rotated):
    """install_v3, enable_linear and enable_attention(window, sinks, rotary) under fp16 autocast against
    the model in torch operations (fp32, no autocast): gradients agree to fp16's precision."""
    config = {"model": {"vocab_size": 97, "max_sequence_length": 160, "n_layers": 2, "n_heads": 4,
                        "d_model": 128, "d_ff": 256}, "method": method}
    torch.manual_seed(5)
    model = build_model(config).to(cuda_device)
    plain = copy.deepcopy(model)
    install_v3(model, core_mode="split" if method == "midpoint" else "reference", mlp_tokens=512,
               swiglu=True, rmsnorm=True, keep_mlp_tiles=True)
    enable_linear(model)
    rotary = Rotary(32, 160, device=cuda_device) if rotated else None
    for m in (model, plain):
        enable_attention(m, window=window, sinks=sinks, rotary=rotary)
    ids = torch.randint(0, 97, (2, 130), device=cuda_device)
    paths.reset()
    with torch.autocast("cuda", dtype=torch.float16):
        loss = F.cross_entropy(model(ids).flatten(0, 1).float(), ids.flatten())
    (1024 * loss).backward()
    assert paths.report()["attention"].keys() == {"hip"}
    truth = F.cross_entropy(plain(ids).flatten(0, 1), ids.flatten())
    truth.backward()
    assert abs(float(loss.detach()) - float(truth.detach())) <= 2e-3 * float(truth.detach())
    for (name, a), b in zip(model.named_parameters(), plain.parameters()):
        rel = float((a.grad / 1024 - b.grad).norm() / b.grad.norm())
        assert rel <= 2e-2, (name, rel)


SMALL = {"model": {"vocab_size": 503, "max_sequence_length": 300, "n_layers": 3, "n_heads": 4,
                   "d_model": 256, "d_ff": 512},
         "step_size": 0.5, "batch": 4, "workload": "a window"}


@pytest.mark.parametrize("method,core", [("midpoint", "split"), ("euler", "reference")])
@pytest.mark.parametrize("window,sinks,rotated", [(40, 3, True), (None, 0, True), (90, 0, False)])
def test_captured_updates_with_a_window_match_eager_ones(cuda_device, monkeypatch, method, core,
                                                         window, sinks, rotated):
    """The whole update of a model with a window captured in a graph and replayed: loss, parameters
    and loss scale are a twin's eager ones, bit for bit, with host synchronisations and the
    twin's updates between the replays."""
    import bench
    from reversability_amd.graph import CapturedStep
    monkeypatch.setitem(bench.TRAIN_CONFIGS, "window",
                        {**SMALL, "method": method, "core_mode": core})
    steps = []
    for _ in range(2):
        step, _, _ = bench.make_train_step(cuda_device, "window")
        rotary = Rotary(64, 300, device=cuda_device) if rotated else None
        enable_attention(step.model, window=window, sinks=sinks, rotary=rotary)
        steps.append(step)
    eager, graphed = steps
    paths.reset()
    captured = CapturedStep(graphed, warmup=3)
    assert paths.report()["attention"].keys() == {"hip"}
    for _ in range(3):  # the capture's warm-up updates
        eager()
    torch.cuda.synchronize()
    before = [p.detach().clone() for p in graphed.model.parameters()]
    for i in range(4):
        print(f"  replay {i}", flush=True)
        loss_g = captured().clone()
        torch.cuda.synchronize()
        loss_e = eager()
        torch.cuda.synchronize()
        assert torch.equal(loss_g, loss_e), (i, float(loss_g), float(loss_e))
        for (name, pe), pg in zip(eager.model.named_parameters(), graphed.model.parameters()):
            assert torch.equal(pe, pg), (i, name)
        assert torch.equal(eager.scaler._scale, graphed.scaler._scale)
    assert all(not torch.equal(b, p) for b, p in zip(before, graphed.model.parameters()))
