"""Fine-tuning updates end to end on the GPU: preference_backward and policy_backward
with FusedAdamW8bit on reversible decoders.

The comparator is plain torch on a copy of the model (modules unpatched, autograd
backward, eager residual updates): log_softmax of fp32-widened logits, the losses
written out.  Bars as in the other model comparisons under fp16 autocast:
per-parameter gradient relative L2 2e-2, loss relative 2e-3 (of the loss plus
one: these losses are near log 2 or 0).  bf16 rounds eight times coarser: 0.16.
"""
from __future__ import annotations

import copy
import math

import pytest
import torch
import torch.nn.functional as F

from reversability_amd import build_model, paths
from reversability_amd.attention import enable_attention
from reversability_amd.embedding import enable_embedding
from reversability_amd.graph import CapturedStep
from reversability_amd.linear import enable_linear
from reversability_amd.optim import FusedAdamW8bit
from reversability_amd.optimized_v3 import install_v3
from reversability_amd.preference import (policy_backward, policy_loss, preference_backward,
                                          preference_loss, sequence_logprobs,
                                          tied_head_logprobs)
from reversability_amd.residual import eager_updates

pytestmark = pytest.mark.gpu

MODEL = {"vocab_size": 1003, "max_sequence_length": 96, "n_layers": 2, "n_heads": 4,
         "d_model": 128, "d_ff": 256}
AMP = {"fp16": torch.float16, "bf16": torch.bfloat16}


def build(method, device, wired, **sizes):
    torch.manual_seed(1337)
    model = build_model({"model": {**MODEL, **sizes}, "method": method}).to(device)
    with torch.no_grad():  # confident enough for gradients that differ from token to token
        model.token_embedding.weight.mul_(8)
    plain = copy.deepcopy(model)
    if method != "baseline":
        plain.backward_mode = "autograd"
    if wired:
        install_v3(model, core_mode="split" if method == "midpoint" else "reference",
                   mlp_tokens=100, swiglu=True, rmsnorm=True)
        enable_linear(model)
        enable_attention(model)
        enable_embedding(model, into_grad=True)
    return model, plain


def batch(device, seqs=6, tokens=48, vocab=1003, seed=0):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(vocab, (seqs, tokens), generator=g)
    labels = ids.roll(-1, 1)
    labels[:, -1] = -100
    labels[:, :7] = -100
    labels[1] = -100  # a sequence without an answer
    labels[2, 20:] = -100
    return ids.to(device), labels.to(device)


def plain_logp(model, ids, labels, precision):
    with torch.autocast("cuda", dtype=AMP[precision]), eager_updates():
        logits = model(ids)
    table = logits.float().log_softmax(-1)
    logp = table.gather(-1, labels.clamp_min(0)[..., None])[..., 0]
    return torch.where(labels != -100, logp, 0.0)


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm().clamp_min(1e-30))


def compare(model, plain, bar):
    for (name, p), q in zip(model.named_parameters(), plain.parameters()):
        assert p.grad is not None and bool(torch.isfinite(p.grad).all()), name
        assert rel(p.grad, q.grad) <= bar, (name, rel(p.grad, q.grad))


# the fused SwiGLU and norms of the wired model take fp16 and fp32
@pytest.mark.parametrize("method,wired,precision", [
    ("midpoint", True, "fp16"), ("euler", True, "fp16"), ("baseline", False, "fp16"),
    ("midpoint", False, "fp16"), ("baseline", False, "bf16"), ("midpoint", False, "bf16")])
def test_preference_update_matches_plain_torch(cuda_device, method, wired, precision):
    model, plain = build(method, cuda_device, wired)
    ids, labels = batch(cuda_device)
    reference = copy.deepcopy(plain)
    with torch.no_grad():
        for p in reference.parameters():
            p.mul_(0.9)
        ref = sequence_logprobs(reference, ids, labels, precision)
        ref_plain = plain_logp(reference, ids, labels, precision)
    scale = 1.0 if precision == "fp16" else 8.0
    assert rel(ref, ref_plain) <= 2e-3 * scale and not ref[labels == -100].any()
    scaler = torch.amp.GradScaler("cuda", init_scale=256.0)
    out = preference_backward(model, ids, labels, ref_plain, 0.1, label_smoothing=0.1,
                              chunk_tokens=77, scaler=scaler, precision=precision)
    s = (plain_logp(plain, ids, labels, precision) - ref_plain).sum(1) * 0.1
    margin = s[:3] - s[3:]
    loss = -(0.9 * F.logsigmoid(margin) + 0.1 * F.logsigmoid(-margin)).mean()
    (loss * 256).backward()
    loss = loss.detach()
    assert abs(float(out.loss - loss)) <= 2e-3 * scale * (1 + float(loss))
    assert rel(torch.cat([out.chosen, out.rejected]), s.detach()) <= 2e-2 * scale
    compare(model, plain, 2e-2 * scale)


@pytest.mark.parametrize("reduction", ["token", "sequence"])
@pytest.mark.parametrize("method,wired", [("midpoint", True), ("baseline", False)])
def test_policy_update_matches_plain_torch(cuda_device, method, wired, reduction):
    model, plain = build(method, cuda_device, wired)
    ids, labels = batch(cuda_device)
    mask = labels != -100
    g = torch.Generator().manual_seed(5)
    with torch.no_grad():
        now = plain_logp(plain, ids, labels, "fp16")
    # ratios away from the clip borders, where the two models' rounding does not decide
    shift = torch.tensor([-0.5, -0.1, 0.0, 0.1, 0.6])
    old = now - shift[torch.randint(5, now.shape, generator=g)].to(cuda_device) * mask
    ref = now + (0.3 * torch.randn(now.shape, generator=g)).to(cuda_device) * mask
    adv = torch.randn(len(ids), generator=g).to(cuda_device)
    out = policy_backward(model, ids, labels, old, adv, ref_logp=ref, clip=(0.2, 0.3),
                          kl_coef=0.05, reduction=reduction)
    logp = plain_logp(plain, ids, labels, "fp16")
    r, a = (logp - old).exp(), adv[:, None]
    term = -torch.minimum(r * a, r.clamp(0.8, 1.3) * a)
    term = (term + 0.05 * ((ref - logp).exp() - (ref - logp) - 1)) * mask
    if reduction == "token":
        loss = term.sum() / mask.sum()
    else:
        loss = (term.sum(1) / mask.sum(1).clamp_min(1)).mean()
    loss.backward()
    loss = loss.detach()
    assert abs(float(out.loss - loss)) <= 2e-3 * (1 + abs(float(loss)))
    r = r.detach()
    clipped = ((a > 0) & (r > 1.3) | (a < 0) & (r < 0.8)) & mask
    assert abs(float(out.clipped) - float(clipped.sum() / mask.sum())) <= 1e-6
    compare(model, plain, 2e-2)


def test_update_is_its_operators(cuda_device):
    """preference_backward's numbers are tied_head_logprobs and preference_loss on the
    model's hidden states; the head's gradient is added to what is there; width that 8
    does not divide and a frozen head work."""
    from reversability_amd.optimized import hidden_states
    model, _ = build("baseline", cuda_device, False, d_model=100)
    ids, labels = batch(cuda_device)
    ref = sequence_logprobs(model, ids, labels)
    with torch.autocast("cuda", dtype=torch.float16):
        hidden = hidden_states(model, ids)
    head = torch.zeros(1024, 100, device=cuda_device, dtype=torch.float16)
    head[:1003] = model.lm_head.weight.detach()
    x = hidden.detach().half().requires_grad_(True)
    head.requires_grad_(True)
    logp = tied_head_logprobs(x, head, 1003, labels)
    assert torch.equal(logp.detach(), ref)
    loss = preference_loss(logp, ref - 0.1, mask=labels != -100).loss
    dx, dhead = torch.autograd.grad(loss, (x, head))
    out = preference_backward(model, ids, labels, ref - 0.1)
    assert torch.equal(out.loss, loss.detach())
    first = [p.grad.clone() for p in model.parameters()]
    # the embedding's part of the tied gradient
    model.zero_grad()
    model.lm_head.weight.requires_grad_(True)
    with torch.autocast("cuda", dtype=torch.float16):
        hidden_states(model, ids).backward(dx.to(hidden.dtype))
    tied = model.lm_head.weight.grad + dhead[:1003].float()
    assert rel(first[0], tied) <= 2e-3  # fp16's rounding of dhead
    model.zero_grad()
    for _ in range(2):
        preference_backward(model, ids, labels, ref - 0.1)
    for p, g in zip(model.parameters(), first):
        assert rel(p.grad, 2 * g) <= 1e-5
    model.zero_grad()
    model.lm_head.weight.requires_grad_(False)
    preference_backward(model, ids, labels, ref - 0.1)
    assert model.lm_head.weight.grad is None
    for p, g in list(zip(model.parameters(), first))[1:]:
        assert rel(p.grad, g) <= 1e-5


def test_fully_unscored_batch_gives_zero_gradients(cuda_device):
    model, _ = build("midpoint", cuda_device, True)
    ids, labels = batch(cuda_device)
    labels.fill_(-100)
    out = preference_backward(model, ids, labels, torch.zeros(ids.shape, device=cuda_device))
    assert abs(float(out.loss) - math.log(2)) <= 1e-7
    assert not any(bool(p.grad.any()) for p in model.parameters())
    out = policy_backward(model, ids, labels, torch.zeros(ids.shape, device=cuda_device),
                          torch.ones(len(ids), device=cuda_device))
    assert [float(t) for t in out] == [0.0, 0.0, 0.0]


def test_captured_finetuning_run_equals_eager(cuda_device):
    """Whole updates -- score, preference and policy losses, scaler, clip, 8-bit AdamW --
    captured and replayed, bit for bit the eager run's."""
    ids, labels = batch(cuda_device)
    runs = []
    for captured in (False, True):
        model, _ = build("midpoint", cuda_device, True)
        frozen = copy.deepcopy(_)
        opt = FusedAdamW8bit(model.parameters(), lr=1e-3, betas=(0.9, 0.95), weight_decay=0.1)
        scaler = torch.amp.GradScaler("cuda", init_scale=256.0)
        adv = torch.linspace(-1, 1, len(ids), device=cuda_device)

        def step():
            ref = sequence_logprobs(frozen, ids, labels)
            opt.zero_grad(set_to_none=True)
            a = preference_backward(model, ids, labels, ref, scaler=scaler)
            b = policy_backward(model, ids, labels, ref, adv, ref_logp=ref, kl_coef=0.1,
                                scaler=scaler)
            opt.unscale_clip_(scaler, 1.0)
            scaler.step(opt)
            scaler.update()
            return torch.stack([a.loss, b.loss])
        losses = []
        if captured:
            replay = CapturedStep(step, warmup=1)
            for _ in range(4):
                losses.append(replay().clone())
                torch.randn(100, device=cuda_device).sum().item()
        else:
            for _ in range(5):
                losses.append(step().clone())
            losses = losses[1:]
        runs.append((torch.stack(losses), [p.detach().clone() for p in model.parameters()]))
        assert "exp_avg_scale" in opt.state[model.lm_head.weight]
    assert torch.equal(runs[0][0], runs[1][0])
    assert all(torch.equal(p, q) for p, q in zip(runs[0][1], runs[1][1]))


def test_finetuning_takes_the_kernels(cuda_device):
    model, _ = build("midpoint", cuda_device, True)
    ids, labels = batch(cuda_device)
    paths.reset()
    with paths.strict():
        ref = sequence_logprobs(model, ids, labels)
        preference_backward(model, ids, labels, ref)
    assert paths.report()["tied_head_logprobs"] == {"mfma": 2}


def test_bad_calls_are_refused(cuda_device):
    model, _ = build("baseline", cuda_device, False)
    ids, labels = batch(cuda_device)
    ref = torch.zeros(ids.shape, device=cuda_device)
    with pytest.raises(ValueError, match="fp16 or bf16"):
        preference_backward(model, ids, labels, ref, precision="fp32")
    with pytest.raises(ValueError, match="labels"):
        preference_backward(model, ids, labels[:, 1:], ref)
    with pytest.raises(ValueError, match="chunk"):
        preference_backward(model, ids, labels, ref, chunk_tokens=0)
    with pytest.raises(ValueError, match="one chosen and one rejected"):
        preference_backward(model, ids[:5], labels[:5], ref[:5])
    with pytest.raises(ValueError, match="ref_logp"):
        preference_backward(model, ids, labels, ref[:, 1:])
    with pytest.raises(ValueError, match="mask"):
        preference_loss(ref, ref, mask=torch.ones(ids.shape, device=cuda_device))
    with pytest.raises(ValueError, match="mask"):
        preference_loss(ref, ref, mask=torch.ones(ids.shape, dtype=torch.bool))
    with pytest.raises(ValueError, match="advantages"):
        policy_loss(ref, ref, ref[:, 0].double())
    with pytest.raises(ValueError, match="advantages"):
        policy_loss(ref, ref, ref[0])
    with pytest.raises(ValueError, match="KL"):
        policy_loss(ref, ref, ref, kl_coef=0.1)
    x = torch.zeros(4, 64, device=cuda_device, dtype=torch.float16)
    head = torch.zeros(128, 64, device=cuda_device, dtype=torch.float16)
    lab = torch.zeros(4, device=cuda_device, dtype=torch.int64)
    for args in ((x.bfloat16(), head, 100, lab), (x.float(), head.float(), 100, lab),
                 (x, head[:100], 100, lab), (x, head, 129, lab), (x, head, 0, lab),
                 (x, head, 100, lab[:3]), (x, head, 100, lab.int()), (x[:, :32], head, 100, lab)):
        with pytest.raises(ValueError, match="tied_head_logprobs"):
            tied_head_logprobs(*args)
    with pytest.raises(ValueError, match="device"):
        tied_head_logprobs(x, head, 100, lab.cpu())
