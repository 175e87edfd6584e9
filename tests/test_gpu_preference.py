"""GPU tests of reversability_amd.preference against plain 64-bit computations.

Tolerances, with u the rounding of the operands' type (2^-11 fp16, 2^-8 bf16) and
S = max_j sum_k |x_k w_jk| of a row:

* a logit: d products summed in fp32, d 2^-24 S.
* a log-probability: two of those (its logit, the log-sum-exp), the exponents' and
  maxima's roundings 4 2^-24 max|z|, v_exp_f32's 2^-23, at most 2^8 additions a lane and
  as many in the joins, 2^-15, and 2^-23 of the logarithm.  Below: ``logp_bound``.
* dx, dhead: each logit gradient is off by u and by that bound (its exponential's
  argument), its products are summed in fp32 (n 2^-24 of the absolute sum for n terms,
  n = vocabulary or rows), the result is rounded, u.  Logit gradients below the 16-bit
  type's range: the scale puts the largest row gradient at 2^14 or more and fp16's
  spacing there ends at 2^-24, so at most 2^-39 of that gradient each.
* the losses: fp64 sums of fp32 terms; a policy term goes through expf and fp32
  arithmetic (2^-20 of its parts), results are rounded to fp32.
"""
from __future__ import annotations

import math

import pytest
import torch

from reversability_amd import preference
from reversability_amd.graph import CapturedStep
from reversability_amd.preference import policy_loss, preference_loss, tied_head_logprobs

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def head_inputs(rows, d, vocab, dtype, seed=0, pad=0, spread=2.0, scale=1.0):
    g = gen(seed)
    padded = -(-vocab // 64) * 64 + pad
    head = torch.zeros(padded, d, device="cuda", dtype=dtype)
    head[:vocab] = (torch.randn(vocab, d, generator=g, device="cuda") * spread / math.sqrt(d)).to(dtype)
    x = torch.randn(rows, d, generator=g, device="cuda").to(dtype)
    labels = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    for at, value in enumerate((0, vocab - 1, -100, min(127, vocab - 1), min(128, vocab - 1),
                                min(255, vocab - 1), min(256, vocab - 1))):
        if at < rows:
            labels[at] = value
    grad = torch.randn(rows, generator=g, device="cuda") * scale
    return x, head, labels, grad


def exact_logp(x, head, vocab, labels, grad=None, held=None):
    """(logp, bound, dx, dx bound, dhead, dhead bound) in 64 bits; ``held``: how far the
    logits' gradients are off as they are held (None: their type's rounding)."""
    u = U[x.dtype]
    held = held or u
    x, w = x.double(), head[:vocab].double()
    valid = labels != -100
    z = x @ w.t()
    spread = (x.abs() @ w.abs().t()).amax(1)
    table = z.log_softmax(1)
    logp = torch.where(valid, table.gather(1, labels.clamp_min(0)[:, None])[:, 0], 0.0)
    lse = z.logsumexp(1)
    bound = (2 * x.shape[1] * 2.0 ** -24 * spread + 4 * 2.0 ** -24 * z.abs().amax(1) + 2.0 ** -15
             + 2.0 ** -23 * lse.abs())
    bound = bound * valid
    if grad is None:
        return logp, bound
    g = (grad.double() * valid)[:, None]
    p = table.exp()
    dz = -p * g
    dz.scatter_add_(1, labels.clamp_min(0)[:, None], g)
    # the error of a logit gradient
    floor = g.abs().max() * 2.0 ** -39
    ddz = dz.abs() * held + (p * g.abs()) * (bound + 2.0 ** -22)[:, None] + floor * valid[:, None]
    dx, dhead = dz @ w, torch.zeros(head.shape, device="cuda", dtype=torch.float64)
    dhead[:vocab] = dz.t() @ x
    bx = ddz @ w.abs() + vocab * 2.0 ** -24 * (dz.abs() @ w.abs()) + u * dx.abs() + 1e-30
    bh = torch.zeros_like(dhead)
    bh[:vocab] = ddz.t() @ x.abs() + len(x) * 2.0 ** -24 * (dz.abs().t() @ x.abs())
    bh += u * dhead.abs()
    bh[:vocab] += 1e-30
    tiny = 2.0 ** -25 if u == 2.0 ** -11 else 0.0  # fp16's last half step, of the results
    return logp, bound, dx, bx + tiny, dhead, bh + tiny * (bh > 0)


def within(got, ref, bound):
    bad = ~((got.double() - ref).abs() <= bound)
    assert not bool(bad.any()), (int(bad.sum()), float((got.double() - ref).abs().max()))


SIZES = [(1, 8, 1), (1, 128, 50257), (3, 64, 2), (7, 72, 64), (51, 256, 1000), (130, 128, 4097),
         (257, 100, 3001), (300, 200, 777), (64, 1, 300), (1000, 384, 4097), (2331, 512, 5000),
         (700, 640, 50257), (5000, 128, 20011), (66, 2048, 130), (20000, 264, 500),
         (70000, 32, 90)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,d,vocab", SIZES)
def test_logprobs_and_gradients(cuda_device, rows, d, vocab, dtype):
    x, head, labels, grad = head_inputs(rows, d, vocab, dtype)
    x.requires_grad_(True)
    head.requires_grad_(True)
    logp = tied_head_logprobs(x, head, vocab, labels)
    dx, dhead = torch.autograd.grad(logp, (x, head), grad)
    assert logp.dtype == torch.float32 and dx.dtype == dhead.dtype == dtype
    ref, bound, rx, bx, rh, bh = exact_logp(x.detach(), head.detach(), vocab, labels, grad)
    within(logp.detach(), ref, bound)
    within(dx, rx, bx)
    within(dhead, rh, bh)
    assert not logp[labels == -100].any() and not dx[labels == -100].any()
    with torch.no_grad():  # the same bits without a graph, and again
        assert torch.equal(tied_head_logprobs(x, head, vocab, labels), logp)
    again = torch.autograd.grad(tied_head_logprobs(x, head, vocab, labels), (x, head), grad)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dhead)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,d,vocab", [(1, 64, 777), (3, 256, 5000), (51, 512, 5000), (51, 96, 64),
                                          (400, 640, 20000), (512, 256, 20000), (511, 8, 300)])
def test_few_rows_hold_their_gradients_twice_as_long(cuda_device, rows, d, vocab, dtype):
    """Up to 512 rows a logit's gradient is a 16-bit number and the 16-bit number of
    what that left out: off by u^2, so that the results are off by their own rounding."""
    x, head, labels, grad = head_inputs(rows, d, vocab, dtype, seed=rows)
    x.requires_grad_(True)
    head.requires_grad_(True)
    dx, dhead = torch.autograd.grad(tied_head_logprobs(x, head, vocab, labels), (x, head), grad)
    _, _, rx, bx, rh, bh = exact_logp(x.detach(), head.detach(), vocab, labels, grad,
                                      held=U[dtype] ** 2)
    within(dx, rx, bx)
    within(dhead, rh, bh)
    # the whole of it: a rounding's error is at most u and 0.58 of it on average (a uniform
    # one), where one of the gradient and one of the result make 0.82
    for got, ref in ((dx, rx), (dhead, rh)):
        if rows >= 51:
            assert float((got.double() - ref).norm()) <= 0.6 * U[dtype] * float(ref.norm())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("chunk", [1, 100, 256, 333])
def test_logprobs_backward_in_chunks(cuda_device, chunk, dtype):
    rows, d, vocab = (333, 136, 1003) if chunk > 1 else (5, 136, 1003)
    x, head, labels, grad = head_inputs(rows, d, vocab, dtype, pad=128)
    x.requires_grad_(True)
    head.requires_grad_(True)
    logp = tied_head_logprobs(x, head, vocab, labels, chunk_tokens=chunk)
    dx, dhead = torch.autograd.grad(logp, (x, head), grad)
    _, _, rx, bx, rh, bh = exact_logp(x.detach(), head.detach(), vocab, labels, grad)
    within(dx, rx, bx)
    within(dhead, rh, bh)
    assert not dhead[vocab:].any()


def test_logprobs_forward_in_chunks(cuda_device, monkeypatch):
    x, head, labels, _ = head_inputs(1000, 128, 999, torch.float16)
    monkeypatch.setattr(preference, "FORWARD_TOKENS", 300)
    ref, bound = exact_logp(x, head, 999, labels)
    within(tied_head_logprobs(x, head, 999, labels), ref, bound)


def test_logprobs_shapes_strides_and_alignment(cuda_device):
    """Leading dimensions; rows with a stride, off a 16-byte boundary; strided
    labels; one gradient only; a head with more padding than it needs."""
    x, head, labels, grad = head_inputs(60, 64, 500, torch.float16, pad=64)
    expected = tied_head_logprobs(x, head, 500, labels)
    three = x.view(3, 4, 5, 64)
    assert torch.equal(tied_head_logprobs(three, head, 500, labels.view(3, 4, 5)),
                       expected.view(3, 4, 5))
    wide = torch.full((60, 80), math.nan, device="cuda", dtype=torch.float16)
    wide[:, 3:67] = x
    strided = wide[:, 3:67]
    spread = torch.full((60, 2), 7, device="cuda")
    spread[:, 1] = labels
    flat = torch.empty(head.numel() + 1, device="cuda", dtype=torch.float16)[1:]
    odd = flat.view(head.shape)
    odd.copy_(head)
    assert torch.equal(tied_head_logprobs(strided, odd, 500, spread[:, 1]), expected)
    x.requires_grad_(True)
    only, = torch.autograd.grad(tied_head_logprobs(x, head, 500, labels), x, grad)
    strided.requires_grad_(True)
    odd.requires_grad_(True)
    sx, sh = torch.autograd.grad(tied_head_logprobs(strided, odd, 500, spread[:, 1]),
                                 (strided, odd), grad)
    assert torch.equal(sx, only)
    head.requires_grad_(True)
    hh, = torch.autograd.grad(tied_head_logprobs(x.detach(), head, 500, labels), head,
                              grad.view(60, 1).expand(60, 2)[:, 0])
    assert torch.equal(hh, sh) and not hh[500:].any()
    none = tied_head_logprobs(x[:0], head, 500, labels[:0])
    assert none.shape == (0,)
    zx, zh = torch.autograd.grad(none.sum(), (x, head))
    assert not zx.any() and not zh.any() and zh.shape == head.shape


def test_logprobs_special_labels_and_values(cuda_device):
    """All tokens unscored; labels outside the vocabulary; a NaN or infinite row
    reaches its own log-probability only; logits far apart; identical ones."""
    x, head, labels, grad = head_inputs(40, 64, 700, torch.float16)
    x.requires_grad_(True)
    head.requires_grad_(True)
    nothing = torch.full_like(labels, -100)
    dx, dhead = torch.autograd.grad(tied_head_logprobs(x, head, 700, nothing), (x, head),
                                    torch.full_like(grad, math.nan))
    assert not dx.any() and not dhead.any()
    wrong = labels.clone()
    wrong[5], wrong[6], wrong[7] = 700, -1, 2 ** 40
    logp = tied_head_logprobs(x, head, 700, wrong)
    good = torch.ones(40, dtype=torch.bool, device="cuda")
    good[5:8] = False
    expected = tied_head_logprobs(x, head, 700, labels)
    assert torch.equal(logp[good], expected[good]) and bool(logp[~good].isnan().all())
    dx, = torch.autograd.grad(logp, x, grad)
    assert bool(dx[~good].isnan().all()) and bool(dx[good].isfinite().all())
    y = x.detach().clone()
    y[9], y[10] = math.nan, math.inf
    logp = tied_head_logprobs(y, head, 700, labels)
    good[5:8], good[9:11] = True, False
    assert torch.equal(logp[good], expected[good]) and bool(logp[~good].isnan().all())
    # logits of +-10^4: the label's probability is 1 or its logarithm far below
    far = torch.zeros(3, 64, device="cuda", dtype=torch.float16)
    far[:, 0] = 1000
    table = torch.zeros(64, 64, device="cuda", dtype=torch.float16)
    table[0, 0], table[1, 0] = 10, -10
    logp = tied_head_logprobs(far, table, 64, torch.tensor([0, 1, 2], device="cuda"))
    # the first: the logarithm of a sum that is 1 but for the roundings of two v_exp (2^-23
    # each) and their product; the others' differences are exact
    assert abs(float(logp[0])) <= 2.0 ** -21 and logp[1:].tolist() == [-20000.0, -10000.0]
    same = tied_head_logprobs(torch.zeros(2, 64, device="cuda", dtype=torch.bfloat16),
                              torch.zeros(1024, 64, device="cuda", dtype=torch.bfloat16), 1000,
                              torch.tensor([0, 999], device="cuda"))
    assert bool(((same + math.log(1000)).abs() <= 2.0 ** -15 + 2.0 ** -23 * 7).all())


@pytest.mark.parametrize("d", [64, 256, 512])
def test_pad_rows_of_the_head_get_zeros(cuda_device, d):
    """Whatever they hold, and beside rows whose gradients are NaN."""
    x, head, labels, grad = head_inputs(40, d, 70, torch.float16, pad=192)
    with torch.no_grad():
        head[70:] = math.nan
    labels[3] = 70
    x.requires_grad_(True)
    head.requires_grad_(True)
    logp = tied_head_logprobs(x, head, 70, labels)
    dx, dhead = torch.autograd.grad(logp, (x, head), grad)
    assert torch.isnan(logp[3]) and torch.isnan(dx[3]).all() and torch.isnan(dhead[:70]).all()
    assert not torch.isnan(torch.cat([logp[:3], logp[4:]])).any()
    assert not torch.isnan(torch.cat([dx[:3], dx[4:]])).any()
    assert not dhead[70:].any() and not torch.isnan(dhead[70:]).any()


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e-5, 1.0, 1e4])
def test_logprobs_gradients_of_any_size(cuda_device, scale):
    """Small gradients do not vanish in the 16-bit logit gradients (bf16 operands hold
    the results), nor large ones overflow."""
    x, head, labels, grad = head_inputs(200, 128, 3000, torch.bfloat16, scale=scale)
    x.requires_grad_(True)
    head.requires_grad_(True)
    dx, dhead = torch.autograd.grad(tied_head_logprobs(x, head, 3000, labels), (x, head), grad)
    _, _, rx, bx, rh, bh = exact_logp(x.detach(), head.detach(), 3000, labels, grad)
    for got, ref, bound in ((dx, rx, bx), (dhead, rh, bh)):
        within(got, ref, bound)
        assert float((got.double() - ref).norm()) <= 2 * U[torch.bfloat16] * float(ref.norm())


def test_logprobs_gradient_against_differences(cuda_device):
    """Directional differences of the kernel's own forward: x moves by exact fp16
    steps.  D(h) = phi' + c h^2 + ..., so Richardson's (4 D(h) - D(2h)) / 3 is off by a
    fraction of D(2h) - D(h); the log-probabilities' own error enters as sum |g| 2^-14 /
    h."""
    x, head, labels, grad = head_inputs(100, 64, 600, torch.float16)
    x = (x.float().clamp(-3.5, 3.5) * 64).round().div(64).half()
    v = torch.where(torch.rand(100, 64, generator=gen(9), device="cuda") < 0.5, -1.0, 1.0)
    x.requires_grad_(True)
    dx, = torch.autograd.grad(tied_head_logprobs(x, head, 600, labels), x, grad)

    def phi(h):
        moved = (x.detach().float() + h * v).half()
        return float((tied_head_logprobs(moved, head, 600, labels).double() * grad).sum())
    h = 2.0 ** -6
    d1, d2 = ((phi(k) - phi(-k)) / (2 * k) for k in (h, 2 * h))
    slope = float((dx.double() * v).sum())
    rounding = float(grad.abs().sum()) * 2.0 ** -14 / h + 2.0 ** -10 * float(dx.double().abs().sum())
    assert abs((4 * d1 - d2) / 3 - slope) <= abs(d2 - d1) + rounding
    assert abs(slope) > 3 * rounding  # the test sees the gradient


def test_logprobs_captured(cuda_device):
    """Forward and backward captured once; every replay against the eager result, new
    inputs in place, eager work between."""
    x, head, labels, grad = head_inputs(500, 128, 2000, torch.float16)
    xs = x.clone().requires_grad_(True)
    hs = head.clone().requires_grad_(True)

    def step():
        logp = tied_head_logprobs(xs, hs, 2000, labels, chunk_tokens=300)
        return (logp.detach(), *torch.autograd.grad(logp, (xs, hs), grad))
    captured = CapturedStep(step)
    for seed in range(3):
        new = head_inputs(500, 128, 2000, torch.float16, seed=seed + 1)
        with torch.no_grad():
            xs.copy_(new[0])
            hs.copy_(new[1])
        labels.copy_(new[2])
        grad.copy_(new[3])
        out = [t.clone() for t in captured()]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_logprobs_on_another_stream(cuda_device):
    x, head, labels, grad = head_inputs(300, 128, 2000, torch.bfloat16)
    x.requires_grad_(True)
    expected, = torch.autograd.grad(tied_head_logprobs(x, head, 2000, labels), x, grad)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, = torch.autograd.grad(tied_head_logprobs(x, head, 2000, labels), x, grad)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, expected)


# ---------------------------------------------------------------------------
# preference loss
# ---------------------------------------------------------------------------
def some_mask(kind, shape, seed=1):
    if kind == "none":
        return None
    mask = torch.rand(shape, generator=gen(seed), device="cuda") < 0.6
    mask[::3] = False  # rows without a token
    return mask


def exact_preference(logp, ref, beta, mask, smoothing, average):
    logp = logp.detach().double().requires_grad_(True)
    on = torch.ones_like(logp, dtype=torch.bool) if mask is None else mask
    diff = torch.where(on, logp, 0.0) - torch.where(on, ref.double(), 0.0)
    s = diff.sum(1)
    if average:
        s = s / on.sum(1).clamp(min=1)
    chosen, rejected = (beta * s).chunk(2)
    m = chosen - rejected
    loss = -((1 - smoothing) * torch.nn.functional.logsigmoid(m)
             + smoothing * torch.nn.functional.logsigmoid(-m)).mean()
    dlogp, = torch.autograd.grad(loss, logp)
    size = diff.detach().abs().sum(1).max()
    return loss.detach(), chosen.detach(), rejected.detach(), dlogp, float(size)


@pytest.mark.parametrize("kind", ["none", "some"])
@pytest.mark.parametrize("average,smoothing,beta", [(False, 0.0, 0.1), (True, 0.1, 0.5),
                                                    (False, 0.5, 0.3)])
@pytest.mark.parametrize("pairs,tokens", [(1, 1), (1, 17), (5, 3), (3, 64), (64, 512), (7, 1001),
                                          (3, 2049), (2, 40000), (3000, 5), (1100, 2050),
                                          (20000, 1)])
def test_preference_loss(cuda_device, pairs, tokens, average, smoothing, beta, kind):
    g = gen(pairs * 10007 + tokens)
    ref = -torch.empty(2 * pairs, tokens, device="cuda").exponential_(0.5, generator=g)
    logp = ref + 0.3 * torch.randn(2 * pairs, tokens, generator=g, device="cuda")
    mask = some_mask(kind, logp.shape)
    leaf = logp.clone().requires_grad_(True)
    out = preference_loss(leaf, ref, beta, mask=mask, label_smoothing=smoothing, average=average)
    upstream = torch.tensor(3.0, device="cuda")
    dlogp, = torch.autograd.grad(out.loss, leaf, upstream)
    loss, chosen, rejected, ref_grad, size = exact_preference(logp, ref, beta, mask, smoothing,
                                                              average)
    # each difference is rounded to fp32 (2^-24 of it and its operands' spread)
    off = 2.0 ** -23 * (size + 1) * beta
    within(out.loss.detach(), loss, 2 * off + 2.0 ** -23 * loss.abs())
    within(out.chosen, chosen, off + 2.0 ** -23 * chosen.abs())
    within(out.rejected, rejected, off + 2.0 ** -23 * rejected.abs())
    within(dlogp, 3 * ref_grad, 2.0 ** -22 * 3 * ref_grad.abs()
           + 3 * 2 * off * beta / pairs * (ref_grad != 0))
    assert torch.equal(preference_loss(logp, ref, beta, mask=mask, label_smoothing=smoothing,
                                       average=average).loss, out.loss.detach())


def test_preference_masked_values_are_never_used(cuda_device):
    logp = torch.randn(8, 50, device="cuda")
    ref = torch.randn(8, 50, device="cuda")
    mask = some_mask("some", (8, 50))
    results = []
    for fill in (0.0, math.nan, math.inf, -3.0e38):
        a = torch.where(mask, logp, fill).requires_grad_(True)
        out = preference_loss(a, torch.where(mask, ref, -fill), mask=mask)
        dlogp, = torch.autograd.grad(out.loss, a)
        results.append((out.loss.detach(), out.chosen, out.rejected, dlogp))
    for other in results[1:]:
        assert all(torch.equal(x, y) for x, y in zip(results[0], other))
    assert not results[0][3][~mask].any()


@pytest.mark.parametrize("tokens", [50, 2500])
def test_preference_strides_and_alignment(cuda_device, tokens):
    base = torch.randn(6, tokens + 9, device="cuda")
    ref = torch.randn(6, tokens + 9, device="cuda")
    mask = some_mask("some", (6, tokens + 9))
    views = [(base[:, 3:3 + tokens], ref[:, 1:1 + tokens], mask[:, 5:5 + tokens]),
             (base.t().contiguous().t()[:, :tokens], ref[0, :tokens].expand(6, tokens),
              mask.t().contiguous().t()[:, :tokens])]
    for a, b, m in views:
        dense = [t.contiguous().clone() for t in (a, b, m)]
        leaves = [t.detach().requires_grad_(True) for t in (a, dense[0])]
        out = [preference_loss(leaf, r, 0.2, mask=k)
               for leaf, r, k in zip(leaves, (b, dense[1]), (m, dense[2]))]
        grads = [torch.autograd.grad(o.loss, leaf)[0] for o, leaf in zip(out, leaves)]
        # the order of a row's sum may differ with its alignment: fp64 sums
        for x, y in ((out[0].loss, out[1].loss), (out[0].chosen, out[1].chosen),
                     (out[0].rejected, out[1].rejected), (grads[0], grads[1])):
            within(x.detach(), y.detach().double(), 2.0 ** -23 * y.detach().double().abs())


def test_preference_extremes(cuda_device):
    """Margins that overflow exp, no tokens at all, an infinite log-probability."""
    logp = torch.tensor([[5e5], [-5e5], [0.0], [0.0]], device="cuda", requires_grad=True)
    out = preference_loss(logp, torch.zeros(4, 1, device="cuda"), 1.0)
    dlogp, = torch.autograd.grad(out.loss, logp)
    assert float(out.loss.detach()) == 250000.0
    assert dlogp.flatten().tolist() == [0.0, -0.5, 0.0, 0.5]
    empty = torch.zeros(4, 0, device="cuda", requires_grad=True)
    out = preference_loss(empty, empty.detach())
    dlogp, = torch.autograd.grad(out.loss, empty)
    assert dlogp.shape == (4, 0) and abs(float(out.loss.detach()) - math.log(2)) <= 2.0 ** -24
    bad = torch.tensor([[-math.inf], [0.0]], device="cuda")
    assert float(preference_loss(bad, torch.zeros(2, 1, device="cuda")).loss) == math.inf
    bad = torch.tensor([[math.nan], [0.0]], device="cuda")
    assert math.isnan(float(preference_loss(bad, torch.zeros(2, 1, device="cuda")).loss))


# ---------------------------------------------------------------------------
# policy loss
# ---------------------------------------------------------------------------
def exact_policy(logp, old, adv, ref, mask, clip, kl_coef, reduction):
    """(loss, kl, clipped, dlogp) in 64 bits and the size of the loss's terms."""
    on = torch.ones_like(logp, dtype=torch.bool) if mask is None else mask
    zero = torch.zeros((), device="cuda", dtype=torch.float64)
    lp = torch.where(on, logp.detach().double(), zero).requires_grad_(True)
    old = torch.where(on, old.double(), zero)
    adv = adv.double()[:, None] if adv.ndim == 1 else adv.double()
    adv = torch.where(on, adv, zero)
    ratio = (lp - old).exp()
    term = -torch.minimum(ratio * adv, ratio.clamp(1 - clip[0], 1 + clip[1]) * adv)
    k = torch.zeros_like(lp)
    if ref is not None:
        shift = torch.where(on, ref.double(), zero) - lp
        k = torch.expm1(shift) - shift
        term = term + kl_coef * k
    n = on.sum().clamp(min=1)
    if reduction == "token":
        loss = torch.where(on, term, zero).sum() / n
    else:
        loss = (torch.where(on, term, zero).sum(1) / on.sum(1).clamp(min=1)).sum() / len(on)
    dlogp, = torch.autograd.grad(loss, lp)
    r = ratio.detach()
    out = ((adv > 0) & (r > 1 + clip[1])) | ((adv < 0) & (r < 1 - clip[0]))
    size = term.detach().abs() + (1 + r) * adv.abs()
    if ref is not None:
        size = size + abs(kl_coef) * (2 + shift.detach().exp() + shift.detach().abs())
    return (loss.detach(), torch.where(on, k.detach(), zero).sum() / n,
            (out & on).sum() / n, dlogp, float(size.max()))


@pytest.mark.parametrize("reduction", ["token", "sequence"])
@pytest.mark.parametrize("kind,with_ref,per_token,clip", [
    ("none", False, False, (0.2, 0.2)), ("some", True, False, (0.2, 0.28)),
    ("some", True, True, (0.1, 0.3)), ("some", False, True, (0.0, 0.0))])
@pytest.mark.parametrize("seqs,tokens", [(1, 1), (5, 333), (3, 4), (64, 512), (2, 30001),
                                         (30000, 1), (9000, 3), (1, 2_200_000)])
def test_policy_loss(cuda_device, seqs, tokens, kind, with_ref, per_token, clip, reduction):
    g = gen(seqs * 101 + tokens)
    shape = (seqs, tokens)
    old = -torch.empty(shape, device="cuda").exponential_(0.5, generator=g)
    logp = old + 0.2 * torch.randn(shape, generator=g, device="cuda")
    ref = old + 0.2 * torch.randn(shape, generator=g, device="cuda") if with_ref else None
    adv = torch.randn(shape if per_token else shape[:1], generator=g, device="cuda")
    mask = some_mask(kind, shape)
    kl = 0.05 if with_ref else 0.0
    leaf = logp.clone().requires_grad_(True)
    out = policy_loss(leaf, old, adv, ref_logp=ref, mask=mask, clip=clip, kl_coef=kl,
                      reduction=reduction)
    dlogp, = torch.autograd.grad(out.loss, leaf, torch.tensor(5.0, device="cuda"))
    loss, k, clipped, grad, size = exact_policy(logp, old, adv, ref, mask, clip, kl, reduction)
    # a term: exp of an argument rounded once (2^-24 of up to 32), 2^-23 of its own, and
    # fp32 sums of a few parts
    each = 2.0 ** -19 * size
    within(out.loss.detach(), loss, each)
    within(out.kl, k, 2.0 ** -19 * 4)
    within(out.clipped, clipped, 2.0 ** -23)
    weight = torch.full((seqs, 1), 1.0, device="cuda", dtype=torch.float64)
    on = torch.ones(shape, device="cuda") if mask is None else mask.double()
    weight = (1 / on.sum().clamp(min=1) if reduction == "token"
              else 1 / on.sum(1, keepdim=True).clamp(min=1) / seqs) * weight
    within(dlogp, 5 * grad, 5 * each * weight + 2.0 ** -22 * 5 * grad.abs())
    assert not dlogp[on == 0].any()
    again = policy_loss(logp, old, adv, ref_logp=ref, mask=mask, clip=clip, kl_coef=kl,
                        reduction=reduction)
    assert torch.equal(again.loss, out.loss.detach()) and torch.equal(again.kl, out.kl)


def test_policy_at_the_clip_borders(cuda_device):
    """Ratios one fp32 step to either side of a border: the gradient is there up to the
    border and gone behind it.  Zero advantages have neither."""
    low, high = math.log1p(-0.2), math.log1p(0.25)
    rows = []
    for border, adv in ((high, 1.0), (low, -1.0), (high, -1.0), (low, 1.0), (high, 0.0)):
        near = torch.tensor(border, dtype=torch.float32)
        for step in (-1, 0, 1):
            x = near
            if step:
                x = torch.nextafter(near, torch.tensor(step * math.inf))
            rows.append((float(x), adv))
    logp = torch.tensor([r[0] for r in rows], device="cuda").view(-1, 1).requires_grad_(True)
    adv = torch.tensor([r[1] for r in rows], device="cuda")
    out = policy_loss(logp, torch.zeros(len(rows), 1, device="cuda"), adv, clip=(0.2, 0.25))
    dlogp, = torch.autograd.grad(out.loss, logp)
    expected = [(a > 0 and x > high) or (a < 0 and x < low) for x, a in rows]
    got = [a != 0 and d == 0 for (_, a), d in zip(rows, dlogp.flatten().tolist())]
    assert got == expected and 0 < sum(expected) < len(rows)
    assert abs(float(out.clipped) - sum(expected) / len(rows)) <= 2.0 ** -23
    assert not dlogp[-3:].any()


def test_policy_masked_values_are_never_used(cuda_device):
    shape = (6, 37)
    old, logp, ref, adv = (torch.randn(shape, device="cuda") for _ in range(4))
    mask = some_mask("some", shape)
    results = []
    for fill in (0.0, math.nan, math.inf, -3.0e38):
        a = torch.where(mask, logp, fill).requires_grad_(True)
        out = policy_loss(a, torch.where(mask, old, fill), torch.where(mask, adv, -fill),
                          ref_logp=torch.where(mask, ref, -fill), mask=mask, kl_coef=0.1)
        dlogp, = torch.autograd.grad(out.loss, a)
        results.append((out.loss.detach(), out.kl, out.clipped, dlogp))
    for other in results[1:]:
        assert all(torch.equal(x, y) for x, y in zip(results[0], other))
    nothing = torch.zeros(shape, device="cuda", dtype=torch.bool)
    for reduction in ("token", "sequence"):
        a = torch.full(shape, math.nan, device="cuda", requires_grad=True)
        out = policy_loss(a, old, adv, ref_logp=ref, mask=nothing, kl_coef=0.1,
                          reduction=reduction)
        dlogp, = torch.autograd.grad(out.loss, a)
        assert [float(t.detach()) for t in out] == [0.0, 0.0, 0.0] and not dlogp.any()
    empty = torch.zeros(3, 0, device="cuda", requires_grad=True)
    out = policy_loss(empty, empty.detach(), torch.zeros(3, device="cuda"), reduction="sequence")
    dlogp, = torch.autograd.grad(out.loss, empty)
    assert float(out.loss.detach()) == 0.0 and dlogp.shape == (3, 0)


def test_policy_strides_and_alignment(cuda_device):
    wide = [torch.randn(6, 61, device="cuda") for _ in range(4)]
    mask = some_mask("some", (6, 61))
    logp, old, ref, adv = (t[:, at:at + 50] for at, t in enumerate(wide))
    adv = adv[:, :1].expand(6, 50)
    for reduction in ("token", "sequence"):
        results = []
        for dense in (False, True):
            args = [t.contiguous() if dense else t for t in (logp, old, adv, ref, mask[:, 7:57])]
            leaf = args[0].detach().requires_grad_(True)
            out = policy_loss(leaf, args[1], args[2], ref_logp=args[3], mask=args[4], kl_coef=0.2,
                              reduction=reduction)
            results.append((out.loss.detach(), out.kl, out.clipped,
                            torch.autograd.grad(out.loss, leaf)[0]))
        assert all(torch.equal(x, y) for x, y in zip(*results))
    same = policy_loss(logp, old, wide[3][:, 3].contiguous())  # one advantage per row
    spread = policy_loss(logp, old, wide[3][:, 3:4].expand(6, 50))
    assert torch.equal(same.loss, spread.loss)


@pytest.mark.parametrize("which", ["preference", "policy"])
def test_losses_against_differences(cuda_device, which):
    """Central differences of the 32-bit loss along a random direction: truncation
    estimated from two steps, plus the loss's own rounding over the step."""
    g = gen(3)
    old, ref = (-torch.rand(8, 40, generator=g, device="cuda") for _ in range(2))
    logp = old + 0.05 * torch.randn(8, 40, generator=g, device="cuda")
    v = torch.randn(8, 40, generator=g, device="cuda")
    adv = torch.randn(8, generator=g, device="cuda")

    def value(t):
        if which == "preference":
            return preference_loss(t, ref, 0.3, label_smoothing=0.1).loss
        return policy_loss(t, old, adv, ref_logp=ref, clip=(0.9, 9.0), kl_coef=0.5).loss
    leaf = logp.clone().requires_grad_(True)
    dlogp, = torch.autograd.grad(value(leaf), leaf)
    h = 2.0 ** -7
    d1, d2 = ((float(value(logp + k * v)) - float(value(logp - k * v))) / (2 * k)
              for k in (h, 2 * h))
    slope = float((dlogp.double() * v).sum())
    rounding = 2.0 ** -22 * (1 + float(value(logp).abs())) / h
    assert abs((4 * d1 - d2) / 3 - slope) <= abs(d2 - d1) + rounding
    assert abs(slope) > 3 * rounding


def test_losses_captured_and_on_another_stream(cuda_device):
    shape = (12, 700)
    old, ref, logp = (-torch.rand(shape, device="cuda") for _ in range(3))
    adv = torch.randn(12, device="cuda")
    mask = some_mask("some", shape)
    logp.requires_grad_(True)

    def step():
        a = preference_loss(logp, ref, mask=mask)
        b = policy_loss(logp, old, adv, ref_logp=ref, mask=mask, kl_coef=0.1,
                        reduction="sequence")
        return [a.loss.detach(), a.chosen, b.loss.detach(), b.kl, b.clipped,
                *torch.autograd.grad(a.loss + b.loss, logp)]
    captured = CapturedStep(step)
    for _ in range(3):
        with torch.no_grad():
            logp.copy_(-torch.rand(shape, device="cuda"))
        out = [t.clone() for t in captured()]
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(out, there))


@pytest.mark.parametrize("shift", [1e-6, 1e-3, 0.1, 0.9, 1.5])
def test_policy_kl_of_close_models(cuda_device, shift):
    """exp(s) - s - 1 and its gradient keep their digits where they are small."""
    g = gen(17)
    # multiples of 2^-22 up to 2: sums and differences are exact
    grid = lambda t: (t * 2.0 ** 22).round() * 2.0 ** -22
    logp = grid(-0.5 * torch.rand(6, 500, generator=g, device="cuda"))
    ref = logp + grid(shift * torch.randn(6, 500, generator=g, device="cuda").clamp(-1, 1))
    s = ref.double() - logp.double()
    assert torch.equal((ref - logp).double(), s)
    leaf = logp.clone().requires_grad_(True)
    out = policy_loss(leaf, logp, torch.zeros(6, device="cuda"), ref_logp=ref, kl_coef=1.0)
    dlogp, = torch.autograd.grad(out.loss, leaf)
    k = torch.expm1(s) - s
    # relative, in units of 2^-24: the series 1.5 (its last step and coefficient; the
    # terms before shrink), the square and the product 2, its end 2^-3, the mean's rounding
    # 1; from 1 on exp's 2 of up to 4.5 and two roundings, of a value of 0.37 (s = -1) or
    # 0.72 (s = 1) and more: 16
    within(out.kl, k.mean(), 16 * 2.0 ** -24 * k.mean())
    within(out.loss.detach(), k.mean(), 17 * 2.0 ** -24 * k.mean())
    # k and s add to exp(s) - 1: at s = -1, where they cancel most, 0.37 and 1 leave 0.63, so
    # a relative error of 16 of k is 10 of the sum; its rounding, 1 / n and the products 4
    grad = -torch.expm1(s) / s.numel()
    within(dlogp, grad, 14 * 2.0 ** -24 * grad.abs())


@pytest.mark.parametrize("tokens", [0, 40, 9000])
def test_policy_without_sequences(cuda_device, tokens):
    logp = torch.zeros(0, tokens, device="cuda", requires_grad=True)
    for mask in (None, torch.ones(0, tokens, device="cuda", dtype=torch.bool)):
        for reduction in ("token", "sequence"):
            out = policy_loss(logp, logp.detach(), torch.zeros(0, device="cuda"), mask=mask,
                              reduction=reduction)
            dlogp, = torch.autograd.grad(out.loss, logp)
            assert [float(t.detach()) for t in out] == [0.0, 0.0, 0.0]
            assert dlogp.shape == (0, tokens)


def test_statistics_may_change_before_the_backward(cuda_device):
    """An in-place change of a returned statistic (as an all-reduce makes it) leaves the
    backward as it is."""
    old, ref, logp = (-torch.rand(4, 30, device="cuda") for _ in range(3))
    adv = torch.randn(4, device="cuda")
    logp.requires_grad_(True)
    for call in (lambda: preference_loss(logp, ref),
                 lambda: policy_loss(logp, old, adv, ref_logp=ref, kl_coef=0.1)):
        plain, = torch.autograd.grad(call().loss, logp)
        out = call()
        for t in out[1:]:
            t.mul_(0.5)
        changed, = torch.autograd.grad(out.loss, logp)
        assert torch.equal(changed, plain) and plain.any()
