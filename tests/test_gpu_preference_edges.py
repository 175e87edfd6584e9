"""Edges of the log-probabilities and the policy loss: not-a-numbers and infinities in the
head, against 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

from reversability_amd.preference import policy_loss, tied_head_logprobs

pytestmark = pytest.mark.gpu


def operands(rows, d, vocab, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    head = torch.zeros(-(-vocab // 64) * 64, d, device="cuda", dtype=dtype)
    head[:vocab] = (torch.randn(vocab, d, generator=g, device="cuda") / math.sqrt(d)).to(dtype)
    x = torch.randn(rows, d, generator=g, device="cuda").to(dtype)
    labels = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    if rows > 2:
        labels[2] = -100
    return x, head, labels


# both sides of width 256, of 64 and 128 rows, and enough tiles for 256 x 256 ones
NAN_SIZES = [(5, 512, 321), (100, 512, 321), (700, 264, 321), (9, 1024, 50257),
             (300, 512, 50257), (2100, 512, 12305), (5, 256, 321), (300, 64, 12305)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,d,vocab", NAN_SIZES)
def test_nan_in_a_row_of_the_head_reaches_every_token(cuda_device, rows, d, vocab, dtype):
    """A logit that is no number leaves no log-probability of its row a number: in the
    first columns, the last whole block of them, and alone among padding."""
    x, head, labels = operands(rows, d, vocab, dtype)
    assert bool(tied_head_logprobs(x, head, vocab, labels).isfinite().all())
    scored = labels != -100
    for first, last in ((0, 1), (vocab // 2, vocab // 2 + 1), (vocab - 1, vocab),
                        (vocab - 17, vocab), (0, vocab)):
        broken = head.clone()
        broken[first:last] = math.nan
        logp = tied_head_logprobs(x, broken, vocab, labels)
        assert bool(logp[scored].isnan().all()) and not logp[~scored].any(), (first, last)
    # behind the vocabulary it reaches nothing
    broken = head.clone()
    broken[vocab:] = math.nan
    assert torch.equal(tied_head_logprobs(x, broken, vocab, labels),
                       tied_head_logprobs(x, head, vocab, labels))


@pytest.mark.parametrize("rows,d,vocab", NAN_SIZES)
def test_infinite_logits(cuda_device, rows, d, vocab):
    """A head row of an infinity: a logit of -inf counts for nothing, one of +inf leaves
    its row without a log-probability."""
    x, head, labels = operands(rows, d, vocab, torch.bfloat16, seed=1)
    at = min(vocab - 1, 320)
    head[at] = 0
    head[at, 3] = math.inf
    head[vocab - 1, 5] = -math.inf
    x[:, 3] = x[:, 3].abs() + 1
    x[::2, 3] *= -1
    x[:, 5] = x[:, 5].abs() + 1
    logp = tied_head_logprobs(x, head, vocab, labels).double()
    z = x.double() @ head[:vocab].double().t()
    ref = z.log_softmax(1).gather(1, labels.clamp_min(0)[:, None])[:, 0]
    ref = torch.where(labels == -100, 0.0, ref)
    assert torch.equal(logp.isnan(), ref.isnan())
    assert torch.equal(logp.isinf(), ref.isinf())
    ok = ref.isfinite()
    assert bool(((logp - ref)[ok].abs() <= 1e-3).all())  # fp32 sums of d products: below 1e-4


@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_kl_gradient_of_tokens_far_from_the_reference(cuda_device, sign):
    """d/dlogp of exp(s) - s - 1, s = ref - logp, is 1 - exp(s): no difference of large
    numbers.  In units of 2^-24 of it: expf 2 of exp(s), which is at most 0.59 (s <= -1)
    or 1.59 (s >= 1) times the value; the subtraction, 1 / n, its product and the
    coefficient's 1 each: 7.2 at most."""
    g = torch.Generator(device="cuda").manual_seed(3)
    # multiples of 2^-16 up to 128: sums and differences are exact
    grid = lambda t: (t * 2.0 ** 16).round() * 2.0 ** -16
    logp = grid(-40 * torch.rand(6, 500, generator=g, device="cuda"))
    ref = logp + sign * grid(1 + 39 * torch.rand(6, 500, generator=g, device="cuda"))
    s = ref.double() - logp.double()
    assert torch.equal((ref - logp).double(), s)
    leaf = logp.clone().requires_grad_(True)
    out = policy_loss(leaf, logp, torch.zeros(6, device="cuda"), ref_logp=ref, kl_coef=1.0)
    dlogp, = torch.autograd.grad(out.loss, leaf)
    grad = -torch.expm1(s) / s.numel()
    assert bool(((dlogp.double() - grad).abs() <= 8 * 2.0 ** -24 * grad.abs()).all())


def test_kl_gradient_of_an_impossible_reference(cuda_device):
    """A reference probability of 0: an infinite term whose gradient is the coefficient."""
    logp = torch.tensor([[-1.0, -2.0]], device="cuda", requires_grad=True)
    out = policy_loss(logp, logp.detach(), torch.zeros(1, device="cuda"), kl_coef=0.5,
                      ref_logp=torch.tensor([[-math.inf, -2.0]], device="cuda"))
    out.loss.backward()
    assert float(out.loss.detach()) == float(out.kl) == math.inf
    assert logp.grad.tolist() == [[0.25, 0.0]]


@pytest.mark.parametrize("reduction", ["token", "sequence"])
def test_kl_as_a_statistic_alone(cuda_device, reduction):
    """A reference with a coefficient of 0: its KL estimate is returned, and an infinite
    one (s = 100) leaves the loss and its gradient as they are without it."""
    g = torch.Generator(device="cuda").manual_seed(4)
    old = -torch.rand(3, 50, generator=g, device="cuda")
    old[1, 7] = -101.0
    ref = old.clone()
    ref[1, 7] = -1.0
    adv = torch.randn(3, generator=g, device="cuda")
    logp, plain = (old.clone().requires_grad_(True) for _ in range(2))
    out = policy_loss(logp, old, adv, ref_logp=ref, reduction=reduction)
    bare = policy_loss(plain, old, adv, reduction=reduction)
    assert float(out.kl) == math.inf and torch.equal(out.loss, bare.loss)
    out.loss.backward()
    bare.loss.backward()
    assert torch.equal(logp.grad, plain.grad) and bool(logp.grad.isfinite().all())


# up to 512 rows and more, both sides of width 256, products in one piece and split
APART_SIZES = [(9, 256, 5000), (300, 512, 5000), (600, 128, 20000), (700, 640, 8000),
               (2100, 512, 12305), (20000, 64, 500)]


@pytest.mark.parametrize("few", [False, True])
@pytest.mark.parametrize("rows,d,vocab", APART_SIZES)
def test_gradients_of_tokens_far_apart(cuda_device, rows, d, vocab, few):
    """fp16, token gradients over 2^30: a small one's input gradient is its own, not what a
    larger one's scale leaves of it (the softmax's part takes most of the label's away
    here: the head's rows are much alike).  ``few``: one token is large, the others
    2^-24 of it and less.

    A logit's gradient is off by u of it and, in fp16's last range, by half a step at the scale
    that brings its token's gradient to 2^14 or more: 2^-39 of that; by its exponential's
    argument, d 2^-24 and a few more units of sum |x w|; the sums of n products by n
    2^-24.  The head's gradient takes x at a scale of the token too: off by 2^-25 where the
    largest |g| max|x| is at 2^28 or more, times a logit gradient of up to 2^15: by
    2^-38 of that largest one, times dz / g."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    u = 2.0 ** -11
    head = torch.zeros(-(-vocab // 64) * 64, d, device="cuda", dtype=torch.float16)
    head[:vocab] = 0.25 + 0.05 * torch.randn(vocab, d, generator=g, device="cuda")
    x = (torch.randn(rows, d, generator=g, device="cuda") / math.sqrt(d)).half()
    labels = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    labels[rows // 2] = -100
    low = 24 * torch.ones(rows, device="cuda") if few else torch.zeros(rows, device="cuda")
    grad = 2.0 ** (15 - low - (6 if few else 30) * torch.rand(rows, generator=g, device="cuda"))
    grad[0] = 2.0 ** 15
    grad[rows // 2] = 2.0 ** 30  # not scored: not looked at
    x.requires_grad_(True)
    head.requires_grad_(True)
    dx, dhead = torch.autograd.grad(tied_head_logprobs(x, head, vocab, labels), (x, head), grad)
    xd, w = x.detach().double(), head.detach()[:vocab].double()
    on = labels != -100
    gd = (grad.double() * on)[:, None]
    z = xd @ w.t()
    p = z.softmax(1)
    share = -p  # dz / g
    share.scatter_add_(1, labels.clamp_min(0)[:, None], torch.ones_like(gd))
    argument = (2 * d + 8) * 2.0 ** -24 * (xd.abs() @ w.abs().t()).amax(1, keepdim=True) + 2.0 ** -14
    off = share.abs() * u + p * argument + 2.0 ** -39
    rx = gd * (share @ w)
    bx = gd.abs() * (off @ w.abs() + vocab * 2.0 ** -24 * (share.abs() @ w.abs()))
    bx += u * rx.abs() + 2.0 ** -25
    assert bool(((dx.double() - rx).abs() <= bx).all()), float(((dx.double() - rx).abs() / bx).max())
    rh = (gd * share).t() @ xd
    largest = float((gd[:, 0].abs() * xd.abs().amax(1)).max())
    bh = (gd.abs() * off).t() @ xd.abs() + rows * 2.0 ** -24 * ((gd * share).abs().t() @ xd.abs())
    bh += largest * 2.0 ** -38 * share[on].abs().sum(0)[:, None] + u * rh.abs() + 2.0 ** -25
    assert bool(((dhead[:vocab].double() - rh).abs() <= bh).all())
    assert not dx[rows // 2].any() and not dhead[vocab:].any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,d,vocab", NAN_SIZES)
def test_columns_masked_with_the_lowest_value(cuda_device, rows, d, vocab, dtype):
    """A vocabulary whose first columns, and one in five of the others, are masked by the
    type's lowest value (times a constant input): as if they were not there, also
    for the gradients of the others, and a masked label's log-probability is as low."""
    x, head, labels = operands(rows, d, vocab, dtype, seed=2)
    masked = torch.rand(vocab, generator=torch.Generator().manual_seed(9)) < 0.2
    masked[:min(256, vocab - 1)] = True
    masked[vocab - 1] = False
    masked = masked.cuda()
    x[:, 1] = 1.0
    head[:vocab, 1] = torch.where(masked, torch.finfo(dtype).min, 0.0).to(dtype)
    kept = (~masked).nonzero()[:, 0]
    place = torch.randint(0, len(kept), (rows,), device="cuda")
    place[min(2, rows - 1)] = 0
    small = -(-len(kept) // 64) * 64
    other = torch.zeros(small, d, device="cuda", dtype=dtype)
    other[:len(kept)] = head[kept]
    a, b = ((t.clone().requires_grad_(True), u.clone().requires_grad_(True))
            for t, u in ((x, head), (x, other)))
    one = tied_head_logprobs(*a, vocab, kept[place])
    two = tied_head_logprobs(*b, len(kept), place)
    assert bool(((one - two).abs() <= 1e-4).all())  # other tiles: sums in another order
    weight = torch.randn(rows, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    got = torch.autograd.grad(one, a, weight)
    ref = torch.autograd.grad(two, b, weight)
    # both sides are rounded twice, and another order moves a rounding: 2^-8 at the most in
    # fp16 and 2^-6 in bf16 of the largest entry
    near = {torch.float16: 2.0 ** -8, torch.bfloat16: 2.0 ** -6}[dtype]
    assert float((got[0] - ref[0]).abs().max()) <= near * float(ref[0].abs().max())
    assert float((got[1][kept] - ref[1][:len(kept)]).abs().max()) <= near * float(ref[1].abs().max())
    assert not got[1][:vocab][masked].any()
    labels[0] = 0
    low = tied_head_logprobs(x, head, vocab, labels)
    assert bool(low.isfinite().all()) and float(low[0]) < 0.99 * torch.finfo(dtype).min


@pytest.mark.parametrize("lowest", [-1.0, 1.0])
@pytest.mark.parametrize("rows,d,vocab", NAN_SIZES)
def test_rows_out_of_range_have_no_log_probability(cuda_device, rows, d, vocab, lowest):
    x, head, labels = operands(rows, d, vocab, torch.bfloat16, seed=2)
    x[:, 1] = 1.0
    head[:vocab, 1] = lowest * torch.finfo(torch.bfloat16).max
    logp = tied_head_logprobs(x, head, vocab, labels)
    assert bool(logp[labels != -100].isnan().all()) and not logp[labels == -100].any()
