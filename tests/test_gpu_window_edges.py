"""Windowed attention's gradients of gradients far below 1, where fp16 has few digits left."""
from __future__ import annotations

import math

import pytest
import torch

from reversability_amd.attention import window_attention
from test_gpu_window import make, sight, worst

pytestmark = pytest.mark.gpu

SMALL = [  # batch, seq, heads, kv, hd, window, sinks
    (1, 1, 1, 1, 32, 1, 0),
    (2, 700, 4, 2, 64, 65, 130),
    (1, 2500, 2, 1, 32, 2500, 0),
    (1, 2100, 4, 2, 128, 900, 3),
    (12, 1100, 8, 2, 64, 300, 4),  # queries in two launches
]


def gradient(qkv, dout, heads, kv, window, sinks):
    x = qkv.detach().clone().requires_grad_(True)
    out = window_attention(x, heads, window, sinks, kv_heads=kv)
    return torch.autograd.grad(out, x, dout)[0]


def parts(qkv, dout, heads, kv, window, sinks):
    """One sequence in fp64, [heads, seq, ..]: q, k, v, dO, P, dS (k and v repeated)."""
    seq, hd, group = len(qkv), qkv.shape[1] // (heads + 2 * kv), heads // kv
    x = qkv.double().view(seq, heads + 2 * kv, hd).transpose(0, 1)
    q = x[:heads].contiguous()
    k, v = (t.repeat_interleave(group, 0).contiguous()
            for t in (x[heads:heads + kv], x[heads + kv:]))
    do = dout.double().view(seq, heads, hd).transpose(0, 1).contiguous()
    score = (q @ k.transpose(1, 2).contiguous()) / math.sqrt(hd)
    p = torch.softmax(score.masked_fill(~sight(seq, window, sinks, x.device), -math.inf), -1)
    dp = do @ v.transpose(1, 2).contiguous()
    return q, k, v, do, p, p * (dp - (do * (p @ v)).sum(-1, keepdim=True))


def turn(t):
    return t.transpose(1, 2).contiguous()


def share(t, kv):
    """The sum over the query heads of a key head."""
    return t.view(kv, -1, *t.shape[1:]).sum(1)


def heads_of(t, hd):
    return t.view(len(t), -1, hd).transpose(0, 1)


@pytest.mark.parametrize("batch,seq,heads,kv,hd,window,sinks", SMALL)
@pytest.mark.parametrize("power", [4, 9, 13])
def test_fp16_gradients_scale(cuda_device, batch, seq, heads, kv, hd, window, sinks, power):
    """The gradient is linear in dO.  Of 2^-power dO, where both are fp16 numbers, it is 2^-power times
    that of dO but for the two final roundings, half a step of each, and

    * in dK for dS: dO v and its sums are taken of fp16 subnormals in one of the calls, whose fp32
      sums may differ in their last digits, and a dS next to a border then rounds to the other
      side, a step of u |dS| * 2 from where it was;
    * in dV for those digits alone (P does not depend on dO): seq terms, 2^-24 of each at most."""
    qkv, dout = make(batch, seq, heads, kv, hd, torch.float16, cuda_device, seed=seq)
    # multiples of 2^-10 with every head's largest at most 1/2 and at least 1/4
    rows = dout.double().view(-1, hd)
    rows = (rows / rows.abs().amax(1, keepdim=True) * 400).round() / 1024
    dout = rows.view(dout.shape).half()
    small = (dout.double() * 2.0 ** -power).half()
    assert torch.equal(small.double() * 2.0 ** power, dout.double())
    whole = gradient(qkv, dout, heads, kv, window, sinks).double()
    got = gradient(qkv, small, heads, kv, window, sinks).double()
    u, least, scale = 2.0 ** -11, 2.0 ** -25, 2.0 ** -power  # half a step, and of subnormals
    for b in range(batch):
        q, _, _, do, p, ds = parts(qkv[b], dout[b], heads, kv, window, sinks)
        dk = 2 * u * (turn(ds.abs()) @ q.abs()) / math.sqrt(hd)
        dv = seq * 2.0 ** -24 * (turn(p) @ do.abs())
        off = torch.cat([torch.zeros_like(q), share(dk, kv), share(dv, kv)]) * scale
        ref, mine = heads_of(whole[b], hd) * scale, heads_of(got[b], hd)
        off = off + u * ref.abs() + least * scale  # (the rounding of ``whole``)
        tol = off + torch.maximum(u * (ref.abs() + off), torch.full_like(ref, least))
        assert worst(mine, ref, tol) <= 1.0


@pytest.mark.parametrize("batch,seq,heads,kv,hd,window,sinks", SMALL)
def test_fp16_gradients_of_unlike_sizes(cuda_device, batch, seq, heads, kv, hd, window, sinks):
    """Stretches of queries and heads whose gradients differ by up to 2^14, against fp64.  P and dS are
    rounded to fp16, dS times a power of two that brings the largest |dO| of a query (in dQ) or of
    64 (in dK) to 1/4 at least (up to 2^15): what is lost of a term below 2^-14 is half a step of 2^-24 over that
    power, thus at most 4 * 2^-25 max |dO|, or 2^-25 * 2^-15."""
    qkv, dout = make(batch, seq, heads, kv, hd, torch.float16, cuda_device, seed=seq)
    g = torch.Generator().manual_seed(8)
    stretches = -(-seq // 37)
    power = -torch.randint(0, 15, (batch, stretches, heads), generator=g).double()
    power = power.repeat_interleave(37, 1)[:, :seq].to(cuda_device)
    dout = (dout.double().view(batch, seq, heads, hd) * 2.0 ** power.unsqueeze(-1))
    dout = dout.view(batch, seq, -1).half()
    got = gradient(qkv, dout, heads, kv, window, sinks)
    u, sub, s = 2.0 ** -11, 2.0 ** -25, 1 / math.sqrt(hd)
    bad = 0.0
    for b in range(batch):
        q, k, v, do, p, ds = parts(qkv[b], dout[b], heads, kv, window, sinks)
        top = do.abs().amax(-1)
        top64 = torch.nn.functional.pad(top, (0, -seq % 64)).view(heads, -1, 64).amax(-1)
        top64 = top64.repeat_interleave(64, 1)[:, :seq]
        # D is off by the roundings of O and of P in it, each of them u at most
        base = u * ds.abs() + p * u * (do.abs() * (p @ v.abs() + (p @ v).abs())).sum(-1, True)
        few = (p > 0).double()
        lost = lambda largest: base + few * sub * (4 * largest).clamp(2.0 ** -15, 1).unsqueeze(-1)
        grad = [s * (ds @ k), s * (turn(ds) @ q), turn(p) @ do]
        tol = [s * (lost(top) @ k.abs()), s * (turn(lost(top64)) @ q.abs()),
               u * (turn(p) @ do.abs()) + sub * (turn(few) @ do.abs())]
        grad, tol = (torch.cat([t[0], share(t[1], kv), share(t[2], kv)]) for t in (grad, tol))
        tol = 2 * (tol + u * grad.abs() + sub)
        bad = max(bad, worst(heads_of(got[b], hd), grad, tol))
    print(f"  {bad:.3f} of the bound", flush=True)
    assert bad <= 1.0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_large_scores_by_their_roundings(cuda_device, dtype):
    """Scores of up to +-10^3, where single tokens take whole rows.  Beside the roundings of P and of the
    output: a score is a sum in fp32 of hd products, off by d = (hd + 1) 2^-24 sum |q k| s, then of
    2^-22 of its size (times log2 e, less the maximum); weights move with it, and the output by
    sum P (d + its mean) |v - out| in the first order (twice for the rest)."""
    seq, heads, hd, window, sinks = 400, 2, 64, 50, 3
    qkv, _ = make(1, seq, heads, heads, hd, dtype, cuda_device, spread=6.0)
    qkv[..., :2 * heads * hd] *= 4
    out = window_attention(qkv, heads, window, sinks)[0].view(seq, heads, hd).transpose(0, 1).double()
    q, k, v, _, p, _ = parts(qkv[0], torch.zeros_like(qkv[0, :, :heads * hd]), heads, heads, window,
                             sinks)
    s, u = 1 / math.sqrt(hd), torch.finfo(dtype).eps / 2
    sub = torch.finfo(dtype).smallest_normal * u
    score = (q @ turn(k)).abs() * s
    off = (hd + 1) * 2.0 ** -24 * (q.abs() @ turn(k.abs())) * s + 2.0 ** -22 * score
    off = off + (p * off).sum(-1, keepdim=True)
    ref = p @ v
    few = (p > 0).sum(-1, keepdim=True)
    tol = 2 * (u * (p @ v.abs()) + u * ref.abs() + sub * (1 + few * v.abs().amax()))
    for h in range(heads):  # [seq, seq, hd] at a time
        tol[h] += 2 * ((p[h] * off[h]).unsqueeze(-1) * (v[h] - ref[h].unsqueeze(1)).abs()).sum(1)
    print(f"  {worst(out, ref, tol):.3f} of the bound; tolerance at most {float(tol.max()):.4f}",
          flush=True)
    assert worst(out, ref, tol) <= 1.0
