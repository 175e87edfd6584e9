"""Windowed attention with sinks and the rotation of queries and keys against fp64.

With u half a step of the type (eps / 2): the kernels round the weights P to the type
before P V and the output once, so

    |out - ref| <= 2 (u P|V| + u |ref| + tiny)

(twice those terms, the second half for fp32 scores, exponentials and sums: below 2^-14 of them
at these sizes, against u >= 2^-11).  Backward: P and dS are rounded, D = sum dO O is
taken of the rounded output (off by at most u (P|V| + |O|) an element), and the gradients
are rounded once:

    |ddS| <= u |dS| + P u sum |dO| (P|V| + |O|)
    |ddV| <= 2 (u P^T |dO| + u |dV|),  |ddQ| <= 2 (s |ddS| |K| + u |dQ|),  dK alike

tiny and the subnormal terms: half the type's smallest number per P or dS.
"""
from __future__ import annotations

import math

import pytest
import torch

from reversability_amd import attention
from reversability_amd.attention import Rotary, rotate_qkv, window_attention

pytestmark = pytest.mark.gpu

CASES = [  # batch, seq, heads, kv, hd, window, sinks
    (1, 1, 1, 1, 32, 1, 0),
    (2, 77, 8, 8, 32, 32, 4),
    (1, 130, 4, 2, 64, 1, 0),      # a token sees itself alone
    (1, 129, 4, 1, 64, 64, 1),
    (2, 300, 6, 2, 128, 100, 7),
    (1, 700, 3, 3, 64, 65, 130),   # sinks of more than one block of keys
    (1, 513, 2, 1, 128, 200, 600),  # sinks beyond the sequence: causal
    (1, 1000, 10, 2, 64, 1, 3),
    (1, 2053, 2, 1, 32, 5000, 0),  # a window beyond the sequence
    (3, 640, 5, 5, 128, 128, 64),
    (1, 1500, 16, 2, 32, 96, 2),
]


def make(batch, seq, heads, kv, hd, dtype, device, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    qkv = spread * torch.randn(batch, seq, (heads + 2 * kv) * hd, generator=g)
    dout = torch.randn(batch, seq, heads * hd, generator=g)
    return qkv.to(dtype).to(device), dout.to(dtype).to(device)


def sight(seq, window, sinks, device):
    i = torch.arange(seq, device=device)
    gap = i[:, None] - i
    return (gap >= 0) & ((gap < window) | (i < sinks))


def reference(qkv, dout, heads, kv, window, sinks):
    """fp64 output and gradient with their bounds, [batch, seq, ...]."""
    batch, seq, width = qkv.shape
    hd = width // (heads + 2 * kv)
    u = torch.finfo(qkv.dtype).eps / 2
    sub = torch.finfo(qkv.dtype).smallest_normal * torch.finfo(qkv.dtype).eps / 2
    s = 1 / math.sqrt(hd)
    x = qkv.double().view(batch, seq, heads + 2 * kv, hd).transpose(1, 2)
    group = heads // kv
    q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    k, v = (t.repeat_interleave(group, 1).contiguous() for t in (k, v))
    do = dout.double().view(batch, seq, heads, hd).transpose(1, 2).contiguous()
    score = (q @ k.transpose(2, 3).contiguous()) * s
    p = torch.softmax(score.masked_fill(~sight(seq, window, sinks, qkv.device), -math.inf), -1)
    out = p @ v
    pv = p @ v.abs()
    n = (p > 0).sum(-1, keepdim=True)
    out_tol = 2 * (u * pv + u * out.abs() + sub * (1 + n * v.abs().amax()))
    pt = p.transpose(2, 3).contiguous()
    dp = do @ v.transpose(2, 3).contiguous()
    ds = p * (dp - (do * out).sum(-1, keepdim=True))
    ds_tol = u * ds.abs() + p * u * (do.abs() * (pv + out.abs())).sum(-1, keepdim=True) + (
        sub * (p > 0))
    dq, dv, dk = s * (ds @ k), pt @ do, s * (ds.transpose(2, 3).contiguous() @ q)
    dq_tol = s * (ds_tol @ k.abs())
    dk_tol = s * (ds_tol.transpose(2, 3).contiguous() @ q.abs())
    dv_tol = u * (pt @ do.abs()) + sub * ((pt > 0).double() @ do.abs())

    def share(t):
        return t.view(batch, kv, group, seq, hd).sum(2)
    grad = torch.cat([dq, share(dk), share(dv)], 1)
    tol = 2 * (torch.cat([dq_tol, share(dk_tol), share(dv_tol)], 1) + u * grad.abs() + sub)
    pack = lambda t: t.transpose(1, 2).reshape(batch, seq, -1)
    return pack(out), pack(out_tol), pack(grad), pack(tol)


def worst(got, ref, tol):
    return float(((got.double() - ref).abs() / tol).max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch,seq,heads,kv,hd,window,sinks", CASES)
def test_forward_and_backward(cuda_device, batch, seq, heads, kv, hd, window, sinks, dtype):
    qkv, dout = make(batch, seq, heads, kv, hd, dtype, cuda_device, seed=seq)
    out_ref, out_tol, grad_ref, grad_tol = reference(qkv, dout, heads, kv, window, sinks)
    x = qkv.requires_grad_(True)
    out = window_attention(x, heads, window, sinks, kv_heads=kv)
    assert out.dtype == dtype and out.shape == dout.shape
    first = worst(out, out_ref, out_tol)
    print(f"  forward {first:.3f} of the bound", flush=True)
    assert first <= 1.0
    grad, = torch.autograd.grad(out, x, dout)
    second = worst(grad, grad_ref, grad_tol)
    print(f"  backward {second:.3f} of the bound", flush=True)
    assert second <= 1.0
    again = window_attention(x, heads, window, sinks, kv_heads=kv)
    assert torch.equal(again, out)
    assert torch.equal(torch.autograd.grad(again, x, dout)[0], grad)


def test_gradient_against_differences(cuda_device):
    """d loss / d qkv along a random direction, by central differences in fp64 of the formula."""
    qkv, dout = make(1, 150, 4, 2, 32, torch.float16, cuda_device, seed=3)
    x = qkv.requires_grad_(True)
    grad, = torch.autograd.grad(window_attention(x, 4, 20, 2, kv_heads=2), x, dout)
    g = torch.Generator().manual_seed(4)
    step = torch.randn(qkv.shape, generator=g).double().to(cuda_device)

    def loss(h):
        y = (qkv.detach().double() + h * step).view(1, 150, 8, 32).transpose(1, 2)
        q, k, v = y[:, :4], *(t.repeat_interleave(2, 1) for t in (y[:, 4:6], y[:, 6:]))
        s = (q @ k.transpose(2, 3).contiguous()) / math.sqrt(32)
        p = torch.softmax(s.masked_fill(~sight(150, 20, 2, qkv.device), -math.inf), -1)
        return ((p @ v).transpose(1, 2).reshape(1, 150, -1) * dout.double()).sum()
    want = float((loss(1e-4) - loss(-1e-4)) / 2e-4)
    got = float((grad.double() * step).sum())
    _, _, _, tol = reference(qkv.detach(), dout, 4, 2, 20, 2)
    assert abs(got - want) <= float((tol * step.abs()).sum()) + 1e-6 * abs(want)


def test_strided_and_misaligned_operands(cuda_device):
    qkv, dout = make(2, 90, 4, 2, 64, torch.bfloat16, cuda_device)
    want = window_attention(qkv, 4, 30, 2, kv_heads=2)
    wide = torch.full((2, 90, 8 * 64 + 3), float("nan"), device=cuda_device, dtype=qkv.dtype)
    wide[..., 3:] = qkv
    assert torch.equal(window_attention(wide[..., 3:], 4, 30, 2, kv_heads=2), want)
    turned = qkv.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(window_attention(turned, 4, 30, 2, kv_heads=2), want)
    x = qkv.requires_grad_(True)
    grad, = torch.autograd.grad(window_attention(x, 4, 30, 2, kv_heads=2), x, dout)
    sparse = torch.zeros(2, 90, 512, device=cuda_device, dtype=qkv.dtype)[..., ::2]
    sparse.copy_(dout)
    got, = torch.autograd.grad(window_attention(x, 4, 30, 2, kv_heads=2), x, sparse)
    assert torch.equal(got, grad)


def test_empty_batch(cuda_device):
    for shape in ((0, 5, 96), (2, 0, 96)):
        x = torch.zeros(shape, device=cuda_device, dtype=torch.float16, requires_grad=True)
        out = window_attention(x, 1, 3)
        out.sum().backward()
        assert out.shape == (*shape[:2], 32) and x.grad.shape == shape


def test_window_of_everything_is_causal_attention(cuda_device):
    qkv, dout = make(2, 500, 4, 4, 64, torch.float16, cuda_device)
    out = window_attention(qkv, 4, 500)
    ref, tol, _, _ = reference(qkv, dout, 4, 4, 500, 0)
    causal = attention.causal_attention(qkv, 4)
    assert float(((out.double() - causal.double()).abs() / (2 * tol)).max()) <= 1.0


def test_large_scores(cuda_device):
    """Scores of +-10^3: single tokens take whole rows."""
    qkv, dout = make(1, 400, 2, 2, 64, torch.float16, cuda_device, spread=6.0)
    qkv[..., :256] *= 4
    ref, tol, _, _ = reference(qkv, dout, 2, 2, 50, 3)
    # the fp32 scores are off by 64 products of up to 2^9, 2^-24 of each: 2^-9 in the exponent
    out = window_attention(qkv, 2, 50, 3)
    assert torch.isfinite(out).all()
    assert float(((out.double() - ref).abs() / (tol + 2 ** -8 * qkv.abs().max())).max()) <= 1.0


def test_another_stream(cuda_device):
    qkv, dout = make(2, 300, 4, 2, 64, torch.float16, cuda_device)
    x = qkv.requires_grad_(True)
    want = window_attention(x, 4, 40, 2, kv_heads=2)
    grad, = torch.autograd.grad(want, x, dout)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = window_attention(x, 4, 40, 2, kv_heads=2)
        got, = torch.autograd.grad(out, x, dout)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want) and torch.equal(got, grad)


def test_captured(cuda_device):
    """Forward and backward in a graph, replayed with other inputs."""
    base, dout = make(1, 600, 6, 2, 64, torch.bfloat16, cuda_device)
    x = base.clone().requires_grad_(True)

    def step():
        out = window_attention(x, 6, 100, 4, kv_heads=2)
        return out, torch.autograd.grad(out, x, dout)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        fresh, _ = make(1, 600, 6, 2, 64, torch.bfloat16, cuda_device, seed=seed + 5)
        with torch.no_grad():
            x.copy_(fresh)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        y = fresh.requires_grad_(True)
        out = window_attention(y, 6, 100, 4, kv_heads=2)
        grad, = torch.autograd.grad(out, y, dout)
        assert torch.equal(held[0], out) and torch.equal(held[1], grad)


def test_refusals(cuda_device):
    qkv, _ = make(1, 8, 4, 2, 32, torch.float16, cuda_device)
    for bad in (dict(qkv=qkv.float()), dict(qkv=qkv[0]), dict(heads=3), dict(kv_heads=3),
                dict(qkv=qkv[..., :-32]), dict(window=0), dict(sinks=-1)):
        with pytest.raises(ValueError):
            window_attention(**{**dict(qkv=qkv, heads=4, window=3, sinks=1, kv_heads=2), **bad})
    x = qkv.clone().requires_grad_(True)
    grad, = torch.autograd.grad(window_attention(x, 4, 3, kv_heads=2).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):  # no second derivative
        grad.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(qkv, torch.ones_like(qkv))
        with pytest.raises((RuntimeError, NotImplementedError)):
            window_attention(dual, 4, 3, kv_heads=2)
    rotary = Rotary(32, 8, device=cuda_device)
    positions = torch.zeros(1, 8, device=cuda_device, dtype=torch.int32)
    for bad in (dict(rotary=Rotary(64, 8, device=cuda_device)), dict(positions=positions.long()),
                dict(positions=positions[0]), dict(positions=positions.cpu()),
                dict(rotary=Rotary(32, 8, device="cpu")), dict(rotary=Rotary(
                    32, 7, device=cuda_device))):
        with pytest.raises(ValueError):
            rotate_qkv(**{**dict(qkv=qkv, heads=4, rotary=rotary, kv_heads=2), **bad})


def test_gradients_of_a_frozen_input_and_twice(cuda_device):
    """Without gradients the same values; two backward passes through one graph agree."""
    qkv, dout = make(2, 200, 4, 2, 64, torch.float16, cuda_device)
    with torch.no_grad():
        frozen = window_attention(qkv, 4, 30, 2, kv_heads=2)
    x = qkv.clone().requires_grad_(True)
    out = window_attention(x, 4, 30, 2, kv_heads=2)
    assert torch.equal(out, frozen)
    first, = torch.autograd.grad(out, x, dout, retain_graph=True)
    second, = torch.autograd.grad(out, x, dout)
    assert torch.equal(first, second)


@pytest.mark.parametrize("hd", [64, 128])
def test_many_sequences_are_as_few(cuda_device, hd):
    """A batch whose queries are launched in two parts: each sequence as in a smaller batch."""
    heads, kv, seq, window, sinks = 6, 2, 300, 70, 3
    qkv, dout = make(80, seq, heads, kv, hd, torch.float16, cuda_device, seed=3)

    def grads(first, last):
        x = qkv[first:last].detach().clone().requires_grad_(True)
        out = window_attention(x, heads, window, sinks, kv_heads=kv)
        return out.detach(), torch.autograd.grad(out, x, dout[first:last].contiguous())[0]
    out, got = grads(0, 80)
    own = slice(0, heads * hd)
    for first in range(0, 80, 20):
        few, part = grads(first, first + 20)
        assert torch.equal(out[first:first + 20], few)
        assert torch.equal(got[first:first + 20, :, own], part[:, :, own])
    rows = torch.tensor([0, 41, 79], device=cuda_device)
    out_ref, out_tol, ref, tol = reference(qkv.detach()[rows], dout[rows], heads, kv, window, sinks)
    assert worst(out[rows], out_ref, out_tol) <= 1.0
    assert worst(got[rows], ref, tol) <= 1.0


def test_long_sequences_and_sinks(cuda_device):
    """Sinks summed over many queries keep their digits: errors as on short sequences."""
    heads, kv, hd, window, sinks = 2, 1, 64, 128, 3
    qkv, dout = make(1, 9000, heads, kv, hd, torch.bfloat16, cuda_device, seed=5)
    x = qkv.requires_grad_(True)
    out = window_attention(x, heads, window, sinks, kv_heads=kv)
    got, = torch.autograd.grad(out, x, dout)
    out_ref, out_tol, ref, tol = reference(qkv.detach(), dout, heads, kv, window, sinks)
    assert worst(out, out_ref, out_tol) <= 1.0
    assert worst(got, ref, tol) <= 1.0
    # of the sinks' keys and values the roundings of P and dS are made up for: what is left is the
    # final rounding, D's (its output kept twice: 2^-16 of it) and fp32 sums of 9000 terms
    u = torch.finfo(torch.bfloat16).eps / 2
    part = slice(heads * hd, None)
    left = (got[0, :sinks, part].double() - ref[0, :sinks, part]).abs()
    loose = tol[0, :sinks, part]  # 2 (u of every term + u of the sum): u^2 of the terms stay
    bound = u * ref[0, :sinks, part].abs() + 4 * u * loose + 2 ** -14 * loose
    assert float((left / bound).max()) <= 1.0


# ---------------------------------------------------------------------------
# rotation
# ---------------------------------------------------------------------------
def turned(x, positions, base, interleaved, sign=1.0):
    """x [..., heads, hd] in fp64 turned by positions [...]."""
    half = x.shape[-1] // 2
    angle = positions.double()[..., None, None] * base ** (
        -torch.arange(half, device=x.device, dtype=torch.float64) / half)
    cos, sin = angle.cos(), sign * angle.sin()
    x = x.double()
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    y = (a * cos - b * sin, a * sin + b * cos)
    size = (a.abs() * cos.abs() + b.abs() * sin.abs(), a.abs() * sin.abs() + b.abs() * cos.abs())
    join = (lambda t: torch.stack(t, -1).flatten(-2)) if interleaved else (
        lambda t: torch.cat(t, -1))
    return join(y), join(size)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("batch,seq,heads,kv,hd", [(1, 1, 1, 1, 32), (2, 33, 6, 2, 64),
                                                   (1, 130, 5, 5, 128)])
def test_rotation(cuda_device, batch, seq, heads, kv, hd, interleaved, dtype):
    """One rounding to the type, and fp32 products, sums and table: 4 x 2^-24 of the terms."""
    qkv, _ = make(batch, seq, heads, kv, hd, dtype, cuda_device, seed=seq)
    grad, _ = make(batch, seq, heads, kv, hd, dtype, cuda_device, seed=seq + 1)
    rotary = Rotary(hd, 100_001, interleaved=interleaved, device=cuda_device)
    g = torch.Generator().manual_seed(7)
    far = torch.randint(0, 100_001, (batch, seq), generator=g, dtype=torch.int32).to(cuda_device)
    far[-1, -1] = 100_000
    u = torch.finfo(dtype).eps / 2
    sub = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    for positions in (None, far):
        at = (torch.arange(seq, device=cuda_device).expand(batch, seq) if positions is None
              else positions)
        x = qkv.clone().requires_grad_(True)
        out = rotate_qkv(x, heads, rotary, positions, kv_heads=kv)
        back, = torch.autograd.grad(out, x, grad)
        for got, source, sign in ((out, qkv, 1.0), (back, grad, -1.0)):
            got, source = (t.detach().view(batch, seq, heads + 2 * kv, hd) for t in (got, source))
            assert torch.equal(got[:, :, heads + kv:], source[:, :, heads + kv:])
            ref, size = turned(source[:, :, :heads + kv], at, 10000.0, interleaved, sign)
            tol = u * ref.abs() + 4 * 2 ** -24 * size + sub
            assert worst(got[:, :, :heads + kv], ref, tol) <= 1.0


def test_rotation_outside_its_table(cuda_device):
    qkv, _ = make(1, 4, 2, 2, 32, torch.float16, cuda_device)
    rotary = Rotary(32, 10, device=cuda_device)
    positions = torch.tensor([[3, 10, -1, 9]], device=cuda_device, dtype=torch.int32)
    out = rotate_qkv(qkv, 2, rotary, positions).view(4, 6, 32)
    assert out[1:3, :4].isnan().all() and not out[1:3, 4:].isnan().any()
    assert not out[0].isnan().any() and not out[3].isnan().any()
    with pytest.raises(ValueError, match="positions of the Rotary table"):
        rotate_qkv(qkv.new_zeros(1, 11, 192), 2, rotary)


def test_rotation_of_nothing_and_strides(cuda_device):
    rotary = Rotary(32, 64, device=cuda_device)
    empty = torch.zeros(2, 0, 192, device=cuda_device, dtype=torch.float16, requires_grad=True)
    rotate_qkv(empty, 2, rotary).sum().backward()
    assert empty.grad.shape == empty.shape
    qkv, _ = make(2, 40, 2, 2, 32, torch.float16, cuda_device)
    want = rotate_qkv(qkv, 2, rotary)
    assert torch.equal(rotate_qkv(qkv.transpose(0, 1).contiguous().transpose(0, 1), 2, rotary),
                       want)


# ---------------------------------------------------------------------------
# a model trained with them
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("method", ["baseline", "midpoint", "euler"])
@pytest.mark.parametrize("rotated", [False, True])
def test_enable_attention_trains_with_a_window(cuda_device, method, rotated):
    """The model under fp16 autocast against itself in torch operations (fp32, no autocast):
    gradients agree to fp16's precision."""
    import copy

    from reversability_amd import build_model, paths
    config = {"model": {"vocab_size": 97, "max_sequence_length": 160, "n_layers": 2, "n_heads": 4,
                        "d_model": 128, "d_ff": 256}, "method": method}
    torch.manual_seed(5)
    model = build_model(config).to(cuda_device)
    plain = copy.deepcopy(model)
    rotary = Rotary(32, 160, device=cuda_device) if rotated else None
    for m in (model, plain):
        attention.enable_attention(m, window=24, sinks=2, rotary=rotary)
    ids = torch.randint(0, 97, (2, 130), device=cuda_device)
    paths.reset()
    with torch.autocast("cuda", dtype=torch.float16):
        loss = torch.nn.functional.cross_entropy(model(ids).flatten(0, 1).float(), ids.flatten())
    (1024 * loss).backward()
    assert paths.report()["attention"].keys() == {"hip"}
    loss64 = torch.nn.functional.cross_entropy(plain(ids).flatten(0, 1), ids.flatten())
    loss64.backward()
    assert abs(float(loss) - float(loss64)) <= 2e-3 * float(loss64)
    for (name, a), b in zip(model.named_parameters(), plain.parameters()):
        rel = float((a.grad / 1024 - b.grad).norm() / b.grad.norm())
        assert rel <= 2e-2, (name, rel)


def test_enable_attention_without_window_is_as_before(cuda_device):
    from reversability_amd import build_model
    config = {"model": {"vocab_size": 97, "max_sequence_length": 64, "n_layers": 1, "n_heads": 4,
                        "d_model": 128, "d_ff": 256}, "method": "baseline"}
    model = build_model(config).to(cuda_device)
    ids = torch.randint(0, 97, (2, 64), device=cuda_device)
    with torch.autocast("cuda", dtype=torch.float16), torch.no_grad():
        attention.enable_attention(model)
        before = model(ids)
        attention.enable_attention(model, window=8)
        windowed = model(ids)
        attention.enable_attention(model)
        after = model(ids)
    assert torch.equal(before, after) and not torch.equal(before, windowed)
