"""GPU parity of FusedAdamW8bit (rv_adamw8_step) with the update written out in torch.

The comparator does the kernel's arithmetic in separate fp32 operations and its
codes in integers; the roundings are the same operation by operation, so codes,
scales and fp32 moments are compared bit for bit.  The parameter's update goes
through other operations on the two sides.  In units of 2^-24 of it, the kernel:
square root 1, the correction's reciprocal 1 and the product with it 1, eps 1, v_rcp_f32
2 (1 ulp), the products with m and the learning rate 1 and 1, the learning rate's
own rounding 1; torch: square root, division, eps, division, product 1 each.  14 in
all, 7 x 2^-23 of the update, and two roundings of the parameter.  Against 64 bits: a stored moment is off by at most half a step of e4m3
(2^-4 of the value, or 2^-10 of the block's unit below its smallest normal number)
for exp_avg and by less than a whole one for exp_avg_sq.
"""
from __future__ import annotations

import copy
import math

import pytest
import torch

from reversability_amd.graph import CapturedStep
from reversability_amd.optim import FusedAdamW, FusedAdamW8bit

pytestmark = pytest.mark.gpu

BLOCK = 32
SHAPES = [(33,), (64, 96), (1, 1), (1031, 7), (4096,), (257,), (31,), (2, 50001)]
BETAS, LR, DECAY, EPS = (0.9, 0.95), 1e-2, 0.1, 1e-8


def mix(h):
    h = (h ^ (h >> 16)) * 0x85EBCA6B & 0xFFFFFFFF
    h = (h ^ (h >> 13)) * 0xC2B2AE35 & 0xFFFFFFFF
    return h ^ (h >> 16)


def blocks_of(t):
    flat = t.reshape(-1)
    return torch.nn.functional.pad(flat, (0, -flat.numel() % BLOCK)).view(-1, BLOCK)


def scale_of(t):
    """The scale byte of each block of an fp32 tensor."""
    t = torch.where(torch.isfinite(t), t, 0.0).abs()
    return ((blocks_of(t).amax(1).view(torch.int32) >> 23) - 7).clamp_min(0)


def scaled(t, byte):
    """t in its blocks' units, exactly (fp64)."""
    return blocks_of(t).double() * (127.0 - byte.double()).exp2().unsqueeze(1)


def decode(codes, byte, shape):
    value = blocks_of(codes.float()).double() * (byte.double() - 127).exp2().unsqueeze(1)
    return value.reshape(-1)[:math.prod(shape)].view(shape).float()


def random_codes(v, byte, seed, place, step, first=False):
    """``first``: of the first moment, signed, with a key of its own."""
    q = scaled(v.abs() if first else v, byte).float()
    key = mix((mix((seed + 0x9E3779B9 * (place + 1)) & 0xFFFFFFFF) + step) & 0xFFFFFFFF)
    if first:
        key = mix((key + 0x9E3779B9) & 0xFFFFFFFF)
    index = torch.arange(q.numel(), device=q.device).view_as(q)
    bits = mix(((index >> 1) + key) & 0xFFFFFFFF)
    noise = ((bits >> 16 * (index & 1) & 0xFFFF) << 4 | 8).int()
    normal = ((q.view(torch.int32) + noise) >> 20) - 960
    tiny = (torch.where(q < 1, q, 0.0) * 512 + noise.float() * 2.0 ** -20).int()
    code = torch.where(q < 2.0 ** -6, tiny, normal)
    if not first:
        code = torch.where((code == 0) & (q > 0), 1, code)
    code = torch.where(torch.isfinite(q), code, 0x7F).reshape(-1)[:v.numel()].view(v.shape)
    return code | torch.signbit(v).int() << 7 if first else code


class Plain:
    """The update in separate torch operations, state as the optimizer stores it."""

    def __init__(self, params, seed=0, betas=BETAS, lr=LR, decay=DECAY):
        self.p = [p.clone() for p in params]
        self.seed, self.betas, self.lr, self.decay = seed, betas, lr, decay
        self.step = 0
        self.state = [None] * len(params)

    def update(self, grads):
        self.step += 1
        b1, b2 = self.betas
        for at, (p, g) in enumerate(zip(self.p, grads)):
            if self.state[at] is None:
                m, v = torch.zeros_like(p), torch.zeros_like(p)
            else:
                mc, ms, vc, vs = self.state[at]
                m, v = decode(mc, ms, p.shape), decode(vc, vs, p.shape)
            m = m * b1 + g * (1 - b1)
            v = v * b2 + g * (1 - b2) * g
            # tensor divisors: by a number torch multiplies with its reciprocal
            second = torch.tensor(math.sqrt(1 - b2 ** self.step), device=p.device)
            update = m / (v.sqrt() / second + EPS)
            p.copy_(p * (1 - self.lr * self.decay) - update * (self.lr / (1 - b1 ** self.step)))
            ms, vs = scale_of(m), scale_of(v)
            q = scaled(m, ms).float().reshape(-1)[:m.numel()].view(m.shape)
            mc = torch.where(torch.isfinite(q), q, math.nan).to(torch.float8_e4m3fn)
            if 1 - b1 < 2.0 ** -4:
                mc = random_codes(m, ms, self.seed, at, self.step, first=True).to(
                    torch.uint8).view(torch.float8_e4m3fn)
            vc = random_codes(v, vs, self.seed, at, self.step).to(torch.uint8)
            self.state[at] = (mc, ms, vc.view(torch.float8_e4m3fn), vs)


def make(dev, shapes=SHAPES, **options):
    g = torch.Generator().manual_seed(3)
    params = [(0.02 * torch.randn(*s, generator=g)).to(dev).requires_grad_(True) for s in shapes]
    options = {"lr": LR, "betas": BETAS, "eps": EPS, "weight_decay": DECAY, "min_8bit_numel": 1,
               **options}
    return params, FusedAdamW8bit(params, **options)


def grads_for(params, seed, scale=1e-2):
    """Gradients whose elements differ by orders of magnitude, zeros among them."""
    g = torch.Generator().manual_seed(1000 + seed)
    out = []
    for p in params:
        t = torch.randn(p.shape, generator=g) * scale
        t *= 10.0 ** (-6 * torch.rand(p.shape, generator=g) ** 3)
        t[torch.rand(p.shape, generator=g) < 0.05] = 0
        out.append(t.to(p.device))
    return out


def bits(t):
    return t.reshape(-1).view(torch.uint8).view(*t.shape, -1).squeeze(-1)


def same_state(opt, params, plain):
    for at, p in enumerate(params):
        st, (mc, ms, vc, vs) = opt.state[p], plain.state[at]
        assert st["exp_avg"].dtype == torch.float8_e4m3fn and st["exp_avg"].shape == p.shape
        assert torch.equal(st["exp_avg_scale"].int(), ms.int()), (at, "exp_avg_scale")
        assert torch.equal(st["exp_avg_sq_scale"].int(), vs.int()), (at, "exp_avg_sq_scale")
        m, v = bits(st["exp_avg"]), bits(st["exp_avg_sq"])
        # -0 and 0 are one value
        assert torch.equal(torch.where(m == 0x80, 0, m), torch.where(bits(mc) == 0x80, 0, bits(mc))), at
        assert torch.equal(v, bits(vc)), (at, int((v != bits(vc)).sum()))


@pytest.mark.parametrize("betas,seed", [((0.9, 0.95), 0), ((0.9, 0.999), 12345),
                                        ((0.0, 0.0), 2 ** 32 - 1), ((0.95, 0.99), 9)])
def test_matches_written_out_update(cuda_device, betas, seed):
    params, opt = make(cuda_device, betas=betas, seed=seed)
    plain = Plain([p.detach() for p in params], seed, betas)
    for step in range(4):
        grads = grads_for(params, step)
        before = [p.clone() for p in plain.p]
        for p, g in zip(params, grads):
            p.grad = g
        opt.step()
        plain.update(grads)
        same_state(opt, params, plain)
        for p, q, b in zip(params, plain.p, before):
            eps = 2.0 ** -23
            step_size = (q - b).abs() + LR * DECAY * b.abs()  # at least the update
            bound = 7 * eps * step_size + 2 * eps * torch.maximum(q.abs(), b.abs()) + 1e-38
            assert bool(((p.detach() - q).abs() <= bound).all())
            q.copy_(p.detach())  # the bound is one step's: the next starts from one value


def test_stored_moments_against_64_bits(cuda_device):
    params, opt = make(cuda_device)
    old = [(torch.zeros_like(p).double(), torch.zeros_like(p).double()) for p in params]
    for step in range(3):
        for p, g in zip(params, grads_for(params, step)):
            p.grad = g
        opt.step()
        for at, p in enumerate(params):
            g, (m, v) = p.grad.double(), old[at]
            m = BETAS[0] * m + (1 - BETAS[0]) * g
            v = BETAS[1] * v + (1 - BETAS[1]) * g * g
            got = [t.double() for t in opt.moments(p)]
            units = [(opt.state[p][k].double() - 127).exp2().repeat_interleave(BLOCK)
                     [:p.numel()].view(p.shape) for k in ("exp_avg_scale", "exp_avg_sq_scale")]
            # half a step (and 2^-22 for fp32's own roundings); a whole one for v
            near = torch.maximum(m.abs() * 2.0 ** -4, units[0] * 2.0 ** -10) + m.abs() * 2.0 ** -22
            whole = torch.maximum(v * 2.0 ** -3, units[1] * 2.0 ** -9) + v * 2.0 ** -22
            assert bool(((got[0] - m).abs() <= near).all()) and bool(((got[1] - v).abs() <= whole).all())
            assert bool(((got[1] > 0) | (v < 1e-40)).all())  # a v > 0 stays > 0
            old[at] = got


def test_second_moment_keeps_its_expectation(cuda_device):
    """With beta2 = 0.999 a step moves v by at most 0.1% of it, a hundredth of a step
    of e4m3.  v starts at E[g^2] of one gradient and has to reach that of a four times
    larger one: (1 - 0.999^2000) = 86% of the way, where rounding to nearest does not
    move at all.  The rounding's variance per element: a step of at most v / 8, up
    or down with p (1 - p), p <= 0.008 x 4; summed over 1 / (1 - b2^2) = 500 steps
    sd < 0.36 v, and the mean over 65536 elements within 5 sd / 256 < 1%; twice that."""
    p = torch.zeros(65536, device=cuda_device, requires_grad=True)
    opt = FusedAdamW8bit([p], lr=0.0, betas=(0.9, 0.999), weight_decay=0.0)
    p.grad = torch.full_like(p, 1.0)
    opt.step()
    # every element of v is now 0.001; make it 1
    opt.state[p]["exp_avg_sq_scale"].fill_(127 - 7)
    opt.state[p]["exp_avg_sq"].copy_(torch.full_like(p, 128.0).detach())
    p.grad = torch.full_like(p, 2.0)
    for _ in range(2000):
        opt.step()
    expected = 4 - 3 * 0.999 ** 2000
    assert abs(float(opt.moments(p)[1].mean()) - expected) <= 0.02 * expected


def test_first_moment_keeps_its_expectation(cuda_device):
    """As above for m with beta1 = 0.99, where a zero gradient takes 1% of it a step
    (to nearest nothing): from values of both signs to 0.99^200 = 13% of them.  The
    rounding's variance: a step of at most m / 8, up or down with p (1 - p), p <= 0.16;
    summed over 1 / (1 - b1^2) = 50 steps, with m above the value at the end, sd < 0.33
    times the start; the mean over 32768 elements within 5 sd / 181 < 1% of the start.
    A beta1 at the border of the rule still falls to zero by the nearest values."""
    p = torch.zeros(65536, device=cuda_device, requires_grad=True)
    start = torch.where(torch.arange(65536, device=cuda_device) % 2 == 0, 0.9, -1.1)
    for beta1, steps in ((0.99, 200), (0.9375, 400)):
        opt = FusedAdamW8bit([p], lr=0.0, betas=(beta1, 0.999), weight_decay=0.0)
        p.grad = start / (1 - beta1)
        opt.step()
        p.grad = torch.zeros_like(p)
        for _ in range(steps):
            opt.step()
        m = opt.moments(p)[0].double()
        left = beta1 ** steps
        for at in (0, 1):
            assert abs(float(m[at::2].mean()) - float(start[at]) * left) <= 0.011


def test_specials(cuda_device):
    """NaN and infinities stay in their elements and leave their block's scale alone;
    a zero gradient leaves zeros."""
    p = torch.zeros(96, device=cuda_device, requires_grad=True)
    opt = FusedAdamW8bit([p], lr=LR, betas=BETAS, min_8bit_numel=1)
    g = torch.linspace(0.1, 1, 96)
    g[3], g[40], g[41] = math.nan, math.inf, -math.inf
    g[64:] = 0
    p.grad = g.to(cuda_device)
    opt.step()
    m, v = (t.cpu() for t in opt.moments(p))
    bad = torch.zeros(96, dtype=torch.bool)
    bad[[3, 40, 41]] = True
    assert torch.equal(torch.isnan(m), bad) and torch.equal(torch.isnan(v), bad)
    good = ~bad & (g != 0)
    assert bool(((m - 0.1 * g)[good].abs() <= 0.1 * g[good] * 2.0 ** -4 * 1.001).all())
    assert not m[64:].any() and not v[64:].any() and not p.detach()[64:].any()
    assert bool(torch.isfinite(p.detach().cpu()[~bad]).all())


@pytest.mark.parametrize("magnitude", [1e-30, 1e-22, 1e-12, 1e6, 1e18])
def test_magnitudes(cuda_device, magnitude):
    """Moments of any size fp32 holds: g^2 of 1e-30 and 1e-22 leaves fp32's normal
    range, and so does v's scale byte (0 at the least)."""
    params, opt = make(cuda_device, shapes=[(4096,)])
    plain = Plain([p.detach() for p in params])
    g = torch.Generator().manual_seed(5)
    for step in range(2):
        grad = (torch.rand(4096, generator=g) + 0.5).mul_(magnitude).to(cuda_device)
        params[0].grad = grad
        opt.step()
        plain.update([grad])
    m, _ = opt.moments(params[0])
    assert torch.equal(m, decode(*plain.state[0][:2], (4096,)))
    if 1e-20 < magnitude < 1e18:
        same_state(opt, params, plain)
    assert bool(torch.isfinite(params[0]).all())


def test_unaligned_tensors_match_aligned(cuda_device):
    """A parameter and gradient off a 16-byte boundary, codes off a 4-byte one."""
    n = 5003
    store = [torch.randn(n + 8, device=cuda_device) for _ in range(2)]
    runs = []
    for shift in (0, 1):
        p = torch.empty(n + 8, device=cuda_device)[shift:shift + n]
        p.copy_(store[0][:n])
        p.requires_grad_(True)
        g = torch.empty(n + 8, device=cuda_device)[shift:shift + n]
        g.copy_(store[1][:n])
        p.grad = g
        opt = FusedAdamW8bit([p], lr=LR, betas=BETAS, seed=9)
        opt.step()
        if shift:
            for k in ("exp_avg", "exp_avg_sq"):
                moved = torch.empty(n + 4, device=cuda_device, dtype=torch.uint8)[1:1 + n]
                moved.copy_(bits(opt.state[p][k]))
                opt.state[p][k] = moved.view(torch.float8_e4m3fn)
        opt.step()
        runs.append([p.detach().clone(), *(bits(opt.state[p][k]) for k in (
            "exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale"))])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_small_tensors_and_many_tensors(cuda_device):
    """Tensors below min_8bit_numel take FusedAdamW's update; 100 tensors take more
    than one launch; frozen and gradient-free ones are left alone."""
    shapes = [(4095,), (4096,)] + [(64, 65 + i) for i in range(98)]
    params, opt = make(cuda_device, shapes=shapes, min_8bit_numel=4096)
    other = [p.detach().clone().requires_grad_(True) for p in params]
    fp32 = FusedAdamW(other, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY)
    plain = Plain([p.detach() for p in params])
    untouched = params[7].detach().clone()
    for step in range(2):
        grads = grads_for(params, step)
        for p, q, g in zip(params, other, grads):
            p.grad, q.grad = g, g.clone()
        params[7].grad = None
        opt.step()
        fp32.step()
        plain.update(grads)
    assert torch.equal(params[0], other[0]) and "exp_avg_scale" not in opt.state[params[0]]
    assert torch.equal(opt.state[params[0]]["exp_avg_sq"], fp32.state[other[0]]["exp_avg_sq"])
    assert torch.equal(params[7], untouched) and not opt.state[params[7]]
    for at in (1, 50, 99):
        st = opt.state[params[at]]
        assert torch.equal(bits(st["exp_avg_sq"]), bits(plain.state[at][2]))


def test_gradscaler_overflow_and_clip(cuda_device):
    """An overflow changes nothing; unscale_clip_ multiplies as it does for fp32."""
    params, opt = make(cuda_device)
    scaler = torch.amp.GradScaler("cuda", init_scale=1024.0)
    grads = grads_for(params, 0)
    for p, g in zip(params, grads):
        p.grad = g * 1024
    scaler.scale(torch.zeros((), device=cuda_device))
    norm = opt.unscale_clip_(scaler, 0.5)
    scaler.step(opt)
    scaler.update()
    coef = (torch.full_like(norm, 0.5) / (norm + 1e-6)).clamp(max=1)
    plain = Plain([p.detach() for p in params])
    plain.update([g * coef for g in grads])
    same_state(opt, params, plain)
    before = [p.detach().clone() for p in params]
    states = [{k: t.clone() for k, t in opt.state[p].items()} for p in params]
    params[2].grad.fill_(math.inf)
    opt.unscale_clip_(scaler, 0.5)
    scaler.step(opt)
    scaler.update()
    for p, b, st in zip(params, before, states):
        assert torch.equal(p, b)
        assert all(torch.equal(bits(opt.state[p][k]), bits(t)) for k, t in st.items())


def test_state_dict_round_trip(cuda_device):
    params, opt = make(cuda_device, seed=77, min_8bit_numel=64)
    for p, g in zip(params, grads_for(params, 0)):
        p.grad = g
    opt.step()
    twins = [p.detach().clone().requires_grad_(True) for p in params]
    other = FusedAdamW8bit(twins, lr=1.0, min_8bit_numel=64)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    for step in range(1, 3):
        for p, q, g in zip(params, twins, grads_for(params, step)):
            p.grad, q.grad = g, g.clone()
        opt.step()
        other.step()
    for p, q in zip(params, twins):
        assert torch.equal(p, q)
        assert all(torch.equal(bits(opt.state[p][k]), bits(other.state[q][k]))
                   and opt.state[p][k].dtype == other.state[q][k].dtype for k in opt.state[p])
    with pytest.raises(ValueError, match="8 bits"):
        FusedAdamW(twins).load_state_dict(opt.state_dict())
    # a fp32 run goes on with its fp32 moments
    plain = FusedAdamW(twins)
    plain.step()
    resumed = FusedAdamW8bit(twins, min_8bit_numel=64)
    resumed.load_state_dict(plain.state_dict())
    resumed.step()
    assert all(resumed.state[q]["exp_avg"].dtype == torch.float32 for q in twins)


def test_moments_of_another_size_are_refused(cuda_device):
    """Such a checkpoint (another width or vocabulary) changes nothing."""
    def made(shape):
        p = torch.ones(shape, device=cuda_device, requires_grad=True)
        p.grad = torch.ones_like(p)
        return p, FusedAdamW8bit([p], lr=LR, min_8bit_numel=64)
    small, source = made((40, 64))
    source.step()
    plain = FusedAdamW([small])
    plain.step()
    for state in (source.state_dict(), plain.state_dict()):
        p, opt = made((80, 64))
        with pytest.raises(ValueError, match="shape"):
            opt.load_state_dict(state)
        assert not opt.state[p]
    for key, wrong in (("exp_avg_scale", torch.zeros(79, dtype=torch.uint8)),
                       ("exp_avg_sq", torch.zeros(40, 64))):
        state = copy.deepcopy(source.state_dict())
        state["state"][0][key] = wrong.to(cuda_device)
        with pytest.raises(ValueError, match="8-bit"):
            made((40, 64))[1].load_state_dict(state)


def test_captured_updates_equal_eager_ones(cuda_device):
    """Replays advance the device's step count, and with it the random bits."""
    runs = []
    for captured in (False, True):
        params, opt = make(cuda_device, seed=4)
        for p, g in zip(params, grads_for(params, 0)):
            p.grad = g
        if captured:
            step = CapturedStep(lambda: opt.step(), warmup=1)
            for _ in range(4):
                step()
                torch.randn(1000, device=cuda_device).sum().item()  # eager work between
        else:
            for _ in range(5):
                opt.step()
        torch.cuda.synchronize()
        runs.append([t.clone() for p in params for t in (
            p.detach(), bits(opt.state[p]["exp_avg"]), bits(opt.state[p]["exp_avg_sq"]))])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_another_stream(cuda_device):
    params, opt = make(cuda_device)
    plain = Plain([p.detach() for p in params])
    grads = grads_for(params, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for p, g in zip(params, grads):
            p.grad = g
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    plain.update(grads)
    same_state(opt, params, plain)


def test_refused_before_anything_changes(cuda_device):
    p, q = (torch.zeros(64, 80, device=cuda_device, requires_grad=True) for _ in range(2))
    opt = FusedAdamW8bit([p, q], lr=LR, min_8bit_numel=1)
    p.grad = torch.ones_like(p)
    q.grad = torch.ones(80, 64, device=cuda_device).t()
    with pytest.raises(ValueError, match="contiguous"):
        opt.step()
    assert not p.detach().any() and not opt.state[p]
    q.grad = torch.ones_like(q)
    opt.step()
    assert float(opt.state[p]["step"]) == 1 and bool(p.detach().all())
    with pytest.raises(ValueError, match="contiguous"):
        r = torch.zeros(64, 80, device=cuda_device).t().requires_grad_(True)
        r.grad = torch.ones_like(r)
        FusedAdamW8bit([r], min_8bit_numel=1).step()
