"""The operators of fine-tuning a decoder from preferences or rewards, as measurable cases.

  logp    log-probabilities of labels under the tied head, with or without the
          gradients of the hidden states and the head (tied_head_logprobs)
  pref    the preference loss over pairs of sequences and its gradient
          (preference_loss)
  policy  the clipped policy loss with a KL term and its gradient (policy_loss)
  adamw8  AdamW with its moments in 8 bits (FusedAdamW8bit)

With ``own`` false ``run`` computes the same from elementary torch operations.

Sizes are the decoder configurations this repository trains and benchmarks
(width 256, 7 layers, 512 tokens; width 1024, 12 layers, 2048 tokens; vocabulary
50257), the small and odd shapes of its tests, and the ranges between them.
"""
import math

import torch

own = False

VOCAB = 50257
SCALE = 1024.0  # loss scale of an fp16 backward, one at which a single token stays finite
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
BETAS, LR, DECAY, EPS = (0.9, 0.95), 6e-4, 0.1, 1e-8
BLOCK = 32  # elements of a moment that share one exponent
SMALL = 4096  # tensors with fewer elements keep their moments in 32 bits


def listed():
    return [
        # scoring a few short sequences: all latency
        {"name": "logp_3x17", "kind": "logp", "rows": 51, "d": 256, "vocab": VOCAB,
         "dtype": "fp16", "train": False},
        # the narrow decoder's whole batch scored by the frozen reference model
        {"name": "logp_33x512", "kind": "logp", "rows": 33 * 512, "d": 256, "vocab": VOCAB,
         "dtype": "fp16", "train": False},
        # a training step of a mid-sized decoder on two odd-length sequences, bf16
        {"name": "logp_train_2x777", "kind": "logp", "rows": 2 * 777, "d": 512, "vocab": 32000,
         "dtype": "bf16", "train": True},
        # the narrow decoder's whole batch, trained
        {"name": "logp_train_33x512", "kind": "logp", "rows": 33 * 512, "d": 256, "vocab": VOCAB,
         "dtype": "fp16", "train": True},
        # the wide decoder's whole batch, trained
        {"name": "logp_train_16x2048", "kind": "logp", "rows": 16 * 2048, "d": 1024,
         "vocab": VOCAB, "dtype": "fp16", "train": True},
        # one pair of short answers: all latency
        {"name": "pref_1x17", "kind": "pref", "pairs": 1, "tokens": 17, "average": False,
         "smooth": 0.0},
        # the narrow decoder's context, an ordinary batch, length-normalised
        {"name": "pref_64x512", "kind": "pref", "pairs": 64, "tokens": 512, "average": True,
         "smooth": 0.1},
        # a large collected batch over the wide decoder's context
        {"name": "pref_2048x2048", "kind": "pref", "pairs": 2048, "tokens": 2048,
         "average": False, "smooth": 0.0},
        # a few odd-length answers
        {"name": "policy_5x333", "kind": "policy", "seqs": 5, "tokens": 333, "kl": 0.05,
         "per_token": False, "reduction": "sequence"},
        # a large collected batch over the wide decoder's context, an advantage per token
        {"name": "policy_4096x2048", "kind": "policy", "seqs": 4096, "tokens": 2048, "kl": 0.05,
         "per_token": True, "reduction": "token"},
        # one layer of the narrow decoder with its embeddings
        {"name": "adamw8_256", "kind": "adamw8", "d": 256, "f": 1024, "vocab": VOCAB,
         "seq": 512},
        # one layer of a wide decoder with its embeddings
        {"name": "adamw8_1280", "kind": "adamw8", "d": 1280, "f": 5120, "vocab": VOCAB,
         "seq": 2048},
    ]


def _log(rng, low, high):
    """An integer spread over the logarithm of [low, high]."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["logp", "logp", "logp", "pref", "policy", "adamw8"])
    if kind == "logp":
        d = 8 * rng.randint(8, 128) if rng.random() < 0.3 else 128 * rng.randint(1, 8)
        return {"kind": kind, "rows": _log(rng, 1, 16 * 2048), "d": d,
                "vocab": _log(rng, 1000, VOCAB), "dtype": rng.choice(["fp16", "fp16", "bf16"]),
                "train": rng.random() < 0.6}
    if kind == "pref":
        tokens = _log(rng, 1, 4096)
        return {"kind": kind, "pairs": _log(rng, 1, 2 ** 22 // tokens), "tokens": tokens,
                "average": rng.random() < 0.5, "smooth": rng.choice([0.0, 0.1])}
    if kind == "policy":
        tokens = _log(rng, 1, 4096)
        return {"kind": kind, "seqs": _log(rng, 1, 2 ** 23 // tokens), "tokens": tokens,
                "kl": rng.choice([0.0, 0.05]), "per_token": rng.random() < 0.5,
                "reduction": rng.choice(["token", "sequence"])}
    d = 64 * rng.randint(2, 20)
    return {"kind": kind, "d": d, "f": rng.choice([3, 4]) * d, "vocab": _log(rng, 1000, VOCAB),
            "seq": rng.choice([512, 1024, 2048])}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda").mul_(std)


def _answers(g, seqs, tokens):
    """Which tokens of a padded batch are scored: an answer behind its prompt,
    ended at its own length; one sequence in 32 has none."""
    at = torch.arange(tokens, device="cuda")
    first = torch.randint(0, max(1, tokens // 3), (seqs, 1), generator=g, device="cuda")
    length = torch.randint(1, tokens + 1, (seqs, 1), generator=g, device="cuda")
    mask = (at >= first) & (at < first + length)
    mask[31::32] = False
    return mask


def _inputs(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    if kind == "logp":
        rows, d, vocab, t = case["rows"], case["d"], case["vocab"], DTYPES[case["dtype"]]
        padded = -(-vocab // 64) * 64
        head = torch.zeros(padded, d, device="cuda", dtype=t)
        head[:vocab] = _randn(g, vocab, d, std=2 / math.sqrt(d)).to(t)
        labels = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        # every second token is one that the model is confident of
        x = _randn(g, rows, d)
        x[::2] += 2 * head[labels[::2]].float()
        labels[torch.arange(rows, device="cuda") % 512 < 96 * (rows > 512)] = -100  # prompts
        grad = _randn(g, rows, std=(SCALE if case["dtype"] == "fp16" else 1.0) / rows)
        return {"x": x.to(t), "head": head, "labels": labels, "grad": grad, "vocab": vocab}
    if kind == "pref":
        shape = (2 * case["pairs"], case["tokens"])
        mask = _answers(g, *shape)
        ref = -torch.empty(shape, device="cuda").exponential_(0.5, generator=g)
        logp = ref + _randn(g, *shape, std=0.3)
        return {"logp": logp, "ref": ref, "mask": mask}
    if kind == "policy":
        shape = (case["seqs"], case["tokens"])
        mask = _answers(g, *shape)
        old = -torch.empty(shape, device="cuda").exponential_(0.5, generator=g)
        logp = old + _randn(g, *shape, std=0.2)
        ref = old + _randn(g, *shape, std=0.2) if case["kl"] else None
        adv = _randn(g, *(shape if case["per_token"] else shape[:1]))
        return {"logp": logp, "old": old, "ref": ref, "mask": mask, "adv": adv}
    d, f = case["d"], case["f"]
    shapes = [(case["vocab"], d), (case["seq"], d), (d,), (3 * d, d), (d, d), (d,), (2 * f, d),
              (d, f), (d,)]
    params = [_randn(g, *s, std=0.02) for s in shapes]
    grads = [_randn(g, *s, std=0.05) for s in shapes]
    moments = []
    for s in shapes:  # the moments some steps into a run
        n = math.prod(s)
        m, v = _randn(g, n, std=0.012), _randn(g, n, std=0.05).square_()
        if n < SMALL:
            moments.append((m.view(s), v.view(s)))
        else:
            blocks = -(-n // BLOCK)
            scales = [torch.full((blocks,), 127 - e, device="cuda", dtype=torch.uint8)
                      for e in (12, 9)]
            codes = [(t * 2.0 ** e).to(torch.float8_e4m3fn).view(s)
                     for t, e in ((m, 12), (v, 9))]
            moments.append((codes[0], codes[1], scales[0], scales[1]))
    return {"params": params, "grads": grads, "moments": moments, "seed": seed % 1000}


def prepare(case, seed):
    kind = case["kind"]
    state = _inputs(case, seed)
    state.update(case)
    if kind == "logp" and case["train"]:
        state["x"].requires_grad_(True)
        state["head"].requires_grad_(True)
    elif kind in ("pref", "policy"):
        state["logp"].requires_grad_(True)
    elif kind == "adamw8":
        state["step"] = 100
        if own:
            state["opt"] = _optimizer(state)
    return state


def _optimizer(state):
    """FusedAdamW8bit as its run of 100 steps left it."""
    from reversability_amd.optim import FusedAdamW8bit
    params = [torch.nn.Parameter(p) for p in state["params"]]
    opt = FusedAdamW8bit(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY,
                         seed=state["seed"])
    step = torch.full((), 100.0, device="cuda")
    for p, grad, moments in zip(params, state["grads"], state["moments"]):
        p.grad = grad
        names = ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")
        opt.state[p].update(zip(names, moments), step=step)
    return opt


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return {"logp": _logp, "pref": _pref, "policy": _policy, "adamw8": _adamw8}[state["kind"]](state)


def _logp(s):
    if own:
        from reversability_amd.preference import tied_head_logprobs
        if not s["train"]:
            with torch.no_grad():
                return {"logp": tied_head_logprobs(s["x"], s["head"], s["vocab"], s["labels"])}
        logp = tied_head_logprobs(s["x"], s["head"], s["vocab"], s["labels"])
        dx, dhead = torch.autograd.grad(logp, (s["x"], s["head"]), s["grad"])
        return {"logp": logp.detach(), "dx": dx, "dhead": dhead}
    x, head = s["x"].detach().float(), s["head"].detach().float()
    labels, valid = s["labels"].clamp_min(0).unsqueeze(1), s["labels"] >= 0
    z = x @ head[:s["vocab"]].t()
    top = z.max(1, keepdim=True).values
    e = (z - top).exp_()
    total = e.sum(1, keepdim=True)
    logp = (z.gather(1, labels) - top - total.log()).squeeze(1)
    logp = torch.where(valid, logp, 0.0)
    if not s["train"]:
        return {"logp": logp}
    del z
    g = torch.where(valid, s["grad"], 0.0).unsqueeze(1)
    dz = e.mul_(-g / total)
    dz.scatter_add_(1, labels, g)
    dx = (dz @ head[:s["vocab"]]).to(s["x"].dtype)
    dhead = torch.zeros_like(s["head"])
    dhead[:s["vocab"]] = (dz.t() @ x).to(s["x"].dtype)
    return {"logp": logp, "dx": dx, "dhead": dhead}


BETA = 0.1


def _pref(s):
    if own:
        from reversability_amd.preference import preference_loss
        loss, chosen, rejected = preference_loss(s["logp"], s["ref"], BETA, mask=s["mask"],
                                                 label_smoothing=s["smooth"],
                                                 average=s["average"])
        dlogp, = torch.autograd.grad(loss, s["logp"])
        return {"loss": loss.detach(), "chosen": chosen, "rejected": rejected, "dlogp": dlogp}
    pairs, eps = s["pairs"], s["smooth"]
    logp, mask = s["logp"].detach(), s["mask"]
    # sums over long answers of small differences: 64 bits
    ratio = torch.where(mask, logp - s["ref"], 0.0).sum(1, dtype=torch.float64)
    share = 1.0 / mask.sum(1).clamp_min(1) if s["average"] else torch.ones_like(ratio)
    reward = BETA * ratio * share
    margin = reward[:pairs] - reward[pairs:]
    soft = (-margin.abs()).exp().log1p()  # log(1 + exp(-|margin|))
    loss = ((1 - eps) * (soft + (-margin).clamp_min(0))
            + eps * (soft + margin.clamp_min(0))).mean()
    slope = (1 / (1 + (-margin).exp()) - (1 - eps)) * (BETA / pairs)
    slope = (torch.cat([slope, -slope]) * share).float().unsqueeze(1)
    reward = reward.float()
    return {"loss": loss.float(), "chosen": reward[:pairs], "rejected": reward[pairs:],
            "dlogp": torch.where(mask, slope, 0.0)}


CLIP = (0.2, 0.28)


def _policy(s):
    if own:
        from reversability_amd.preference import policy_loss
        loss, kl, clipped = policy_loss(s["logp"], s["old"], s["adv"], ref_logp=s["ref"],
                                        mask=s["mask"], clip=CLIP, kl_coef=s["kl"],
                                        reduction=s["reduction"])
        dlogp, = torch.autograd.grad(loss, s["logp"])
        return {"loss": loss.detach(), "kl": kl, "clipped": clipped, "dlogp": dlogp}
    logp, old, mask = s["logp"].detach(), s["old"], s["mask"]
    adv = s["adv"] if s["per_token"] else s["adv"].unsqueeze(1)
    ratio = (logp - old).exp()
    # the clip borders: 64 bits, so that a ratio next to one falls on its side of it
    delta = logp.double() - old.double()
    high = (adv > 0) & (delta > math.log1p(CLIP[1]))
    low = (adv < 0) & (delta < math.log1p(-CLIP[0]))
    clipped = high | low
    bound = torch.where(high, 1 + CLIP[1], torch.where(low, 1 - CLIP[0], ratio))
    term = -bound * adv
    slope = torch.where(clipped, 0.0, -ratio * adv)
    count = mask.sum()
    kl = torch.zeros((), device="cuda")
    if s["kl"]:
        shift = s["ref"] - logp
        away = shift.exp()
        gap = away - shift - 1
        kl = (torch.where(mask, gap, 0.0).sum(dtype=torch.float64) / count.clamp_min(1)).float()
        term = term + s["kl"] * gap
        slope = slope + s["kl"] * (1 - away)
    if s["reduction"] == "token":
        weight = (1.0 / count.clamp_min(1)).double()
        loss = torch.where(mask, term, 0.0).sum(dtype=torch.float64) * weight
    else:
        weight = (1.0 / mask.sum(1).clamp_min(1).double() / s["seqs"]).unsqueeze(1)
        loss = (torch.where(mask, term, 0.0).sum(1, dtype=torch.float64) * weight[:, 0]).sum()
    share = (clipped & mask).sum() / count.clamp_min(1)
    return {"loss": loss.float(), "kl": kl, "clipped": share.float(),
            "dlogp": torch.where(mask, slope * weight.float(), 0.0)}


def _mix(h):
    """The 32-bit finalizer of MurmurHash3 on int64 tensors or numbers."""
    h = (h ^ (h >> 16)) * 0x85EBCA6B & 0xFFFFFFFF
    h = (h ^ (h >> 13)) * 0xC2B2AE35 & 0xFFFFFFFF
    return h ^ (h >> 16)


def _decode(codes, exponent):
    """fp32 values of a moment's e4m3 codes and its blocks' exponents, in whole blocks."""
    flat = codes.reshape(-1).float()
    flat = torch.nn.functional.pad(flat, (0, -flat.numel() % BLOCK)).view(-1, BLOCK)
    return flat * (exponent.int() << 23).view(torch.float32).unsqueeze(1)


def _exponents(t):
    """The exponent byte of each block: its largest magnitude in [2^7, 2^8) of it."""
    top = t.abs().amax(1)
    return ((top.view(torch.int32) >> 23) - 7).clamp_min(0)


def _adamw8(s):
    if own:
        opt = s["opt"]
        opt.step()
        params = opt.param_groups[0]["params"]
        moments = [[opt.state[p][k] for k in ("exp_avg", "exp_avg_sq", "exp_avg_scale",
                                              "exp_avg_sq_scale") if k in opt.state[p]]
                   for p in params]
        return {"params": [p.detach() for p in params], "moments": moments}
    s["step"] += 1
    b1, b2 = BETAS
    first = LR / (1 - b1 ** s["step"])
    second = math.sqrt(1 - b2 ** s["step"])
    for at, (p, g, moments) in enumerate(zip(s["params"], s["grads"], s["moments"])):
        n, small = p.numel(), p.numel() < SMALL
        if small:
            m, v, g = moments[0], moments[1], g
        else:
            m, v = _decode(moments[0], moments[2]), _decode(moments[1], moments[3])
            g = torch.nn.functional.pad(g.reshape(-1), (0, -n % BLOCK)).view(-1, BLOCK)
        m = m * b1 + g * (1 - b1)
        v = v * b2 + g * (1 - b2) * g
        update = m / (v.sqrt() / second + EPS)
        p.mul_(1 - LR * DECAY).sub_(update.reshape(-1)[:n].view(p.shape) * first)
        if small:
            moments[0].copy_(m)
            moments[1].copy_(v)
            continue
        em, ev = _exponents(m), _exponents(v)
        # powers of two: exact (two factors, each of them a normal number)
        m = (m * torch.exp2(64.0 - em.float()).unsqueeze(1)) * 2.0 ** 63
        v = (v * torch.exp2(64.0 - ev.float()).unsqueeze(1)) * 2.0 ** 63
        key = _mix((s["seed"] + 0x9E3779B9 * (at + 1)) & 0xFFFFFFFF)
        key = _mix((key + s["step"]) & 0xFFFFFFFF)
        index = torch.arange(v.numel(), device="cuda").view_as(v)
        noise = _mix(((index >> 1) + key) & 0xFFFFFFFF) >> 16 * (index & 1) & 0xFFFF
        noise = (noise << 4 | 8).int()
        code = ((v.view(torch.int32) + noise) >> 20) - 960
        tiny = (v * 512 + noise.float() * 2.0 ** -20).int()
        code = torch.where(v < 2.0 ** -6, tiny, code).clamp_min((v > 0).int())
        moments[0].view(-1).copy_(m.reshape(-1)[:n].to(torch.float8_e4m3fn))
        moments[1].view(torch.uint8).view(-1).copy_(code.reshape(-1)[:n])
        moments[2].copy_(em)
        moments[3].copy_(ev)
    return {"params": s["params"], "moments": [list(m) for m in s["moments"]]}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "logp":
        rows, d, vocab = case["rows"], case["d"], case["vocab"]
        # x, head and labels once, logp; trained: the gradients of both, and g
        return {"bytes": (rows * d + vocab * d) * 2 * (2 if case["train"] else 1)
                + rows * (16 if case["train"] else 12),
                "flops": (6 if case["train"] else 2) * rows * d * vocab}
    if kind == "pref":
        n = 2 * case["pairs"] * case["tokens"]
        return {"bytes": n * 13 + case["pairs"] * 8, "flops": n * 3}
    if kind == "policy":
        n = case["seqs"] * case["tokens"]
        per = 13 + 4 * case["per_token"] + 4 * bool(case["kl"])
        return {"bytes": n * per + 4 * case["seqs"], "flops": n * 20}
    d, f = case["d"], case["f"]
    n = (case["vocab"] + case["seq"]) * d + 4 * d * d + 3 * d * f
    return {"bytes": 16.125 * n + 28 * 3 * d, "flops": 16 * n}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    return {"logp": _logp64, "pref": _pref64, "policy": _policy64, "adamw8": _adamw64}[
        case["kind"]](case, s)


def _logp64(case, s):
    x, w = s["x"].double(), s["head"][:case["vocab"]].double()
    labels, rows = s["labels"], case["rows"]
    logp = torch.zeros(rows, device="cuda", dtype=torch.float64)
    dx = torch.zeros_like(x)
    dhead = torch.zeros(s["head"].shape, device="cuda", dtype=torch.float64)
    for at in range(0, rows, 2048):
        keep = (labels[at:at + 2048] != -100).nonzero()[:, 0] + at
        table = torch.log_softmax(x[keep] @ w.t(), dim=1)
        spot = (torch.arange(len(keep), device="cuda"), labels[keep])
        logp[keep] = table[spot]
        if case["train"]:
            # gradient of sum g logp: g times the one-hot label minus the softmax
            d = table.exp_().neg_()
            d[spot] += 1
            d *= s["grad"][keep].double().unsqueeze(1)
            dx[keep] = d @ w
            dhead[:case["vocab"]] += d.t().contiguous() @ x[keep]
        del table
    return {"logp": logp, "dx": dx, "dhead": dhead} if case["train"] else {"logp": logp}


def _pref64(case, s):
    logp = s["logp"].double().requires_grad_(True)
    on = s["mask"].double()
    score = ((logp - s["ref"].double()) * on).sum(1)
    if case["average"]:
        score = score / on.sum(1).clamp(min=1)
    chosen, rejected = (BETA * score).chunk(2)
    yes = torch.nn.functional.logsigmoid(chosen - rejected)
    no = torch.nn.functional.logsigmoid(rejected - chosen)
    loss = -((1 - case["smooth"]) * yes + case["smooth"] * no).mean()
    dlogp, = torch.autograd.grad(loss, logp)
    return {"loss": loss.detach(), "chosen": chosen.detach(), "rejected": rejected.detach(),
            "dlogp": dlogp}


def _policy64(case, s):
    logp = s["logp"].double().requires_grad_(True)
    on, old = s["mask"].double(), s["old"].double()
    adv = s["adv"].double().reshape(case["seqs"], -1)
    ratio = torch.exp(logp - old)
    objective = torch.minimum(ratio * adv, ratio.clamp(1 - CLIP[0], 1 + CLIP[1]) * adv)
    loss, kl = -objective, torch.zeros_like(logp)
    if case["kl"]:
        shift = s["ref"].double() - logp
        kl = torch.expm1(shift) - shift
        loss = loss + case["kl"] * kl
    total = on.sum().clamp(min=1)
    if case["reduction"] == "token":
        loss = (loss * on).sum() / total
    else:
        loss = ((loss * on).sum(1) / on.sum(1).clamp(min=1)).mean()
    dlogp, = torch.autograd.grad(loss, logp)
    ratio = ratio.detach()
    out = ((adv > 0) & (ratio > 1 + CLIP[1])) | ((adv < 0) & (ratio < 1 - CLIP[0]))
    return {"loss": loss.detach(), "kl": (kl.detach() * on).sum() / total,
            "clipped": (out * on).sum() / total, "dlogp": dlogp}


def _adamw64(case, s):
    """Parameters, and the 32-bit moments of the small tensors; a moment in 8 bits is what
    the values before the rounding are in their block's scale (the exponents are whole
    numbers, without a value here)."""
    params, moments = [], []
    for p, g, state in zip(s["params"], s["grads"], s["moments"]):
        g, n = g.double().reshape(-1), g.numel()
        old = [t.reshape(-1).to(torch.float32).double() for t in state[:2]]
        if len(state) == 4:
            old = [t * torch.pow(2.0, e.double() - 127).repeat_interleave(BLOCK)[:n]
                   for t, e in zip(old, state[2:])]
        m = BETAS[0] * old[0] + (1 - BETAS[0]) * g
        v = BETAS[1] * old[1] + (1 - BETAS[1]) * g * g
        mhat, vhat = m / (1 - BETAS[0] ** 101), v / (1 - BETAS[1] ** 101)
        new = p.double().reshape(-1) * (1 - LR * DECAY) - LR * mhat / (vhat.sqrt() + EPS)
        params.append(new.view(p.shape))
        if len(state) == 2:
            moments.append([m.view(p.shape), v.view(p.shape)])
            continue
        scaled = []
        for t in (m, v):
            blocks = torch.nn.functional.pad(t, (0, -n % BLOCK)).view(-1, BLOCK)
            unit = torch.floor(torch.log2(blocks.abs().amax(1).clamp_min(1e-300))) - 7
            scaled.append((blocks * torch.pow(2.0, -unit).unsqueeze(1)).reshape(-1)[:n].view(p.shape))
        moments.append([scaled[0], scaled[1], None, None])
    return {"params": params, "moments": moments}
