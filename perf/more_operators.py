"""Attention over a part of the sequence and over a paged cache, as measurable cases.

  window  causal attention with a sliding window and first tokens that stay visible
          (sinks), with the gradient of the packed qkv (window_attention)
  rotate  rotation of q and k by position, with its gradient (rotate_qkv)
  append  where new tokens go in a paged cache, and their rotated keys and values
          written there (cache_plan, append_kv)
  cached  attention of new tokens over the cache: one token a sequence, a chunk of a
          prompt, or a tree of drafted tokens (cached_attention)

With ``own`` false ``run`` computes the same from elementary torch operations.

Sizes are the decoder configurations this repository trains and benchmarks (8 heads
of 32 over 512 tokens, 20 heads of 64), the odd shapes of its tests, and generic ones
with heads of 128 and shared keys and values.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
BASE = 10000.0
TABLE = 1 << 17  # positions that a rotation table holds


def listed():
    return [
        # two short sequences of the narrow decoder: all latency
        {"name": "window_2x77", "kind": "window", "batch": 2, "seq": 77, "heads": 8, "kv": 8,
         "hd": 32, "window": 32, "sinks": 4, "dtype": "fp16"},
        # the narrow decoder's whole batch, trained with a short window
        {"name": "window_33x512", "kind": "window", "batch": 33, "seq": 512, "heads": 8, "kv": 8,
         "hd": 32, "window": 128, "sinks": 4, "dtype": "fp16"},
        # a wide decoder with shared keys and values on sequences of odd length, bf16
        {"name": "window_3x1999", "kind": "window", "batch": 3, "seq": 1999, "heads": 20, "kv": 4,
         "hd": 64, "window": 500, "sinks": 3, "dtype": "bf16"},
        # long documents: what a window is for
        {"name": "window_2x16384", "kind": "window", "batch": 2, "seq": 16384, "heads": 10,
         "kv": 10, "hd": 128, "window": 2048, "sinks": 4, "dtype": "bf16"},
        # one short sequence of the narrow decoder: all latency
        {"name": "rotate_1x33", "kind": "rotate", "batch": 1, "seq": 33, "heads": 8, "kv": 8,
         "hd": 32, "pairs": False, "packed": False, "dtype": "fp16"},
        # a wide decoder's whole batch, documents packed one behind the other
        {"name": "rotate_16x2048", "kind": "rotate", "batch": 16, "seq": 2048, "heads": 20,
         "kv": 4, "hd": 64, "pairs": True, "packed": True, "dtype": "bf16"},
        # a decoding step of a few sequences in the narrow decoder's context: all latency
        {"name": "append_37x1", "kind": "append", "seqs": 37, "longest": 512, "query": 1,
         "heads": 8, "kv": 8, "hd": 32, "page": 16, "rotary": "halves", "dtype": "fp16"},
        # four prompts of odd lengths taken in at once
        {"name": "append_4x4096", "kind": "append", "seqs": 4, "longest": 9000, "query": 4096,
         "heads": 32, "kv": 8, "hd": 128, "page": 64, "rotary": "halves", "dtype": "bf16"},
        # one sequence in the narrow decoder's context answers: all latency
        {"name": "decode_1x200", "kind": "cached", "seqs": 1, "longest": 200, "query": 1,
         "heads": 8, "kv": 8, "hd": 32, "page": 16, "tree": False, "window": 0, "sinks": 0,
         "dtype": "fp16"},
        # a serving batch: sequences of 100 to 65536 tokens, a token each
        {"name": "decode_33x65536", "kind": "cached", "seqs": 33, "longest": 65536, "query": 1,
         "heads": 32, "kv": 8, "hd": 128, "page": 64, "tree": False, "window": 0, "sinks": 0,
         "dtype": "bf16"},
        # drafted trees of up to 64 tokens are checked in one pass
        {"name": "tree_8x4000", "kind": "cached", "seqs": 8, "longest": 4000, "query": 64,
         "heads": 20, "kv": 4, "hd": 64, "page": 32, "tree": True, "window": 0, "sinks": 0,
         "dtype": "bf16"},
        # the next chunks of long prompts, with the window they were trained with
        {"name": "chunk_4x12000", "kind": "cached", "seqs": 4, "longest": 12000, "query": 512,
         "heads": 16, "kv": 2, "hd": 128, "page": 16, "tree": False, "window": 4096, "sinks": 4,
         "dtype": "fp16"},
    ]


def _log(rng, low, high):
    """An integer spread over the logarithm of [low, high]."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["window", "window", "rotate", "append", "cached", "cached", "cached"])
    hd, kv = rng.choice([32, 64, 128]), rng.randint(1, 10)
    heads = kv * (1 if rng.random() < 0.4 else rng.randint(1, 8))
    case = {"kind": kind, "heads": heads, "kv": kv, "hd": hd,
            "dtype": rng.choice(["fp16", "bf16"])}
    if kind == "window":
        # the plain form goes over the whole square of every head
        per = heads * hd
        seq = _log(rng, 1, min(16384, math.isqrt(2 * 10 * 16384 ** 2 * 128 // per)))
        most = max(1, 2 * 10 * 16384 ** 2 * 128 // (per * seq * seq))
        most = min(most, 33 * 512 * 8 * 32 * 8 // (per * seq) + 1)
        window = _log(rng, 1, min(4096, seq + 8))
        sinks = rng.choice([0, 1, 4, _log(rng, 1, 200)])
        batch = _log(rng, 1, most)
        largest = work(listed()[3])["flops"]
        case.update(batch=batch, seq=seq, window=window, sinks=sinks)
        while case["batch"] > 1 and work(case)["flops"] > largest:
            case["batch"] //= 2
        while work(case)["flops"] > largest:
            case["window"] //= 2
        return case
    if kind == "rotate":
        tokens = 16 * 2048 * 28 * 64 // ((heads + 2 * kv) * hd)
        seq = _log(rng, 1, min(8192, tokens))
        case.update(batch=_log(rng, 1, max(1, tokens // seq)), seq=seq,
                    pairs=rng.random() < 0.5, packed=rng.random() < 0.5)
        return case
    case["page"] = rng.choice([16, 32, 64, 128])
    if kind == "append":
        tokens = 4 * 4096 * 48 * 128 // ((heads + 2 * kv) * hd)
        seqs = _log(rng, 1, 256)
        query = _log(rng, 1, max(1, min(8192, tokens // seqs)))
        case.update(seqs=seqs, query=query, longest=query + _log(rng, 1, 8192),
                    rotary=rng.choice(["none", "halves", "pairs"]))
        return case
    shape = rng.choice(["one", "one", "tree", "chunk"])
    query = {"one": 1, "tree": rng.randint(2, 64), "chunk": _log(rng, 2, 2048)}[shape]
    seqs = _log(rng, 1, 256 if shape == "one" else 32)
    held = 33 * 10000 * 8 * 128 // (kv * hd * seqs)  # tokens a sequence of the largest case's cache
    longest = query + _log(rng, 1, max(1, min(65536, held)))
    windowed = rng.random() < 0.4
    case.update(seqs=seqs, longest=longest, query=query, tree=shape == "tree",
                window=_log(rng, 1, 8192) if windowed else 0,
                sinks=rng.choice([0, 1, 4, 64]) if windowed else 0)
    largest = work(listed()[11])["flops"]
    while query > 1 and case["seqs"] > 1 and work(case)["flops"] > largest:
        case["seqs"] //= 2
    while query > 1 and work(case)["flops"] > largest:
        case["longest"] = query + max(1, (case["longest"] - query) // 2)
        if case["longest"] == query + 1:
            break
    return case


# ---------------------------------------------------------------------------
# what a batch of sequences looks like
# ---------------------------------------------------------------------------
def _batch(case):
    """(new tokens, tokens held with the new ones) of each sequence: the first is the
    longest, others spread over the logarithm; one of every eight slots is idle."""
    rng = random.Random(f"{case['seqs']} {case['longest']} {case['query']}")
    new, held = [], []
    for i in range(case["seqs"]):
        if i % 8 == 5:
            new.append(0)
            held.append(0)
            continue
        n = case["query"] if i == 0 else rng.randint(-(-case["query"] // 3), case["query"])
        low = min(case["longest"], n + 100)
        total = case["longest"] if i == 0 else _log(rng, low, case["longest"])
        new.append(n)
        held.append(total)
    return new, held


def _visible(case, position):
    """How many of the tokens 0 .. position a token there sees."""
    if not case["window"]:
        return position + 1
    inside = min(position + 1, case["window"])
    return inside + min(case["sinks"], position + 1 - inside)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device=DEVICE).mul_(std)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, device=DEVICE, dtype=dtype)


def _trees(counts, seed):
    """A random tree of each sequence's new tokens: a token sees its path from the root."""
    rng = random.Random(seed)
    masks = []
    for n in counts:
        paths = []
        for i in range(n):
            above = paths[rng.randint(max(0, i - 9), i - 1)] if i else 0
            paths.append(above | 1 << i)
        masks += paths
    return [m - (1 << 64) if m >> 63 else m for m in masks]


def _inputs(case, seed):
    g = _gen(seed)
    t, heads, kv, hd = DTYPES[case["dtype"]], case["heads"], case["kv"], case["hd"]
    width = (heads + 2 * kv) * hd
    if case["kind"] in ("window", "rotate"):
        batch, seq = case["batch"], case["seq"]
        qkv = _randn(g, batch, seq, width)
        if case["kind"] == "window":
            # queries lean towards the first keys, as trained ones do
            lean = _randn(g, kv, 1, hd, std=0.4)
            qkv[..., :heads * hd].view(batch, seq, kv, -1, hd).add_(lean)
            qkv[:, :4, heads * hd:(heads + kv) * hd].view(batch, -1, kv, hd).add_(2 * lean[:, 0])
            return {"qkv": qkv.to(t), "grad": _randn(g, batch, seq, heads * hd, std=0.5).to(t)}
        positions = None
        if case["packed"]:  # documents one behind the other
            first = torch.rand(batch, seq, generator=g, device=DEVICE) < 4 / seq
            at = torch.arange(seq, device=DEVICE).expand(batch, seq)
            positions = (at - torch.where(first, at, 0).cummax(1).values).int()
        return {"qkv": qkv.to(t), "grad": _randn(g, batch, seq, width, std=0.5).to(t),
                "positions": positions}
    new, held = _batch(case)
    page, per = case["page"], -(-case["longest"] // case["page"])
    pages = sum(-(-n // page) for n in held) + 3  # some belong to nobody here
    order = torch.randperm(pages, generator=g, device=DEVICE).int()
    table, at = torch.zeros(case["seqs"], per, device=DEVICE, dtype=torch.int32), 0
    for i, n in enumerate(held):
        count = -(-n // page)
        table[i, :count] = order[at:at + count]
        at += count
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    state = {"table": table, "lengths": _ints(held), "starts": _ints(starts), "new": new,
             "held": held,
             "keys": _randn(g, pages, kv, page, hd).to(t),
             "values": _randn(g, pages, kv, page, hd).to(t)}
    if case["kind"] == "append":
        state["qkv"] = _randn(g, starts[-1], width).to(t)
    else:
        state["q"] = _randn(g, starts[-1], heads, hd, std=1.5).to(t)
        state["tree"] = _ints(_trees(new, seed), torch.int64) if case["tree"] else None
    return state


def _rotary(case):
    from reversability_amd.attention import Rotary
    style = case.get("rotary", "pairs" if case.get("pairs") else "halves")
    return None if style == "none" else Rotary(case["hd"], TABLE, base=BASE,
                                               interleaved=style == "pairs", device=DEVICE)


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if case["kind"] in ("window", "rotate"):
        state["qkv"].requires_grad_(True)
    if own and case["kind"] in ("rotate", "append"):
        state["rotary"] = _rotary(case)
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return {"window": _window, "rotate": _rotate, "append": _append, "cached": _cached}[
        state["case"]["kind"]](state["case"], state)


def _softmax(scores, mask):
    """Softmax over the last axis where ``mask`` is set; rows without any are zeros."""
    scores = scores.masked_fill_(~mask, -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    return scores.div_(scores.sum(-1, keepdim=True).clamp_min(1e-30))


def _window(case, s):
    if own:
        from reversability_amd.attention import window_attention
        out = window_attention(s["qkv"], case["heads"], case["window"], case["sinks"],
                               kv_heads=case["kv"])
        dqkv, = torch.autograd.grad(out, s["qkv"], s["grad"])
        return {"out": out.detach(), "dqkv": dqkv}
    batch, seq, heads, kv, hd = (case[k] for k in ("batch", "seq", "heads", "kv", "hd"))
    t, group, scale = s["qkv"].dtype, heads // kv, 1 / math.sqrt(hd)
    qkv = s["qkv"].detach().view(batch, seq, heads + 2 * kv, hd).transpose(1, 2)
    grad = s["grad"].view(batch, seq, heads, hd).transpose(1, 2)
    out = torch.empty(batch, heads, seq, hd, device=DEVICE, dtype=t)
    dqkv = torch.empty(batch, heads + 2 * kv, seq, hd, device=DEVICE, dtype=t)
    at = torch.arange(seq, device=DEVICE)
    gap = at.unsqueeze(1) - at
    mask = (gap >= 0) & ((gap < case["window"]) | (at < case["sinks"]))
    step = max(1, (1 << 28) // (kv * seq * seq))  # sequences at a time, one head of each group
    for b in range(0, batch, step):
        part = slice(b, b + step)
        k, v = (qkv[part, heads + i * kv:heads + (i + 1) * kv].float().contiguous()
                for i in (0, 1))
        dk, dv = torch.zeros_like(k), torch.zeros_like(v)
        for j in range(group):
            rows = slice(j, heads, group)
            q, do = (x[part, rows].float().contiguous() for x in (qkv, grad))
            p = _softmax((q @ k.transpose(2, 3).contiguous()).mul_(scale), mask)
            out[part, rows] = (p @ v).to(t)
            dv += p.transpose(2, 3).contiguous() @ do
            ds = do @ v.transpose(2, 3).contiguous()
            ds.sub_((ds * p).sum(-1, keepdim=True)).mul_(p).mul_(scale)
            dqkv[part, rows] = (ds @ k).to(t)
            dk += ds.transpose(2, 3).contiguous() @ q
            del p, ds
        dqkv[part, heads:heads + kv] = dk.to(t)
        dqkv[part, heads + kv:] = dv.to(t)
    return {"out": out.transpose(1, 2).reshape(batch, seq, -1),
            "dqkv": dqkv.transpose(1, 2).reshape(batch, seq, -1)}


def _turn(x, positions, pairs, back=False):
    """x [tokens, heads, hd] in 32 bits, turned by its positions' angles (64 bits)."""
    half = x.shape[-1] // 2
    rate = BASE ** (-torch.arange(half, device=DEVICE, dtype=torch.float64) / half)
    angle = positions.double().unsqueeze(1) * rate
    cos, sin = angle.cos().float().unsqueeze(1), angle.sin().float().unsqueeze(1)
    if back:
        sin = -sin
    a, b = (x[..., 0::2], x[..., 1::2]) if pairs else (x[..., :half], x[..., half:])
    turned = (a * cos - b * sin, a * sin + b * cos)
    return torch.stack(turned, -1).flatten(-2) if pairs else torch.cat(turned, -1)


def _rotate(case, s):
    heads, kv, hd = case["heads"], case["kv"], case["hd"]
    if own:
        from reversability_amd.attention import rotate_qkv
        out = rotate_qkv(s["qkv"], heads, s["rotary"], s["positions"], kv_heads=kv)
        dqkv, = torch.autograd.grad(out, s["qkv"], s["grad"])
        return {"out": out.detach(), "dqkv": dqkv}
    shape = s["qkv"].shape
    at = torch.arange(case["seq"], device=DEVICE).expand(shape[:2])
    positions = (at if s["positions"] is None else s["positions"]).reshape(-1)
    done = []
    for x, back in ((s["qkv"].detach(), False), (s["grad"], True)):
        y = x.reshape(-1, heads + 2 * kv, hd).clone()
        y[:, :heads + kv] = _turn(y[:, :heads + kv].float(), positions, case["pairs"],
                                  back).to(x.dtype)
        done.append(y.view(shape))
    return {"out": done[0], "dqkv": done[1]}


def _append(case, s):
    heads, kv, hd, page = (case[k] for k in ("heads", "kv", "hd", "page"))
    if own:
        from reversability_amd.cache import append_kv, cache_plan
        slots, positions = cache_plan(s["table"], s["lengths"], s["starts"], s["qkv"].shape[0],
                                      page)
        q = append_kv(s["qkv"], heads, s["keys"], s["values"], slots, s["rotary"], positions)
        return {"q": q, "keys": s["keys"], "values": s["values"], "slots": slots,
                "positions": positions}
    new = (s["starts"][1:] - s["starts"][:-1]).long()
    owner = torch.repeat_interleave(torch.arange(case["seqs"], device=DEVICE), new,
                                    output_size=s["qkv"].shape[0])
    at = torch.arange(s["qkv"].shape[0], device=DEVICE)
    positions = s["lengths"].long()[owner] - s["starts"].long()[owner + 1] + at
    slots = s["table"][owner, positions // page].long() * page + positions % page
    x = s["qkv"].view(-1, heads + 2 * kv, hd)
    q, k = x[:, :heads], x[:, heads:heads + kv]
    if case["rotary"] != "none":
        q, k = (_turn(y.float(), positions, case["rotary"] == "pairs").to(x.dtype)
                for y in (q, k))
    s["keys"][slots // page, :, slots % page] = k
    s["values"][slots // page, :, slots % page] = x[:, heads + kv:]
    return {"q": q, "keys": s["keys"], "values": s["values"], "slots": slots,
            "positions": positions.int()}


def _cached(case, s):
    heads, kv, hd, page = (case[k] for k in ("heads", "kv", "hd", "page"))
    if own:
        from reversability_amd.cache import cached_attention
        return {"out": cached_attention(
            s["q"], s["keys"], s["values"], s["table"], s["lengths"], s["starts"], case["query"],
            tree=s["tree"], window=case["window"] or None, sinks=case["sinks"])}
    out, first, group = torch.empty_like(s["q"]), 0, heads // kv
    for i, (n, total) in enumerate(zip(s["new"], s["held"])):
        if not n:
            continue
        rows = s["table"][i, :-(-total // page)].long()
        k, v = (x[rows].transpose(0, 1).reshape(kv, -1, hd)[:, :total].float()
                for x in (s["keys"], s["values"]))
        q = s["q"][first:first + n].float().view(n, kv, group, hd)
        q = q.permute(1, 2, 0, 3).reshape(kv, group * n, hd)
        mask = _sight(case, n, total, None if s["tree"] is None else s["tree"][first:first + n])
        scores = (q @ k.transpose(1, 2).contiguous()).mul_(1 / math.sqrt(hd))
        p = _softmax(scores.view(kv, group, n, total), mask).view(kv, group * n, total)
        mixed = (p @ v).view(kv, group, n, hd).permute(2, 0, 1, 3)
        out[first:first + n] = mixed.reshape(n, heads, hd).to(out.dtype)
        first += n
    return {"out": out}


def _sight(case, n, total, tree):
    """[n, total]: which tokens of a sequence its n new ones see."""
    at = torch.arange(total, device=DEVICE)
    context = total - n
    if tree is None:
        place = at
        mask = at <= at[context:].unsqueeze(1)
    else:
        bits = tree.unsqueeze(1) >> torch.arange(n, device=DEVICE) & 1
        place = torch.cat([at[:context], context + bits.sum(1) - 1])
        mask = torch.cat([torch.ones(n, context, device=DEVICE, dtype=torch.bool), bits == 1], 1)
    if case["window"]:
        far = place[context:].unsqueeze(1) - place >= case["window"]
        mask &= ~far | (place < case["sinks"])
    return mask


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    kind, heads, kv, hd = (case[k] for k in ("kind", "heads", "kv", "hd"))
    width = (heads + 2 * kv) * hd
    if kind == "window":
        full, tokens = min(case["seq"], case["window"]), case["batch"] * case["seq"]
        pairs = full * (full + 1) // 2 + (case["seq"] - full) * full
        far = case["seq"] - full  # tokens that see sinks behind their window
        few = min(case["sinks"], far)
        pairs += few * (few + 1) // 2 + (far - few) * few
        # qkv and the output's gradient read, the output and qkv's gradient written
        return {"bytes": tokens * 2 * (2 * width + 2 * heads * hd),
                "flops": 14 * hd * heads * case["batch"] * pairs}
    if kind == "rotate":
        tokens = case["batch"] * case["seq"]
        return {"bytes": tokens * (8 * width + 4 * case["packed"]),
                "flops": tokens * 6 * (heads + kv) * hd}
    new, held = _batch(case)
    if kind == "append":
        turned = case["rotary"] != "none"
        per = 2 * ((heads if turned else 0) + 2 * kv) * hd  # a query that is not turned stays
        return {"bytes": sum(new) * (per * 2 + 12),
                "flops": 3 * sum(new) * (heads + kv) * hd * turned}
    seen = pairs = 0
    for n, total in zip(new, held):
        if not n:
            continue
        pairs += sum(_visible(case, p) for p in range(total - n, total)) if not case["tree"] else (
            n * _visible(case, total - n))
        near = total if not case["window"] else min(total, case["window"] + n - 1)
        seen += near + min(case["sinks"], total - near)
    return {"bytes": seen * kv * hd * 4 + sum(new) * heads * hd * 4,
            "flops": 4 * hd * heads * pairs}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    kind = case["kind"]
    if kind == "window" and case["heads"] * case["batch"] * case["seq"] ** 2 > 1 << 31:
        return None  # over twenty seconds
    if kind == "cached" and work(case)["flops"] > 1 << 37:
        return None
    return {"window": _window64, "rotate": _rotate64, "append": _append64,
            "cached": _cached64}[kind](case, _inputs(case, seed))


def _attend64(q, k, v, seen):
    """Attention of q [heads, n, hd] over k, v [heads, m, hd] where ``seen`` [n, m]."""
    score = torch.matmul(q, k.transpose(1, 2).contiguous()) / q.shape[-1] ** 0.5
    weight = torch.softmax(score.where(seen, score.new_tensor(-math.inf)), dim=2)
    return torch.matmul(torch.where(seen.any(1)[:, None], weight, 0.0), v)


def _window64(case, s):
    heads, kv, hd = case["heads"], case["kv"], case["hd"]
    i = torch.arange(case["seq"], device=DEVICE)[:, None]
    j = torch.arange(case["seq"], device=DEVICE)[None]
    seen = torch.logical_and(j <= i, torch.logical_or(i < j + case["window"], j < case["sinks"]))
    outs, grads = [], []
    for row, grad in zip(s["qkv"], s["grad"]):
        x = row.double().requires_grad_(True)
        q, k, v = x.reshape(case["seq"], -1, hd).permute(1, 0, 2).split((heads, kv, kv))
        mixed = _attend64(q, k.repeat_interleave(heads // kv, 0),
                          v.repeat_interleave(heads // kv, 0), seen)
        out = mixed.permute(1, 0, 2).reshape(case["seq"], heads * hd)
        grads.append(torch.autograd.grad(out, x, grad.double())[0])
        outs.append(out.detach())
    return {"out": torch.stack(outs), "dqkv": torch.stack(grads)}


def _spin64(x, positions, pairs, sign=1):
    """x [tokens, heads, hd] as complex numbers times exp(i angle)."""
    n, h, hd = x.shape
    z = x.double()
    z = z.view(n, h, hd // 2, 2) if pairs else z.view(n, h, 2, hd // 2).transpose(2, 3)
    z = torch.view_as_complex(z.contiguous())
    index = torch.arange(hd // 2, device=DEVICE, dtype=torch.float64)
    angle = positions.double()[:, None] / torch.pow(BASE, 2 * index / hd)
    z = torch.view_as_real(z * torch.polar(torch.ones_like(angle), sign * angle)[:, None])
    return z.reshape(n, h, hd) if pairs else z.transpose(2, 3).reshape(n, h, hd)


def _rotate64(case, s):
    turning = case["heads"] + case["kv"]
    positions = s["positions"]
    if positions is None:
        positions = torch.arange(case["seq"], device=DEVICE).repeat(case["batch"])
    out = {}
    for name, x, sign in (("out", s["qkv"], 1), ("dqkv", s["grad"], -1)):
        parts = x.double().reshape(-1, turning + case["kv"], case["hd"])
        out[name] = torch.cat([_spin64(parts[:, :turning], positions.reshape(-1), case["pairs"],
                                       sign), parts[:, turning:]], 1).reshape(x.shape)
    return out


def _append64(case, s):
    page, rows = case["page"], s["qkv"].view(-1, case["heads"] + 2 * case["kv"], case["hd"])
    slots, positions = [], []
    for i, (n, total) in enumerate(zip(s["new"], s["held"])):
        pages = s["table"][i].tolist()
        for p in range(total - n, total):
            positions.append(p)
            slots.append(pages[p // page] * page + p % page)
    slots, positions = _ints(slots, torch.int64), _ints(positions)
    q, k, v = rows.double().split((case["heads"], case["kv"], case["kv"]), 1)
    if case["rotary"] != "none":
        q, k = (_spin64(x, positions, case["rotary"] == "pairs") for x in (q, k))
    result = {"q": q, "slots": slots, "positions": positions}
    for name, x in (("keys", k), ("values", v)):
        cache = s[name].double().transpose(1, 2).reshape(-1, case["kv"], case["hd"])
        cache[slots] = x
        result[name] = cache.view(-1, page, case["kv"], case["hd"]).transpose(1, 2)
    return result


def _cached64(case, s):
    page, heads, kv = case["page"], case["heads"], case["kv"]
    caches = [s[name].transpose(1, 2).reshape(-1, kv, case["hd"]) for name in ("keys", "values")]
    masks = None if s["tree"] is None else s["tree"].tolist()
    outs = []
    for i, (n, total) in enumerate(zip(s["new"], s["held"])):
        if not n:
            continue
        first, context = sum(s["new"][:i]), total - n
        j = torch.arange(total, device=DEVICE)
        flat = s["table"][i].long()[j // page] * page + j % page
        k, v = (c[flat].double().permute(1, 0, 2).repeat_interleave(heads // kv, 0)
                for c in caches)
        if masks is None:
            place, seen = j, j[None] <= context + torch.arange(n, device=DEVICE)[:, None]
        else:
            paths = [[m >> b & 1 for b in range(n)] for m in masks[first:first + n]]
            place = torch.cat([j[:context], _ints([context - 1 + sum(p) for p in paths],
                                                  torch.int64)])
            seen = torch.ones(n, total, device=DEVICE, dtype=torch.bool)
            seen[:, context:] = _ints(paths, torch.bool)
        if case["window"]:
            near = place[context:, None] < place[None] + case["window"]
            seen = seen & (near | (place < case["sinks"])[None])
        q = s["q"][first:first + n].double().permute(1, 0, 2)
        outs.append(_attend64(q, k, v, seen).permute(1, 0, 2))
    return {"out": torch.cat(outs)}
