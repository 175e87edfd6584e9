"""A paged cache: where tokens go, their keys and values, and the attention over them,
against plain computations in fp64.

With u half a step of the type: the weights are rounded to it before the product with the
values and the output once, so |out - ref| <= 2 (u P|V| + u |ref|) plus half the type's
smallest number per weight (twice the terms: the second half for fp32 scores,
exponentials, sums and the joining of stretches, below 2^-13 of them at these sizes).
"""
from __future__ import annotations

import math
import random

import pytest
import torch

from reversability_amd.attention import Rotary, rotate_qkv
from reversability_amd.cache import append_kv, cache_plan, cached_attention

pytestmark = pytest.mark.gpu


def batch_of(new, held, page, device, seed=0, spare=2, wide=1):
    """(page_table, lengths, starts, pages) with every sequence's pages scattered; entries
    that no token needs name pages that do not exist."""
    rng = random.Random(seed)
    counts = [-(-n // page) for n in held]
    pages = sum(counts) + spare
    order = list(range(pages))
    rng.shuffle(order)
    table = torch.full((len(held), max(counts + [1]) + wide), 1 << 30, dtype=torch.int32)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = torch.tensor(order[at:at + c], dtype=torch.int32)
        at += c
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    as_int = lambda t: torch.tensor(t, dtype=torch.int32, device=device)
    return table.to(device), as_int(held), as_int(starts), pages


def slots_of(table, held, page):
    """Slots of each sequence's tokens, as lists."""
    rows = table.tolist()
    return [[rows[i][t // page] * page + t % page for t in range(n)] for i, n in enumerate(held)]


def filled(table, held, pages, kv, page, hd, dtype, device, seed=1, spread=1.0):
    """A cache whose slots of no token are NaN."""
    g = torch.Generator().manual_seed(seed)
    caches = []
    flat = torch.tensor(sum(slots_of(table, held, page), []), dtype=torch.int64)
    for _ in range(2):
        c = torch.full((pages * page, kv, hd), math.nan, dtype=dtype)
        c[flat] = (spread * torch.randn(len(flat), kv, hd, generator=g)).to(dtype)
        caches.append(c.view(pages, page, kv, hd).transpose(1, 2).contiguous().to(device))
    return caches


def trees(new, seed=0):
    rng = random.Random(seed)
    masks = []
    for n in new:
        paths = []
        for i in range(n):
            paths.append((paths[rng.randint(max(0, i - 5), i - 1)] if i else 0) | 1 << i)
        masks += paths
    return masks


def signed(masks, device):
    return torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64,
                        device=device)


def reference(q, keys, values, table, new, held, masks=None, window=None, sinks=0):
    """fp64 outputs and bounds [tokens, heads, hd]."""
    tokens, heads, hd = q.shape
    pages, kv, page, _ = keys.shape
    u = torch.finfo(q.dtype).eps / 2
    sub = torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps / 2
    flat = [c.transpose(1, 2).reshape(pages * page, kv, hd) for c in (keys, values)]
    out = torch.zeros(tokens, heads, hd, dtype=torch.float64, device=q.device)
    tol, first = torch.zeros_like(out), 0
    for slots, n, total in zip(slots_of(table, held, page), new, held):
        if not n:
            continue
        at = torch.tensor(slots, dtype=torch.int64, device=q.device)
        k, v = (c[at].double().transpose(0, 1).repeat_interleave(heads // kv, 0) for c in flat)
        context = total - n
        seen = torch.zeros(n, total, dtype=torch.bool)
        for i in range(n):
            if masks is None:
                where, visible = context + i, range(0, context + i + 1)
                place = lambda j: j
            else:
                low = (1 << n) - 1
                where = context + bin(masks[first + i] & low).count("1") - 1
                visible = [j for j in range(total)
                           if j < context or masks[first + i] >> (j - context) & 1]
                place = lambda j: j if j < context else (
                    context + bin(masks[first + j - context] & low).count("1") - 1)
            for j in visible:
                if window is None or where - place(j) < window or place(j) < sinks:
                    seen[i, j] = True
        seen = seen.to(q.device)
        score = (q[first:first + n].double().transpose(0, 1)
                 @ k.transpose(1, 2).contiguous()) / math.sqrt(hd)
        p = torch.softmax(score.masked_fill(~seen, -math.inf), -1).nan_to_num(0.0)
        o, pv = p @ v, p @ v.abs()
        out[first:first + n] = o.transpose(0, 1)
        few = seen.sum(1).view(1, n, 1)
        bound = 2 * (u * pv + u * o.abs() + sub * (1 + few * v.abs().max()))
        tol[first:first + n] = bound.transpose(0, 1)
        first += n
    return out, tol


def check(out, ref, tol):
    bad = float(((out.double() - ref).abs() / tol.clamp_min(1e-300)).nan_to_num(math.inf).max())
    print(f"  {bad:.3f} of the bound", flush=True)
    assert bad <= 1.0


ONE = [([1], [1]), ([1], [17]), ([1, 0, 1, 1], [5, 0, 300, 64]), ([1] * 3, [33, 2000, 700])]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,hd,page", [(1, 1, 32, 16), (8, 8, 32, 64), (10, 2, 64, 32),
                                              (8, 1, 128, 16), (34, 2, 64, 128), (40, 1, 128, 256)])
@pytest.mark.parametrize("new,held", ONE)
def test_one_token_each(cuda_device, new, held, heads, kv, hd, page, dtype):
    table, lengths, starts, pages = batch_of(new, held, page, cuda_device)
    keys, values = filled(table, held, pages, kv, page, hd, dtype, cuda_device)
    g = torch.Generator().manual_seed(2)
    q = (2 * torch.randn(sum(new), heads, hd, generator=g)).to(dtype).to(cuda_device)
    out = cached_attention(q, keys, values, table, lengths, starts, 1)
    check(out, *reference(q, keys, values, table, new, held))
    assert torch.equal(out, cached_attention(q, keys, values, table, lengths, starts, 1))
    # a bound on the lengths below the truth changes the division of the work, not what it gives
    check(cached_attention(q, keys, values, table, lengths, starts, 1, max_length=20),
          *reference(q, keys, values, table, new, held))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,hd,page", [(2, 2, 32, 16), (6, 2, 64, 64), (8, 2, 128, 32)])
@pytest.mark.parametrize("new,held", [([7], [7]), ([1, 40, 0, 3], [1, 41, 9, 3]),
                                      ([130, 64], [130, 1000]), ([17, 33], [2049, 33])])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (20, 3), (100, 40)])
def test_chunks(cuda_device, new, held, heads, kv, hd, page, dtype, window, sinks):
    table, lengths, starts, pages = batch_of(new, held, page, cuda_device)
    keys, values = filled(table, held, pages, kv, page, hd, dtype, cuda_device)
    g = torch.Generator().manual_seed(2)
    q = (2 * torch.randn(sum(new), heads, hd, generator=g)).to(dtype).to(cuda_device)
    out = cached_attention(q, keys, values, table, lengths, starts, max(new), window=window,
                           sinks=sinks)
    check(out, *reference(q, keys, values, table, new, held, window=window, sinks=sinks))


@pytest.mark.parametrize("heads,kv,hd,page", [(4, 4, 32, 16), (10, 2, 64, 32), (8, 1, 128, 64)])
@pytest.mark.parametrize("new,held", [([1], [1]), ([64], [64]), ([5, 0, 23, 64], [5, 0, 500, 1000]),
                                      ([33, 2], [2081, 34])])
@pytest.mark.parametrize("window,sinks", [(None, 0), (2, 0), (9, 4), (300, 40)])
def test_trees(cuda_device, new, held, heads, kv, hd, page, window, sinks):
    dtype = torch.bfloat16
    table, lengths, starts, pages = batch_of(new, held, page, cuda_device)
    keys, values = filled(table, held, pages, kv, page, hd, dtype, cuda_device)
    g = torch.Generator().manual_seed(2)
    q = (2 * torch.randn(sum(new), heads, hd, generator=g)).to(dtype).to(cuda_device)
    masks = trees(new)
    out = cached_attention(q, keys, values, table, lengths, starts, 64,
                           tree=signed(masks, cuda_device), window=window, sinks=sinks)
    check(out, *reference(q, keys, values, table, new, held, masks, window, sinks))


def test_a_chain_is_a_chunk(cuda_device):
    new, held = [30, 64], [130, 64]
    table, lengths, starts, pages = batch_of(new, held, 16, cuda_device)
    keys, values = filled(table, held, pages, 2, 16, 64, torch.float16, cuda_device)
    q = torch.randn(94, 4, 64, device=cuda_device).half()
    chain = [(2 << i) - 1 for n in new for i in range(n)]
    args = (q, keys, values, table, lengths, starts, 64)
    for span in ({}, {"window": 10, "sinks": 2}):
        ref, tol = reference(q, keys, values, table, new, held, **span)
        check(cached_attention(*args, **span), ref, tol)
        check(cached_attention(*args, tree=signed(chain, cuda_device), **span), ref, tol)


def test_masks_that_leave_nothing(cuda_device):
    """A token whose mask is empty and that has no context gets zeros; bits of tokens that its
    sequence does not have are not read."""
    new, held = [3, 2], [3, 12]
    table, lengths, starts, pages = batch_of(new, held, 16, cuda_device)
    keys, values = filled(table, held, pages, 1, 16, 32, torch.float16, cuda_device)
    q = torch.randn(5, 2, 32, device=cuda_device).half()
    masks = [0, 1, -8 & ((1 << 64) - 1), 0, 1 << 40 | 2]
    out = cached_attention(q, keys, values, table, lengths, starts, 3,
                           tree=signed(masks, cuda_device))
    assert out[0].eq(0).all() and out[2].eq(0).all()
    check(out, *reference(q, keys, values, table, new, held, [0, 1, 0, 0, 2]))


def test_rows_of_no_sequence_are_left(cuda_device):
    new, held = [2, 1], [40, 7]
    table, lengths, starts, pages = batch_of(new, held, 16, cuda_device)
    keys, values = filled(table, held, pages, 2, 16, 32, torch.float16, cuda_device)
    q = torch.randn(9, 4, 32, device=cuda_device).half()
    out = torch.full_like(q, 7.0)
    got = cached_attention(q, keys, values, table, lengths, starts, 2, out=out)
    assert got is out and out[3:].eq(7).all()
    check(out[:3], *reference(q[:3], keys, values, table, new, held))


def test_lengths_that_do_not_fit(cuda_device):
    """New tokens that a sequence does not hold see nothing in front of its first; a length beyond
    the page table is cut to it; pages that do not exist hold nothing."""
    table, _, starts, pages = batch_of([3], [32], 16, cuda_device, wide=0)
    keys, values = filled(table, [32], pages, 1, 16, 32, torch.float16, cuda_device)
    q = torch.randn(3, 1, 32, device=cuda_device).half()
    as_int = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda_device)
    short = cached_attention(q, keys, values, table, as_int(1), starts, 3)
    assert short[:2].eq(0).all()
    check(short[2:], *reference(q[2:], keys, values, table, [1], [1]))
    long = cached_attention(q, keys, values, table, as_int(4000), starts, 3)
    check(long, *reference(q, keys, values, table, [3], [32]))
    none = cached_attention(q, keys, values, table, as_int(-5), starts, 3)
    assert none.eq(0).all()
    # without its second page: as if the first were all (the new tokens lie behind it)
    lost = table.clone()
    for bad in (-1, pages, 1 << 30):
        lost[0, 1] = bad
        part = cached_attention(q, keys, values, lost, as_int(32), starts, 3)
        first = [reference(q[i:i + 1], keys, values, table, [1], [16]) for i in range(3)]
        check(part, torch.cat([r for r, _ in first]), torch.cat([t for _, t in first]))


def test_long_sequences_in_stretches(cuda_device):
    """Lengths of every order in one batch, cut into stretches of which many are empty."""
    new, held = [1, 1, 0, 1, 1], [20000, 3, 0, 5000, 129]
    table, lengths, starts, pages = batch_of(new, held, 64, cuda_device)
    keys, values = filled(table, held, pages, 2, 64, 128, torch.bfloat16, cuda_device)
    q = (3 * torch.randn(4, 8, 128, device=cuda_device)).bfloat16()
    out = cached_attention(q, keys, values, table, lengths, starts, 1)
    check(out, *reference(q, keys, values, table, new, held))
    spans = dict(window=4500, sinks=70)
    out = cached_attention(q, keys, values, table, lengths, starts, 1, **spans)
    check(out, *reference(q, keys, values, table, new, held, **spans))


def test_offsets_beyond_32_bits(cuda_device):
    """A cache of more than 2^31 elements; the tokens lie in its last pages."""
    pages, kv, page, hd = 70_000, 4, 64, 128
    keys, values = (torch.empty(pages, kv, page, hd, device=cuda_device, dtype=torch.float16)
                    for _ in range(2))
    assert keys.numel() > 1 << 31
    held = [150]
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32, device=cuda_device)
    ids = table[0].long()
    for c in (keys, values):
        c[ids] = torch.randn(3, kv, page, hd, device=cuda_device).half()
    lengths = torch.tensor(held, dtype=torch.int32, device=cuda_device)
    starts = torch.tensor([0, 2], dtype=torch.int32, device=cuda_device)
    slots, positions = cache_plan(table, lengths, starts, 2, page)
    assert slots.tolist() == [(pages - 2) * 64 + 20, (pages - 2) * 64 + 21]
    qkv = torch.randn(2, (8 + 2 * kv) * hd, device=cuda_device).half()
    q = append_kv(qkv, 8, keys, values, slots)
    out = cached_attention(q, keys, values, table, lengths, starts, 2)
    small = [c[ids] for c in (keys, values)]
    near = torch.tensor([[0, 1, 2]], dtype=torch.int32)
    check(out, *reference(q, *small, near, [2], held))
    x = qkv.view(2, 8 + 2 * kv, hd)
    assert torch.equal(keys[pages - 2, :, 20:22].transpose(0, 1), x[:, 8:8 + kv])
    assert torch.equal(values[pages - 2, :, 20:22].transpose(0, 1), x[:, 8 + kv:])


def test_strided_operands_and_tables(cuda_device):
    new, held = [2, 3], [50, 20]
    table, lengths, starts, pages = batch_of(new, held, 16, cuda_device)
    keys, values = filled(table, held, pages, 2, 16, 64, torch.float16, cuda_device)
    q = torch.randn(5, 4, 64, device=cuda_device).half()
    want = cached_attention(q, keys, values, table, lengths, starts, 3)
    wide = torch.zeros(5, 512, device=cuda_device).half()
    wide[:, 8:264] = q.view(5, 256)
    views = [wide[:, 8:264].view(5, 4, 64), q.transpose(0, 1).contiguous().transpose(0, 1)]
    odd = torch.zeros(5, 4 * 64 + 1, device=cuda_device).half()
    odd[:, 1:] = q.view(5, 256)
    views.append(odd[:, 1:].unflatten(1, (4, 64)))
    big = torch.full((2, 40), -3, dtype=torch.int32, device=cuda_device)
    big[:, 4:4 + table.shape[1]] = table
    for view in views:
        assert torch.equal(cached_attention(view, keys, values, table, lengths, starts, 3), want)
    assert torch.equal(cached_attention(q, keys, values, big[:, 4:4 + table.shape[1]], lengths,
                                        starts, 3), want)
    assert torch.equal(cached_attention(q, keys, values, table.t().contiguous().t(), lengths,
                                        starts, 3), want)


# ---------------------------------------------------------------------------
# appending
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("page", [16, 64])
def test_plan(cuda_device, page):
    new, held = [3, 0, 1, 20], [40, 9, 1, 20]
    table, lengths, starts, _ = batch_of(new, held, page, cuda_device)
    slots, positions = cache_plan(table, lengths, starts, 30, page)
    want = [s for slots_, n, t in zip(slots_of(table, held, page), new, held)
            for s in slots_[t - n:]]
    assert slots.tolist() == want + [-1] * 6
    places = [p for n, t in zip(new, held) for p in range(t - n, t)]
    assert positions.tolist() == places + [0] * 6
    masks = trees(new) + [0] * 6
    tree_slots, tree_positions = cache_plan(table, lengths, starts, 30, page,
                                            tree=signed(masks, cuda_device))
    assert torch.equal(tree_slots, slots)
    base = [t - n for n, t in zip(new, held) for _ in range(n)]
    assert tree_positions.tolist() == [c + bin(m).count("1") - 1
                                       for c, m in zip(base, masks)] + [0] * 6


def test_plan_of_tokens_without_pages(cuda_device):
    table = torch.tensor([[2, -1]], dtype=torch.int32, device=cuda_device)
    as_int = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda_device)
    slots, _ = cache_plan(table, as_int(17), as_int(0, 2), 2, 16)
    assert slots.tolist() == [47, -1]  # the second's page is missing
    slots, _ = cache_plan(table, as_int(40), as_int(0, 2), 2, 16)
    assert slots.tolist() == [-1, -1]  # past the table
    slots, positions = cache_plan(table, as_int(1), as_int(0, 2), 2, 16)
    assert slots.tolist() == [-1, 32] and positions.tolist() == [0, 0]
    empty, _ = cache_plan(table, as_int(1), as_int(0, 0), 0, 16)
    assert empty.shape == (0,)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,hd,page", [(1, 1, 32, 16), (6, 2, 64, 64), (10, 5, 128, 32)])
@pytest.mark.parametrize("style", [None, False, True])
def test_append(cuda_device, heads, kv, hd, page, style, dtype):
    """Bit for bit what rotate_qkv gives, at the slots; nothing else of the cache changes."""
    n, pages = 37, 12
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(n, (heads + 2 * kv) * hd, generator=g).to(dtype).to(cuda_device)
    keys, values = (torch.randn(pages, kv, page, hd, generator=g).to(dtype).to(cuda_device)
                    for _ in range(2))
    slots = torch.randperm(pages * page, generator=g)[:n].to(cuda_device)
    slots[5], slots[11], slots[20] = -1, pages * page, -(1 << 40)
    kept = [i for i in range(n) if i not in (5, 11, 20)]
    positions = torch.randint(0, 5000, (n,), generator=g, dtype=torch.int32).to(cuda_device)
    x = qkv
    rotary = None
    if style is not None:
        rotary = Rotary(hd, 5000, interleaved=style, device=cuda_device)
        x = rotate_qkv(qkv.unsqueeze(0), heads, rotary, positions.unsqueeze(0), kv_heads=kv)[0]
    x = x.view(n, heads + 2 * kv, hd)
    want = [c.clone() for c in (keys, values)]
    for c, part in zip(want, (x[:, heads:heads + kv], x[:, heads + kv:])):
        c[slots[kept] // page, :, slots[kept] % page] = part[kept]
    q = append_kv(qkv, heads, keys, values, slots, rotary, positions)
    assert torch.equal(q, x[:, :heads])
    assert torch.equal(keys, want[0]) and torch.equal(values, want[1])
    # strided rows, and none
    wide = torch.zeros(n, qkv.shape[1] + 16, device=cuda_device, dtype=dtype)
    wide[:, 8:-8] = qkv
    again = append_kv(wide[:, 8:-8], heads, keys, values, slots, rotary, positions)
    assert torch.equal(again, q) and torch.equal(keys, want[0])
    none = append_kv(qkv[:0], heads, keys, values, slots[:0], rotary, positions[:0])
    assert none.shape == (0, heads, hd)


def test_move(cuda_device):
    """All read before any is written; slots outside the cache are passed over."""
    from reversability_amd.cache import PagedCache
    held = PagedCache(2, 3, 16, 2, 32, torch.bfloat16, cuda_device)
    held.keys.normal_()
    held.values.normal_()
    before = [t.clone().transpose(2, 3).reshape(2, 48, 2, 32) for t in (held.keys, held.values)]
    as_slots = lambda *v: torch.tensor(v, dtype=torch.int64, device=cuda_device)
    held.move(as_slots(0, 17, 40, 5, -1, 48), as_slots(17, 40, 3, -1, 6, 7))
    for side, was in zip((held.keys, held.values), before):
        now = side.transpose(2, 3).reshape(2, 48, 2, 32)
        want = was.clone()
        want[:, [17, 40, 3]] = was[:, [0, 17, 40]]
        assert torch.equal(now, want)
    held.move(as_slots(), as_slots())


@pytest.mark.parametrize("heads,kv,hd,page", [(2, 2, 32, 16), (8, 2, 64, 32), (4, 1, 128, 16)])
@pytest.mark.parametrize("new,held", [([1], [90]), ([3], [90]), ([14], [75]), ([50, 2], [333, 40])])
@pytest.mark.parametrize("kind", ["chunk", "tree", "window"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_values_that_are_not_finite(cuda_device, heads, kv, hd, page, new, held, kind, bad):
    """A key or value that is not finite reaches the rows that see it, and in V the columns where
    it stands, and nothing else."""
    dtype = torch.bfloat16
    table, lengths, starts, pages = batch_of(new, held, page, cuda_device)
    keys, values = filled(table, held, pages, kv, page, hd, dtype, cuda_device, spread=0.5)
    g = torch.Generator().manual_seed(2)
    q = torch.randn(sum(new), heads, hd, generator=g).to(dtype).to(cuda_device)
    masks = trees(new) if kind == "tree" else None
    span = dict(window=20, sinks=2) if kind == "window" else {}
    slots = slots_of(table, held, page)
    for which, (n, total) in enumerate(zip(new, held)):
        # in front of the window, at its edge and among the new tokens
        spots = {5: (0, 3), max(0, total - n - 19): (0, 7), total - n // 2 - 1: (kv - 1, hd - 1)}
        for t, (head, column) in spots.items():
            slot = slots[which][t]
            values[slot // page, head, slot % page, column] = bad
        slot = slots[which][max(0, total - n - 21)]
        if kind == "window":  # outside every window
            keys[slot // page, :, slot % page] = bad
    out = cached_attention(q, keys, values, table, lengths, starts, max(new),
                           tree=None if masks is None else signed(masks, cuda_device), **span)
    clean = [c.nan_to_num(0.0, 0.0, 0.0) for c in (keys, values)]
    ref, tol = reference(q, *clean, table, new, held, masks, **span)
    # the same with the bad values marked: a row of ones where a row and column sees one
    mark = (~torch.isfinite(values)).to(dtype)
    for slot in set(range(pages * page)) - set(sum(slots, [])):
        mark[slot // page, :, slot % page] = 0
    hit, _ = reference(q, clean[0], mark, table, new, held, masks, **span)
    touched = hit > 0
    assert touched.any() and not touched.all()
    assert not torch.isfinite(out[touched]).any()
    if bad == math.inf:
        assert (out[touched] == math.inf).all()
    assert torch.isfinite(out[~touched]).all()
    check(out[~touched], ref[~touched], tol[~touched])


def test_infinite_scores_beside_a_value_that_is_not_finite(cuda_device):
    """Keys that no weight is left for, in front of a value that is made up for key by key."""
    table, lengths, starts, pages = batch_of([2], [100], 16, cuda_device)
    keys, values = filled(table, [100], pages, 1, 16, 32, torch.float16, cuda_device)
    slots = slots_of(table, [100], 16)[0]
    for j in range(70):
        keys[slots[j] // 16, 0, slots[j] % 16, 0] = -math.inf
    q = torch.zeros(2, 1, 32, device=cuda_device, dtype=torch.float16)
    q[:, 0, 0] = 1.0
    ref, tol = reference(q, keys, values, table, [2], [100])
    values[slots[99] // 16, 0, slots[99] % 16, 3] = math.nan  # the second token's own
    out = cached_attention(q, keys, values, table, lengths, starts, 2)
    check(out[:1], ref[:1], tol[:1])
    assert out[1, 0, 3].isnan() and out[1, 0, :3].isfinite().all()


def test_two_calls_at_once(cuda_device):
    """Calls on two streams, each with stretches of its own to join, and one after the other."""
    new, held = [1, 1, 1], [3000, 700, 1999]
    table, lengths, starts, pages = batch_of(new, held, 16, cuda_device)
    keys, values = filled(table, held, pages, 2, 16, 64, torch.float16, cuda_device)
    g = torch.Generator().manual_seed(5)
    qs = [torch.randn(3, 8, 64, generator=g).half().to(cuda_device) for _ in range(8)]
    call = lambda q: cached_attention(q, keys, values, table, lengths, starts, 1)
    want = [call(q) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i, q in enumerate(qs):
        with torch.cuda.stream(streams[i % 2]):
            got.append(call(q))
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_captured_step(cuda_device):
    """Plan, append and attention in two graphs that are alive together, replayed with other
    tokens, lengths and pages than they were captured with."""
    heads, kv, hd, page, rows = 8, 2, 64, 16, 6
    rotary = Rotary(hd, 4096, device=cuda_device)
    table, lengths, starts, pages = batch_of([1] * 4, [700, 90, 33, 16], page, cuda_device)
    keys, values = filled(table, [700, 90, 33, 16], pages, kv, page, hd, torch.float16,
                          cuda_device)
    qkv = torch.randn(rows, (heads + 2 * kv) * hd, device=cuda_device).half()

    def step():
        slots, positions = cache_plan(table, lengths, starts, rows, page)
        q = append_kv(qkv, heads, keys, values, slots, rotary, positions)
        return cached_attention(q, keys, values, table, lengths, starts, 1,
                                out=torch.zeros_like(q))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        graphs.append((graph, held))
    for seed, (new, total) in enumerate([([1] * 4, [700, 90, 33, 16]), ([1, 0, 1, 1], [9, 0, 500, 2]),
                                         ([0, 1, 0, 0], [0, 704, 0, 0])]):
        other, more, first, count = batch_of(new, total, page, cuda_device, seed=seed + 3)
        fresh = filled(other, total, pages, kv, page, hd, torch.float16, cuda_device, seed=seed)
        table.fill_(-1)
        table[:, :other.shape[1]] = other[:, :table.shape[1]]
        lengths.copy_(more)
        starts.copy_(first)
        qkv.normal_()
        for graph, held in graphs:
            keys.copy_(fresh[0])
            values.copy_(fresh[1])
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            after = [keys.clone(), values.clone()]
            got = held.clone()
            keys.copy_(fresh[0])
            values.copy_(fresh[1])
            assert torch.equal(got, step())
            assert all(torch.equal(a.nan_to_num(9), b.nan_to_num(9))
                       for a, b in zip(after, (keys, values)))


# ---------------------------------------------------------------------------
# a model over its cache
# ---------------------------------------------------------------------------
def _model(method, device, window, sinks, rotated, precision_fused):
    from reversability_amd import build_model
    from reversability_amd.attention import enable_attention
    from reversability_amd.linear import enable_linear
    from reversability_amd.optimized_v3 import install_v3
    config = {"model": {"vocab_size": 97, "max_sequence_length": 256, "n_layers": 3, "n_heads": 4,
                        "d_model": 128, "d_ff": 256}, "method": method}
    torch.manual_seed(9)
    model = build_model(config).to(device)
    if precision_fused:
        install_v3(model, core_mode="split" if method == "midpoint" else "reference",
                   mlp_tokens=64, swiglu=True, rmsnorm=True)
        enable_linear(model)
    rotary = Rotary(32, 256, device=device) if rotated else None
    enable_attention(model, window=window, sinks=sinks, rotary=rotary)
    return model


@pytest.mark.parametrize("method,fused", [("baseline", False), ("midpoint", False),
                                          ("midpoint", True), ("euler", False),
                                          ("euler", True), ("baseline", True)])
@pytest.mark.parametrize("window,sinks,rotated", [(None, 0, False), (20, 2, True)])
@pytest.mark.parametrize("precision", ["fp16", "bf16"])
def test_decode_matches_whole_sequences(cuda_device, method, fused, window, sinks, rotated,
                                        precision):
    """Prompts in chunks, then single tokens, then a checked tree of drafts: the logits are the
    model's own forward pass's on the whole sequences, within twice the type's roundings of
    values of their size (a layer rounds each of its products once)."""
    from reversability_amd.cache import CacheBatch, PagedCache, decode
    from reversability_amd.optimized import amp_context
    if fused and precision == "bf16":
        pytest.skip("the fused MLP is fp16's")
    dtype = {"fp16": torch.float16, "bf16": torch.bfloat16}[precision]
    model = _model(method, cuda_device, window, sinks, rotated, fused)
    g = torch.Generator().manual_seed(3)
    lens = [150, 7, 64]
    text = [torch.randint(0, 97, (n,), generator=g).to(cuda_device) for n in lens]

    def whole(ids):
        with torch.no_grad(), amp_context(ids.device, precision):
            return model(ids.unsqueeze(0))[0].float()
    cache = PagedCache.for_model(model, pages=20, page_size=16, dtype=dtype)
    order = torch.randperm(20, generator=g)
    table = torch.full((3, 12), -1, dtype=torch.int32)
    table[0, :11], table[1, :2], table[2, :5] = order[:11].int(), order[11:13].int(), order[13:18].int()
    table = table.to(cuda_device)
    as_int = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda_device)

    def feed(parts, done, tree=None, pad=0):
        new = [len(p) for p in parts]
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        ids = torch.cat([*parts, parts[0].new_zeros(pad)])
        held = [d + n for d, n in zip(done, new)]
        batch = CacheBatch(table, as_int(held), as_int(starts), max(new + [1]), 256, tree)
        out = decode(model, ids, cache, batch, precision=precision).float()
        return [out[a:b] for a, b in zip(starts, starts[1:])], held

    limit = 24 * torch.finfo(dtype).eps  # logits are of order 1 and less: 3 layers, 8 roundings
    done, got = [0, 0, 0], [[], [], []]
    for cut in ([100, 3, 40], [40, 0, 20], [9, 3, 3]):
        parts = [t[d:d + c] for t, d, c in zip(text, done, cut)]
        outs, done = feed(parts, done, pad=2)
        for a, o in zip(got, outs):
            a.append(o)
    outs, done = feed([t[d:d + 1] for t, d in zip(text, done)], done)
    for a, o in zip(got, outs):
        a.append(o)
    assert done == lens
    for ids, parts in zip(text, got):
        assert (torch.cat(parts) - whole(ids)).abs().max() <= limit
    # a tree behind each text: two branches, and the second's path kept
    tree = torch.tensor([0b1, 0b11, 0b101, 0b1101] * 3, dtype=torch.int64, device=cuda_device)
    drafts = [torch.randint(0, 97, (4,), generator=g).to(cuda_device) for _ in range(3)]
    outs, after = feed(drafts, done, tree=tree)
    for ids, draft, o in zip(text, drafts, outs):
        for path in ([0], [0, 1], [0, 2], [0, 2, 3]):
            want = whole(torch.cat([ids, draft[path]]))[-1]
            assert (o[path[-1]] - want).abs().max() <= limit
    batch = CacheBatch(table, as_int(after), as_int([0, 4, 8, 12]), 4, 256)
    slots, _ = cache_plan(table, batch.lengths, batch.starts, 12, 16)
    cache.move(slots.view(3, 4)[:, [2, 3]].reshape(-1), slots.view(3, 4)[:, [1, 2]].reshape(-1))
    kept = [d + 3 for d in done]
    last = [torch.randint(0, 97, (1,), generator=g).to(cuda_device) for _ in range(3)]
    outs, _ = feed(last, kept)
    for ids, draft, end, o in zip(text, drafts, last, outs):
        want = whole(torch.cat([ids, draft[[0, 2, 3]], end]))[-1]
        assert (o[0] - want).abs().max() <= limit


def test_decode_of_chosen_rows_and_refusals(cuda_device):
    from reversability_amd.cache import CacheBatch, PagedCache, decode
    model = _model("midpoint", cuda_device, 20, 2, True, False)
    cache = PagedCache.for_model(model, pages=4, page_size=16)
    as_int = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda_device)
    batch = CacheBatch(as_int([[0, 1], [2, 3]]), as_int([5, 3]), as_int([0, 5, 8]), 5, 32)
    ids = torch.randint(0, 97, (8,), device=cuda_device)
    whole = decode(model, ids, cache, batch)
    rows = torch.tensor([4, 7], device=cuda_device)
    # (the head's product over fewer rows may round otherwise)
    assert torch.allclose(decode(model, ids, cache, batch, rows=rows), whole[rows], atol=2e-3)
    with pytest.raises(ValueError, match="ids"):
        decode(model, ids.view(2, 4), cache, batch)
    with pytest.raises(ValueError, match="type"):
        append_kv(torch.zeros(8, 384, device=cuda_device, dtype=torch.bfloat16), 4,
                  cache.keys[0], cache.values[0], torch.zeros(8, dtype=torch.int64,
                                                             device=cuda_device))


def test_decode_of_a_padded_batch_and_of_nothing(cuda_device):
    """Rows of no sequence in front of and behind the others change neither those nor the cache."""
    from reversability_amd.cache import CacheBatch, PagedCache, decode
    model = _model("euler", cuda_device, 20, 2, True, False)
    caches = [PagedCache.for_model(model, pages=4, page_size=16) for _ in range(2)]
    as_int = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda_device)
    table, lengths = as_int([[0, 1], [2, 3]]), as_int([5, 3])
    ids = torch.randint(0, 97, (14,), device=cuda_device)
    want = decode(model, ids[2:10].clone(), caches[0],
                  CacheBatch(table, lengths, as_int([0, 5, 8]), 5, 32))
    got = decode(model, ids, caches[1], CacheBatch(table, lengths, as_int([2, 7, 10]), 5, 32))
    # (products over more rows may round otherwise)
    assert torch.allclose(got[2:10], want, atol=4e-3)
    assert torch.allclose(caches[0].keys, caches[1].keys, atol=4e-3)
    assert torch.allclose(caches[0].values, caches[1].values, atol=4e-3)
    before = caches[0].keys.clone()
    none = decode(model, ids[:0], caches[0], CacheBatch(table, lengths, as_int([0, 0, 0]), 1, 32))
    assert none.shape == (0, 97) and none.dtype == torch.float16
    assert torch.equal(caches[0].keys, before)


def test_captured_decode(cuda_device):
    """decode in a graph, replayed for other sequences, against eager calls on a cache of their
    own."""
    from reversability_amd.cache import CacheBatch, PagedCache, decode
    from reversability_amd.graph import CapturedStep
    model = _model("midpoint", cuda_device, 20, 2, True, True)
    as_int = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda_device)
    table = as_int([[3, 0, 5], [1, 4, 2]])
    caches = [PagedCache.for_model(model, pages=6, page_size=16) for _ in range(2)]
    prompt = torch.randint(0, 97, (30,), device=cuda_device)
    first = CacheBatch(table, as_int([20, 10]), as_int([0, 20, 30]), 20, 48)
    for cache in caches:
        decode(model, prompt, cache, first)
    ids, lengths = torch.zeros(2, dtype=torch.int64, device=cuda_device), as_int([21, 11])
    batch = CacheBatch(table, lengths, as_int([0, 1, 2]), 1, 48)
    step = CapturedStep(lambda: decode(model, ids, caches[0], batch))
    torch.cuda.synchronize()
    caches[0].keys.copy_(caches[1].keys)  # (the warm-up calls wrote the first token)
    caches[0].values.copy_(caches[1].values)
    for at in range(4):
        ids.copy_(torch.randint(0, 97, (2,), device=cuda_device))
        lengths.copy_(as_int([21 + at, 11 + at]))
        torch.cuda.synchronize()
        got = step().clone()
        torch.cuda.synchronize()
        assert torch.equal(got, decode(model, ids, caches[1], batch))
        assert torch.equal(caches[0].keys, caches[1].keys)


def test_refusals(cuda_device):
    """Arguments that the operators do not take, on the device and before any launch."""
    table, lengths, starts, pages = batch_of([1, 1], [20, 5], 16, cuda_device)
    keys, values = filled(table, [20, 5], pages, 2, 16, 32, torch.float16, cuda_device)
    q = torch.zeros(2, 4, 32, device=cuda_device, dtype=torch.float16)
    good = dict(q=q, keys=keys, values=values, page_table=table, lengths=lengths, starts=starts,
                max_query=1)
    cached_attention(**good)
    wide = torch.zeros(2, 4, 32, device=cuda_device, dtype=torch.int64)
    for bad in (dict(q=q.float()), dict(q=q.bfloat16()), dict(q=q[:, :3]), dict(q=q[..., :16]),
                dict(q=q[0]), dict(values=values[1:]), dict(values=values.bfloat16()),
                dict(keys=keys.transpose(2, 3)), dict(keys=keys[:, :, :8], values=values[:, :, :8]),
                dict(page_table=table.long()), dict(page_table=table[0]), dict(page_table=table[:1]),
                dict(lengths=lengths.long()), dict(starts=starts[1:]), dict(max_query=0),
                dict(max_length=0), dict(window=0), dict(sinks=-1), dict(tree=lengths),
                dict(max_query=65, tree=torch.zeros(100, dtype=torch.int64, device=cuda_device),
                     q=q.new_zeros(100, 4, 32)),
                dict(out=q.float()), dict(out=torch.empty_like(q).transpose(0, 1)), dict(out=q),
                dict(lengths=lengths.cpu())):
        with pytest.raises(ValueError):
            cached_attention(**{**good, **bad})
    with pytest.raises(ValueError, match="no_grad"):
        cached_attention(**{**good, "q": q.clone().requires_grad_(True)})
    with torch.no_grad():
        cached_attention(**{**good, "q": q.clone().requires_grad_(True)})
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q, torch.ones_like(q))
        with pytest.raises(NotImplementedError):
            cached_attention(**{**good, "q": dual})
    qkv = torch.zeros(2, 8 * 32, device=cuda_device, dtype=torch.float16)
    slots = torch.tensor([3, 4], device=cuda_device)
    rotary = Rotary(32, 8, device=cuda_device)
    for bad in (dict(heads=3), dict(heads=5), dict(slots=slots[:1]), dict(slots=slots.int()),
                dict(rotary=rotary), dict(rotary=Rotary(64, 8, device=cuda_device),
                                          positions=slots.int()),
                dict(rotary=rotary, positions=slots), dict(qkv=qkv[:, :-32])):
        with pytest.raises(ValueError):
            append_kv(**{**dict(qkv=qkv, heads=4, keys=keys, values=values, slots=slots), **bad})
    for bad in (dict(page_size=24), dict(tokens=-1), dict(tree=wide[0, 0, :3])):
        with pytest.raises(ValueError):
            cache_plan(**{**dict(page_table=table, lengths=lengths, starts=starts, tokens=2,
                                 page_size=16), **bad})
