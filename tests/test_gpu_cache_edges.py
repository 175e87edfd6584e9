"""Calls at the edges of the paged cache: pages that hold only some of a sequence's new tokens.
Bounds are test_gpu_cache.py's."""
from __future__ import annotations

import math

import pytest
import torch

from reversability_amd.cache import append_kv, cache_plan, cached_attention
from test_gpu_cache import (_model, batch_of, check, filled, reference, signed, slots_of,
                            trees)

pytestmark = pytest.mark.gpu


def seen_by(new, total, kept, masks, window, sinks):
    """[new, kept]: which of the ``kept`` slots the last ``new`` of ``total`` tokens see."""
    context, low = total - new, (1 << new) - 1
    place = list(range(total))
    if masks is not None:
        for i in range(new):
            place[context + i] = context + bin(masks[i] & low).count("1") - 1
    seen = torch.zeros(new, kept, dtype=torch.bool)
    for i in range(new):
        for j in range(kept):
            order = j <= context + i if masks is None else (
                j < context or bool(masks[i] >> (j - context) & 1))
            seen[i, j] = order and (window is None or place[context + i] - place[j] < window
                                    or place[j] < sinks)
    return seen


def attend(q, k, v, seen):
    """fp64 outputs of q [n, heads, hd] over k, v [kept, kv, hd], and their bounds."""
    heads, hd = q.shape[1:]
    u = torch.finfo(q.dtype).eps / 2
    sub = torch.finfo(q.dtype).smallest_normal * u
    k, v = (t.double().transpose(0, 1).repeat_interleave(heads // k.shape[1], 0).contiguous()
            for t in (k, v))
    seen = seen.to(q.device)
    score = q.double().transpose(0, 1).contiguous() @ k.transpose(1, 2).contiguous() / math.sqrt(hd)
    p = torch.softmax(score.masked_fill(~seen, -math.inf), -1).nan_to_num(0.0)
    out = p @ v
    few = seen.sum(1).view(1, -1, 1)
    tol = 2 * (u * (p @ v.abs()) + u * out.abs() + sub * (1 + few * v.abs().max()))
    return out.transpose(0, 1), tol.transpose(0, 1)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,hd", [(2, 2, 32), (8, 2, 64), (12, 1, 128)])
@pytest.mark.parametrize("new,over", [(4, 2), (1, 0), (30, 29), (30, 5), (64, 1)])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("window,sinks", [(None, 0), (9, 3)])
def test_pages_that_hold_some_of_the_new_tokens(cuda_device, new, over, heads, kv, hd, dtype, tree,
                                                window, sinks):
    """Plan, append and attention agree on where the new tokens are: those that the pages hold see
    themselves and what is in front of them, the ``over`` others what is held."""
    page, kept = 16, 80
    total = kept + over
    table, _, starts, pages = batch_of([new], [kept], page, cuda_device, wide=0)
    lengths = torch.tensor([total], dtype=torch.int32, device=cuda_device)
    held = total - new  # the context
    keys, values = filled(table, [held], pages, kv, page, hd, dtype, cuda_device)
    g = torch.Generator().manual_seed(4)
    qkv = (1.5 * torch.randn(new, (heads + 2 * kv) * hd, generator=g)).to(dtype).to(cuda_device)
    masks = trees([new]) if tree else None
    bits = signed(masks, cuda_device) if tree else None
    slots, _ = cache_plan(table, lengths, starts, new, page, tree=bits)
    every = slots_of(table, [kept], page)[0]
    assert slots.tolist() == every[held:] + [-1] * over
    q = append_kv(qkv, heads, keys, values, slots)
    out = cached_attention(q, keys, values, table, lengths, starts, new, tree=bits, window=window,
                           sinks=sinks)
    at = torch.tensor(every, device=cuda_device)
    k, v = (c.transpose(1, 2).reshape(-1, kv, hd)[at] for c in (keys, values))
    check(out, *attend(q, k, v, seen_by(new, total, kept, masks, window, sinks)))


def test_outputs_in_the_cache_are_refused(cuda_device):
    table, lengths, starts, pages = batch_of([1, 1], [20, 5], 16, cuda_device)
    keys, values = filled(table, [20, 5], pages, 2, 16, 32, torch.float16, cuda_device)
    q = torch.randn(2, 4, 32, device=cuda_device).half()
    for side in (keys, values):
        before = side.clone()
        for first in (0, side.numel() - 256):
            out = side.view(-1)[first:first + 256].view(2, 4, 32)
            with pytest.raises(ValueError, match="overlap"):
                cached_attention(q, keys, values, table, lengths, starts, 1, out=out)
        assert torch.equal(side.nan_to_num(9), before.nan_to_num(9))


def test_lone_rows_of_any_stride(cuda_device):
    """One token, one sequence, one head, one page: torch lets the stride of a size of one be
    anything, and calls it contiguous."""
    table, lengths, starts, pages = batch_of([1], [40], 16, cuda_device)
    keys, values = filled(table, [40], pages, 2, 16, 64, torch.float16, cuda_device)
    plain = torch.randn(1, 4, 64, device=cuda_device).half()
    want = cached_attention(plain, keys, values, table, lengths, starts, 1)
    wide = torch.zeros(1, 515, device=cuda_device, dtype=torch.float16)
    wide[:, :256] = plain.view(1, 256)
    shifted = torch.zeros(1, 515, device=cuda_device, dtype=torch.float16)
    shifted[:, 1:257] = plain.view(1, 256)
    for q in (plain.transpose(0, 1).contiguous().transpose(0, 1), wide[:, :256].view(1, 4, 64),
              shifted[:, 1:257].view(1, 4, 64), plain.as_strided(plain.shape, (0, 64, 1)),
              plain.as_strided(plain.shape, (3, 64, 1))):
        out = torch.empty_like(want)
        assert torch.equal(cached_attention(q, keys, values, table, lengths, starts, 1), want)
        assert cached_attention(q, keys, values, table, lengths, starts, 1, out=out) is out
        assert torch.equal(out, want)
    turned = table.reshape(-1, 1).clone().t()  # one sequence: strides (1, 1)
    assert turned.stride() == (1, 1) and torch.equal(turned, table)
    assert torch.equal(cached_attention(plain, keys, values, turned, lengths, starts, 1), want)
    slots, positions = cache_plan(table, lengths, starts, 1, 16)
    for got, ref in zip(cache_plan(turned, lengths, starts, 1, 16), (slots, positions)):
        assert torch.equal(got, ref)
    lone = table[:, :1]  # one page, of every stride
    few = torch.tensor([9], dtype=torch.int32, device=cuda_device)
    first = cached_attention(plain, keys, values, lone.contiguous(), few, starts, 1)
    for strides in ((1, 1), (0, 7), (7, 0), (1, 5)):
        odd = lone.as_strided((1, 1), strides)
        assert torch.equal(cached_attention(plain, keys, values, odd, few, starts, 1), first)
    # one row to append, from rows of a stride that no two rows could have
    qkv = torch.randn(1, 512, device=cuda_device).half()
    after = []
    for rows in (qkv, torch.cat([qkv, qkv[:, :3]], 1)[:, :512], qkv.as_strided((1, 512), (5, 1)),
                 torch.cat([qkv[:, :1], qkv], 1)[:, 1:], qkv.as_strided((1, 1, 512), (7, 3, 1))):
        kept = [c.clone() for c in (keys, values)]
        q = append_kv(rows, 4, *kept, slots)
        assert torch.equal(q, qkv[:, :256].view(1, 4, 64))
        # (q, a view of such rows, goes on to the attention)
        after.append([cached_attention(q, *kept, table, lengths, starts, 1), *kept])
    for other in after[1:]:
        assert all(torch.equal(a.nan_to_num(9), b.nan_to_num(9)) for a, b in zip(after[0], other))
    # one head
    table, lengths, starts, pages = batch_of([2], [20], 16, cuda_device)
    keys, values = filled(table, [20], pages, 1, 16, 32, torch.float16, cuda_device)
    q = torch.randn(2, 1, 32, device=cuda_device).half()
    want = cached_attention(q, keys, values, table, lengths, starts, 2)
    odd = q.as_strided((2, 1, 32), (32, 5, 1))
    assert torch.equal(cached_attention(odd, keys, values, table, lengths, starts, 2), want)


@pytest.fixture
def marked_memory():
    """New tensors that nothing is written to hold NaN."""
    torch.use_deterministic_algorithms(True, warn_only=True)
    assert torch.utils.deterministic.fill_uninitialized_memory
    yield
    torch.use_deterministic_algorithms(False)


@pytest.mark.parametrize("method,fused", [("baseline", False), ("midpoint", True), ("euler", False)])
def test_decode_appends_nothing_that_was_not_computed(cuda_device, marked_memory, method, fused):
    """Rows of no sequence, and tokens past ``max_query``: finite logits, keys and values, and the
    other sequence's as without them."""
    from reversability_amd.cache import CacheBatch, PagedCache, decode
    model = _model(method, cuda_device, 20, 2, True, fused)
    as_int = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda_device)
    table = as_int([[0, 1], [2, 3]])
    ids = torch.randint(0, 97, (12,), device=cuda_device)
    caches = [PagedCache.for_model(model, pages=4, page_size=16) for _ in range(2)]
    # five new tokens and two where two are allowed; three rows of no sequence
    logits = decode(model, ids, caches[0], CacheBatch(table, as_int([5, 2]), as_int([1, 6, 8]), 2, 32))
    assert torch.isfinite(logits).all()
    assert all(torch.isfinite(t).all() for t in (caches[0].keys, caches[0].values))
    want = decode(model, ids[6:8].clone(), caches[1],
                  CacheBatch(table[1:], as_int([2]), as_int([0, 2]), 2, 32))
    # (products over more rows may round otherwise)
    assert torch.allclose(logits[6:8], want, atol=4e-3)
    for a, b in ((caches[0].keys, caches[1].keys), (caches[0].values, caches[1].values)):
        assert torch.allclose(a[:, 2:], b[:, 2:], atol=4e-3)


@pytest.mark.parametrize("heads,kv,hd,page", [(4, 4, 32, 16), (10, 2, 64, 32), (8, 1, 128, 64)])
@pytest.mark.parametrize("new,held", [([64], [64]), ([5, 0, 23, 64], [5, 0, 500, 1000]),
                                      ([33, 2], [2081, 34])])
@pytest.mark.parametrize("window,sinks", [(None, 0), (2, 0), (300, 40)])
def test_trees_in_fp16(cuda_device, new, held, heads, kv, hd, page, window, sinks):
    """Up to 512 rows that share a key head, at every head size."""
    table, lengths, starts, pages = batch_of(new, held, page, cuda_device)
    keys, values = filled(table, held, pages, kv, page, hd, torch.float16, cuda_device)
    g = torch.Generator().manual_seed(2)
    q = (2 * torch.randn(sum(new), heads, hd, generator=g)).half().to(cuda_device)
    masks = trees(new)
    out = cached_attention(q, keys, values, table, lengths, starts, 64,
                           tree=signed(masks, cuda_device), window=window, sinks=sinks)
    check(out, *reference(q, keys, values, table, new, held, masks, window, sinks))


@pytest.mark.parametrize("method", ["baseline", "midpoint", "euler"])
def test_decode_of_fused_models_in_bf16(cuda_device, method):
    """install_v3 without its fp16 MLP: the logits are the model's own on the whole sequence, within
    twice bf16's roundings of values of order 1 (3 layers of 8)."""
    from reversability_amd import build_model
    from reversability_amd.attention import enable_attention
    from reversability_amd.cache import CacheBatch, PagedCache, decode
    from reversability_amd.optimized import amp_context
    from reversability_amd.optimized_v3 import install_v3
    config = {"model": {"vocab_size": 97, "max_sequence_length": 256, "n_layers": 3, "n_heads": 4,
                        "d_model": 128, "d_ff": 256}, "method": method}
    torch.manual_seed(9)
    model = build_model(config).to(cuda_device)
    install_v3(model, core_mode="split" if method == "midpoint" else "reference", rmsnorm=True)
    enable_attention(model, window=20, sinks=2)
    ids = torch.randint(0, 97, (50,), device=cuda_device)
    with torch.no_grad(), amp_context(cuda_device, "bf16"):
        want = model(ids.unsqueeze(0))[0].float()
    cache = PagedCache.for_model(model, pages=4, page_size=16, dtype=torch.bfloat16)
    as_int = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda_device)
    got = []
    for first, last in ((0, 30), (30, 49), (49, 50)):
        batch = CacheBatch(as_int([[2, 0, 3, 1]]), as_int([last]), as_int([0, last - first]),
                           last - first, 64)
        got.append(decode(model, ids[first:last], cache, batch, precision="bf16").float())
    assert (torch.cat(got) - want).abs().max() <= 24 * torch.finfo(torch.bfloat16).eps


def test_decode_runs_on_its_tensors_device(cuda_device, monkeypatch):
    """Every module of the model runs while the cache's device is the current one."""
    from reversability_amd import cache as module
    depth, seen = [0], []

    class Guard(module._DeviceGuard):
        def __enter__(self):
            assert self.index == cuda_device.index
            depth[0] += 1
            return super().__enter__()

        def __exit__(self, *exc):
            depth[0] -= 1
            return super().__exit__(*exc)
    monkeypatch.setattr(module, "_DeviceGuard", Guard)
    model = _model("midpoint", cuda_device, 20, 2, True, True)
    for name, part in model.named_modules():
        part.register_forward_pre_hook(lambda *_, name=name: seen.append((name, depth[0])))
    as_int = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda_device)
    held = module.PagedCache.for_model(model, pages=2, page_size=16)
    batch = module.CacheBatch(as_int([[0, 1]]), as_int([3]), as_int([0, 3]), 3, 32)
    module.decode(model, torch.randint(0, 97, (3,), device=cuda_device), held, batch)
    names = {name for name, _ in seen}
    assert {"token_embedding", "blocks.0.attn.qkv", "blocks.2.mlp", "lm_head"} <= names
    assert all(inside for _, inside in seen) and depth[0] == 0


def test_weight_casts_stay_on_their_stream(cuda_device):
    """Two threads that answer at once, each on a stream of its own: a cast that one of them made is
    not handed to the other, whose stream does not wait for it."""
    from reversability_amd import mlp
    w = torch.randn(64, 64, device=cuda_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with mlp.weight_cast_cache():
        for make in (lambda: mlp.prefetch_casts([w]), lambda: None):
            make()
            own = mlp.cast_weight(w)
            assert mlp.cast_weight(w) is own
            with torch.cuda.stream(side):
                other = mlp.cast_weight(w)
                assert other is not own and other.data_ptr() != own.data_ptr()
            side.synchronize()
            assert torch.equal(own, other) and mlp.cast_weight(w) is own


def test_decode_on_two_threads(cuda_device):
    """Two threads, streams and caches, one model: each thread's logits and cache are those of its
    calls one after the other."""
    import threading

    from reversability_amd.cache import CacheBatch, PagedCache, decode
    model = _model("midpoint", cuda_device, 20, 2, True, True)
    as_int = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda_device)
    ids = torch.randint(0, 97, (2, 24), device=cuda_device)

    def answer(which):
        cache = PagedCache.for_model(model, pages=2, page_size=16)
        out = []
        for n in range(8):
            batch = CacheBatch(as_int([[1, 0]]), as_int([3 * n + 3]), as_int([0, 3]), 3, 32)
            out.append(decode(model, ids[which, 3 * n:3 * n + 3], cache, batch))
        torch.cuda.current_stream().synchronize()
        return torch.cat(out), cache.keys, cache.values
    want = [answer(i) for i in (0, 1)]
    torch.cuda.synchronize()
    got = [None, None]

    def run(which):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[which] = answer(which)
    threads = [threading.Thread(target=run, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
