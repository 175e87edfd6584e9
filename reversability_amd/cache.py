"""Answering with a model: a paged cache of keys and values, and the attention of new
tokens over it, on gfx950 kernels.

The reference trains and evaluates whole sequences (src/reversibility/model.py:26-45);
sampled answers, as ``preference.policy_backward`` takes them, need one token at a time.

* ``PagedCache``: keys and values of every layer in pages of 16 to 256 tokens.
* ``cache_plan``: where the new tokens of a batch of sequences go, and their positions.
* ``append_kv``: the packed projection's keys and values into the cache, keys and
  queries rotated by position on the way.
* ``cached_attention``: attention of the new tokens over the cache -- one token a sequence,
  a chunk of a prompt, or a tree of drafted tokens -- with the window and the sinks of
  ``attention.window_attention``.
* ``decode(model, ...)``: a model's logits for new tokens, with the settings of
  ``attention.enable_attention``.

A batch of sequences is described on the device (so that a captured call can be replayed
with other sequences): ``page_table`` int32 [sequences, pages of the longest], ``lengths``
int32 [sequences]: tokens a sequence holds, the new ones included, ``starts`` int32
[sequences + 1]: sequence b's new tokens are rows starts[b] .. starts[b + 1] - 1 of the
batch.  A sequence without new tokens is passed over, and so are rows behind the last one
(a padded batch).  A tree of drafted tokens is an int64 mask per new token: bit i says that
it sees the i-th new token of its sequence (its path from the root, itself included).

Nothing here is differentiable, and there is no CPU fallback.
"""
from __future__ import annotations

import functools
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import paths
from ._hip import _check, _DeviceGuard, _stream, library
from .attention import _CODES, HEAD_DIMS, Rotary, check_window, packed_heads
from .kernels_v3 import add_rms_norm
from .mlp import prefetch_casts, weight_cast_cache
from .optimized import _AMP_DTYPES, amp_context
from .residual import euler_step, midpoint_step

PAGE_SIZES = (16, 32, 64, 128, 256)


# These operators run once a layer and token, on calls of a few microseconds: what is checked is
# checked without building anything.
def _no_graph(what: str, *tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                raise ValueError(f"{what} is not differentiable: call it under torch.no_grad()")
    if getattr(forward_ad, "_current_level", 0) >= 0:  # (no dual tensors outside a level)
        for t in tensors:
            if forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{what} has no forward-mode derivative")


def _check_cache(keys: torch.Tensor, values: torch.Tensor, what: str) -> None:
    if (not keys.is_cuda or keys.dtype not in _CODES or keys.ndim != 4 or not keys.numel()
            or keys.shape[2] not in PAGE_SIZES or keys.shape[3] not in HEAD_DIMS):
        raise ValueError(f"{what} needs a CUDA (ROCm device) fp16 or bf16 cache [pages, kv_heads, "
                         f"page size in {PAGE_SIZES}, head size in {HEAD_DIMS}]; no silent "
                         "fallback")
    if (values.shape != keys.shape or values.dtype != keys.dtype or values.device != keys.device
            or not keys.is_contiguous() or not values.is_contiguous()
            or keys.data_ptr() % 16 or values.data_ptr() % 16):
        raise ValueError(f"{what} needs contiguous, 16-byte aligned keys and values of one shape")


def _ints(t: torch.Tensor, shape: tuple, like: torch.Tensor, what: str,
          dtype=torch.int32) -> torch.Tensor:
    if t.dtype != dtype or tuple(t.shape) != shape or t.device != like.device:
        raise ValueError(f"{what} must be {str(dtype)[6:]} {list(shape)} on the cache's device")
    return t.contiguous()


def _row_stride(t: torch.Tensor, width: int) -> int:
    """The stride of rows of ``width``.  That of a lone row may be anything (torch ignores it, and
    ``contiguous()`` leaves it): it has no next row, and gets its width."""
    return t.stride(0) if t.shape[0] > 1 else width


def _sequences(page_table, lengths, starts, like, what):
    """The batch's description, checked; the page table keeps its row stride, which is returned
    behind it."""
    if (page_table.dtype != torch.int32 or page_table.ndim != 2 or not page_table.numel()
            or page_table.device != like.device):
        raise ValueError(f"{what} needs an int32 page_table [sequences, pages] on its device")
    seqs = page_table.shape[0]
    columns = page_table.shape[1]
    if page_table.stride(1) != 1 or _row_stride(page_table, columns) < columns:
        page_table = page_table.contiguous()
    return (page_table, _row_stride(page_table, columns), _ints(lengths, (seqs,), like, "lengths"),
            _ints(starts, (seqs + 1,), like, "starts"))


def cache_plan(page_table: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor,
               tokens: int, page_size: int, tree: Optional[torch.Tensor] = None) -> tuple:
    """(slots int64 [tokens], positions int32 [tokens]) of a batch's rows: a slot is page *
    page_size + row of the cache, -1 for rows of no sequence and tokens that their sequence's
    pages do not hold (or whose page is negative); a position counts from the sequence's
    first token (with ``tree``: the last token in front of the new ones, plus the token's
    bits)."""
    if not page_table.is_cuda or page_size not in PAGE_SIZES or tokens < 0:
        raise ValueError(f"cache_plan needs CUDA (ROCm device) tensors, a page size in "
                         f"{PAGE_SIZES} and tokens >= 0")
    table, ld, lengths, starts = _sequences(page_table, lengths, starts, page_table, "cache_plan")
    if tree is not None:
        tree = _ints(tree, (tokens,), table, "tree", torch.int64)
    slots = torch.empty(tokens, device=table.device, dtype=torch.int64)
    positions = torch.empty(tokens, device=table.device, dtype=torch.int32)
    with _DeviceGuard(table):
        if tokens:
            _check(library().rv_cache_plan(
                table.data_ptr(), ld, table.shape[1], lengths.data_ptr(),
                starts.data_ptr(), None if tree is None else tree.data_ptr(), table.shape[0],
                tokens, page_size, slots.data_ptr(), positions.data_ptr(), _stream(table)),
                "rv_cache_plan")
    return slots, positions


def append_kv(qkv: torch.Tensor, heads: int, keys: torch.Tensor, values: torch.Tensor,
              slots: torch.Tensor, rotary: Optional[Rotary] = None,
              positions: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Writes the keys and values of packed rows ``qkv`` [..., (heads + 2 kv_heads) hd] into
    their ``slots`` (int64, one per row) of a layer's ``keys`` and ``values`` [pages, kv_heads,
    page size, hd], and returns the queries [rows, heads, hd].  With ``rotary``, queries and
    keys are rotated by ``positions`` (int32, one per row; outside the table: NaN) as
    ``rotate_qkv`` does; without, the queries are a view of ``qkv``.  A slot outside the cache
    is not written; the slots of one call must differ.  All of one type, fp16 or bf16."""
    _check_cache(keys, values, "append_kv")
    _no_graph("append_kv", qkv, keys, values)
    kv, hd = packed_heads(qkv, heads, keys.shape[1], "append_kv")
    if qkv.dtype != keys.dtype or qkv.device != keys.device or hd != keys.shape[3]:
        raise ValueError("append_kv needs qkv of the cache's type, head size and device")
    rows = qkv if qkv.ndim == 2 else qkv.reshape(-1, qkv.shape[-1])
    n, width = rows.shape
    ld = _row_stride(rows, width)
    if rows.stride(1) != 1 or ld % 8 or ld < width:
        rows, ld = rows.contiguous(), width
    if rows.data_ptr() % 16:
        rows, ld = rows.clone(memory_format=torch.contiguous_format), width
    slots = _ints(slots, (n,), keys, "slots", torch.int64)
    turn = (None, 0, None, False)
    if rotary is None:
        q = rows[:, :heads * hd].view(n, heads, hd)
    else:
        rotary.check(qkv, hd, "append_kv")
        if positions is None:
            raise ValueError("append_kv needs positions to rotate by")
        positions = _ints(positions, (n,), keys, "positions")
        turn = (rotary.table.data_ptr(), rotary.positions, positions.data_ptr(),
                rotary.interleaved)
        q = torch.empty(n, heads, hd, device=qkv.device, dtype=qkv.dtype)
    paths.took("append_kv", "hip")
    if n:
        with _DeviceGuard(keys):
            _check(library().rv_append_kv(
                rows.data_ptr(), ld, q.data_ptr() if rotary is not None else None,
                keys.data_ptr(), values.data_ptr(), slots.data_ptr(), n, heads, kv, hd,
                _CODES[keys.dtype], keys.shape[0], keys.shape[2], *turn, _stream(keys)),
                "rv_append_kv")
    return q


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(*sizes) -> int:
    nbytes = library().rv_cached_attn_workspace_bytes(*sizes)
    if nbytes < 0:
        _check(-nbytes, "rv_cached_attn_workspace_bytes")
    return nbytes


def cached_attention(q: torch.Tensor, keys: torch.Tensor, values: torch.Tensor,
                     page_table: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor,
                     max_query: int, *, max_length: Optional[int] = None,
                     tree: Optional[torch.Tensor] = None, window: Optional[int] = None,
                     sinks: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of a batch's new tokens over the cache they were appended to.

    ``q`` [tokens, heads, hd] of the cache's type; ``keys`` and ``values`` a layer's [pages,
    kv_heads, page size, hd]; heads a multiple of kv_heads.  ``max_query``: the most new
    tokens of a sequence (later ones are passed over).  ``max_length``: the most tokens that
    a sequence holds, for the division of the work (None: what the page table can hold; a
    longer sequence is still right, but slower).  ``tree`` int64 [tokens]: masks of drafted
    tokens (``max_query`` at most 64).  A new token sees the slots up to its own, or with
    ``tree`` its context and what its mask has; with ``window`` of these the tokens less than
    ``window`` positions before it and the first ``sinks`` positions.  A token that sees
    nothing gets zeros.  Returns ``out`` (contiguous, q's shape and type; None: a new
    tensor; memory of its own), whose rows of no sequence are left as they were.

    New tokens that their sequence's pages have no room for see what the pages hold, the others
    are where ``cache_plan`` puts them (a sequence without room for its first new token is
    cut to its pages).
    Slots that no sequence's tokens hold are never used, whatever they contain.  Scores,
    statistics and sums in fp32, the weights rounded to the cache's type for the product with
    the values.  Deterministic."""
    _check_cache(keys, values, "cached_attention")
    _no_graph("cached_attention", q, keys, values)
    pages, kv, page, hd = keys.shape
    if (q.ndim != 3 or q.dtype != keys.dtype or q.device != keys.device or q.shape[2] != hd
            or not q.shape[1] or q.shape[1] % kv):
        raise ValueError("cached_attention needs q [tokens, heads, hd] of the cache's type, head "
                         "size and device, heads a multiple of its kv_heads")
    check_window(window, sinks, "cached_attention")
    tokens, heads = q.shape[:2]
    table, table_ld, lengths, starts = _sequences(page_table, lengths, starts, keys,
                                                  "cached_attention")
    held = table.shape[1] * page
    if max_query < 1 or (max_length is not None and max_length < 1):
        raise ValueError("cached_attention needs max_query and max_length >= 1")
    max_query, max_length = min(max_query, max(1, tokens)), min(max_length or held, held)
    if tree is not None:
        tree = _ints(tree, (tokens,), keys, "tree", torch.int64)
        if max_query > 64:
            raise ValueError("cached_attention takes trees of at most 64 tokens a sequence")
    q_ld = _row_stride(q, heads * hd)
    if (q.stride(2) != 1 or q.stride(1) != hd or q_ld % 8 or q_ld < heads * hd
            or q.data_ptr() % 16):
        q, q_ld = q.contiguous(), heads * hd
        q = q if q.data_ptr() % 16 == 0 else q.clone()
    if out is None:
        out = (torch.empty_like(q) if q.is_contiguous() else
               torch.empty(tokens, heads, hd, device=q.device, dtype=q.dtype))
    elif (out.shape != q.shape or out.dtype != q.dtype or out.device != q.device
          or not out.is_contiguous() or out.data_ptr() % 16):
        raise ValueError("out must be a contiguous, 16-byte aligned tensor like q")
    else:
        first, last = out.data_ptr(), out.data_ptr() + out.numel() * 2
        for t, values_of in ((q, q_ld * (tokens - 1) + heads * hd), (keys, keys.numel()),
                             (values, keys.numel())):
            if tokens and first < t.data_ptr() + values_of * 2 and t.data_ptr() < last:
                raise ValueError("out must not overlap q, keys or values")
    paths.took("cached_attention", "hip")
    if not tokens:
        return out
    lib, span = library(), (window or 0, sinks if window else 0)
    sizes = (tokens, table.shape[0], heads, kv, hd)
    nbytes = _workspace_bytes(*sizes, max_query, max_length, *span)
    with _DeviceGuard(q):
        ws = torch.empty(nbytes, device=q.device, dtype=torch.uint8) if nbytes else None
        _check(lib.rv_cached_attn(
            q.data_ptr(), q_ld, keys.data_ptr(), values.data_ptr(), table.data_ptr(),
            table_ld, table.shape[1], lengths.data_ptr(), starts.data_ptr(),
            None if tree is None else tree.data_ptr(), *sizes, _CODES[q.dtype], pages, page,
            max_query, max_length, *span, out.data_ptr(), None if ws is None else ws.data_ptr(),
            nbytes, _stream(q)), "rv_cached_attn")
    return out


# ---------------------------------------------------------------------------
# a model over its cache
# ---------------------------------------------------------------------------
class PagedCache:
    """Keys and values of every layer of a model: ``keys[layer]`` and ``values[layer]`` are
    [pages, kv_heads, page_size, head_dim].  Which pages belong to which sequence is the
    caller's (its page table)."""

    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.float16, device="cuda"):
        if (layers < 1 or pages < 1 or page_size not in PAGE_SIZES or kv_heads < 1
                or head_dim not in HEAD_DIMS or dtype not in _CODES):
            raise ValueError(f"PagedCache needs fp16 or bf16 pages of {PAGE_SIZES} tokens and a "
                             f"head size in {HEAD_DIMS}")
        self.page_size = page_size
        both = torch.zeros(2, layers, pages, kv_heads, page_size, head_dim, device=device,
                           dtype=dtype)
        self.keys, self.values = both[0], both[1]

    @classmethod
    def for_model(cls, model, pages: int, page_size: int = 64,
                  dtype: torch.dtype = torch.float16) -> "PagedCache":
        attn = model.blocks[0].attn
        return cls(len(model.blocks), pages, page_size, attn.n_heads, attn.head_dim, dtype,
                   model.lm_head.weight.device)

    @torch.no_grad()
    def move(self, source: torch.Tensor, target: torch.Tensor) -> None:
        """Copies the tokens at the slots ``source`` to the slots ``target`` (int64 [n]) in every
        layer, all read before any is written: what is kept of a checked tree goes behind its
        context.  A pair with a slot outside the cache (as ``cache_plan``'s -1) is passed over;
        the others' targets must differ."""
        layers, pages, kv, size, hd = self.keys.shape
        n = _ints(source, tuple(source.shape), self.keys, "source", torch.int64).numel()
        if source.ndim != 1:
            raise ValueError("move needs lists of slots")
        target = _ints(target, (n,), self.keys, "target", torch.int64)
        _check_cache(self.keys[0], self.values[0], "move")
        inside = (source >= 0) & (source < pages * size)
        target = torch.where(inside, target, -1)
        at = source.clamp(0, pages * size - 1)
        page, row = at // size, at % size
        # packed rows of kv heads each: queries (not read), keys, values
        rows = torch.empty(layers, n, 3, kv, hd, device=self.keys.device, dtype=self.keys.dtype)
        for i, side in ((1, self.keys), (2, self.values)):
            rows[:, :, i] = side[:, page, :, row].transpose(0, 1)
        for layer in range(layers if n else 0):
            append_kv(rows[layer].view(n, -1), kv, self.keys[layer], self.values[layer], target)


class CacheBatch(NamedTuple):
    """A batch of sequences over a ``PagedCache``; see the module's first lines."""
    page_table: torch.Tensor
    lengths: torch.Tensor
    starts: torch.Tensor
    max_query: int   # most new tokens of a sequence
    max_length: int  # most tokens that a sequence holds
    tree: Optional[torch.Tensor] = None


@torch.no_grad()
def decode(model, ids: torch.Tensor, cache: PagedCache, batch: CacheBatch,
           rows: Optional[torch.Tensor] = None, precision: str = "fp16") -> torch.Tensor:
    """Logits of ``model`` for the batch's new tokens ``ids`` (int64 [tokens]), whose keys and
    values are appended to ``cache``: [tokens, vocab], or of the rows ``rows`` (int64) alone.

    The model is a ``BaselineLM`` or ``ReversibleLM`` with what was enabled on it; a window,
    sinks and a rotation are those of ``enable_attention``.  Logits are what the model's own
    forward pass gives for the whole sequences, but for roundings; dropout is not applied.
    Logits of rows of no sequence have no meaning (their ids must be of the vocabulary all the
    same); no sequence may have more than ``batch.max_query`` of them (those past it attend to
    nothing).  ``batch.max_length`` must
    not exceed the model's ``max_sequence_length``, nor the positions of its ``Rotary``
    (positions past the former, which only a wrong max_length lets through, are taken as its
    last).  The keys and values of one call's tokens need slots of their own: sequences may
    share pages of tokens that all of them hold, not those that new tokens go to; tokens that the
    page table has no room for are not kept.

    The modules' weights are read, their parts called one by one: forward hooks on the model, a
    block or its ``attn`` do not run (and on the fused path those of ``mlp_norm`` do not)."""
    from .optimized_v3 import castable_weights
    if precision not in _AMP_DTYPES or _AMP_DTYPES[precision] != cache.keys.dtype:
        raise ValueError("decode needs fp16 or bf16 precision, that of its cache")
    if ids.ndim != 1 or ids.dtype != torch.int64 or ids.device != cache.keys.device:
        raise ValueError("ids must be int64 [tokens] on the cache's device")
    limit = model.config.max_sequence_length
    if batch.max_length > limit:
        raise ValueError("sequence exceeds max_sequence_length")
    if len(model.blocks) != cache.keys.shape[0]:
        raise ValueError("decode needs a cache of the model's layers")
    rotary = getattr(model.blocks[0].attn, "_rv_rotary", None)
    if rotary is not None and batch.max_length > rotary.positions:
        raise ValueError("sequence exceeds the positions of the Rotary table")
    if not ids.shape[0]:
        return torch.empty(0, model.lm_head.weight.shape[0], device=ids.device,
                           dtype=cache.keys.dtype)
    slots, positions = cache_plan(batch.page_table, batch.lengths, batch.starts, ids.shape[0],
                                  cache.page_size, batch.tree)

    # what the attention does not write (rows of no sequence or past max_query) are zeros, not what the
    # memory held: the layers behind it append keys made from them
    first = model.blocks[0].attn
    seen = torch.zeros(ids.shape[0], first.n_heads, first.head_dim, device=ids.device,
                       dtype=cache.keys.dtype)

    def attend(layer, x):
        attn = model.blocks[layer].attn
        keys, values = cache.keys[layer], cache.values[layer]
        q = append_kv(attn.qkv(x), attn.n_heads, keys, values, slots,
                      getattr(attn, "_rv_rotary", None), positions)
        mixed = cached_attention(q, keys, values, batch.page_table, batch.lengths, batch.starts,
                                 batch.max_query, max_length=batch.max_length, tree=batch.tree,
                                 window=getattr(attn, "_rv_window", None),
                                 sinks=getattr(attn, "_rv_sinks", 0), out=seen)
        return attn.proj(mixed.flatten(1).unsqueeze(0))

    # (the fused layers launch on the current device)
    with _DeviceGuard(ids), weight_cast_cache(), amp_context(ids.device, precision):
        if precision == "fp16":
            prefetch_casts(castable_weights(model))
        where = positions.clamp(max=limit - 1)
        x = (model.token_embedding(ids) + model.position_embedding(where)).unsqueeze(0)
        hidden = model.final_norm(_stack(model, x, attend))[0]
        return model.lm_head(hidden if rows is None else hidden[rows])


def _stack(model, x, attend):
    """The blocks on x [1, tokens, d], their attention being ``attend(layer, normalized x)``:
    ``BaselineLM.forward`` and ``ReversibleLM.core`` without a graph."""
    method = getattr(model, "method", None)
    p = q = x
    for layer, block in enumerate(model.blocks):
        if method is None:
            x = x + attend(layer, block.attn_norm(x))
            x = x + block.mlp(block.mlp_norm(x))
        elif method == "midpoint":
            force = attend(layer, block.attn_norm(q))
            mlp = block.mlp(add_rms_norm(q, force, block.mlp_norm)[1])
            p, q = q, midpoint_step(p, force, mlp, 2 * model.step_size, +1)
        else:
            q, normed = add_rms_norm(q, attend(layer, block.attn_norm(p)), block.mlp_norm)
            p = euler_step(p, block.mlp(normed), +1)
    return x if method is None else q if method == "midpoint" else p
