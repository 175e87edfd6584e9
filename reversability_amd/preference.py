"""Fine-tuning from preferences and rewards: log-probabilities of the tied head
and the losses on them, on gfx950 kernels.

The reference trains with one summed cross-entropy (src/reversibility/
kernels.py:56-85, optimized_v3.py:151-192).  Training the same models on pairs
of answers or on sampled answers with rewards needs the log-probability of
every token with a gradient of its own:

* ``tied_head_logprobs(x16, head16, vocab, labels)``: the log-probability of each
  label under the tied head, differentiable.  The logits stay in registers
  (``rv_head_logp_fwd``): the forward keeps one fp32 log-sum-exp per token, and the
  backward makes the products again, a chunk of tokens at a time.  Log-
  probabilities come from the fp32 accumulators, without the Half-logsoftmax
  rounding of ``cross_entropy_sum``: ratios of two models' probabilities are
  exponentials of small differences of them.
* ``preference_loss(logp, ref_logp, ...)``: logistic loss on paired log ratios.
* ``policy_loss(logp, old_logp, advantages, ...)``: clipped policy loss with a KL
  term.

``sequence_logprobs`` scores a batch with a model (the reference or behaviour
policy); ``preference_backward`` and ``policy_backward`` run one update's forward
and backward the way ``cached_head_backward`` does for the cross-entropy: hidden
states, head and loss without a graph over the vocabulary, one core backward.

A label of -100 marks a token that is not scored (its log-probability is 0);
masks are bool tensors, True where a token counts.  Masked tokens are never
used, whatever they hold.  There is no CPU fallback.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd.forward_ad import unpack_dual
from torch.autograd.function import once_differentiable

from . import paths
from ._hip import RV_BF16, RV_F16, RV_F32, _check, _DeviceGuard, _stream, library
from .kernels import IGNORE_INDEX, VOCAB_ALIGN
from .mlp import prefetch_casts, weight_cast_cache
from .optimized import _AMP_DTYPES, amp_context, hidden_states

_CODES = {torch.float16: RV_F16, torch.bfloat16: RV_BF16}
# tokens per launch of the forward (its partial statistics: 8 bytes per token and tile of
# columns, of 64 to the whole vocabulary) and bytes of one chunk's logit gradients in the backward
FORWARD_TOKENS = 1 << 16
GRADIENT_BYTES = 1 << 32


# ---------------------------------------------------------------------------
# log-probabilities of the tied head
# ---------------------------------------------------------------------------
def _rows16(t: torch.Tensor, width: int) -> torch.Tensor:
    """``t`` [..., d] as the kernels read it: dense rows of ``width`` (zeros behind t's
    own columns), 16-byte aligned."""
    d = t.shape[-1]
    if d != width:
        out = t.new_zeros(*t.shape[:-1], width)
        out[..., :d] = t
        return out
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _workspace(nbytes: int, like: torch.Tensor, what: str):
    if nbytes < 0:
        _check(-nbytes, what)
    return torch.empty(nbytes, device=like.device, dtype=torch.uint8) if nbytes else None


def _logp_forward(x, head, vocab, labels, want_lse=True):
    """(logp, lse or None), fp32 of the labels' shape, of dense operands."""
    rows, d = labels.numel(), x.shape[-1]
    lib, code = library(), _CODES[x.dtype]
    logp = torch.empty(labels.shape, device=x.device, dtype=torch.float32)
    lse = torch.empty_like(logp) if want_lse else None
    with _DeviceGuard(x):
        for at in range(0, rows, FORWARD_TOKENS):
            n = min(FORWARD_TOKENS, rows - at)
            nbytes = lib.rv_head_logp_workspace_bytes(n, d, vocab)
            ws = _workspace(nbytes, x, "rv_head_logp_workspace_bytes")
            _check(lib.rv_head_logp_fwd(
                x.data_ptr() + at * d * 2, head.data_ptr(), n, d, vocab, code,
                labels.data_ptr() + at * 8, IGNORE_INDEX, logp.data_ptr() + at * 4,
                lse.data_ptr() + at * 4 if want_lse else None, ws.data_ptr(), nbytes, _stream(x)), "rv_head_logp_fwd")
    return logp, lse


def _logp_backward(x, head, vocab, labels, lse, grad, dx=None, dw=None, accumulate=False,
                   chunk_tokens=None):
    """Gradients for ``grad`` (fp32 [rows]) into dx [rows, d] of x's type and dw
    [vocab or padded, d] of x's type or fp32 (added to it with ``accumulate``); either
    may be None.  ``dw`` of x's type takes one chunk only.  All dense."""
    rows, d = x.shape
    padded = head.shape[0]
    lib, code = library(), _CODES[x.dtype]
    step = min(rows, chunk_of(padded, d, chunk_tokens))
    out = (None, vocab, code) if dw is None else (
        dw.data_ptr(), dw.shape[0], RV_F32 if dw.dtype == torch.float32 else code)
    with _DeviceGuard(x):
        nbytes = lib.rv_head_logp_bwd_workspace_bytes(step, d, vocab, padded)
        ws = _workspace(nbytes, x, "rv_head_logp_bwd_workspace_bytes")
        for at in range(0, rows, step):
            n = min(step, rows - at)
            if n < step:  # a short last chunk has a plan of its own
                nbytes = lib.rv_head_logp_bwd_workspace_bytes(n, d, vocab, padded)
                if nbytes > ws.numel():
                    ws = _workspace(nbytes, x, "rv_head_logp_bwd_workspace_bytes")
            _check(lib.rv_head_logp_bwd(
                x.data_ptr() + at * d * 2, head.data_ptr(), n, d, vocab, padded, code,
                labels.data_ptr() + at * 8, IGNORE_INDEX, lse.data_ptr() + at * 4,
                grad.data_ptr() + at * 4, dx.data_ptr() + at * d * 2 if dx is not None else None,
                *out, accumulate or at > 0, ws.data_ptr(), ws.numel(), _stream(x)),
                "rv_head_logp_bwd")


def max_chunk(padded: int) -> int:
    """Tokens whose 16-bit logit gradients over ``padded`` columns fill GRADIENT_BYTES
    (at most 2^22, what one call takes)."""
    return min(1 << 22, max(256, GRADIENT_BYTES // (2 * padded) // 256 * 256))


def chunk_of(padded: int, d: int, chunk_tokens: Optional[int]) -> int:
    """Tokens that the backward takes at a time (one call: fewer than 2^34 elements of x)."""
    return min(chunk_tokens or max_chunk(padded), ((1 << 34) - 1) // d)


class TiedHeadLogProbs(torch.autograd.Function):
    """log softmax(x head[:vocab]^T) at the labels; see ``tied_head_logprobs``."""

    @staticmethod
    def forward(ctx, x, head, vocab, labels, chunk_tokens):
        width = -(-x.shape[1] // 8) * 8
        labels = labels.contiguous()
        logp, lse = _logp_forward(_rows16(x, width), _rows16(head, width), vocab, labels)
        ctx.save_for_backward(x, head, labels, lse)
        ctx.vocab, ctx.chunk_tokens, ctx.width = vocab, chunk_tokens, width
        return logp

    @staticmethod
    @once_differentiable
    def backward(ctx, gradient):
        x, head, labels, lse = ctx.saved_tensors
        need_x, need_head = ctx.needs_input_grad[:2]
        rows, d = x.shape
        if not rows:
            return (torch.zeros_like(x) if need_x else None,
                    torch.zeros_like(head) if need_head else None, None, None, None)
        width, padded = ctx.width, head.shape[0]
        grad = gradient.contiguous()
        dx = x.new_empty(rows, width) if need_x else None
        one = rows <= chunk_of(padded, width, ctx.chunk_tokens)
        dw = (torch.empty(padded, width, device=x.device,
                          dtype=head.dtype if one else torch.float32) if need_head else None)
        _logp_backward(_rows16(x, width), _rows16(head, width), ctx.vocab, labels, lse, grad, dx,
                       dw, chunk_tokens=ctx.chunk_tokens)
        if need_head and not one:
            dw = dw.to(head.dtype)
        if width != d:
            dx, dw = (t if t is None else t[:, :d] for t in (dx, dw))
        return dx, dw, None, None, None


def tied_head_logprobs(x16: torch.Tensor, head16: torch.Tensor, vocab: int, labels: torch.Tensor,
                       chunk_tokens: Optional[int] = None) -> torch.Tensor:
    """fp32 log-probability of each label under the tied head, differentiable in
    ``x16`` and ``head16``.

    ``x16`` [..., d] and ``head16`` [padded, d] are both fp16 or both bf16 (d of any
    size; multiples of 8 need no copies); head16's rows past ``vocab`` are padding, as
    ``padded_head`` makes it, up to a multiple of VOCAB_ALIGN (their gradient is
    zero).  ``labels`` int64 of x16's leading shape, the result's shape; a label of
    -100 gives 0 and no gradient, another one outside [0, vocab) gives NaN (in its
    gradients too).  Products are summed in fp32 and the logits never rounded.  The
    backward holds ``chunk_tokens`` tokens' logit gradients in 16 bits at a time
    (default: as many as fill GRADIENT_BYTES, 4 GiB; fewer take less memory), in fp16 scaled
    by a power of two for each token, so that a small gradient of x16 does not depend on
    larger ones of other tokens
    (up to 512 tokens as two 16-bit numbers each); gradients come in the operands' type.
    As in any product, a NaN or an infinity in an unscored token's row of ``x16`` reaches
    the gradient of the head.  A row whose largest logit is beyond 2^126 in magnitude has
    no log-probability (NaN); lower logits than -2^126 count for nothing.
    """
    shape, table = x16.shape, head16.shape
    # a dual tensor requires no gradient: without an autograd node its tangent would vanish
    if unpack_dual(x16).tangent is not None or unpack_dual(head16).tangent is not None:
        raise NotImplementedError("tied_head_logprobs has no forward-mode derivative")
    if (x16.dtype not in _CODES or head16.dtype != x16.dtype or len(shape) < 1 or len(table) != 2
            or not x16.is_cuda or shape[-1] != table[1] or not table[1]
            or table[0] % VOCAB_ALIGN or not 0 < vocab <= table[0]
            or labels.dtype != torch.int64 or labels.shape != shape[:-1]):
        raise ValueError("tied_head_logprobs needs CUDA fp16 or bf16 x [..., d], a padded head "
                         "[padded, d] of the same type and int64 labels [...]")
    if head16.device != x16.device or labels.device != x16.device:
        raise ValueError("tied_head_logprobs needs its head and labels on x's device")
    if chunk_tokens is not None and not 1 <= chunk_tokens <= 1 << 22:
        raise ValueError("tied_head_logprobs needs chunk_tokens in [1, 2^22]")
    paths.took("tied_head_logprobs", "mfma")
    if torch.is_grad_enabled() and (x16.requires_grad or head16.requires_grad):
        return TiedHeadLogProbs.apply(x16.reshape(-1, table[1]), head16, vocab,
                                      labels.reshape(-1), chunk_tokens).reshape(labels.shape)
    width = -(-table[1] // 8) * 8
    return _logp_forward(_rows16(x16, width), _rows16(head16, width), vocab, labels.contiguous(),
                         want_lse=False)[0]


# ---------------------------------------------------------------------------
# losses on token log-probabilities
# ---------------------------------------------------------------------------
def _rows(t: torch.Tensor) -> torch.Tensor:
    """A [sequences, tokens] operand with dense rows."""
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def _tokens(t: torch.Tensor, like: torch.Tensor, what: str) -> torch.Tensor:
    if t.dtype != torch.float32 or t.shape != like.shape or t.device != like.device:
        raise ValueError(f"{what} must be fp32, of logp's shape and on its device")
    return _rows(t)


def _mask(mask, like: torch.Tensor):
    if mask is None:
        return None
    if mask.dtype != torch.bool or mask.shape != like.shape or mask.device != like.device:
        raise ValueError("mask must be a bool tensor of logp's shape on its device")
    return _rows(mask)


def _check_logp(logp: torch.Tensor, what: str) -> None:
    if not logp.is_cuda or logp.dtype != torch.float32 or logp.ndim != 2:
        raise ValueError(f"{what} needs CUDA (ROCm device) fp32 logp [sequences, tokens]; "
                         "no silent fallback")


def _at(t) -> tuple:
    """(address, row stride) of an optional [sequences, tokens] operand."""
    return (None, 0) if t is None else (t.data_ptr(), t.stride(0))


# The two Functions below are called on small batches too, where the host's work is
# what they take: few allocations (outputs and workspace cut from one) and no zeros
# made for the outputs without a gradient.  Pieces of one allocation share its version
# count, so none is handed to save_for_backward: a caller may change the returned
# statistics in place (an all-reduce) before the backward pass.  fp32 values of the
# workspace's share:
def _floats(nbytes: int, what: str) -> int:
    if nbytes < 0:
        _check(-nbytes, what)
    return -(-nbytes // 4)


class PreferenceLoss(torch.autograd.Function):
    """See ``preference_loss``."""

    @staticmethod
    def forward(ctx, logp, ref, mask, beta, smoothing, average):
        seqs, tokens = logp.shape
        lib, pairs, dev = library(), seqs // 2, logp.device
        rows = _rows(logp)
        with _DeviceGuard(logp):
            nbytes = lib.rv_pref_loss_workspace_bytes(pairs, tokens)
            # the workspace first: its fp64 sums need the allocation's alignment
            sizes = (_floats(nbytes, "rv_pref_loss_workspace_bytes"), pairs, pairs)
            ws, chosen, rejected = torch.empty(
                sum(sizes), device=dev, dtype=torch.float32).split(sizes)
            coef = torch.empty(seqs, device=dev, dtype=torch.float32)
            loss = torch.empty((), device=dev, dtype=torch.float32)
            _check(lib.rv_pref_loss(
                rows.data_ptr(), rows.stride(0), *_at(ref), *_at(mask), pairs, tokens, beta,
                smoothing, average, loss.data_ptr(), chosen.data_ptr(), coef.data_ptr(),
                ws.data_ptr(), nbytes, _stream(logp)), "rv_pref_loss")
        ctx.save_for_backward(coef, mask)
        ctx.shape = (seqs, tokens)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(chosen, rejected)
        return loss, chosen, rejected

    @staticmethod
    @once_differentiable
    def backward(ctx, gradient, *_):
        if gradient is None:
            return None, None, None, None, None, None
        coef, mask = ctx.saved_tensors
        dlogp = torch.empty(ctx.shape, device=coef.device, dtype=torch.float32)
        _check(library().rv_pref_grad(coef.data_ptr(), *_at(mask), gradient.data_ptr(), *ctx.shape,
                                      dlogp.data_ptr(), _stream(coef)), "rv_pref_grad")
        return dlogp, None, None, None, None, None


class PreferenceResult(NamedTuple):
    loss: torch.Tensor      # fp32 scalar, differentiable
    chosen: torch.Tensor    # [pairs] rewards beta * sum (logp - ref_logp)
    rejected: torch.Tensor  # [pairs]


def preference_loss(logp: torch.Tensor, ref_logp: torch.Tensor, beta: float = 0.1, *,
                    mask: Optional[torch.Tensor] = None, label_smoothing: float = 0.0,
                    average: bool = False) -> PreferenceResult:
    """Logistic preference loss on paired log ratios, the mean over pairs.

    ``logp`` fp32 [2 pairs, tokens]: the chosen answers, then the rejected ones in the
    same order; ``ref_logp`` the reference model's; ``mask`` the tokens that count
    (None: all).  With s the sum of logp - ref_logp over a row's counted tokens
    (``average``: their mean; 0 for a row without any) and m = beta (s_chosen -
    s_rejected), a pair's loss is -(1 - label_smoothing) log sigmoid(m) -
    label_smoothing log sigmoid(-m).  The gradient reaches ``logp`` alone.  Sums in
    fp64, deterministic."""
    _check_logp(logp, "preference_loss")
    if not logp.shape[0] or logp.shape[0] % 2:
        raise ValueError("preference_loss needs one chosen and one rejected row per pair")
    if not 0.0 <= label_smoothing <= 0.5:
        raise ValueError("label_smoothing must be in [0, 0.5]")
    return PreferenceResult(*PreferenceLoss.apply(
        logp, _tokens(ref_logp, logp, "ref_logp"), _mask(mask, logp), beta, label_smoothing,
        bool(average)))


class PolicyLoss(torch.autograd.Function):
    """See ``policy_loss``."""

    @staticmethod
    def forward(ctx, logp, old, ref, adv, mask, clip, kl_coef, per_sequence):
        seqs, tokens = logp.shape
        lib, dev = library(), logp.device
        rows = _rows(logp)
        slope = (torch.empty(seqs, tokens, device=dev, dtype=torch.float32)
                 if ctx.needs_input_grad[0] else None)
        with _DeviceGuard(logp):
            nbytes = lib.rv_policy_loss_workspace_bytes(seqs, tokens, per_sequence)
            # the workspace first: its fp64 sums need the allocation's alignment
            sizes = (_floats(nbytes, "rv_policy_loss_workspace_bytes"), 1, 1, 1)
            ws, kl, clipped, factor = torch.empty(
                sum(sizes), device=dev, dtype=torch.float32).split(sizes)
            loss = torch.empty((), device=dev, dtype=torch.float32)
            _check(lib.rv_policy_loss(
                rows.data_ptr(), rows.stride(0), *_at(old), *_at(ref), adv.data_ptr(),
                adv.stride(0), adv.stride(1) if adv.ndim == 2 else 0, *_at(mask), seqs, tokens,
                *clip, kl_coef, per_sequence, loss.data_ptr(), kl.data_ptr(),
                slope.data_ptr() if slope is not None else None, ws.data_ptr(), nbytes,
                _stream(logp)), "rv_policy_loss")
        ctx.save_for_backward(slope)
        ctx.factor = factor
        ctx.set_materialize_grads(False)
        kl, clipped = kl.reshape(()), clipped.reshape(())
        ctx.mark_non_differentiable(kl, clipped)
        return loss, kl, clipped

    @staticmethod
    @once_differentiable
    def backward(ctx, gradient, *_):
        if gradient is None:
            return None, None, None, None, None, None, None, None
        slope, = ctx.saved_tensors
        dlogp = torch.empty_like(slope)
        _check(library().rv_policy_grad(slope.data_ptr(), ctx.factor.data_ptr(), gradient.data_ptr(),
                                        slope.numel(), dlogp.data_ptr(), _stream(slope)),
               "rv_policy_grad")
        return dlogp, None, None, None, None, None, None, None


class PolicyResult(NamedTuple):
    loss: torch.Tensor     # fp32 scalar, differentiable
    kl: torch.Tensor       # mean KL estimate over all counted tokens (0 without ref_logp)
    clipped: torch.Tensor  # share of the counted tokens whose ratio is clipped


def policy_loss(logp: torch.Tensor, old_logp: torch.Tensor, advantages: torch.Tensor, *,
                ref_logp: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                clip: tuple[float, float] = (0.2, 0.2), kl_coef: float = 0.0,
                reduction: str = "token") -> PolicyResult:
    """Clipped policy loss with a KL term.

    ``logp`` fp32 [sequences, tokens] of the model that is trained, ``old_logp`` of the
    one that sampled the answers, ``advantages`` fp32 [sequences] or [sequences,
    tokens], ``mask`` the tokens that count (None: all).  With r = exp(logp - old_logp)
    a token's loss is -min(r A, clamp(r, 1 - clip[0], 1 + clip[1]) A), plus kl_coef
    (exp(d) - d - 1), d = ref_logp - logp, if ``ref_logp`` is given (kl_coef 0: its
    mean is returned, the loss has no such term).  ``reduction`` "token": the mean over
    all counted tokens; "sequence": the mean over all sequences of each one's mean.
    Nothing counted gives 0.  Where the ratio is clipped the
    first term has no gradient (at the border itself it has).  The gradient reaches
    ``logp`` alone.  Sums in fp64, deterministic."""
    _check_logp(logp, "policy_loss")
    low, high = (float(c) for c in clip)
    if not (0.0 <= low < 1.0 and 0.0 <= high < float("inf")):
        raise ValueError("clip needs 0 <= clip[0] < 1 and 0 <= clip[1]")
    if reduction not in ("token", "sequence"):
        raise ValueError("reduction must be token or sequence")
    if (advantages.dtype != torch.float32 or advantages.device != logp.device
            or advantages.shape not in (logp.shape, logp.shape[:1])):
        raise ValueError("advantages must be fp32 [sequences] or [sequences, tokens] on logp's "
                         "device")
    if kl_coef != 0.0 and ref_logp is None:
        raise ValueError("a KL term needs ref_logp")
    ref = None if ref_logp is None else _tokens(ref_logp, logp, "ref_logp")
    return PolicyResult(*PolicyLoss.apply(
        logp, _tokens(old_logp, logp, "old_logp"), ref, advantages, _mask(mask, logp), (low, high),
        kl_coef, reduction == "sequence"))


# ---------------------------------------------------------------------------
# one update of a model
# ---------------------------------------------------------------------------
def _compute_dtype(model, ids, precision) -> torch.dtype:
    if precision not in _AMP_DTYPES:
        raise ValueError("the tied head's log-probabilities need fp16 or bf16 precision")
    if ids.device.type != "cuda" or model.lm_head.weight.dtype != torch.float32:
        raise ValueError("the tied head's log-probabilities need an fp32 model and CUDA (ROCm "
                         "device) tokens; no silent fallback")
    return _AMP_DTYPES[precision]


def _head16(weight: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """The head's rows in ``dtype`` as the kernels read them (width a multiple of 8),
    with zero rows up to a multiple of VOCAB_ALIGN."""
    vocab, d = weight.shape
    padded, width = -(-vocab // VOCAB_ALIGN) * VOCAB_ALIGN, -(-d // 8) * 8
    make = torch.empty if width == d else torch.zeros
    head = make(padded, width, device=weight.device, dtype=dtype)
    head[:vocab, :d].copy_(weight)
    head[vocab:].zero_()
    return head


def _labels(ids, labels):
    if labels.dtype != torch.int64 or labels.shape != ids.shape or labels.device != ids.device:
        raise ValueError("labels must be int64, of the ids' shape and on their device")
    return labels.reshape(-1).contiguous()


@torch.no_grad()
def sequence_logprobs(model, ids: torch.Tensor, labels: torch.Tensor,
                      precision: str = "fp16") -> torch.Tensor:
    """fp32 [batch, tokens] log-probabilities of ``labels`` (0 where -100) under
    ``model``, without a graph: a reference or behaviour policy's score of a batch."""
    from .optimized_v3 import castable_weights
    dtype = _compute_dtype(model, ids, precision)
    targets = _labels(ids, labels)
    with weight_cast_cache(), amp_context(ids.device, precision):
        if precision == "fp16":
            prefetch_casts(castable_weights(model))
        hidden = hidden_states(model, ids)
    weight = model.lm_head.weight
    head = _head16(weight, dtype)
    x = _rows16(hidden.reshape(-1, hidden.shape[-1]).to(dtype), head.shape[1])
    paths.took("tied_head_logprobs", "mfma")
    return _logp_forward(x, head, weight.shape[0], targets, want_lse=False)[0].reshape(ids.shape)


def _loss_backward(model, ids, labels, loss_of, chunk_tokens, scaler, precision):
    """Forward, loss and backward of one batch: ``loss_of(logp [batch, tokens])``
    returns a result whose first item is the loss.  Gradients are added to the
    parameters' ``.grad``."""
    from .optimized_v3 import castable_weights
    if not torch.is_grad_enabled():
        raise ValueError("an update needs gradients enabled")
    dtype = _compute_dtype(model, ids, precision)
    targets = _labels(ids, labels)
    if chunk_tokens is not None and not 1 <= chunk_tokens <= 1 << 22:
        raise ValueError("chunk size in [1, 2^22] required")
    with weight_cast_cache():  # weights are constant until the optimizer step
        if precision == "fp16":
            prefetch_casts(castable_weights(model))
        with amp_context(ids.device, precision):
            hidden = hidden_states(model, ids)
        if not hidden.requires_grad:  # before the head's gradient is added
            raise ValueError("an update needs gradients of the hidden states")
        weight = model.lm_head.weight
        vocab, d = weight.shape
        flat = hidden.detach().reshape(-1, d)
        head = _head16(weight, dtype)
        x = _rows16(flat.to(dtype), head.shape[1])
        paths.took("tied_head_logprobs", "mfma")
        logp, lse = _logp_forward(x, head, vocab, targets)
        with torch.enable_grad():
            leaf = logp.reshape(ids.shape).requires_grad_(True)
            result = loss_of(leaf)
            scaled = result[0] if scaler is None else scaler.scale(result[0])
            grad, = torch.autograd.grad(scaled, leaf)
        dx = torch.empty_like(x)
        sink, first = None, weight.grad is None
        direct = False
        if weight.requires_grad:
            direct = d == x.shape[1] and (first or (
                weight.grad.is_contiguous() and weight.grad.dtype == torch.float32
                and weight.grad.data_ptr() % 16 == 0))
            # the head's gradient goes straight into the tied weight's
            sink = (weight.grad if direct and not first else
                    torch.empty(vocab, x.shape[1], device=x.device, dtype=torch.float32))
        if targets.numel():
            _logp_backward(x, head, vocab, targets, lse, grad.reshape(-1), dx, sink,
                           accumulate=direct and not first, chunk_tokens=chunk_tokens)
        elif sink is not None and not (direct and not first):
            sink.zero_()
        if sink is not None and first:
            weight.grad = sink if direct else sink[:, :d].contiguous()
        elif sink is not None and not direct:
            weight.grad.add_(sink[:, :d])
        del head, x, sink, grad
        with amp_context(ids.device, precision):
            hidden.backward(dx[:, :d].to(hidden.dtype).reshape_as(hidden))
    return type(result)(result[0].detach(), *result[1:])


def preference_backward(model, ids: torch.Tensor, labels: torch.Tensor, ref_logp: torch.Tensor,
                        beta: float = 0.1, *, label_smoothing: float = 0.0, average: bool = False,
                        chunk_tokens: Optional[int] = None, scaler=None,
                        precision: str = "fp16") -> PreferenceResult:
    """One preference update's forward and backward: ``preference_loss`` of
    ``model`` on ids [2 pairs, tokens] (chosen rows, then rejected ones), scored where
    ``labels`` are not -100, against ``ref_logp`` (``sequence_logprobs`` of the
    reference model).  Parameter gradients are added to ``.grad`` (times the scaler's
    factor)."""
    def loss_of(logp):
        return preference_loss(logp, ref_logp, beta, mask=labels != IGNORE_INDEX,
                               label_smoothing=label_smoothing, average=average)
    return _loss_backward(model, ids, labels, loss_of, chunk_tokens, scaler, precision)


def policy_backward(model, ids: torch.Tensor, labels: torch.Tensor, old_logp: torch.Tensor,
                    advantages: torch.Tensor, *, ref_logp: Optional[torch.Tensor] = None,
                    clip: tuple[float, float] = (0.2, 0.2), kl_coef: float = 0.0,
                    reduction: str = "token", chunk_tokens: Optional[int] = None, scaler=None,
                    precision: str = "fp16") -> PolicyResult:
    """One policy update's forward and backward: ``policy_loss`` of ``model`` on ids
    [sequences, tokens], scored where ``labels`` are not -100.  Parameter gradients
    are added to ``.grad`` (times the scaler's factor)."""
    def loss_of(logp):
        return policy_loss(logp, old_logp, advantages, ref_logp=ref_logp,
                           mask=labels != IGNORE_INDEX, clip=clip, kl_coef=kl_coef,
                           reduction=reduction)
    return _loss_backward(model, ids, labels, loss_of, chunk_tokens, scaler, precision)
