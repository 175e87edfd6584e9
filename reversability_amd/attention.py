"""Causal self-attention on the gfx950 MFMA kernels (src/reversibility/model.py:26-45).

The reference's ``CausalSelfAttention`` projects to a packed ``qkv`` of width
``3 d``, views it as ``[B, T, 3, H, hd]``, permutes it into three strided
``[B, H, T, hd]`` tensors for ``F.scaled_dot_product_attention(is_causal=True)``,
and transposes the result back to ``[B, T, d]`` for the output projection;
autograd then stacks ``dq, dk, dv`` back into the packed layout.  Here the
kernels read ``qkv`` in the layout the qkv GEMM wrote, write the output in the
layout the output GEMM reads, and write the gradient straight into a packed
``dqkv`` (``rv_attn_fwd`` / ``rv_attn_bwd``, csrc/attention.hip): no permute,
transpose or concatenation copies.  Forward keeps the base-2 log-sum-exp per
query; backward is deterministic (no atomics).

``enable_attention(model)`` patches every block's ``attn.forward``; calls the
kernels do not cover (no fp16 ``qkv`` -- i.e. not under fp16 autocast --, head
sizes other than 32/64/128, dropout in training mode, CPU tensors) keep the
reference computation, recorded in ``paths.report()`` (or raising under
``paths.strict()``).

Beside it, without a counterpart in the reference: ``window_attention``, causal
attention with a sliding window and first tokens that stay visible (sinks), fp16 or
bf16, with query heads that may share key and value heads; and ``rotate_qkv``, the
rotation of queries and keys by position, from a ``Rotary`` table.
``enable_attention(model, window=, sinks=, rotary=)`` trains a model with them, and
``cache.decode`` answers with the same settings.
"""
from __future__ import annotations

import math
import types
from typing import Optional

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import linear as _linear
from . import paths
from ._hip import RV_BF16, RV_F16, RV_F32, _check, _DeviceGuard, _stream, library
from .mlp import cast_operands, splitk_workspace

HEAD_DIMS = (32, 64, 128)


def supported(qkv: torch.Tensor, heads: int, dropout: float = 0.0) -> bool:
    if not (qkv.is_cuda and qkv.dtype == torch.float16 and qkv.ndim == 3 and dropout == 0.0):
        return False
    width = qkv.shape[-1]
    return width % (3 * heads) == 0 and width // (3 * heads) in HEAD_DIMS


class CausalAttention(torch.autograd.Function):
    """``qkv`` fp16 ``[B, T, 3 d]`` -> causal attention output fp16 ``[B, T, d]``."""

    @staticmethod
    def forward(ctx, qkv, heads):
        batch, seq, width = qkv.shape
        d = width // 3
        qkv = qkv.contiguous()
        out = torch.empty(batch, seq, d, device=qkv.device, dtype=torch.float16)
        lse = torch.empty(batch * heads, seq, device=qkv.device, dtype=torch.float32)
        _check(library().rv_attn_fwd(qkv.data_ptr(), batch, seq, heads, d // heads,
                                     out.data_ptr(), lse.data_ptr(), _stream(qkv)), "rv_attn_fwd")
        ctx.save_for_backward(qkv, out, lse)
        ctx.heads = heads
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        qkv, out, lse = ctx.saved_tensors
        batch, seq, width = qkv.shape
        heads = ctx.heads
        lib = library()
        dout = dout.to(torch.float16).contiguous()
        dqkv = torch.empty_like(qkv)
        nbytes = lib.rv_attn_bwd_workspace_bytes(batch, seq, heads)
        if nbytes < 0:
            _check(-nbytes, "rv_attn_bwd_workspace_bytes")
        ws = torch.empty(nbytes // 4, device=qkv.device, dtype=torch.float32)
        _check(lib.rv_attn_bwd(qkv.data_ptr(), out.data_ptr(), dout.data_ptr(), lse.data_ptr(),
                               batch, seq, heads, width // 3 // heads, dqkv.data_ptr(),
                               ws.data_ptr(), nbytes, _stream(qkv)), "rv_attn_bwd")
        return dqkv, None


class AttentionLayer(torch.autograd.Function):
    """``proj(causal_attention(qkv(x)))`` of one layer under fp16 autocast as one
    autograd node: the same kernels on the same values as ``FusedLinear``,
    ``CausalAttention`` and ``FusedLinear`` in turn, with one launch for the
    operand casts and one for the two weight gradients (reduced over the
    rows in another fixed order than each alone).  The weights' fp16 casts live
    from forward to backward (2 bytes per weight), and qkv, its log-sum-exp and the
    attention output to the end of the backward, where three nodes free them one
    after the other (8 bytes per token and column more at the input gradient)."""

    @staticmethod
    def forward(ctx, x, w_qkv, w_proj, heads):
        batch, seq, d = x.shape
        rows, out_f = batch * seq, w_proj.shape[0]
        lib, st = library(), _stream(x)
        x16, qkv16, proj16 = cast_operands(x.reshape(rows, d).contiguous(), w_qkv, w_proj)
        dev = x.device
        qkv = torch.empty(rows, 3 * d, device=dev, dtype=torch.float16)
        mixed = torch.empty(rows, d, device=dev, dtype=torch.float16)
        lse = torch.empty(batch * heads, seq, device=dev, dtype=torch.float32)
        y = torch.empty(batch, seq, out_f, device=dev, dtype=torch.float16)
        ws, nbytes = splitk_workspace(x16, rows, 3 * d, d)
        _check(lib.rv_linear_fwd_ws(x16.data_ptr(), d, qkv16.data_ptr(), rows, d, 3 * d,
                                    qkv.data_ptr(), ws.data_ptr() if nbytes else None, nbytes,
                                    st), "rv_linear_fwd")
        _check(lib.rv_attn_fwd(qkv.data_ptr(), batch, seq, heads, d // heads, mixed.data_ptr(),
                               lse.data_ptr(), st), "rv_attn_fwd")
        ws, nbytes = splitk_workspace(x16, rows, out_f, d)
        _check(lib.rv_linear_fwd_ws(mixed.data_ptr(), d, proj16.data_ptr(), rows, d, out_f,
                                    y.data_ptr(), ws.data_ptr() if nbytes else None, nbytes, st),
               "rv_linear_fwd")
        ctx.save_for_backward(x16, w_qkv, w_proj, qkv16, proj16, qkv, mixed, lse)
        ctx.heads, ctx.x_dtype, ctx.shape = heads, x.dtype, (batch, seq, d)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gradient):
        x16, w_qkv, w_proj, qkv16, proj16, qkv, mixed, lse = ctx.saved_tensors
        (batch, seq, d), heads, out_f = ctx.shape, ctx.heads, w_proj.shape[0]
        rows = batch * seq
        lib, st, dev = library(), _stream(x16), x16.device
        dy = gradient.reshape(rows, out_f).to(torch.float16).contiguous()
        dx = dw_qkv = dw_proj = None
        need_x, need_qkv, need_proj = ctx.needs_input_grad[:3]
        if need_x or need_qkv:
            dmixed = torch.empty_like(mixed)
            ws, nbytes = splitk_workspace(dy, rows, d, out_f)
            _check(lib.rv_linear_dx_ws(dy.data_ptr(), proj16.data_ptr(), rows, d, out_f,
                                       dmixed.data_ptr(), RV_F16, ws.data_ptr() if nbytes else None,
                                       nbytes, st), "rv_linear_dx")
            dqkv = torch.empty_like(qkv)
            nbytes = lib.rv_attn_bwd_workspace_bytes(batch, seq, heads)
            if nbytes < 0:
                _check(-nbytes, "rv_attn_bwd_workspace_bytes")
            ws = torch.empty(nbytes // 4, device=dev, dtype=torch.float32)
            _check(lib.rv_attn_bwd(qkv.data_ptr(), mixed.data_ptr(), dmixed.data_ptr(), lse.data_ptr(),
                                   batch, seq, heads, d // heads, dqkv.data_ptr(), ws.data_ptr(),
                                   nbytes, st), "rv_attn_bwd")
            del dmixed, ws  # free for the buffers below
        if need_x:
            dx = torch.empty(batch, seq, d, device=dev, dtype=ctx.x_dtype)
            ws, nbytes = splitk_workspace(dqkv, rows, d, 3 * d)
            code = RV_F32 if ctx.x_dtype == torch.float32 else RV_F16
            _check(lib.rv_linear_dx_ws(dqkv.data_ptr(), qkv16.data_ptr(), rows, d, 3 * d,
                                       dx.data_ptr(), code, ws.data_ptr() if nbytes else None,
                                       nbytes, st), "rv_linear_dx")
        if need_qkv and need_proj:
            dw_qkv, dw_proj = torch.empty_like(w_qkv), torch.empty_like(w_proj)
            nbytes = lib.rv_linear_dw_pair_workspace_bytes(rows, d, 3 * d, d, out_f)
            if nbytes < 0:
                _check(-nbytes, "rv_linear_dw_pair_workspace_bytes")
            ws = torch.empty(nbytes // 4, device=dev, dtype=torch.float32) if nbytes else None
            _check(lib.rv_linear_dw_pair(
                dqkv.data_ptr(), x16.data_ptr(), d, 3 * d, dw_qkv.data_ptr(), dy.data_ptr(),
                mixed.data_ptr(), d, out_f, dw_proj.data_ptr(), rows, 0,
                ws.data_ptr() if nbytes else None, nbytes, st), "rv_linear_dw_pair")
        elif need_qkv:  # the other projection is frozen
            dw_qkv = _linear.weight_grad(dqkv.view(rows, 3 * d), x16, w_qkv)
        elif need_proj:
            dw_proj = _linear.weight_grad(dy, mixed, w_proj)
        return dx, dw_qkv, dw_proj, None


def _layer_supported(attn: torch.nn.Module, x: torch.Tensor, dropout: float) -> bool:
    """Whether ``AttentionLayer`` is what the layer's own modules would compute
    on their kernels, one after the other."""
    qkv, proj = attn.qkv, attn.proj
    return (x.ndim == 3 and x.numel() > 0 and dropout == 0.0 and _linear.plain_layer(qkv)
            and _linear.plain_layer(proj)
            and _linear.supported(x, qkv.weight, None) and proj.weight.is_cuda
            and proj.weight.dtype == torch.float32 and proj.weight.is_contiguous()
            and proj.weight.shape[0] % 128 == 0 and proj.weight.shape[1] == x.shape[-1]
            and qkv.weight.shape[0] == 3 * x.shape[-1] and x.shape[-1] % attn.n_heads == 0
            and x.shape[-1] // attn.n_heads in HEAD_DIMS)


def causal_attention(qkv: torch.Tensor, heads: int) -> torch.Tensor:
    """Causal attention of a packed fp16 ``qkv`` on the kernels; raises on inputs
    they do not cover."""
    if not supported(qkv, heads):
        raise ValueError("fused attention needs a CUDA fp16 qkv [B, T, 3 d] with head size "
                         f"in {HEAD_DIMS}")
    return CausalAttention.apply(qkv, heads)


def reference_attention(qkv: torch.Tensor, heads: int, dropout: float = 0.0) -> torch.Tensor:
    """The reference's computation (model.py:40-45) on a packed ``qkv``."""
    batch, length, width = qkv.shape
    d = width // 3
    q, k, v = qkv.view(batch, length, 3, heads, d // heads).permute(2, 0, 3, 1, 4).unbind(0)
    mixed = F.scaled_dot_product_attention(q, k, v, dropout_p=dropout, is_causal=True)
    return mixed.transpose(1, 2).reshape(batch, length, d)


# ---------------------------------------------------------------------------
# windows, sinks and rotation
# ---------------------------------------------------------------------------
_CODES = {torch.float16: RV_F16, torch.bfloat16: RV_BF16}


def _dense(t: torch.Tensor) -> torch.Tensor:
    """``t`` contiguous and 16-byte aligned, as the kernels read it."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def packed_heads(qkv: torch.Tensor, heads: int, kv_heads: Optional[int], what: str) -> tuple:
    """(kv_heads, head size) of packed rows [..., (heads + 2 kv_heads) head size]; raises
    on what the kernels do not cover."""
    kv = heads if kv_heads is None else kv_heads
    if heads < 1 or kv < 1 or heads % kv:
        raise ValueError(f"{what} needs heads that are a multiple of kv_heads")
    width = qkv.shape[-1] if qkv.ndim else 0
    hd = width // (heads + 2 * kv)
    if (not qkv.is_cuda or qkv.dtype not in _CODES or hd not in HEAD_DIMS
            or hd * (heads + 2 * kv) != width):
        raise ValueError(f"{what} needs CUDA (ROCm device) fp16 or bf16 rows of (heads + 2 "
                         f"kv_heads) heads of size in {HEAD_DIMS}; no silent fallback")
    return kv, hd


class WindowAttention(torch.autograd.Function):
    """See ``window_attention``."""

    @staticmethod
    def forward(ctx, qkv, heads, kv, window, sinks):
        batch, seq, width = qkv.shape
        hd = width // (heads + 2 * kv)
        x = _dense(qkv)
        out = torch.empty(batch, seq, heads * hd, device=x.device, dtype=x.dtype)
        rest = torch.empty_like(out) if ctx.needs_input_grad[0] else None
        lse = torch.empty(batch * heads, seq, device=x.device, dtype=torch.float32)
        if out.numel():
            with _DeviceGuard(x):
                _check(library().rv_window_attn_fwd(
                    x.data_ptr(), batch, seq, heads, kv, hd, _CODES[x.dtype], window, sinks,
                    out.data_ptr(), None if rest is None else rest.data_ptr(), lse.data_ptr(),
                    _stream(x)), "rv_window_attn_fwd")
        ctx.save_for_backward(x, out, rest, lse)
        ctx.sizes = (batch, seq, heads, kv, hd)
        ctx.span = (window, sinks)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        x, out, rest, lse = ctx.saved_tensors
        dqkv = torch.empty_like(x)
        if out.numel():
            lib, dout = library(), _dense(dout)
            nbytes = lib.rv_window_attn_bwd_workspace_bytes(*ctx.sizes, *ctx.span)
            if nbytes < 0:
                _check(-nbytes, "rv_window_attn_bwd_workspace_bytes")
            with _DeviceGuard(x):
                ws = torch.empty(nbytes, device=x.device, dtype=torch.uint8)
                _check(lib.rv_window_attn_bwd(
                    x.data_ptr(), out.data_ptr(), rest.data_ptr(), dout.data_ptr(),
                    lse.data_ptr(), *ctx.sizes,
                    _CODES[x.dtype], *ctx.span, dqkv.data_ptr(), ws.data_ptr(), nbytes,
                    _stream(x)), "rv_window_attn_bwd")
        return dqkv, None, None, None, None


def check_window(window: Optional[int], sinks: int, what: str) -> None:
    if window is not None and window < 1:
        raise ValueError(f"{what} needs a window of at least one token")
    if sinks < 0:
        raise ValueError(f"{what} needs sinks >= 0")


def window_attention(qkv: torch.Tensor, heads: int, window: int, sinks: int = 0, *,
                     kv_heads: Optional[int] = None) -> torch.Tensor:
    """Causal attention with a sliding window and sinks, differentiable in ``qkv``.

    ``qkv`` fp16 or bf16 [B, T, (heads + 2 kv_heads) hd], hd 32, 64 or 128: the query
    heads, then the key heads, then the value heads (``kv_heads`` None: as many as
    query heads); query head h reads key and value head h // (heads // kv_heads).  Query
    i sees key j <= i where i - j < ``window`` or j < ``sinks``.  Returns [B, T, heads hd] in
    qkv's type.  Scores, softmax statistics and sums are held in fp32; the weights are
    rounded to qkv's type for the product with the values, as are the scores'
    gradients (in fp16 times a power of two that goes by the size of the gradient that
    comes in: they keep their digits however small it is).  Deterministic.  As in any product, a NaN or an infinity in a key or value
    may reach queries that do not see it (and so may one in a query or gradient reach the
    gradients of keys it does not see)."""
    if qkv.ndim != 3:
        raise ValueError("window_attention needs qkv [B, T, (heads + 2 kv_heads) hd]")
    kv, _ = packed_heads(qkv, heads, kv_heads, "window_attention")
    check_window(window, sinks, "window_attention")
    return WindowAttention.apply(qkv, heads, kv, window, sinks)


class Rotary:
    """Cosines and sines by position for heads of size ``head_dim``: pair i of a head turns by
    position * base^(-2 i / head_dim).  Pairs are the columns (i, i + head_dim / 2), or (2 i,
    2 i + 1) if ``interleaved``.  ``table`` fp32 [positions, head_dim / 2, 2], made in 64
    bits."""

    def __init__(self, head_dim: int, positions: int, base: float = 10000.0,
                 interleaved: bool = False, device="cuda"):
        if head_dim not in HEAD_DIMS or positions < 1 or not base > 0.0:
            raise ValueError(f"Rotary needs a head size in {HEAD_DIMS}, positions >= 1 and "
                             "base > 0")
        self.head_dim, self.positions = head_dim, positions
        self.base, self.interleaved = float(base), bool(interleaved)
        rate = torch.arange(0, head_dim, 2, dtype=torch.float64, device=device)
        rate = rate.mul_(-math.log(self.base) / head_dim).exp_()
        at = torch.arange(positions, dtype=torch.float64, device=device)
        angle = at.unsqueeze(1) * rate
        self.table = torch.empty(*angle.shape, 2, dtype=torch.float32, device=device)
        torch.cos(angle, out=self.table[..., 0])  # rounded on the way
        torch.sin(angle, out=self.table[..., 1])

    def to(self, device) -> "Rotary":
        """A copy with its table on ``device``."""
        other = object.__new__(Rotary)
        other.__dict__.update(self.__dict__, table=self.table.to(device))
        return other

    def check(self, like: torch.Tensor, head_dim: int, what: str) -> None:
        if self.head_dim != head_dim or self.table.device != like.device:
            raise ValueError(f"{what} needs a Rotary of its head size on its device")


class RotateQKV(torch.autograd.Function):
    """See ``rotate_qkv``."""

    @staticmethod
    def _turn(x, ctx, back):
        y = torch.empty_like(x)
        if y.numel():
            rotary, (heads, kv, hd) = ctx.rotary, ctx.heads
            with _DeviceGuard(x):
                _check(library().rv_rotate_qkv(
                    x.data_ptr(), y.data_ptr(), x.shape[0] * x.shape[1], x.shape[1], heads, kv, hd,
                    _CODES[x.dtype], rotary.table.data_ptr(), rotary.positions,
                    None if ctx.positions is None else ctx.positions.data_ptr(),
                    rotary.interleaved, back, _stream(x)), "rv_rotate_qkv")
        return y

    @staticmethod
    def forward(ctx, qkv, heads, kv, hd, rotary, positions):
        ctx.rotary, ctx.heads = rotary, (heads, kv, hd)
        ctx.save_for_backward(positions)
        ctx.positions = positions
        out = RotateQKV._turn(_dense(qkv), ctx, False)
        del ctx.positions
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, gradient):
        ctx.positions, = ctx.saved_tensors
        out = RotateQKV._turn(_dense(gradient), ctx, True)
        del ctx.positions
        return out, None, None, None, None, None


def rotate_qkv(qkv: torch.Tensor, heads: int, rotary: Rotary,
               positions: Optional[torch.Tensor] = None, *,
               kv_heads: Optional[int] = None) -> torch.Tensor:
    """``qkv`` [B, T, (heads + 2 kv_heads) hd], fp16 or bf16, with its queries and keys rotated
    by their positions (int32 [B, T]; None: 0 .. T - 1), values as they are; differentiable in
    ``qkv``.  Products in fp32, rounded once.  A position outside the table gives NaN
    queries and keys."""
    if qkv.ndim != 3:
        raise ValueError("rotate_qkv needs qkv [B, T, (heads + 2 kv_heads) hd]")
    kv, hd = packed_heads(qkv, heads, kv_heads, "rotate_qkv")
    rotary.check(qkv, hd, "rotate_qkv")
    if positions is None:
        if qkv.shape[1] > rotary.positions:
            raise ValueError("sequence exceeds the positions of the Rotary table")
    elif (positions.dtype != torch.int32 or positions.shape != qkv.shape[:2]
          or positions.device != qkv.device):
        raise ValueError("positions must be int32 [B, T] on qkv's device")
    else:
        positions = positions.contiguous()
    return RotateQKV.apply(qkv, heads, kv, hd, rotary, positions)


def reference_rotation(qkv: torch.Tensor, heads: int, rotary: Rotary) -> torch.Tensor:
    """``rotate_qkv`` of as many key heads as query heads in torch operations, for calls the
    kernels do not cover."""
    batch, length, width = qkv.shape
    x = qkv.view(batch, length, 3, heads, -1)
    turn = rotary.table[:length].to(qkv.device).unsqueeze(1).unsqueeze(1)  # [T, 1, 1, hd/2, 2]
    cos, sin = turn.unbind(-1)
    y, half = x[:, :, :2], rotary.head_dim // 2
    a, b = (y[..., 0::2], y[..., 1::2]) if rotary.interleaved else (y[..., :half], y[..., half:])
    pair = (a * cos - b * sin, a * sin + b * cos)
    y = torch.stack(pair, -1).flatten(-2) if rotary.interleaved else torch.cat(pair, -1)
    return torch.cat([y.to(qkv.dtype), x[:, :, 2:]], 2).reshape(batch, length, width)


def reference_window_attention(qkv: torch.Tensor, heads: int, window: Optional[int], sinks: int,
                               dropout: float = 0.0) -> torch.Tensor:
    """``window_attention`` of as many key heads as query heads by torch's attention with a
    mask, for calls the kernels do not cover."""
    if window is None:
        return reference_attention(qkv, heads, dropout)
    batch, length, width = qkv.shape
    d = width // 3
    q, k, v = qkv.view(batch, length, 3, heads, d // heads).permute(2, 0, 3, 1, 4).unbind(0)
    at = torch.arange(length, device=qkv.device)
    gap = at.unsqueeze(1) - at
    mask = (gap >= 0) & ((gap < window) | (at < sinks))
    mixed = F.scaled_dot_product_attention(q, k, v, attn_mask=mask, dropout_p=dropout)
    return mixed.transpose(1, 2).reshape(batch, length, d)


def _local_forward(attn, x, dropout):
    """The attention of a layer with a window, a rotation, or both."""
    qkv, heads, rotary = attn.qkv(x), attn.n_heads, attn._rv_rotary
    window, sinks = attn._rv_window, attn._rv_sinks
    hd = qkv.shape[-1] // (3 * heads)
    if qkv.ndim == 3 and rotary is not None and qkv.shape[1] > rotary.positions:
        raise ValueError("sequence exceeds the positions of the Rotary table")
    if (qkv.is_cuda and qkv.dtype in _CODES and qkv.ndim == 3 and dropout == 0.0
            and hd in HEAD_DIMS):
        paths.took("attention", "hip")
        if rotary is not None:
            qkv = rotate_qkv(qkv, heads, rotary)
        # (no window: one of the whole sequence)
        mixed = window_attention(qkv, heads, window or max(1, qkv.shape[1]), sinks)
    else:
        paths.took("attention", "sdpa",
                   f"windowed attention needs a CUDA fp16 or bf16 qkv, head size in {HEAD_DIMS} "
                   f"and no dropout (got {qkv.dtype} on {qkv.device.type}, head size {hd}, "
                   f"dropout {dropout})")
        if rotary is not None:
            qkv = reference_rotation(qkv, heads, rotary)
        mixed = reference_window_attention(qkv, heads, window, sinks, dropout)
    return attn.proj(mixed)


def enable_attention(model: torch.nn.Module, window: Optional[int] = None, sinks: int = 0,
                     rotary: Optional[Rotary] = None) -> None:
    """Route every block's attention through the fused kernels where they apply.

    ``window`` (None: all earlier tokens) and ``sinks`` limit what a token sees, as in
    ``window_attention``; ``rotary`` rotates queries and keys by position
    (``rotate_qkv``).  Calls that the kernels do not cover compute the same in torch."""
    check_window(window, sinks, "enable_attention")
    if rotary is not None:
        sizes = {block.attn.head_dim for block in model.blocks}
        if sizes - {rotary.head_dim}:
            raise ValueError("enable_attention needs a Rotary of the model's head size")

    def forward(attn, x):
        dropout = attn.dropout if attn.training else 0.0
        if attn._rv_window is not None or attn._rv_rotary is not None:
            return _local_forward(attn, x, dropout)
        if _layer_supported(attn, x, dropout):
            paths.took("linear", "mfma")
            paths.took("attention", "hip")
            paths.took("linear", "mfma")
            return AttentionLayer.apply(x, attn.qkv.weight, attn.proj.weight, attn.n_heads)
        qkv = attn.qkv(x)
        if supported(qkv, attn.n_heads, dropout):
            paths.took("attention", "hip")
            mixed = CausalAttention.apply(qkv, attn.n_heads)
        else:
            paths.took("attention", "sdpa",
                       f"attention kernels need a CUDA fp16 qkv, head size in {HEAD_DIMS} and no "
                       f"dropout (got {qkv.dtype} on {qkv.device.type}, head size "
                       f"{qkv.shape[-1] // (3 * attn.n_heads)}, dropout {dropout})")
            mixed = reference_attention(qkv, attn.n_heads, dropout)
        return attn.proj(mixed)
    for block in model.blocks:
        block.attn._rv_window, block.attn._rv_sinks = window, sinks
        block.attn._rv_rotary = rotary
        block.attn.forward = types.MethodType(forward, block.attn)
