"""Preference and policy operators and the 8-bit AdamW on the CPU: their refusals, and
the C ABI's argument checks (no kernel is launched)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from reversability_amd import _hip, build_model
from reversability_amd.optim import FusedAdamW8bit
from reversability_amd.preference import (max_chunk, policy_loss, preference_backward,
                                          preference_loss, tied_head_logprobs)

NULL, BAD_SIZE, UNSUPPORTED, WORKSPACE = 1, 2, 3, 4
FAKE = ctypes.c_void_p(4096)  # never dereferenced: validation fails first
ODD = ctypes.c_void_p(4100)


def test_cpu_tensors_are_refused():
    x, head = torch.zeros(2, 64).half(), torch.zeros(64, 64).half()
    with pytest.raises(ValueError, match="CUDA"):
        tied_head_logprobs(x, head, 64, torch.zeros(2, dtype=torch.int64))
    logp = torch.zeros(2, 3)
    with pytest.raises(ValueError, match="CUDA"):
        preference_loss(logp, logp)
    with pytest.raises(ValueError, match="CUDA"):
        policy_loss(logp, logp, torch.zeros(2))
    model = build_model({"model": {"vocab_size": 31, "max_sequence_length": 8, "n_layers": 1,
                                   "n_heads": 2, "d_model": 8, "d_ff": 16}})
    ids = torch.zeros(2, 4, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        preference_backward(model, ids, ids, logp)
    p = torch.zeros(5000, requires_grad=True)
    p.grad = torch.zeros(5000)
    with pytest.raises(ValueError, match="CUDA"):
        FusedAdamW8bit([p]).step()


@pytest.mark.parametrize("options", [{"min_8bit_numel": 0}, {"seed": -1}, {"seed": 2 ** 32},
                                     {"lr": -1.0}, {"betas": (0.9, 1.0)}, {"amsgrad": True}])
def test_optimizer_options_are_checked(options):
    with pytest.raises(ValueError):
        FusedAdamW8bit([torch.zeros(3, requires_grad=True)], **options)


def test_chunks_fill_their_bytes():
    assert max_chunk(50304) == (1 << 32) // (2 * 50304) // 256 * 256
    assert max_chunk(64) * 128 <= 1 << 32 and max_chunk(1 << 30) == 256


def test_head_logp_argument_checks():
    lib = _hip.library()
    f16, bf16, f32 = _hip.RV_F16, _hip.RV_BF16, _hip.RV_F32
    need = lib.rv_head_logp_workspace_bytes(51, 256, 50257)
    assert need > 0

    def fwd(x=FAKE, head=FAKE, rows=51, d=256, vocab=50257, dtype=f16, labels=FAKE, logp=FAKE,
            ws=FAKE, nbytes=need):
        return lib.rv_head_logp_fwd(x, head, rows, d, vocab, dtype, labels, -100, logp, FAKE, ws,
                                    nbytes, None)
    assert fwd(x=None) == fwd(labels=None) == fwd(logp=None) == NULL
    assert fwd(rows=0) == fwd(vocab=0) == fwd(d=-8) == BAD_SIZE
    assert fwd(d=100) == fwd(dtype=f32) == fwd(x=ODD) == fwd(head=ODD) == UNSUPPORTED
    assert fwd(ws=None) == fwd(nbytes=need - 1) == fwd(ws=ODD) == WORKSPACE
    assert lib.rv_head_logp_workspace_bytes(0, 256, 10) == -BAD_SIZE
    assert lib.rv_head_logp_workspace_bytes(5, 4, 10) == -UNSUPPORTED
    ws = lib.rv_head_logp_bwd_workspace_bytes(51, 256, 50257, 50304)
    assert ws > 51 * 50304 * 2
    assert lib.rv_head_logp_bwd_workspace_bytes(51, 256, 50257, 50240) == -BAD_SIZE
    assert lib.rv_head_logp_bwd_workspace_bytes((1 << 22) + 1, 256, 64, 64) == -UNSUPPORTED

    def bwd(d=256, padded=50304, dtype=f16, lse=FAKE, grad=FAKE, dx=FAKE, dw=FAKE, dw_rows=50257,
            dw_dtype=f16, accumulate=0, space=FAKE, nbytes=ws):
        return lib.rv_head_logp_bwd(FAKE, FAKE, 51, d, 50257, padded, dtype, FAKE, -100, lse, grad,
                                    dx, dw, dw_rows, dw_dtype, accumulate, space, nbytes, None)
    assert bwd(lse=None) == bwd(grad=None) == NULL
    assert bwd(padded=50240) == bwd(dw_rows=50258) == BAD_SIZE
    assert bwd(padded=50300) == bwd(d=4) == bwd(dx=ODD) == bwd(dw=ODD) == UNSUPPORTED
    assert bwd(padded=1 << 23) == UNSUPPORTED  # a tile's rows pass 32-bit offsets
    assert bwd(accumulate=1) == bwd(dw_dtype=bf16) == bwd(dtype=f32, dw_dtype=f32) == UNSUPPORTED
    assert bwd(space=None) == bwd(nbytes=ws - 1) == WORKSPACE


def test_loss_argument_checks():
    lib = _hip.library()
    need = lib.rv_pref_loss_workspace_bytes(4, 100)

    def pref(logp=FAKE, ld=100, pairs=4, tokens=100, loss=FAKE, ws=FAKE, nbytes=need):
        return lib.rv_pref_loss(logp, ld, FAKE, 100, None, 0, pairs, tokens, 0.1, 0.0, 0, loss,
                                FAKE, FAKE, ws, nbytes, None)
    assert pref(logp=None) == pref(loss=None) == NULL
    assert pref(pairs=0) == pref(tokens=-1) == pref(ld=-1) == BAD_SIZE
    assert pref(ws=None) == pref(nbytes=0) == pref(ws=ctypes.c_void_p(4097)) == WORKSPACE
    assert pref(tokens=1 << 31) == pref(pairs=1 << 30) == UNSUPPORTED
    assert lib.rv_pref_loss_workspace_bytes(0, 5) == -BAD_SIZE
    assert lib.rv_pref_grad(FAKE, None, 0, FAKE, 4, 100, ODD, None) == UNSUPPORTED
    assert lib.rv_pref_grad(None, None, 0, FAKE, 4, 100, FAKE, None) == NULL
    assert lib.rv_pref_grad(None, None, 0, None, 4, 0, None, None) == 0

    need = lib.rv_policy_loss_workspace_bytes(4, 100, 1)

    def policy(logp=FAKE, seqs=4, low=0.2, high=0.2, row=1, loss=FAKE, slope=FAKE, nbytes=need):
        return lib.rv_policy_loss(logp, 100, FAKE, 100, None, 0, FAKE, row, 0, None, 0, seqs, 100,
                                  low, high, 0.0, 1, loss, FAKE, slope, FAKE, nbytes, None)
    assert policy(logp=None) == policy(loss=None) == NULL
    assert policy(seqs=-1) == policy(low=1.0) == policy(low=-0.1) == policy(high=-1.0) == BAD_SIZE
    assert policy(low=float("nan")) == policy(high=float("nan")) == policy(row=-1) == BAD_SIZE
    assert policy(slope=ODD) == UNSUPPORTED and policy(nbytes=need - 1) == WORKSPACE
    assert lib.rv_policy_grad(ODD, FAKE, FAKE, 5, FAKE, None) == UNSUPPORTED
    assert lib.rv_policy_grad(None, FAKE, FAKE, 5, FAKE, None) == NULL
    assert lib.rv_policy_grad(None, None, None, 0, None, None) == 0


def test_adamw8_argument_checks():
    lib = _hip.library()
    assert lib.rv_adamw8_block() == 32 and lib.rv_adamw8_max_tensors() >= 1
    one = (ctypes.c_void_p * 1)(4096)
    none = (ctypes.c_void_p * 1)(None)

    def step(count=1, p=one, ms=one, numel=100, t=FAKE):
        return lib.rv_adamw8_step(count, p, one, one, ms, one, one, (ctypes.c_int64 * 1)(numel),
                                  (ctypes.c_uint32 * 1)(0), 0, 1e-3, 0.9, 0.95, 1e-8, 0.1, t, None,
                                  None, None, None)
    assert step(count=0) == 0
    assert step(count=-1) == step(numel=0) == BAD_SIZE
    assert step(count=1000) == UNSUPPORTED
    assert step(p=None) == step(p=none) == step(ms=none) == step(t=None) == NULL
