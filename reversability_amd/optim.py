"""AdamW on one multi-tensor HIP kernel, a drop-in for torch.optim.AdamW.

The training step of the reference (scripts/benchmark_optimized.py:38-40,
66-80; scripts/train_baseline.py:270-284) runs ``torch.optim.AdamW(params,
lr, betas=(0.9, 0.95), weight_decay=0.1)`` behind ``torch.amp.GradScaler``:
``unscale_``, ``clip_grad_norm_``, ``scaler.step``, ``scaler.update``.
``FusedAdamW`` keeps that constructor and that driving sequence and replaces
torch's per-operation multi-tensor kernels with one pass over parameters,
gradients and both moments (``rv_adamw_step``), in torch's arithmetic order.

It declares ``_step_supports_amp_scaling``: ``GradScaler.step`` then hands it
the device ``found_inf`` flag (and ``grad_scale`` when gradients were not
unscaled first) instead of synchronising on the host; an overflowing step
changes no parameter, moment or step count.  The step count is a device
tensor per parameter group (shared by the group's ``state[p]["step"]``).
Supported: fp32 dense CUDA parameters, amsgrad=False, maximize=False; other
configurations raise.

``unscale_clip_(scaler, max_norm)`` stands for the reference's
``scaler.unscale_(opt); torch.nn.utils.clip_grad_norm_(params, max_norm)``
(scripts/train_baseline.py:278-280) in one read of the gradients: it computes
the norm of the unscaled gradients and the clip coefficient on the device
(``rv_grad_sq_partials`` / ``rv_grad_clip_coef``), records the overflow flag
with the scaler as ``unscale_`` does, and leaves both multiplies to the next
``step()``, which applies them as it reads each gradient
(``rv_adamw_step_clipped``) -- the values the two passes would have written.
Between the two calls ``p.grad`` still holds the scaled, unclipped gradient.

``FusedAdamW8bit`` is the same optimizer with the moments of large tensors in 8
bits (no counterpart in the reference).
"""
from __future__ import annotations

import ctypes

import torch
from torch.optim import Optimizer

from ._hip import _check, _DeviceGuard, _stream, library


class FusedAdamW(Optimizer):
    _step_supports_amp_scaling = True

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
                 amsgrad=False, *, maximize=False, foreach=None, capturable=False,
                 differentiable=False, fused=None):
        if amsgrad or maximize or differentiable:
            raise ValueError("FusedAdamW supports amsgrad=False, maximize=False, "
                             "differentiable=False")
        if not 0.0 <= lr or not 0.0 <= eps or not 0.0 <= weight_decay:
            raise ValueError("Invalid learning rate, epsilon or weight decay")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"Invalid betas: {betas}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def _group_params(self, group):
        """A group's parameters with elements and a gradient; raises for what the kernels do
        not take (they read everything through its address) and changes nothing."""
        params = [p for p in group["params"] if p.grad is not None and p.numel()]
        if not params:
            return params
        dev = params[0].device
        for p in params:
            g = p.grad
            if p.dtype != torch.float32 or not p.is_cuda or g.is_sparse:
                raise ValueError("FusedAdamW requires dense CUDA (ROCm device) FP32 parameters")
            if p.device != dev or not (p.is_contiguous() and g.is_contiguous()):
                raise ValueError("FusedAdamW requires contiguous parameters and gradients, a "
                                 "group's on one device")
            st = self.state.get(p)
            if st and "exp_avg" in st and (st["exp_avg"].device != dev
                                           or st["exp_avg_sq"].device != dev):
                raise ValueError("FusedAdamW's state must be on its parameter's device")
        step = self._step_count(group)
        if step is not None and not (torch.is_tensor(step) and step.dtype == torch.float32
                                     and step.device == dev):
            raise ValueError("FusedAdamW's state needs its step count as an fp32 tensor on the "
                             "parameters' device")
        return params

    def _step_count(self, group):
        for p in group["params"]:
            st = self.state.get(p)
            if st and "step" in st:
                return st["step"]
        return None

    def _group_state(self, group, params):
        """The group's step count; makes the state that ``params`` lack."""
        step = self._step_count(group)
        if step is None:
            step = torch.zeros((), device=params[0].device, dtype=torch.float32)
        for p in params:
            st = self.state[p]
            if "exp_avg" not in st:
                st.update(self._new_moments(p))
            st["step"] = step
        return step

    def _check_shapes(self, state_dict):
        """Moments of another size than the parameter's are refused: the kernels would
        read past them."""
        for p, st in self._saved(state_dict):
            for name in ("exp_avg", "exp_avg_sq"):
                if name in st and st[name].shape != p.shape:
                    raise ValueError(f"{name} of shape {tuple(st[name].shape)} for a parameter "
                                     f"of shape {tuple(p.shape)}")

    def _saved(self, state_dict):
        """Each parameter and what the checkpoint holds for it."""
        places = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        return [(p, state_dict["state"].get(i, {})) for i, p in zip(places, params)]

    def _place_state(self):
        """What the kernels read through its address, after loading (torch leaves it as the
        checkpoint had it): one step count per group, fp32, on the parameters' device
        and apart from the checkpoint's; moments in the order of their elements."""
        for group in self.param_groups:
            step = None
            for p in group["params"]:
                st = self.state.get(p, {})
                if "step" in st:
                    if step is None:
                        step = torch.as_tensor(st["step"]).to(p.device, torch.float32,
                                                              copy=True).reshape(())
                    st["step"] = step
                for name in ("exp_avg", "exp_avg_sq"):
                    if name in st:
                        st[name] = st[name].contiguous()

    def _new_moments(self, p):
        return {k: torch.zeros_like(p, memory_format=torch.preserve_format)
                for k in ("exp_avg", "exp_avg_sq")}

    def load_state_dict(self, state_dict):
        if any("exp_avg_scale" in st for st in state_dict["state"].values()):
            raise ValueError("these moments are in 8 bits: load them into FusedAdamW8bit")
        self._check_shapes(state_dict)
        super().load_state_dict(state_dict)
        self._place_state()

    @torch.no_grad()
    def unscale_clip_(self, scaler, max_norm: float) -> torch.Tensor:
        """``scaler.unscale_(self)`` + ``clip_grad_norm_(all parameters with a
        gradient, max_norm)`` (norm type 2); returns the total norm of the
        unscaled gradients (a device scalar).  ``scaler`` may be None (clip
        only)."""
        from torch.amp.grad_scaler import OptState
        lib = library()
        params = [p for group in self.param_groups for p in group["params"]
                  if p.grad is not None and p.numel()]
        if not params:
            return torch.zeros(())
        dev = params[0].device
        for p in params:
            if p.grad.dtype != torch.float32 or not p.grad.is_contiguous() or p.grad.device != dev:
                raise ValueError("unscale_clip_ requires contiguous fp32 gradients on one device")
        state = None
        inv = None
        if scaler is not None and scaler.is_enabled():
            state = scaler._per_optimizer_states[id(self)]
            if state["stage"] is OptState.UNSCALED:
                raise RuntimeError("unscale_() has already been called on this optimizer since "
                                   "the last update().")
            if state["stage"] is OptState.STEPPED:
                raise RuntimeError("unscale_() is being called after step().")
            inv = scaler._scale.double().reciprocal().float()
        limit = lib.rv_adamw_max_tensors()
        groups = [params[i:i + limit] for i in range(0, len(params), limit)]
        numels = [(ctypes.c_int64 * len(g))(*[p.numel() for p in g]) for g in groups]
        counts = [lib.rv_grad_chunks(n, len(g)) for n, g in zip(numels, groups)]
        for c in counts:
            if c < 0:
                _check(-c, "rv_grad_chunks")
        total_chunks = sum(counts)
        work = torch.empty(2 * total_chunks + 3, device=dev, dtype=torch.float32)
        partials, flags = work[:total_chunks], work[total_chunks:2 * total_chunks]
        total, coef, found = (work[2 * total_chunks + i:2 * total_chunks + i + 1]
                              for i in range(3))
        with _DeviceGuard(params[0]):
            stream = _stream(params[0])
            first = 0
            for g, n, c in zip(groups, numels, counts):
                ptrs = (ctypes.c_void_p * len(g))(*[p.grad.data_ptr() for p in g])
                _check(lib.rv_grad_sq_partials(len(g), ptrs, n,
                                               inv.data_ptr() if inv is not None else None,
                                               partials.data_ptr(), flags.data_ptr(), first, stream),
                       "rv_grad_sq_partials")
                first += c
            _check(lib.rv_grad_clip_coef(partials.data_ptr(), flags.data_ptr(), total_chunks,
                                         float(max_norm), total.data_ptr(), coef.data_ptr(),
                                         found.data_ptr(), stream), "rv_grad_clip_coef")
        if state is not None:
            state["found_inf_per_device"] = {dev: found.reshape(())}
            state["stage"] = OptState.UNSCALED
        self._pending = (inv, coef)
        return total.reshape(())

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        lib = library()
        found_inf = getattr(self, "found_inf", None)
        grad_scale = getattr(self, "grad_scale", None)
        # every refusal comes before anything is launched or forgotten
        work = [(group, self._group_params(group)) for group in self.param_groups]
        pending_inv, clip = getattr(self, "_pending", (None, None))
        self._pending = (None, None)
        for group, params in work:
            if not params:
                continue
            step = self._group_state(group, params)
            dev = params[0].device
            with _DeviceGuard(params[0]):
                stream = _stream(params[0])
                fi = found_inf.to(dev, torch.float32) if found_inf is not None else None
                inv = (grad_scale.to(dev, torch.float64).reciprocal().to(torch.float32)
                       if grad_scale is not None else pending_inv)
                _check(lib.rv_adamw_advance(step.data_ptr(),
                                            fi.data_ptr() if fi is not None else None, stream),
                       "rv_adamw_advance")
                device = (step.data_ptr(), *(t.data_ptr() if t is not None else None
                                             for t in (fi, inv, clip)), stream)
                self._update(lib, group, params, device)
        return loss

    def _update(self, lib, group, params, device):
        """One update of a group's ``params`` (step count, overflow flag, inverse scale
        and clip coefficient on the device, stream: ``device``)."""
        beta1, beta2 = group["betas"]
        limit = lib.rv_adamw_max_tensors()
        for start in range(0, len(params), limit):
            chunk = params[start:start + limit]
            n = len(chunk)
            P = ctypes.c_void_p * n
            ptrs = [P(*[t.data_ptr() for t in ts]) for ts in (
                chunk, [p.grad for p in chunk], [self.state[p]["exp_avg"] for p in chunk],
                [self.state[p]["exp_avg_sq"] for p in chunk])]
            numel = (ctypes.c_int64 * n)(*[p.numel() for p in chunk])
            _check(lib.rv_adamw_step_clipped(
                n, ptrs[0], ptrs[1], ptrs[2], ptrs[3], numel, float(group["lr"]),
                float(beta1), float(beta2), float(group["eps"]), float(group["weight_decay"]),
                *device), "rv_adamw_step_clipped")


# A moment held in 8 bits: its e4m3 values and, under this name, its scale bytes.
_SCALES = {"exp_avg": "exp_avg_scale", "exp_avg_sq": "exp_avg_sq_scale"}


class FusedAdamW8bit(FusedAdamW):
    """``FusedAdamW`` with the moments of large tensors in 8 bits: 2.06 bytes of state
    per parameter instead of 8 (``rv_adamw8_step``).

    A tensor of at least ``min_8bit_numel`` elements keeps ``exp_avg`` and
    ``exp_avg_sq`` as torch.float8_e4m3fn of the parameter's shape with one power of
    two per 32 consecutive elements (``exp_avg_scale``, ``exp_avg_sq_scale``: uint8,
    value = e4m3 * 2^(byte - 127)); smaller ones (norm weights) keep them in fp32.
    The update uses the fp32 moments of its step; what is stored is rounded to
    nearest (``exp_avg`` where beta1 <= 0.9375) or at random with its expectation kept
    (``exp_avg_sq``, and ``exp_avg`` of a larger beta1, whose change per step is below
    half a step of e4m3).  The random bits follow
    from ``seed``, the parameter's place, the step count and the element: a run
    repeats bit for bit.  GradScaler, ``unscale_clip_``, the device-side step count
    and graph capture work as in ``FusedAdamW``; ``moments(p)`` returns a
    parameter's moments in fp32.  A checkpoint of ``FusedAdamW`` can be loaded (its
    moments stay in fp32; a large parameter that it has none for gets 8-bit ones), not
    the other way round.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
                 amsgrad=False, *, min_8bit_numel=4096, seed=0, maximize=False, foreach=None,
                 capturable=False, differentiable=False, fused=None):
        if min_8bit_numel < 1:
            raise ValueError("min_8bit_numel must be positive")
        if not 0 <= seed < 1 << 32:
            raise ValueError("seed must be an unsigned 32-bit number")
        self.min_8bit_numel = min_8bit_numel
        super().__init__(params, lr, betas, eps, weight_decay, amsgrad, maximize=maximize,
                         foreach=foreach, capturable=capturable, differentiable=differentiable,
                         fused=fused)
        self.defaults["seed"] = seed  # saved with the groups: a resumed run goes on alike
        for group in self.param_groups:
            group.setdefault("seed", seed)

    def __getstate__(self):  # of copies and pickles: torch keeps defaults, groups and state
        return {**super().__getstate__(), "min_8bit_numel": self.min_8bit_numel}

    def _new_moments(self, p):
        if p.numel() < self.min_8bit_numel:
            return super()._new_moments(p)
        blocks = -(-p.numel() // library().rv_adamw8_block())
        st = {}
        for name, scale in _SCALES.items():
            codes = torch.zeros(p.shape, device=p.device, dtype=torch.uint8)
            st[name] = codes.view(torch.float8_e4m3fn)
            st[scale] = torch.zeros(blocks, device=p.device, dtype=torch.uint8)
        return st

    def _update(self, lib, group, params, device):
        ordinal = {p: i for i, p in enumerate(q for g in self.param_groups for q in g["params"])}
        small = [p for p in params if "exp_avg_scale" not in self.state[p]]
        large = [p for p in params if "exp_avg_scale" in self.state[p]]
        if small:
            super()._update(lib, group, small, device)
        beta1, beta2 = group["betas"]
        limit = lib.rv_adamw8_max_tensors()
        for start in range(0, len(large), limit):
            chunk = large[start:start + limit]
            n = len(chunk)
            P = ctypes.c_void_p * n
            states = [self.state[p] for p in chunk]
            ptrs = [P(*[t.data_ptr() for t in ts]) for ts in (
                chunk, [p.grad for p in chunk],
                *([st[k] for st in states] for k in ("exp_avg", "exp_avg_scale", "exp_avg_sq",
                                                     "exp_avg_sq_scale")))]
            numel = (ctypes.c_int64 * n)(*[p.numel() for p in chunk])
            places = (ctypes.c_uint32 * n)(*[ordinal[p] for p in chunk])
            _check(lib.rv_adamw8_step(
                n, *ptrs, numel, places, group["seed"], float(group["lr"]), float(beta1),
                float(beta2), float(group["eps"]), float(group["weight_decay"]), *device),
                "rv_adamw8_step")

    @torch.no_grad()
    def moments(self, p) -> tuple:
        """fp32 (exp_avg, exp_avg_sq) of a parameter that has taken a step."""
        st, out = self.state[p], []
        for name, scale in _SCALES.items():
            value = st[name].float()
            if scale in st:
                block = library().rv_adamw8_block()
                # ldexp in two factors: 2^(byte - 127) alone may be no normal number
                exponent = st[scale].double().repeat_interleave(block)[:p.numel()] - 127
                value = (value.double() * exponent.exp2().view(p.shape)).float()
            out.append(value)
        return tuple(out)

    def load_state_dict(self, state_dict):
        """As torch's, which casts every floating or parameter-like state to the
        parameter's type; the 8-bit moments keep theirs."""
        self._check_shapes(state_dict)
        saved = self._saved(state_dict)
        block = library().rv_adamw8_block()
        for p, st in saved:
            for name, scale in _SCALES.items():
                if (scale in st) != (_SCALES["exp_avg"] in st) or scale in st and (
                        st[name].dtype != torch.float8_e4m3fn or st[scale].dtype != torch.uint8
                        or st[scale].numel() != -(-p.numel() // block)):
                    raise ValueError(f"{name} is not the 8-bit moment of its parameter")
        seeds = [g["seed"] for g in self.param_groups]
        Optimizer.load_state_dict(self, state_dict)
        for group, seed in zip(self.param_groups, seeds):
            group.setdefault("seed", seed)  # a plain checkpoint's groups have none
        self._place_state()
        for p, st in saved:
            for name, scale in _SCALES.items():
                if scale in st:
                    for key in (name, scale):
                        t = st[key]
                        bits = t.contiguous().view(torch.uint8).to(p.device, copy=True)
                        self.state[p][key] = bits.view(t.dtype)
