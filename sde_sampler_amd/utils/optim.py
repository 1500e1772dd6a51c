"""AdamW over all tensors of a model at once, with moments in 32 or in 8 bits and gradients clipped by their global norm, in a few launches
(include/sdeh.h: sdeh_adamw_step).  What the reference's trainer does in three passes per optimisation step -- `clip_grad_norm_`, the optimizer,
and not stepping when a gradient is not finite (solver/base.py:409-427) -- is one call here, without a host synchronisation."""
from __future__ import annotations

import itertools

import numpy as np
import torch
from torch.optim.optimizer import _global_optimizer_post_hooks as _global_post
from torch.optim.optimizer import _global_optimizer_pre_hooks as _global_pre

from sde_sampler_amd import _lib as L

__all__ = ["AdamW"]


class _Bucket:
    """The parameters of one group that have one type, their moments in flat buffers (a parameter's part starts at a multiple of
    `L.MOMENT_BLOCK` entries) and the C ABI's table of them."""

    def __init__(self, params, bits: int, first_block: int):
        self.params, self.bits = params, bits
        self.dtype, self.device = params[0].dtype, params[0].device
        self.code = L.dtype_code(self.dtype)
        self.sizes = [p.numel() for p in params]
        blocks = [-(-n // L.MOMENT_BLOCK) for n in self.sizes]
        self.at = [0, *itertools.accumulate(blocks)]  # in blocks
        self.blocks = self.at[-1]
        n = self.blocks * L.MOMENT_BLOCK
        kind = torch.float32 if bits == 32 else torch.uint8
        zeros = lambda n, dtype: torch.zeros(n, device=self.device, dtype=dtype)  # noqa: E731
        self.flat = {"step": zeros(len(params), torch.float32), "exp_avg": zeros(n, kind), "exp_avg_sq": zeros(n, kind)}
        if bits == 8:
            self.flat.update(exp_avg_top=zeros(self.blocks, torch.uint8), exp_avg_sq_top=zeros(self.blocks, torch.uint8))
        # what a step writes and has a version (inference tensors have none)
        self.versioned = [[t for t in ts if not t.is_inference()] for ts in (params, self.flat.values())]
        self.states = []
        self.table = np.zeros((len(params), L.ADAMW_TENSOR_WORDS), dtype=np.int64)
        for i, (p, size, b) in enumerate(zip(params, self.sizes, blocks)):
            lo, b0 = self.at[i] * L.MOMENT_BLOCK, self.at[i]
            s = {"step": self.flat["step"][i], "exp_avg": self.flat["exp_avg"][lo:lo + size].view(p.shape),
                 "exp_avg_sq": self.flat["exp_avg_sq"][lo:lo + size].view(p.shape)}
            if bits == 8:
                s.update(exp_avg_top=self.flat["exp_avg_top"][b0:b0 + b], exp_avg_sq_top=self.flat["exp_avg_sq_top"][b0:b0 + b])
            self.states.append(s)
            top = (s["exp_avg_top"].data_ptr(), s["exp_avg_sq_top"].data_ptr()) if bits == 8 else (0, 0)
            self.table[i, 2:] = (s["exp_avg"].data_ptr(), s["exp_avg_sq"].data_ptr(), *top, s["step"].data_ptr(), size, first_block + b0)

    def rows(self):
        """(the table's rows of the parameters that have a gradient, the gradients, kept alive, and the tensors that a step on these rows writes)"""
        index, dtype = self.device.index, self.dtype
        param, grad, keep, missing = [], [], [], False
        for p, n in zip(self.params, self.sizes):
            g = p.grad
            if g is None:
                missing = True
                param.append(0)
                grad.append(0)
                continue
            if p.get_device() != index or p.dtype != dtype or p.numel() != n or not p.is_contiguous():
                raise RuntimeError(f"AdamW: a parameter of {n} entries ({dtype} on {self.device}) has become {p.numel()} entries, {p.dtype} on {p.device}, "
                                   f"{'contiguous' if p.is_contiguous() else 'not contiguous'} (parameters must be contiguous, and stay what they were)")
            if g.is_sparse or g.get_device() != index or g.dtype != dtype or g.numel() != n:
                raise RuntimeError("AdamW: gradients must be dense and of their parameter's type, size and device")
            if not g.is_contiguous():
                g = g.detach().contiguous()
                keep.append(g)
            param.append(p.data_ptr())
            grad.append(g.data_ptr())
        self.table[:, 0] = param
        self.table[:, 1] = grad
        written, flats = self.versioned
        if not missing:
            return self.table, keep, written + flats
        return self.table[self.table[:, 0] != 0], keep, [p for p in written if p.grad is not None] + flats


class AdamW(torch.optim.Optimizer):
    """Adam with decoupled weight decay (`weight_decay=0`: Adam), as torch.optim.AdamW computes it, plus

    state_bits     32: both moments in fp32, whatever the parameters' type (the state has torch.optim.AdamW's keys and loads its state dicts);
                   8: a byte each, blocks of 256 entries sharing their largest exponent -- 2 bytes a parameter instead of 8.  Rounded
                   stochastically, with bits that follow from (seed, step, place): a run is reproducible, and a slow average still moves.
    max_grad_norm  clip the gradients of all groups together to this norm first (clip_grad_norm_'s formula); `grad_norm` then holds their norm
                   before clipping (0-d tensor).  The `.grad`s themselves stay as they are
    seed           of the rounding of 8-bit moments (it belongs to the state dict)

    `lr` may be a one-element fp32 tensor on the parameters' device (a schedule under a captured graph).  A step never synchronises and, from the second
    on, may be captured (utils/graphs.py: GraphedTrainStep).  Parameters are contiguous fp32, bf16 or fp16 tensors on one HIP device; those without a
    gradient are left alone.  Parameters must not share memory.  A parameter group added later moves the moments: step once, then capture again.
    The state's tensors are views of flat buffers: write into them, do not replace them."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01, *, state_bits: int = 32,
                 max_grad_norm: float | None = None, seed: int = 0):
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: state_bits is 8 or 32, got {state_bits}")
        if max_grad_norm is not None and not max_grad_norm > 0.0:
            raise ValueError(f"AdamW: max_grad_norm must be positive, got {max_grad_norm}")
        self.state_bits, self.max_grad_norm, self.seed = state_bits, max_grad_norm, int(seed)
        self.grad_norm: torch.Tensor | None = None
        self._buckets: list | None = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    @staticmethod
    def _check_group(group):
        lr, (b1, b2) = group["lr"], group["betas"]
        if isinstance(lr, torch.Tensor):
            if not (lr.is_cuda and lr.dtype == torch.float32 and lr.numel() == 1):
                raise ValueError("AdamW: a tensor lr must be one fp32 element on the HIP device")
        elif not lr >= 0.0:
            raise ValueError(f"AdamW: lr must not be negative, got {lr}")
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and group["eps"] >= 0.0 and group["weight_decay"] >= 0.0):
            raise ValueError(f"AdamW: betas in [0, 1), eps and weight_decay >= 0, got {group['betas']}, {group['eps']}, {group['weight_decay']}")

    def add_param_group(self, param_group):
        if isinstance(param_group, dict):  # (anything else is the base class's to refuse)
            self._check_group({**self.defaults, **param_group})
        super().add_param_group(param_group)
        self._buckets = None

    def __getstate__(self):
        return {**super().__getstate__(), "state_bits": self.state_bits, "max_grad_norm": self.max_grad_norm, "seed": self.seed}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._buckets, self.grad_norm = None, None

    # -- state ---------------------------------------------------------------------------------------------------------------------------
    def _plan(self) -> list:
        """[(group, its buckets)]; flat state buffers are made here and take over what `self.state` holds."""
        if self._buckets is not None:
            return self._buckets
        plan, first, device, seen = [], 0, None, set()
        for group in self.param_groups:
            by_type: dict = {}
            for p in group["params"]:
                if not p.is_cuda:
                    raise RuntimeError("AdamW runs on the HIP device only (got a CPU parameter); there is no CPU path in this package")
                if L.dtype_code(p.dtype) is None:
                    raise L.SdehUnsupported(-2, f"AdamW: {p.dtype} (the kernels take float32, bfloat16 and float16)")
                if device is not None and p.device != device:
                    raise L.SdehUnsupported(-2, f"AdamW: parameters on {device} and {p.device} (one optimizer, one device)")
                device = p.device
                if id(p) in seen:
                    raise ValueError("AdamW: a parameter is there twice")
                seen.add(id(p))
                by_type.setdefault(p.dtype, []).append(p)
            if by_type and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("AdamW: the state cannot be made while the stream is capturing (every replay would zero it): step once before")
            buckets = []
            for params in by_type.values():
                bucket = _Bucket(params, self.state_bits, first)
                first += bucket.blocks
                for p, own in zip(params, bucket.states):
                    old = self.state.get(p)
                    if old:
                        self._adopt(own, old)
                    self.state[p] = own
                buckets.append(bucket)
            plan.append((group, buckets))
        self._buckets, self._device = plan, device
        n = sum(len(b.params) for _, bs in plan for b in bs)
        if device is not None:
            self._scratch = torch.empty(max(4, L.load().sdeh_adamw_scratch_floats(n)), device=device, dtype=torch.float32)
            self.grad_norm = torch.zeros((), device=device) if self.max_grad_norm is not None else None
        return plan

    @staticmethod
    def _check_state(own: dict, other: dict) -> None:
        if set(other) != set(own):
            raise ValueError(f"AdamW: a state with {sorted(other)} does not fit one with {sorted(own)} (state_bits differ?)")
        for k, t in own.items():
            s = torch.as_tensor(other[k])
            if s.numel() != t.numel() or (t.dtype == torch.uint8) != (s.dtype == torch.uint8):
                raise ValueError(f"AdamW: {k} is {tuple(s.shape)} {s.dtype}, expected {tuple(t.shape)} {t.dtype}")

    def _adopt(self, own: dict, other: dict) -> None:
        self._check_state(own, other)
        for k, t in own.items():
            t.copy_(torch.as_tensor(other[k]).reshape(t.shape))

    def _check_loaded(self, state_dict) -> None:
        """Refuses what does not fit, before anything is changed.  (Numbers of groups and parameters are the base class's to refuse.)"""
        for group in state_dict["param_groups"]:
            if group.get("amsgrad") or group.get("maximize") or (group.get("weight_decay") and group.get("decoupled_weight_decay") is False):
                raise ValueError("AdamW: a state dict with amsgrad, maximize or coupled weight decay")
            lacks = [k for k in ("lr", "betas", "eps", "weight_decay") if k not in group]
            if lacks:
                raise ValueError(f"AdamW: a state dict whose groups lack {lacks}")
            lr = group["lr"]
            if isinstance(lr, torch.Tensor) and lr.numel() != 1:
                raise ValueError(f"AdamW: a tensor lr must be one element, got {tuple(lr.shape)}")
            self._check_group({**group, "lr": 0.0} if isinstance(lr, torch.Tensor) else group)
        states = {id(p): own for _, buckets in self._plan() for b in buckets for p, own in zip(b.params, b.states)}
        for ours, theirs in zip(self.param_groups, state_dict["param_groups"]):
            for p, i in zip(ours["params"], theirs["params"]):
                if state_dict["state"].get(i):
                    self._check_state(states[id(p)], state_dict["state"][i])

    def state_dict(self):
        """As torch.optim.AdamW's; with 8-bit moments also the seed of their rounding, so that a resumed run rounds as the one it goes on with."""
        out = super().state_dict()
        if self.state_bits == 8:
            out["seed"] = self.seed
        return out

    def load_state_dict(self, state_dict):
        """Values are copied into this optimizer's own buffers, learning rates on the device into their own tensors: a captured step keeps working on them
        (numbers -- a float lr, betas, the seed -- are part of the capture and stay what they were).
        A state dict of torch.optim.AdamW (or Adam, without weight decay) fits 32-bit moments; its flags about how to compute are dropped, those about what
        (amsgrad, maximize) are refused.  A state dict that is refused leaves everything as it was."""
        loaded, held = {}, {}

        # The base class loads groups and their hyperparameters; moments it would cast to the parameters' type.  They are taken out behind the last of the
        # caller's pre-hooks and put in before the first of its post-hooks.
        def take_out(_, state_dict):
            self._check_loaded(state_dict)
            loaded.update(state_dict)
            held.update(buckets=[buckets for _, buckets in self._plan()], norm=self.grad_norm, rates=[group["lr"] for group in self.param_groups])
            return {**state_dict, "state": {}}

        def put_in(_):
            self.seed = int(loaded.get("seed", self.seed))
            self._take_groups(held["rates"])
            # (the same parameters in the same groups: only the groups' dicts are new)
            self._buckets, self.grad_norm = list(zip(self.param_groups, held["buckets"])), held["norm"]
            saved = itertools.chain.from_iterable(g["params"] for g in loaded["param_groups"])
            params = itertools.chain.from_iterable(g["params"] for g in self.param_groups)
            self._take_state({p: loaded["state"].get(i) for i, p in zip(saved, params)})

        hooks = self.register_load_state_dict_pre_hook(take_out), self.register_load_state_dict_post_hook(put_in, prepend=True)
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def _take_groups(self, rates) -> None:
        """Groups as they were loaded; `rates`: the learning rates before."""
        for group, rate in zip(self.param_groups, rates):
            if isinstance(rate, torch.Tensor):
                with torch.no_grad():
                    rate.copy_(torch.as_tensor(group["lr"]).reshape(rate.shape))
                group["lr"] = rate
            elif isinstance(group["lr"], torch.Tensor):  # (from wherever it was loaded to)
                group["lr"] = group["lr"].to(group["params"][0].device, torch.float32)
            for key in ("amsgrad", "maximize", "foreach", "capturable", "differentiable", "fused", "decoupled_weight_decay"):
                group.pop(key, None)

    def _take_state(self, entries: dict) -> None:
        for _, buckets in self._plan():
            for b in buckets:
                for p, own in zip(b.params, b.states):
                    if entries.get(p):
                        self._adopt(own, entries[p])
                    else:
                        for t in own.values():
                            t.zero_()
                    self.state[p] = own

    @torch.no_grad()
    def moments(self) -> tuple[torch.Tensor, torch.Tensor]:
        """The values of all first and of all second moments as two flat fp32 tensors: the parameters in their groups' order (within a group by
        type), each from a multiple of 256 entries on.  With state_bits=32 and one type in one group these are the buffers themselves."""
        flats = []
        for _, buckets in self._plan():
            for b in buckets:
                m, v = b.flat["exp_avg"], b.flat["exp_avg_sq"]
                if b.bits == 8:
                    out = torch.empty(2, m.numel(), device=b.device, dtype=torch.float32)
                    L.call("sdeh_adamw_moments", b.device, m.data_ptr(), b.flat["exp_avg_top"].data_ptr(), v.data_ptr(),
                           b.flat["exp_avg_sq_top"].data_ptr(), b.blocks, out[0].data_ptr(), out[1].data_ptr())
                    m, v = out.unbind()
                flats.append((m, v))
        if len(flats) == 1:
            return flats[0]
        return tuple(torch.cat([f[k] for f in flats]) for k in (0, 1))

    # -- step ----------------------------------------------------------------------------------------------------------------------------
    def step(self, closure=None, *, ok: torch.Tensor | None = None):
        """One step.  ok: an optional one-element bool tensor on the device; where it is False, parameters, moments and step counters stay as they are
        (the decision of `if loss_ok and grad_ok`, solver/base.py:409-421, without a host round trip), and `grad_norm` too."""
        if self._optimizer_step_pre_hooks or self._optimizer_step_post_hooks or _global_pre or _global_post or torch.autograd._profiler_enabled():
            return self._hooked_step(closure, ok=ok)
        return self._step(closure, ok=ok)

    #: torch.optim.Optimizer would wrap `step` for its hooks and the profiler, which costs a quarter of a small model's step: `step` goes through that
    #: wrapper (`_hooked_step`) only when there is a hook or a profiler
    step.hooked = True

    def _step(self, closure=None, *, ok: torch.Tensor | None = None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        groups, tables, keep, written = [], [], [], []
        for group, buckets in self._plan():
            lr, (b1, b2) = group["lr"], group["betas"]
            lr_dev = 0
            if isinstance(lr, torch.Tensor):
                if lr.device != self._device or lr.dtype != torch.float32 or lr.numel() != 1:
                    raise ValueError("AdamW: a tensor lr must be one fp32 element on the parameters' device")
                lr, lr_dev = 0.0, lr.data_ptr()
            for b in buckets:
                rows, held, tensors = b.rows()
                if len(rows):
                    groups.append(L.ADAMW_GROUP.pack(lr, b1, b2, group["eps"], group["weight_decay"], lr_dev, len(rows), b.code, b.bits, 0))
                    tables.append(rows)
                    keep.append(held)
                    written += tensors
        if not groups:
            return loss
        if ok is not None and (ok.device != self._device or ok.numel() != 1 or ok.dtype not in (torch.bool, torch.uint8)):
            raise ValueError(f"AdamW: ok must be one bool on {self._device}, got {tuple(ok.shape)} {ok.dtype} on {ok.device}")
        table = tables[0] if len(tables) == 1 else np.concatenate(tables)
        norm = self.grad_norm
        head = L.ADAMW.pack(self.max_grad_norm or 0.0, 0 if ok is None else ok.data_ptr(), 0 if norm is None else norm.data_ptr(),
                            self.seed & 0xFFFFFFFF, len(groups))
        L.call("sdeh_adamw_step", self._device, head, b"".join(groups), table.ctypes.data, self._scratch.data_ptr())
        if norm is not None and not norm.is_inference():
            written.append(norm)
        # (written behind torch's back: whoever saved one of them for a backward pass, or cached what it held, is told here -- also where `ok` is False,
        # which the host does not know)
        torch.autograd.graph.increment_version(written)
        return loss

    _hooked_step = torch.optim.Optimizer.profile_hook_step(_step)
