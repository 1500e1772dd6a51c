"""Losses over trajectories that were drawn BEFORE the update, with their gradients (include/sdeh.h, ABI v8).

The losses of losses/oc.py simulate the control they differentiate, once per optimisation step.  A batch of trajectories can be used for
several steps when the losses account for the control having moved since: with `v` the control that drove the paths and `u` the one being trained,

    log_ratio = step_log_ratio(u, v, dW, dt)                              # [T, B]: log p_u / p_v of every Euler-Maruyama step
    loss, info = policy_loss(log_ratio.t(), advantage)                    # rows = trajectories
    loss, info = preference_loss(log_ratio.t()[better], log_ratio.t()[worse])

(`Problem.eval(..., noise=)` gives the paths, `noise * dt.sqrt()` the increments; the reference accumulates the same increments of the log-ratio
in losses/oc.py:204-219.)  `policy_loss` and `preference_loss` take any log-probabilities [rows, steps], so they serve sequence models as well.

All functions run on the HIP device, on torch's current stream, never synchronise and may be captured into a graph (a captured backward pass wants
fresh leaves, as any: utils/graphs.py; the `*_and_grad` forms have no autograd graph).  fp32, bf16 and fp16; a log-ratio's sum over the coordinates is
held in 32 bits, the losses' sums over rows and steps in 64 (the policy loss adds the 4 or 8 entries of a 16-byte vector in 32 bits first); results are
fp32, gradients of the type of what they belong to.  Only the first argument(s) -- `control`, `log_prob`, `chosen` and `rejected` -- are differentiated, in
reverse mode and once: everything else is a constant of the graph.
"""
from __future__ import annotations

import torch
from torch.autograd.forward_ad import unpack_dual
from torch.autograd.function import once_differentiable

from sde_sampler_amd import _lib as L

__all__ = ["step_log_ratio", "policy_loss", "policy_loss_and_grad", "preference_loss", "preference_loss_and_grad"]


def _code(name: str, t: torch.Tensor, device=None) -> int:
    if not t.is_cuda:
        raise RuntimeError(f"{name} runs on the HIP device only (got a CPU tensor); there is no CPU path in this package")
    if device is not None and t.device != device:
        raise ValueError(f"{name}: tensors are on {device} and {t.device}")
    code = L.dtype_code(t.dtype)
    if code is None:
        raise L.SdehUnsupported(-2, f"{name}: {t.dtype} (the kernels take float32, bfloat16 and float16)")
    return code


def _no_tangent(name: str, t: torch.Tensor) -> None:
    if unpack_dual(t).tangent is not None:  # (the kernels see its values only; a result without a tangent would pass for a constant)
        raise NotImplementedError(f"{name}: forward-mode differentiation is not implemented")


def _constant(t: torch.Tensor | None) -> torch.Tensor | None:
    return t.detach() if t is not None and t.requires_grad else t


def _once(backward):
    """`once_differentiable` where a graph of the backward pass is asked for; without one (the usual call) there is nothing to guard."""
    guarded = once_differentiable(backward)

    def run(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run


# -- step log-ratio --------------------------------------------------------------------------------------------------------------------------
class _StepLogRatio(torch.autograd.Function):
    @staticmethod
    def forward(ctx, control, behaviour, increments, dt, code):
        ctx.save_for_backward(control, behaviour, increments, dt)
        ctx.code = code
        return _ratio(control, behaviour, increments, dt, code)

    @staticmethod
    @_once
    def backward(ctx, grad):
        control, behaviour, increments, dt = ctx.saved_tensors
        T, B, d = control.shape
        out = torch.empty_like(control)
        grad = grad.float().contiguous()
        L.call("sdeh_step_log_ratio_backward", control.device, control.data_ptr(), None if behaviour is None else behaviour.data_ptr(),
               increments.data_ptr(), dt.data_ptr(), grad.data_ptr(), T, B, d, ctx.code, out.data_ptr())
        return out, None, None, None, None


def _ratio(control, behaviour, increments, dt, code):
    T, B, d = control.shape
    out = torch.empty(T, B, device=control.device, dtype=torch.float32)
    L.call("sdeh_step_log_ratio", control.device, control.data_ptr(), None if behaviour is None else behaviour.data_ptr(),
           increments.data_ptr(), dt.data_ptr(), T, B, d, code, out.data_ptr())
    return out


def step_log_ratio(control: torch.Tensor, behaviour: torch.Tensor | None, increments: torch.Tensor, dt: torch.Tensor) -> torch.Tensor:
    """log p_control(x_{t+1} | x_t) - log p_behaviour(x_{t+1} | x_t) of every Euler-Maruyama step, [T, B] in fp32.

    control     [T, B, d]  u(t, x_t) along the paths; differentiated
    behaviour   [T, B, d]  the control that drove them; None: they are paths of the uncontrolled process
    increments  [T, B, d]  the Brownian increments sqrt(dt) * noise that were added under `behaviour`
    dt          [T]        step sizes
    `control`, `behaviour` and `increments` have one type; tensors that are not contiguous are copied."""
    if control.ndim != 3 or not 1 <= control.shape[2] <= L.MAX_DIM:
        raise ValueError(f"step_log_ratio: control must be [steps, batch, dim] with 1 <= dim <= 2^30, got {tuple(control.shape)}")
    code = _code("step_log_ratio", control)
    _no_tangent("step_log_ratio", control)
    for name, t in (("behaviour", behaviour), ("increments", increments)):
        if t is None and name == "behaviour":
            continue
        if t.shape != control.shape or t.dtype != control.dtype or t.device != control.device:
            raise ValueError(f"step_log_ratio: {name} is {tuple(t.shape)} {t.dtype} on {t.device}, control {tuple(control.shape)} {control.dtype} "
                             f"on {control.device}")
    if dt.shape != control.shape[:1] or dt.device != control.device:
        raise ValueError(f"step_log_ratio: dt must be [{control.shape[0]}] on {control.device}, got {tuple(dt.shape)} on {dt.device}")
    control, increments = control.contiguous(), _constant(increments).contiguous()
    behaviour = None if behaviour is None else _constant(behaviour).contiguous()
    dt = _constant(dt).float().contiguous()
    if torch.is_grad_enabled() and control.requires_grad:
        return _StepLogRatio.apply(control, behaviour, increments, dt, code)
    return _ratio(control, behaviour, increments, dt, code)


# -- clipped policy loss ---------------------------------------------------------------------------------------------------------------------
def _plane(t: torch.Tensor | None):
    return (0, 0, 0) if t is None else (t.data_ptr(), *t.stride())


def _describe_policy(log_prob, advantage, old, ref, mask, clip_low, clip_high, dual_clip, kl_coef, kl, reduction):
    """(the tensors as the kernel takes them, the rest of SdehPolicyLoss)"""
    if log_prob.ndim != 2:
        raise ValueError(f"policy_loss: log_prob must be [rows, steps], got {tuple(log_prob.shape)}")
    dev, shape = log_prob.device, log_prob.shape
    code = _code("policy_loss", log_prob)
    _no_tangent("policy_loss", log_prob)
    for name, t in (("old_log_prob", old), ("ref_log_prob", ref)):
        if t is not None and (t.shape != shape or t.dtype != log_prob.dtype or t.device != dev):
            raise ValueError(f"policy_loss: {name} is {tuple(t.shape)} {t.dtype} on {t.device}, log_prob {tuple(shape)} {log_prob.dtype} on {dev}")
    adv_code = _code("policy_loss", advantage, dev)
    try:
        if advantage.ndim == 2:
            if advantage.shape != shape:
                advantage = advantage.expand(shape)
        elif advantage.ndim != 1 or advantage.shape[0] != shape[0]:
            raise ValueError(f"policy_loss: advantage must be [rows] or [rows, steps], got {tuple(advantage.shape)} for log_prob {tuple(shape)}")
        if mask is not None and mask.shape != shape:
            mask = mask.expand(shape)
    except RuntimeError as exc:
        raise ValueError(f"policy_loss: advantage and mask must broadcast to {tuple(shape)}: {exc}") from None
    if mask is not None and (mask.dtype not in (torch.bool, torch.uint8) or mask.device != dev):
        raise ValueError(f"policy_loss: mask must be bool or uint8 on {dev}, got {mask.dtype} on {mask.device}")
    if kl not in L.KL_ESTIMATORS or reduction not in L.REDUCTIONS:
        raise ValueError(f"policy_loss: kl is one of {list(L.KL_ESTIMATORS)} and reduction one of {list(L.REDUCTIONS)}, got {kl!r} and {reduction!r}")
    if not (clip_low >= 0.0 and clip_high >= 0.0 and (dual_clip is None or dual_clip > 1.0)):
        raise ValueError(f"policy_loss: clip_low, clip_high >= 0 and dual_clip > 1, got {clip_low}, {clip_high}, {dual_clip}")
    rest = (*shape, code, adv_code, L.KL_ESTIMATORS[kl], L.REDUCTIONS[reduction], clip_low, clip_high, dual_clip or 0.0, kl_coef)
    return (log_prob, advantage, old, ref, mask), rest


def _pack_policy(tensors, rest) -> bytes:
    log_prob, advantage, old, ref, mask = tensors
    adv = (advantage.data_ptr(), advantage.stride(0), 0) if advantage.ndim == 1 else _plane(advantage)
    return L.POLICY_LOSS.pack(*_plane(log_prob), *_plane(old), *_plane(ref), *adv, *_plane(mask), *rest)


def _policy_scratch(log_prob, mask, out=None):
    """Scratch of a call; where it needs none, `out` stands for it."""
    n = L.load().sdeh_policy_loss_scratch_floats(*log_prob.shape, mask is not None)
    return out if n == 0 and out is not None else torch.empty(max(n, 4), device=log_prob.device, dtype=torch.float32)


def _loss(out):
    """out[0] as a tensor of its own, on the same memory: a view of `out` could not be changed in place (`loss /= n`) under autograd."""
    return out[0].data


def _policy_info(out):
    _, policy, kl, fraction, valid = out.unbind()
    return {"policy": policy, "kl": kl, "clip_fraction": fraction, "n_valid": valid}


class _PolicyLoss(torch.autograd.Function):
    """The loss now, its gradient when it is asked for: the backward pass reads the inputs again and scales in fp32 before its one rounding, so that a
    scaled loss (gradient accumulation, half-precision loss scaling) loses nothing."""

    @staticmethod
    def forward(ctx, log_prob, advantage, old, ref, mask, rest):
        scratch = _policy_scratch(log_prob, mask)
        out = torch.empty(5, device=log_prob.device, dtype=torch.float32)
        packed = _pack_policy((log_prob, advantage, old, ref, mask), rest)
        L.call("sdeh_policy_loss", log_prob.device, packed, scratch.data_ptr(), 0, None, 1.0, out.data_ptr(), None)
        ctx.save_for_backward(log_prob, advantage, old, ref, mask, scratch)
        ctx.rest, ctx.mask_stride = rest, None if mask is None else mask.stride()
        ctx.mark_non_differentiable(out)
        ctx.set_materialize_grads(False)  # (no zeros for `out`)
        return _loss(out), out

    @staticmethod
    @_once
    def backward(ctx, grad_loss, _):
        if grad_loss is None:
            return None, None, None, None, None, None
        *tensors, scratch = ctx.saved_tensors  # (they may have been away: their addresses are taken anew)
        log_prob, mask = tensors[0], tensors[4]
        counted = mask is None or mask.stride() == ctx.mask_stride  # (the counts in `scratch` are those of the mask's layout)
        grad = torch.empty(log_prob.shape, device=log_prob.device, dtype=log_prob.dtype)
        if grad.numel() == 0:
            return grad, None, None, None, None, None
        scale = grad_loss.float()
        L.call("sdeh_policy_loss", log_prob.device, _pack_policy(tensors, ctx.rest), scratch.data_ptr(), int(counted), scale.data_ptr(), 1.0, None, grad.data_ptr())
        return grad, None, None, None, None, None


def policy_loss(log_prob: torch.Tensor, advantage: torch.Tensor, old_log_prob: torch.Tensor | None = None,
                ref_log_prob: torch.Tensor | None = None, mask: torch.Tensor | None = None, *, clip_low: float = 0.2, clip_high: float = 0.2,
                dual_clip: float | None = None, kl_coef: float = 0.0, kl: str = "k3", reduction: str = "steps") -> tuple[torch.Tensor, dict]:
    """Clipped policy loss with a KL term; returns (loss, info) as `compute_loss` does.

    Per valid entry, with r = exp(log_prob - old_log_prob):  -min(A r, A clip(r, 1 - clip_low, 1 + clip_high))  +  kl_coef * kl, where for A < 0
    the first term is at most -A dual_clip, and kl is an estimate of KL(policy | reference) from k = log_prob - ref_log_prob: "k1" k, "k2" k^2 / 2,
    "k3" exp(-k) - 1 + k.

    log_prob      [rows, steps]  differentiated; any strides
    advantage     [rows], [rows, 1] or [rows, steps]
    old_log_prob  like log_prob; None: log_prob is a log-ratio already (step_log_ratio)
    ref_log_prob  like log_prob; None: no KL term
    mask          bool (or uint8), broadcastable to [rows, steps]; entries it leaves out do not count, whatever they hold
    reduction     "steps": mean over the valid entries; "rows": mean over the rows that have any, of their means; "sum"
    info          0-d fp32 tensors: policy and kl (the two terms, reduced like the loss), clip_fraction, n_valid (exact up to 2^24 entries, rounded
                  beyond; the weights and shares come from the exact number)
    Without a valid entry the loss and its gradient are 0.  A log-probability of -inf in a valid entry gives what the formula gives."""
    tensors, rest = _describe_policy(log_prob, advantage, old_log_prob, ref_log_prob, mask, clip_low, clip_high, dual_clip, kl_coef, kl, reduction)
    x, adv, old, ref, mask = tensors
    if torch.is_grad_enabled() and log_prob.requires_grad:
        loss, out = _PolicyLoss.apply(x, _constant(adv), _constant(old), _constant(ref), mask, rest)
        return loss, _policy_info(out)
    packed = _pack_policy(tensors, rest)
    out = torch.empty(5, device=x.device, dtype=torch.float32)
    scratch = _policy_scratch(x, tensors[4], out)
    L.call("sdeh_policy_loss", x.device, packed, scratch.data_ptr(), 0, None, 1.0, out.data_ptr(), None)
    return _loss(out), _policy_info(out)


def policy_loss_and_grad(log_prob: torch.Tensor, advantage: torch.Tensor, old_log_prob: torch.Tensor | None = None,
                         ref_log_prob: torch.Tensor | None = None, mask: torch.Tensor | None = None, *, clip_low: float = 0.2,
                         clip_high: float = 0.2, dual_clip: float | None = None, kl_coef: float = 0.0, kl: str = "k3", reduction: str = "steps",
                         grad_scale: float = 1.0) -> tuple[torch.Tensor, dict, torch.Tensor]:
    """`policy_loss` and grad_scale * d loss / d log_prob from one pass over the inputs, without an autograd graph: (loss, info, gradient).
    `log_prob.backward(gradient)` hands it to whatever computed log_prob."""
    tensors, rest = _describe_policy(log_prob.detach(), advantage, old_log_prob, ref_log_prob, mask, clip_low, clip_high, dual_clip, kl_coef, kl,
                                     reduction)
    x, packed = tensors[0], _pack_policy(tensors, rest)
    out = torch.empty(5, device=x.device, dtype=torch.float32)
    grad = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    scratch = _policy_scratch(x, tensors[4], out)
    L.call("sdeh_policy_loss", x.device, packed, scratch.data_ptr(), 0, None, grad_scale, out.data_ptr(), grad.data_ptr())
    return _loss(out), _policy_info(out), grad


# -- preference loss -------------------------------------------------------------------------------------------------------------------------
def _describe_preference(chosen, rejected, ref_chosen, ref_rejected, chosen_mask, rejected_mask, beta, label_smoothing, kind, average):
    if chosen.ndim != 2 or rejected.ndim != 2 or chosen.shape[0] != rejected.shape[0] or chosen.shape[0] < 1:
        raise ValueError(f"preference_loss: chosen and rejected must be [pairs, steps] with as many (and at least one) pairs, got {tuple(chosen.shape)} "
                         f"and {tuple(rejected.shape)}")
    code = _code("preference_loss", chosen)
    tensors = []
    for name, x, ref, mask in (("chosen", chosen, ref_chosen, chosen_mask), ("rejected", rejected, ref_rejected, rejected_mask)):
        _no_tangent("preference_loss", x)
        if x.dtype != chosen.dtype or x.device != chosen.device:
            raise ValueError(f"preference_loss: chosen is {chosen.dtype} on {chosen.device}, rejected {x.dtype} on {x.device}")
        if ref is not None and (ref.shape != x.shape or ref.dtype != x.dtype or ref.device != x.device):
            raise ValueError(f"preference_loss: ref_{name} is {tuple(ref.shape)} {ref.dtype} on {ref.device}, {name} {tuple(x.shape)} {x.dtype} on "
                             f"{x.device}")
        if mask is not None:
            if mask.dtype not in (torch.bool, torch.uint8) or mask.device != x.device:
                raise ValueError(f"preference_loss: {name}_mask must be bool or uint8 on {x.device}, got {mask.dtype} on {mask.device}")
            if mask.shape != x.shape:
                try:
                    mask = mask.expand(x.shape)
                except RuntimeError as exc:
                    raise ValueError(f"preference_loss: {name}_mask must broadcast to {tuple(x.shape)}: {exc}") from None
        tensors += [x, ref, mask]
    if kind not in L.PREFERENCE_KINDS:
        raise ValueError(f"preference_loss: kind is one of {list(L.PREFERENCE_KINDS)}, got {kind!r}")
    if not (beta > 0.0 and 0.0 <= label_smoothing < 0.5):
        raise ValueError(f"preference_loss: beta > 0 and 0 <= label_smoothing < 0.5, got {beta} and {label_smoothing}")
    if label_smoothing and kind != "logistic":
        raise ValueError(f"preference_loss: label_smoothing belongs to the logistic kind, got {kind!r}")
    return tensors, (chosen.shape[0], code, L.PREFERENCE_KINDS[kind], bool(average), beta, label_smoothing)


def _pack_preference(tensors, rest) -> bytes:
    x, ref, mask, y, y_ref, y_mask = tensors
    return L.PREFERENCE_LOSS.pack(*_plane(x), *_plane(ref), *_plane(mask), x.shape[1], *_plane(y), *_plane(y_ref), *_plane(y_mask), y.shape[1], *rest)


def _pointer(grad, out):
    return grad.data_ptr() if grad.numel() else out.data_ptr()  # (an empty tensor has no address; nothing is written)


def _preference_forward(packed, chosen, rejected, grads, grad_scale=1.0):
    P = chosen.shape[0]
    out = torch.empty(2 + 4 * P, device=chosen.device, dtype=torch.float32)
    scratch = torch.empty(L.load().sdeh_preference_loss_scratch_floats(packed), device=chosen.device, dtype=torch.float32)
    gc = gr = None
    if grads:
        gc = torch.empty(chosen.shape, device=chosen.device, dtype=chosen.dtype)
        gr = torch.empty(rejected.shape, device=chosen.device, dtype=chosen.dtype)
    L.call("sdeh_preference_loss", chosen.device, packed, scratch.data_ptr(), grad_scale, out.data_ptr(), _pointer(gc, out) if grads else None,
           _pointer(gr, out) if grads else None)
    return out, gc, gr


def _preference_info(out, pairs):
    return {"accuracy": out[1], "chosen_rewards": out[2:2 + pairs], "rejected_rewards": out[2 + pairs:2 + 2 * pairs]}


class _PreferenceLoss(torch.autograd.Function):
    """Loss and the pairs' slopes now; the backward pass spreads the slopes over the valid entries, reading nothing but the masks."""

    @staticmethod
    def forward(ctx, chosen, rejected, ref_chosen, ref_rejected, chosen_mask, rejected_mask, rest):
        packed = _pack_preference((chosen, ref_chosen, chosen_mask, rejected, ref_rejected, rejected_mask), rest)
        out, _, _ = _preference_forward(packed, chosen, rejected, False)
        ctx.save_for_backward(out, chosen_mask, rejected_mask)
        ctx.rest, ctx.shapes, ctx.dtype = rest, (chosen.shape, rejected.shape), chosen.dtype
        ctx.mark_non_differentiable(out)
        ctx.set_materialize_grads(False)
        return _loss(out), out

    @staticmethod
    @_once
    def backward(ctx, grad_loss, _):
        if grad_loss is None:
            return None, None, None, None, None, None, None
        out, chosen_mask, rejected_mask = ctx.saved_tensors
        gc, gr = (torch.empty(s, device=out.device, dtype=ctx.dtype) for s in ctx.shapes)
        scale = grad_loss.float()
        # (the log-probabilities are not read again: the gradients stand in their places)
        packed = L.PREFERENCE_LOSS.pack(_pointer(gc, out), 0, 0, 0, 0, 0, *_plane(chosen_mask), gc.shape[1], _pointer(gr, out), 0, 0, 0, 0, 0,
                                        *_plane(rejected_mask), gr.shape[1], *ctx.rest)
        L.call("sdeh_preference_grad", out.device, packed, out.data_ptr(), scale.data_ptr(), 1.0, _pointer(gc, out), _pointer(gr, out))
        return gc, gr, None, None, None, None, None


def preference_loss(chosen: torch.Tensor, rejected: torch.Tensor, ref_chosen: torch.Tensor | None = None, ref_rejected: torch.Tensor | None = None,
                    chosen_mask: torch.Tensor | None = None, rejected_mask: torch.Tensor | None = None, *, beta: float = 0.1,
                    label_smoothing: float = 0.0, kind: str = "logistic", average: bool = False) -> tuple[torch.Tensor, dict]:
    """Preference loss of paired rows from their log-probabilities; returns (loss, info).

    With s the sum of (log_prob - ref_log_prob) over a row's valid entries (their mean when `average`; 0 for a row without any) and
    h = beta (s_chosen - s_rejected), the mean over the pairs of
      "logistic"  -(1 - label_smoothing) log sigmoid(h) - label_smoothing log sigmoid(-h)
      "hinge"     max(0, 1 - h)
      "square"    (s_chosen - s_rejected - 1 / (2 beta))^2

    chosen, rejected          [pairs, steps], their own number of steps each; differentiated; any strides
    ref_chosen, ref_rejected  like them; None: they are log-ratios already (step_log_ratio)
    *_mask                    bool (or uint8), broadcastable; entries they leave out do not count, whatever they hold
    info                      accuracy (share of the pairs with h > 0), chosen_rewards and rejected_rewards (beta s, [pairs])"""
    keep, rest = _describe_preference(chosen, rejected, ref_chosen, ref_rejected, chosen_mask, rejected_mask, beta, label_smoothing, kind, average)
    if torch.is_grad_enabled() and (chosen.requires_grad or rejected.requires_grad):
        loss, out = _PreferenceLoss.apply(chosen, rejected, _constant(keep[1]), _constant(keep[4]), keep[2], keep[5], rest)
    else:
        out, _, _ = _preference_forward(_pack_preference(keep, rest), chosen, rejected, False)
        loss = _loss(out)
    return loss, _preference_info(out, chosen.shape[0])


def preference_loss_and_grad(chosen: torch.Tensor, rejected: torch.Tensor, ref_chosen: torch.Tensor | None = None,
                             ref_rejected: torch.Tensor | None = None, chosen_mask: torch.Tensor | None = None,
                             rejected_mask: torch.Tensor | None = None, *, beta: float = 0.1, label_smoothing: float = 0.0, kind: str = "logistic",
                             average: bool = False, grad_scale: float = 1.0) -> tuple[torch.Tensor, dict, torch.Tensor, torch.Tensor]:
    """`preference_loss` and grad_scale times its gradients without an autograd graph: (loss, info, gradient of chosen, gradient of rejected)."""
    chosen, rejected = chosen.detach(), rejected.detach()
    keep, rest = _describe_preference(chosen, rejected, ref_chosen, ref_rejected, chosen_mask, rejected_mask, beta, label_smoothing, kind, average)
    out, gc, gr = _preference_forward(_pack_preference(keep, rest), chosen, rejected, True, grad_scale)
    return _loss(out), _preference_info(out, chosen.shape[0]), gc, gr
