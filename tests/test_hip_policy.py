"""Losses over stored trajectories (sde_sampler_amd/losses/policy.py; include/sdeh.h v8) against the formulas in 64 bits.

Tolerances.  h = 2^-24 is half a step of fp32 relative to the value, half(t) that of an output's type.  A result of n roundings of relative size h
over terms of absolute sum S is off by at most n h S; expf is taken as accurate to 2 h (one unit in the last place), its argument's rounding adds
|delta| h.  Each test states its n.  Sums are held in 64 bits except where said."""
import ctypes
import math
import subprocess
from pathlib import Path

import pytest
import torch
import torch.autograd.forward_ad as fwad

from sde_sampler_amd import _lib as L
from sde_sampler_amd.losses import policy as P

H = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
gpu = pytest.mark.gpu


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half a step among the subnormal numbers of a type."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def close(got, want, tol, what=""):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got.double() - want).abs() - tol).max()):.3e} over tolerance"


# -- step log-ratio ------------------------------------------------------------------------------------------------------------------------
def _ratio_case(T, B, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + T + 7 * B + 31 * d)
    dt = (torch.rand(T, generator=g) + 0.5) * 5.0 / T
    v = torch.randn(T, B, d, generator=g)
    u = (v + 0.3 * torch.randn(T, B, d, generator=g)).to(dtype)
    dw = (torch.randn(T, B, d, generator=g) * dt.sqrt()[:, None, None]).to(dtype)
    return u, v.to(dtype), dw, dt, torch.randn(T, B, generator=g)


def _ratio_want(u, v, dw, dt, g):
    u, dw, dt, g = u.double(), dw.double(), dt.double()[:, None, None], g.double()[..., None]
    e = u - (0.0 if v is None else v.double())
    out = (e * dw - 0.5 * dt * e * e).sum(-1)
    size = (e.abs() * (dw.abs() + 0.5 * dt * e.abs())).sum(-1)
    return out, size, g * (dw - dt * e), g.abs() * (dw.abs() + dt * e.abs())


@gpu
@pytest.mark.parametrize("T,B,d", [(1, 1, 1), (3, 5, 1), (1, 4097, 2), (7, 33, 3), (100, 512, 2), (20, 65, 10), (9, 31, 50), (5, 17, 64), (11, 3, 196),
                                   (2, 3, 511), (3, 2, 512), (4, 3, 513), (2, 2, 784), (1, 1, 4099), (400, 1, 7)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_step_log_ratio(T, B, d, dtype):
    u, v, dw, dt, g = _ratio_case(T, B, d, dtype)
    want, size, want_g, size_g = _ratio_want(u, v, dw, dt, g)
    ug = u.cuda().requires_grad_()
    got = P.step_log_ratio(ug, v.cuda(), dw.cuda(), dt.cuda())
    got.backward(g.cuda())
    # a term: difference, product, difference, product (4); a row's sum in fp32: at most d additions
    close(got.detach().cpu(), want, (d + 6) * H * size + 1e-38, "log_ratio")
    close(ug.grad.cpu(), want_g, 5 * H * size_g + half(dtype) * want_g.abs() + tiny(dtype), "grad")
    assert ug.grad.dtype == dtype and got.dtype == torch.float32


@gpu
@pytest.mark.parametrize("d", [3, 50, 600])
def test_step_log_ratio_layouts(d):
    """No behaviour; transposed, offset (unaligned) and broadcast inputs; an expanded cotangent; empty batches."""
    u, v, dw, dt, g = _ratio_case(6, 10, d, torch.float32)
    want, size, want_g, size_g = _ratio_want(u, None, dw, dt, torch.ones_like(g))
    ug = u.cuda().requires_grad_()
    y = P.step_log_ratio(ug, None, dw.cuda(), dt.cuda())
    y.sum().backward()
    close(y.detach().cpu(), want, (d + 6) * H * size)
    close(ug.grad.cpu(), want_g, 6 * H * size_g)
    want, size, _, _ = _ratio_want(u, v, dw, dt, g)
    off = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)]).cuda()[1:].view(t.shape)  # noqa: E731  (4 bytes past a 16-byte border)
    for f in (lambda t: t.transpose(0, 1).contiguous().cuda().transpose(0, 1), off):
        close(P.step_log_ratio(f(u), f(v), f(dw), dt.cuda()).cpu(), want, (d + 6) * H * size)
    one = u[:1].cuda().requires_grad_()
    z = P.step_log_ratio(one.expand(6, -1, -1), v.cuda(), dw.cuda(), dt.cuda())
    z.backward(g.cuda())
    _, _, want_g, size_g = _ratio_want(u[:1].expand(6, -1, -1), v, dw, dt, g)
    close(one.grad.cpu(), want_g.sum(0, keepdim=True), 12 * H * size_g.sum(0, keepdim=True))
    for shape in ((0, 4, d), (4, 0, d)):
        e = torch.zeros(shape, device="cuda", requires_grad=True)
        y = P.step_log_ratio(e, None, e.detach(), torch.ones(shape[0], device="cuda"))
        y.sum().backward()
        assert y.shape == shape[:2] and e.grad.shape == shape


@gpu
def test_step_log_ratio_gradient_against_differences():
    u, v, dw, dt, g = (t.cuda() for t in _ratio_case(4, 3, 5, torch.float32))
    ug = u.clone().requires_grad_()
    P.step_log_ratio(ug, v, dw, dt).backward(g)
    step = 2.0 ** -6
    for i in (0, 17, 59):
        e = torch.zeros_like(u).view(-1)
        e[i] = step
        e = e.view_as(u)
        # quadratic in u: central differences are exact up to rounding
        d = ((P.step_log_ratio(u + e, v, dw, dt) - P.step_log_ratio(u - e, v, dw, dt)) * g).sum() / (2 * step)
        size = float(_ratio_want(u.cpu(), v.cpu(), dw.cpu(), dt.cpu(), g.cpu())[1].max() * g.abs().max().cpu())
        assert abs(float(d - ug.grad.view(-1)[i])) <= 40 * H * (size + 1) / step


@gpu
@pytest.mark.parametrize("d", [1, 3, 5, 6, 10, 50, 196, 513])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("where", ["control", "behaviour", "increments"])
def test_step_log_ratio_keeps_trajectories_apart(d, dtype, where):
    """A trajectory that diverged -- one NaN or infinite coordinate, at a row's first, last or middle place -- has no finite ratio at that step; every other
    ratio and gradient is what it is without it, bit for bit, aligned or not."""
    T, B = 4, 23
    u, v, dw, dt, g = _ratio_case(T, B, d, dtype)
    off = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)]).cuda()[1:].view(t.shape)  # noqa: E731
    for place in (lambda t: t.cuda(), off):
        clean_u = place(u).detach().requires_grad_()
        clean = P.step_log_ratio(clean_u, place(v), place(dw), dt.cuda())
        clean.backward(g.cuda())
        for bad in (math.nan, math.inf, -math.inf):
            case = {"control": u.clone(), "behaviour": v.clone(), "increments": dw.clone()}
            spots = {(0, 0): 0, (1, 7): d - 1, (2, 8): 0, (2, 12): d // 2, (T - 1, B - 1): d - 1}
            for (t, b), k in spots.items():
                case[where][t, b, k] = bad
            x = place(case["control"]).detach().requires_grad_()
            y = P.step_log_ratio(x, place(case["behaviour"]), place(case["increments"]), dt.cuda())
            y.backward(g.cuda())
            hit = torch.zeros(T, B, dtype=torch.bool)
            for t, b in spots:
                hit[t, b] = True
            y, want = y.detach().cpu(), clean.detach().cpu()
            assert torch.equal(~torch.isfinite(y), hit)
            assert torch.equal(y[~hit], want[~hit]) and torch.equal(x.grad.cpu()[~hit], clean_u.grad.cpu()[~hit])


# -- policy loss ---------------------------------------------------------------------------------------------------------------------------
def _policy_case(R, T, dtype, mask="ragged", adv="rows", ref=True, seed=0):
    g = torch.Generator().manual_seed(seed + 13 * R + T)
    lp = (-3 * torch.rand(R, T, generator=g)).to(dtype)
    old = (lp.float() + 0.2 * torch.randn(R, T, generator=g)).to(dtype)
    q = (lp.float() + 0.4 * torch.randn(R, T, generator=g)).to(dtype) if ref else None
    a = torch.randn((R,) if adv == "rows" else (R, T), generator=g) + 0.2
    a.view(-1)[0] = 0.0
    m = None
    if mask == "ragged":
        n = torch.randint(0, T + 1, (R,), generator=g)
        n[R // 2] = 0
        m = torch.arange(T)[None] < n[:, None]
    elif mask == "random":
        m = torch.rand(R, T, generator=g) < 0.6
        m[R // 2] = False
    elif mask == "none valid":
        m = torch.zeros(R, T, dtype=torch.bool)
    return lp, old, q, a, m


def _policy_want(lp, old, ref, adv, mask, clip_low=0.2, clip_high=0.28, dual=None, kl_coef=0.05, kl="k3", reduction="steps"):
    """(loss, policy, kl, clip_fraction, n, gradient, gradient's error bound, loss's error bound) in 64 bits, padding replaced by zeros."""
    live = torch.ones(lp.shape, dtype=torch.bool) if mask is None else mask.expand(lp.shape).bool()
    clean = lambda t: torch.where(live, t.double(), 0.0)  # noqa: E731
    x, o = clean(lp), 0.0 * lp.double() if old is None else clean(old)
    x0 = torch.where(live, lp.double(), 0.0)
    delta = x0 - torch.nan_to_num(o) if old is None else x0 - o
    a = clean((adv[:, None] if adv.ndim == 1 else adv).expand(lp.shape))
    r = delta.exp()
    first, second = a * r, a * r.clamp(1 - clip_low, 1 + clip_high)
    gain = torch.minimum(first, second)
    free = first <= second
    if dual is not None:
        held = (a < 0) & (gain < dual * a)
        gain, free = torch.where(held, dual * a, gain), free & ~held
    k, dk = torch.zeros_like(x0), torch.zeros_like(x0)
    e_k = e_dk = torch.zeros_like(x0)
    if ref is not None:
        d = x0 - clean(ref)
        if kl == "k1":
            k, dk, e_k, e_dk = d, torch.ones_like(d), H * d.abs(), 0 * d
        elif kl == "k2":
            k, dk, e_k, e_dk = d * d / 2, d, 3 * H * d * d, H * d.abs()
        else:
            k, dk = torch.expm1(-d) + d, -torch.expm1(-d)
            # far: exp(-k) to 2 h plus its argument's rounding, two sums; near: ten terms' roundings of a sum below k^2
            e_k = H * torch.where(d.abs() < 0.5, 12 * d * d, (3 + d.abs()) * (-d).exp() + 2 * d.abs() + 2)
            e_dk = e_k + H * dk.abs()
    count = live.sum(1, keepdim=True).double()
    n = count.sum()
    if reduction == "steps":
        w = live / n.clamp(min=1)
    elif reduction == "rows":
        w = live / count.clamp(min=1) / (count > 0).sum().clamp(min=1)
    else:
        w = live.double()
    policy, klm = -(gain * w).sum(), (k * w).sum()
    beta = kl_coef if ref is not None else 0.0
    grad = (beta * dk - torch.where(free, first, 0.0)) * w
    # surrogate: exp (2 + |delta|), product; slope: sum with the KL term; weight and scale: 3 more
    e_first = H * (6 + delta.abs()) * torch.where(free, first.abs(), 0.0)
    e_grad = w * (e_first + beta * e_dk + 6 * H * (beta * dk).abs()) + 5 * H * grad.abs()
    # eight neighbours are added in fp32 before the 64-bit sum (8), weights (3)
    e_policy = (w * (H * (16 + delta.abs()) * gain.abs())).sum()
    e_kl = (w * (e_k + 12 * H * k.abs())).sum()
    frac = (~free & live).sum().double() / n.clamp(min=1)
    return dict(loss=policy + beta * klm, policy=policy, kl=klm, clip_fraction=frac, n_valid=n, grad=grad, e_grad=e_grad, e_policy=e_policy, e_kl=e_kl,
                e_loss=e_policy + beta * e_kl)


def _check_policy(loss, info, grad, want, dtype):
    close(loss.cpu(), want["loss"], want["e_loss"] + 2 * H * want["loss"].abs(), "loss")
    close(info["policy"].cpu(), want["policy"], want["e_policy"] + 2 * H * want["policy"].abs(), "policy")
    close(info["kl"].cpu(), want["kl"], want["e_kl"] + 2 * H * want["kl"].abs(), "kl")
    close(info["clip_fraction"].cpu(), want["clip_fraction"], 2 * H, "clip_fraction")
    assert float(info["n_valid"]) == float(want["n_valid"])
    if grad is not None:
        assert grad.dtype == dtype
        close(grad.cpu(), want["grad"], want["e_grad"] + half(dtype) * want["grad"].abs() * 1.001 + tiny(dtype), "grad")


SHAPES = [(1, 1), (1, 2), (16, 100), (3, 4097), (2048, 5), (1, 20001), (129, 257), (40, 1000), (3, 12288 + 1), (70000, 1)]


@gpu
@pytest.mark.parametrize("R,T", SHAPES)
@pytest.mark.parametrize("mask", [None, "ragged", "random", "none valid"])
@pytest.mark.parametrize("reduction", ["steps", "rows", "sum"])
def test_policy_loss(R, T, mask, reduction):
    dtype = DTYPES[(R + T) % 3]
    kl, dual = ["k1", "k2", "k3"][(R + len(reduction)) % 3], [None, 2.5][T % 2]
    lp, old, ref, adv, m = _policy_case(R, T, dtype, mask, "rows" if (R + T) % 2 else "steps")
    want = _policy_want(lp, old, ref, adv, m, dual=dual, kl=kl, reduction=reduction)
    c = lambda t: None if t is None else t.cuda()  # noqa: E731
    if m is not None:  # padding holds anything
        lp, old = lp.clone(), old.clone()
        lp[~m], old[~m] = -math.inf, math.nan
        ref[~m] = math.inf
    kw = dict(old_log_prob=c(old), ref_log_prob=c(ref), mask=c(m), clip_high=0.28, dual_clip=dual, kl_coef=0.05, kl=kl, reduction=reduction)
    _check_policy(*P.policy_loss_and_grad(c(lp), c(adv), **kw), want, dtype)
    x = c(lp).requires_grad_()
    loss, info = P.policy_loss(x, c(adv), **kw)
    (4.0 * loss).backward()  # (a power of two: scaled exactly)
    want4 = {**want, "grad": 4 * want["grad"], "e_grad": 4 * want["e_grad"]}
    _check_policy(loss.detach(), info, x.grad, want4, dtype)
    with torch.no_grad():
        assert torch.equal(P.policy_loss(x, c(adv), **kw)[0], loss)
    if mask == "none valid":
        assert float(loss.detach()) == 0.0 and not x.grad.any()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,T", [(7, 45), (60, 301)])
def test_policy_loss_layouts(R, T, dtype):
    """Transposed planes, a slice with a row stride, unaligned starts, uint8 and broadcast masks, every type of advantage, log-ratios without `old`."""
    lp, old, ref, adv, m = _policy_case(R, T, dtype, "random", "steps")
    want = _policy_want(lp, old, ref, adv, m)
    tr = lambda t: t.t().contiguous().cuda().t()  # noqa: E731
    wide = lambda t: torch.cat([t, t], 1).cuda()[:, :t.shape[1]]  # noqa: E731
    off = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)]).cuda()[1:].view(t.shape)  # noqa: E731
    kw = dict(clip_high=0.28, kl_coef=0.05)
    for f in (tr, wide, off):
        _check_policy(*P.policy_loss_and_grad(f(lp), f(adv), f(old), f(ref), f(m), **kw), want, dtype)
        x = f(lp).requires_grad_()
        P.policy_loss(x, f(adv), f(old), f(ref), f(m.to(torch.uint8)), **kw)[0].backward()
        close(x.grad.cpu(), want["grad"], want["e_grad"] + half(dtype) * want["grad"].abs() * 1.001 + tiny(dtype))
    for t in DTYPES:
        a = adv.to(t)
        _check_policy(*P.policy_loss_and_grad(lp.cuda(), a.cuda(), old.cuda(), ref.cuda(), m.cuda(), **kw),
                      _policy_want(lp, old, ref, a, m), dtype)
    row = m[:1]
    _check_policy(*P.policy_loss_and_grad(lp.cuda(), adv[:, :1].cuda(), old.cuda(), ref.cuda(), row.cuda(), reduction="rows", **kw),
                  _policy_want(lp, old, ref, adv[:, 0], row, reduction="rows"), dtype)
    ratio = (lp.float() - old.float()).to(dtype)
    _check_policy(*P.policy_loss_and_grad(ratio.cuda(), adv.cuda(), None, None, m.cuda(), **kw), _policy_want(ratio, None, None, adv, m), dtype)
    x = ratio[:1].cuda().requires_grad_()  # one row for all: its gradient is the rows' sum
    P.policy_loss(x.expand(R, T), adv.cuda(), mask=m.cuda(), clip_high=0.28)[0].backward()
    want = _policy_want(ratio[:1].expand(R, T), None, None, adv, m)
    rounded = half(dtype) * want["grad"].abs().sum(0) * (R if dtype != torch.float32 else 2) + R * tiny(dtype)
    close(x.grad.cpu()[0], want["grad"].sum(0), want["e_grad"].sum(0) + 1.01 * rounded + R * H * want["grad"].abs().sum(0))


@gpu
@pytest.mark.parametrize("R,T", [(5, 64), (41, 1003)])
def test_masks_of_any_nonzero_byte(R, T):
    lp, old, ref, adv, m = (t.cuda() for t in _policy_case(R, T, torch.float32, "random", "rows"))
    bytes_ = m.to(torch.uint8) * torch.randint(1, 256, m.shape, device="cuda", dtype=torch.uint8)
    for reduction in ("steps", "rows"):
        a, b = (P.policy_loss_and_grad(lp, adv, old, ref, k, reduction=reduction, kl_coef=0.1) for k in (m, bytes_))
        assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])
    a, b = (P.preference_loss_and_grad(lp, old, None, None, k, k) for k in (m, bytes_))
    assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2]) and torch.equal(a[3], b[3])


@gpu
def test_policy_loss_borders_and_extremes():
    """Either side of the clipping borders by one step of fp32, no clipping at all, ratios that overflow, empty tensors."""
    hi, lo = math.log1p(0.28), math.log1p(-0.2)
    at = torch.tensor([hi, lo], dtype=torch.float32)
    up, down = torch.nextafter(at, at + 1), torch.nextafter(at, at - 1)
    d = torch.stack([up[0], down[0], up[1], down[1]]).repeat(2, 1)
    adv = torch.tensor([1.0, -1.0])
    want = _policy_want(d, None, None, adv, None)
    assert sorted((want["grad"] == 0).nonzero().tolist()) == [[0, 0], [1, 3]]
    loss, info, grad = P.policy_loss_and_grad(d.cuda(), adv.cuda(), clip_high=0.28)
    _check_policy(loss, info, grad, want, torch.float32)
    assert (grad.cpu() == 0).nonzero().tolist() == [[0, 0], [1, 3]]
    loss, info, grad = P.policy_loss_and_grad(d.cuda(), adv.cuda(), clip_low=2.0, clip_high=math.inf)
    assert float(info["clip_fraction"]) == 0.0 and bool((grad != 0).all())
    big = torch.tensor([[100.0, -200.0, 0.0]], device="cuda")
    loss, _, grad = P.policy_loss_and_grad(big, torch.tensor([1.0], device="cuda"), reduction="sum")
    assert torch.equal(grad, torch.tensor([[0.0, -0.0, -1.0]], device="cuda")) and abs(float(loss) + 2.2) < 1e-6
    assert float(P.policy_loss(big, torch.tensor([-1.0], device="cuda"))[0]) == math.inf
    assert float(P.policy_loss(big, torch.tensor([0.0], device="cuda"))[0]) == 0.0
    for shape in ((0, 5), (5, 0)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        loss, info = P.policy_loss(x, torch.zeros(shape[0], device="cuda"), reduction="rows")
        loss.backward()
        assert float(loss) == 0.0 and float(info["n_valid"]) == 0.0 and x.grad.shape == shape


@gpu
@pytest.mark.parametrize("kl", ["k1", "k2", "k3"])
def test_policy_gradient_against_differences(kl):
    """Central differences of the loss in 64 bits (of the formula) and of the kernel's own value, away from the borders."""
    lp, old, ref, adv, m = _policy_case(4, 6, torch.float32, "random", "steps")
    old = lp + 0.05 * torch.randn(4, 6, generator=torch.Generator().manual_seed(1))
    x = lp.cuda().requires_grad_()
    kw = dict(kl_coef=0.7, kl=kl, reduction="sum")
    P.policy_loss(x, adv.cuda(), old.cuda(), ref.cuda(), m.cuda(), **kw)[0].backward()
    step = 2.0 ** -8
    for i in range(24):
        e = torch.zeros(24)
        e[i] = step
        e = e.view(4, 6)
        f = [float(P.policy_loss((lp + s * e).cuda(), adv.cuda(), old.cuda(), ref.cuda(), m.cuda(), **kw)[0]) for s in (1, -1)]
        # third derivatives of exp(+-.) near 1 are below 8: step^2 8 / 6; rounding of two sums of 24 terms below 8
        assert abs((f[0] - f[1]) / (2 * step) - float(x.grad.view(-1)[i])) <= 8 / 6 * step ** 2 * 2 + 24 * 8 * 20 * H / step


# -- preference loss -----------------------------------------------------------------------------------------------------------------------
def _preference_case(N, Tc, Tr, dtype, mask, ref=True, seed=0):
    g = torch.Generator().manual_seed(seed + N + 3 * Tc)
    out = []
    for T in (Tc, Tr):
        x = (-3 * torch.rand(N, T, generator=g)).to(dtype)
        q = (x.float() + 0.3 * torch.randn(N, T, generator=g)).to(dtype) if ref else None
        m = None
        if mask == "ragged":
            n = torch.randint(0, T + 1, (N,), generator=g)
            n[N // 2] = 0
            m = torch.arange(T)[None] < n[:, None]
        elif mask == "random":
            m = torch.rand(N, T, generator=g) < 0.5
        out.append((x, q, m))
    return out


def _preference_want(case, beta=0.1, eps=0.0, kind="logistic", average=False):
    s, w, size, live = [], [], [], []
    for x, q, m in case:
        m = torch.ones(x.shape, dtype=torch.bool) if m is None else m
        d = torch.where(m, x.double() - (0.0 if q is None else q.double()), 0.0)
        n = m.sum(1).double()
        k = 1.0 / n.clamp(min=1) if average else torch.ones_like(n)
        s.append(d.sum(1) * k)
        size.append(d.abs().sum(1) * k * 2.0 ** -50 * max(1, x.shape[1]))
        w.append(k)
        live.append(m)
    gap = s[0] - s[1]
    h = beta * gap
    N = h.numel()
    if kind == "logistic":
        f = torch.nn.functional.logsigmoid
        losses = -(1 - eps) * f(h) - eps * f(-h)
        slope = beta * (eps * torch.sigmoid(h) - (1 - eps) * torch.sigmoid(-h))
        e_loss, e_slope = beta * sum(size), beta * beta * sum(size)
    elif kind == "hinge":
        losses, slope, e_loss, e_slope = (1 - h).clamp(min=0), -beta * (h < 1).double(), beta * sum(size), 0 * h
    else:
        r = gap - 0.5 / beta
        losses, slope, e_loss, e_slope = r * r, 2 * r, 2 * r.abs() * sum(size), 2 * sum(size)
    slope = slope / N
    return dict(loss=losses.mean(), accuracy=(h > 0).double().mean(), chosen_rewards=beta * s[0], rejected_rewards=beta * s[1],
                e_loss=e_loss.mean() + 4 * H * losses.mean(), e_s=[beta * z for z in size], e_slope=e_slope / N,
                grads=[(k * slope * z)[:, None] * m for k, z, m in zip((1, -1), w, live)])


def _check_preference(loss, info, grads, want, dtype, factor=1.0):
    close(loss.cpu(), want["loss"], want["e_loss"], "loss")
    assert float(info["accuracy"]) == float(want["accuracy"].float())
    for name, e in zip(("chosen_rewards", "rejected_rewards"), want["e_s"]):
        close(info[name].cpu(), want[name], 2 * H * want[name].abs() + e, name)
    for got, g in zip(grads, want["grads"]):
        assert got.dtype == dtype
        g = g * factor
        close(got.cpu(), g, 4 * H * g.abs() + factor * want["e_slope"][:, None] + half(dtype) * g.abs() * 1.001 + tiny(dtype), "grad")


@gpu
@pytest.mark.parametrize("N,Tc,Tr", [(1, 1, 1), (16, 100, 100), (5, 3, 800), (300, 64, 65), (2, 1025, 7), (3, 9001, 20011), (1500, 200, 200),
                                     (700, 1100, 900), (9000, 2, 3), (4, 0, 5)])
@pytest.mark.parametrize("mask", [None, "ragged", "random"])
@pytest.mark.parametrize("kind", ["logistic", "hinge", "square"])
def test_preference_loss(N, Tc, Tr, mask, kind):
    dtype = DTYPES[(N + Tc + len(kind)) % 3]
    average = (Tr + len(kind)) % 2 == 1
    eps = 0.1 if kind == "logistic" and Tc % 2 else 0.0
    beta = 0.5 if average else 0.1
    case = _preference_case(N, Tc, Tr, dtype, mask)
    want = _preference_want(case, beta, eps, kind, average)
    (c, qc, mc), (r, qr, mr) = [[None if t is None else t.clone() for t in side] for side in case]
    if mask is not None:
        for x, q, m in ((c, qc, mc), (r, qr, mr)):
            x[~m], q[~m] = math.nan, -math.inf
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    kw = dict(ref_chosen=dev(qc), ref_rejected=dev(qr), chosen_mask=dev(mc), rejected_mask=dev(mr), beta=beta, label_smoothing=eps, kind=kind,
              average=average)
    scale = 2.0 ** 10 if dtype == torch.float16 else 1.0
    loss, info, gc, gr = P.preference_loss_and_grad(dev(c), dev(r), **kw, grad_scale=scale)
    _check_preference(loss, info, (gc, gr), want, dtype, scale)
    x, y = dev(c).requires_grad_(), dev(r).requires_grad_()
    loss2, info = P.preference_loss(x, y, **kw)
    (scale * loss2).backward()
    _check_preference(loss2.detach(), info, (x.grad, y.grad), want, dtype, scale)
    assert torch.equal(loss2.detach(), loss) and torch.equal(x.grad, gc)


@gpu
@pytest.mark.parametrize("N,T", [(6, 50), (3, 5001)])
def test_preference_loss_layouts(N, T):
    case = _preference_case(N, T, T + 3, torch.float32, "random")
    want = _preference_want(case)
    tr = lambda t: t.t().contiguous().cuda().t()  # noqa: E731
    wide = lambda t: torch.cat([t, t], 1).cuda()[:, :t.shape[1]]  # noqa: E731
    off = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)]).cuda()[1:].view(t.shape)  # noqa: E731
    (c, qc, mc), (r, qr, mr) = case
    for f in (tr, wide, off):
        loss, info, gc, gr = P.preference_loss_and_grad(f(c), f(r), f(qc), f(qr), f(mc), f(mr.to(torch.uint8)))
        _check_preference(loss, info, (gc, gr), want, torch.float32)
    want = _preference_want(((c, None, mc[:1].expand_as(c)), (r, None, None)))
    loss, info, gc, gr = P.preference_loss_and_grad(c.cuda(), r.cuda(), chosen_mask=mc[:1].cuda())
    _check_preference(loss, info, (gc, gr), want, torch.float32)
    x = c.cuda().requires_grad_()  # one side only is differentiated; the same row against itself has no margin and no gradient
    P.preference_loss(x, r.cuda())[0].backward()
    close(x.grad.cpu(), _preference_want(((c, None, None), (r, None, None)))["grads"][0], 6 * H)
    x.grad = None
    loss, _ = P.preference_loss(x, x)
    loss.backward()
    assert abs(float(loss) - math.log(2.0)) < 2 * H and not x.grad.any()


@gpu
@pytest.mark.parametrize("h", [0.0, 40.0, -40.0, 800.0, -800.0, math.inf, -math.inf])
def test_preference_loss_saturates(h):
    c, r = torch.tensor([[h]], device="cuda"), torch.zeros(1, 1, device="cuda")
    loss, _, gc, gr = P.preference_loss_and_grad(c, r, beta=1.0)
    want = math.log1p(math.exp(-abs(h))) + max(-h, 0.0) if math.isfinite(h) else (0.0 if h > 0 else math.inf)
    assert float(loss) == pytest.approx(want, rel=2 * H)
    assert float(gc) == pytest.approx(-1 / (1 + math.exp(min(h, 700.0))) if h < 700 else 0.0, rel=4 * H, abs=1e-45) and float(gr) == -float(gc)


@gpu
def test_preference_gradient_against_differences():
    case = _preference_case(5, 7, 9, torch.float32, "random")
    (c, qc, mc), (r, qr, mr) = [[t.cuda() for t in side] for side in case]
    for kind in ("logistic", "square"):
        f = lambda c: P.preference_loss(c, r, qc, qr, mc, mr, beta=0.7, kind=kind)[0]  # noqa: E731
        x = c.clone().requires_grad_()
        f(x).backward()
        step = 2.0 ** -7
        for i in (0, 11, 34):
            e = torch.zeros(35, device="cuda")
            e[i] = step
            e = e.view(5, 7)
            d = (float(f(c + e)) - float(f(c - e))) / (2 * step)
            assert abs(d - float(x.grad.view(-1)[i])) <= step ** 2 + 8 * H * float(f(c).abs() + 1) / step


@gpu
def test_losses_may_be_changed_in_place():
    """`loss /= n` and `loss += other` as gradient accumulation writes them, with and without a gradient; what `info` holds stays as it is."""
    lp, old, ref, adv, m = (t.cuda() for t in _policy_case(6, 40, torch.float32, "random", "rows"))
    for f in (lambda x: P.policy_loss(x, adv, old, ref, m, kl_coef=0.1), lambda x: P.preference_loss(x[:3], x[3:], ref[:3], ref[3:], m[:3], m[3:])):
        x, y = lp.clone().requires_grad_(), lp.clone().requires_grad_()
        loss, info = f(x)
        kept = {k: t.clone() for k, t in info.items()}
        value = loss.detach().clone()
        loss /= 4
        loss += 1
        loss.backward()
        other, _ = f(y)
        (other / 4 + 1).backward()
        assert torch.equal(loss.detach(), value / 4 + 1) and torch.equal(x.grad, y.grad)
        assert all(torch.equal(info[k], kept[k]) and not info[k].requires_grad for k in info)
        z = torch.ones((), device="cuda", requires_grad=True)
        loss, info = f(lp)
        loss += z
        loss.backward()
        assert float(z.grad) == 1.0 and not any(t.requires_grad for t in info.values())


# -- streams, graphs, two calls at once ------------------------------------------------------------------------------------------------------
@gpu
def test_losses_on_another_stream_and_in_a_graph():
    """The gradient of a captured call, replayed on new values with eager work in between, is the eager one bit for bit; two graphs share nothing."""
    def case(seed):
        lp, old, ref, adv, m = (t.cuda() for t in _policy_case(50, 300, torch.float32, "ragged", "rows", seed=seed))
        return lp, adv, old, ref, m

    static = [[t.clone() for t in case(s)] for s in (0, 1)]
    run = lambda a: P.policy_loss_and_grad(*a, kl_coef=0.1, reduction="rows")  # noqa: E731

    def both(a):
        x = a[0].detach().requires_grad_()
        loss, _ = P.policy_loss(x, *a[1:], kl_coef=0.1, reduction="rows")
        pref, _ = P.preference_loss(x[:25], x[25:], a[3][:25], a[3][25:], a[4][:25], a[4][25:])
        return (*run(a)[::2], *torch.autograd.grad(loss + pref, x), loss.detach(), pref.detach())

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(static[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for a in static:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(both(a))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for k in range(4):
        fresh = [case(10 + 2 * k), case(11 + 2 * k)]
        for a, f in zip(static, fresh):
            for t, s in zip(a, f):
                t.copy_(s)
        want = [both(f) for f in fresh]
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(x, y) for x, y in zip(o, w))


@gpu
def test_results_do_not_change_from_call_to_call():
    lp, old, ref, adv, m = (t.cuda() for t in _policy_case(513, 1001, torch.bfloat16, "random", "steps"))
    runs = [P.policy_loss_and_grad(lp, adv, old, ref, m, kl_coef=0.1, reduction="rows") for _ in range(3)]
    assert all(torch.equal(r[0], runs[0][0]) and torch.equal(r[2], runs[0][2]) for r in runs)
    c, r = torch.randn(7, 50001, device="cuda"), torch.randn(7, 40001, device="cuda")
    runs = [P.preference_loss_and_grad(c, r) for _ in range(3)]
    assert all(torch.equal(x[0], runs[0][0]) and torch.equal(x[2], runs[0][2]) for x in runs)


# -- refusals --------------------------------------------------------------------------------------------------------------------------------
def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 3)
    with pytest.raises(RuntimeError, match="HIP device only"):
        P.step_log_ratio(torch.zeros(2, 3, 4), None, torch.zeros(2, 3, 4), torch.ones(2))
    with pytest.raises(RuntimeError, match="HIP device only"):
        P.policy_loss(x, torch.zeros(2))
    with pytest.raises(RuntimeError, match="HIP device only"):
        P.preference_loss(x, x)


@pytest.mark.parametrize("d", [(1 << 30) + 1, (1 << 31) - 1, 1 << 31, (1 << 32) + 7])
def test_step_log_ratio_refuses_dims_past_what_it_indexes(d):
    """Cut to 32 bits a dim of 2^32 + 7 would be 7, and an index of 32 bits that goes on in steps of 256 passes 2^31 behind a row of 2^31 - 1."""
    u = torch.zeros(1).expand(1, 1, d)
    with pytest.raises(ValueError, match="dim"):
        P.step_log_ratio(u, None, u, torch.ones(1))
    if d < 1 << 31:
        lib = L.load()
        assert lib.sdeh_step_log_ratio(64, None, 64, 64, 0, 2, d, 0, 64, None) == lib.sdeh_step_log_ratio(64, None, 64, 64, 1, 1, d, 0, 64, None) == -1
        assert lib.sdeh_step_log_ratio_backward(64, None, 64, 64, 64, 1, 1, d, 0, 64, None) == -1


def test_c_entries_refuse_bad_arguments():
    lib = L.load()
    ok = lambda **k: L.POLICY_LOSS.pack(*(64, 4, 1) * 5, k.get("rows", 2), k.get("steps", 4), k.get("dtype", 0), 0, k.get("kl", 3), k.get("red", 0),  # noqa: E731
                                        k.get("lo", 0.2), k.get("hi", 0.2), k.get("dual", 0.0), 0.0)
    call = lambda p, s=64, o=64, g=None: lib.sdeh_policy_loss(p, s, 0, None, 1.0, o, g, None)  # noqa: E731
    assert call(None) == call(ok(), s=None) == call(ok(), s=72) == call(ok(), o=None) == -1
    for bad in (dict(rows=-1), dict(steps=-1), dict(steps=1 << 31), dict(rows=1 << 40, steps=1 << 30), dict(dtype=3), dict(kl=0), dict(red=3),
                dict(lo=-0.1), dict(hi=math.nan), dict(dual=0.5)):
        assert call(ok(**bad)) == -1, bad
    assert call(L.POLICY_LOSS.pack(*(0, 0, 0) * 5, 2, 4, 0, 0, 3, 0, 0.2, 0.2, 0.0, 0.0)) == -1
    side = (64, 4, 1, 0, 0, 0, 0, 0, 0, 4)
    pref = lambda **k: L.PREFERENCE_LOSS.pack(*k.get("c", side), *side, k.get("pairs", 2), k.get("dtype", 0), k.get("kind", 0), 0, k.get("beta", 0.1),  # noqa: E731
                                              k.get("eps", 0.0))
    assert lib.sdeh_preference_loss(None, 64, 1.0, 64, None, None, None) == -1
    for bad in (dict(pairs=0), dict(dtype=-1), dict(kind=3), dict(beta=0.0), dict(beta=math.nan), dict(eps=0.5), dict(c=(0,) * 9 + (4,)),
                dict(c=(64, 4, 1) + (0,) * 6 + (-1,))):
        assert lib.sdeh_preference_loss(pref(**bad), 64, 1.0, 64, None, None, None) == -1, bad
    assert lib.sdeh_preference_loss(pref(), 72, 1.0, 64, None, None, None) == -1
    assert lib.sdeh_preference_loss(pref(), None, 1.0, 64, None, None, None) == lib.sdeh_preference_loss(pref(), 64, 1.0, 64, 64, None, None) == -1
    assert lib.sdeh_preference_grad(pref(), 64, None, 1.0, None, 64, None) == -1
    assert lib.sdeh_step_log_ratio(64, None, 64, 64, 2, 2, 0, 0, 64, None) == lib.sdeh_step_log_ratio(64, None, None, 64, 2, 2, 2, 0, 64, None) == -1
    assert lib.sdeh_step_log_ratio(64, None, 64, 64, 1 << 31, 1 << 31, 4, 0, 64, None) == -1
    assert lib.sdeh_step_log_ratio_backward(64, None, 64, 64, None, 2, 2, 2, 0, 64, None) == -1
    assert lib.sdeh_step_log_ratio(None, None, None, None, 0, 2, 2, 0, None, None) == 0


def test_packed_structs_match_the_header(tmp_path):
    src = '#include <stdio.h>\n#include "sdeh.h"\nint main(){printf("%zu %zu %zu %zu %zu", sizeof(SdehPolicyLoss), sizeof(SdehPreferenceLoss), ' \
          'sizeof(SdehAdamwGroup), sizeof(SdehAdamw), sizeof(SdehAdamwTensor));return 0;}\n'
    exe = tmp_path / "sizes"
    include = Path(__file__).resolve().parents[1] / "include"
    subprocess.run(["gcc", "-x", "c", "-", "-I", str(include), "-o", str(exe)], input=src.encode(), check=True)
    sizes = list(map(int, subprocess.run([str(exe)], capture_output=True, check=True).stdout.split()))
    assert sizes == [L.POLICY_LOSS.size, L.PREFERENCE_LOSS.size, L.ADAMW_GROUP.size, L.ADAMW.size, L.ADAMW_TENSOR_WORDS * ctypes.sizeof(ctypes.c_int64)]


@gpu
def test_refusals():
    x, a = torch.zeros(3, 4, device="cuda"), torch.zeros(3, device="cuda")
    for kw in (dict(old_log_prob=x[:2]), dict(old_log_prob=x.half()), dict(ref_log_prob=x.cpu()), dict(mask=torch.ones(2, 4, device="cuda", dtype=torch.bool)),
               dict(mask=x), dict(mask=torch.ones(3, 4, dtype=torch.bool)), dict(kl="k4"), dict(reduction="mean"), dict(clip_low=-1.0), dict(dual_clip=1.0)):
        with pytest.raises(ValueError):
            P.policy_loss(x, a, **kw)
    with pytest.raises(ValueError):
        P.policy_loss(x, a[:2])
    with pytest.raises(ValueError):
        P.policy_loss(x[0], a)
    with pytest.raises(L.SdehUnsupported):
        P.policy_loss(x.double(), a)
    for args, kw in (((x, x[:2]), {}), ((x[:0], x[:0]), {}), ((x, x.half()), {}), ((x, x), dict(ref_chosen=x[:, :2])), ((x, x), dict(chosen_mask=x)),
                     ((x, x), dict(rejected_mask=torch.ones(3, 5, device="cuda", dtype=torch.bool))), ((x, x), dict(kind="hing")), ((x, x), dict(beta=0.0)),
                     ((x, x), dict(label_smoothing=0.5)), ((x, x), dict(kind="hinge", label_smoothing=0.1))):
        with pytest.raises(ValueError):
            P.preference_loss(*args, **kw)
    u, dt = torch.zeros(2, 3, 4, device="cuda"), torch.ones(2, device="cuda")
    for args in ((u[0], None, u[0], dt), (u, u[:1], u, dt), (u, None, u.half(), dt), (u, None, u, dt[:1]), (u, None, u, dt.cpu()), (u[..., :0], None, u[..., :0], dt)):
        with pytest.raises(ValueError):
            P.step_log_ratio(*args)


@gpu
def test_gradients_are_differentiable_once():
    x = torch.randn(3, 5, device="cuda", requires_grad=True)
    u = torch.randn(3, 5, 2, device="cuda", requires_grad=True)
    for f, t in ((lambda: P.policy_loss(x, torch.ones(3, device="cuda"))[0], x), (lambda: P.preference_loss(x, -x)[0], x),
                 (lambda: P.step_log_ratio(u, None, u.detach(), torch.ones(3, device="cuda")).sum(), u)):
        (first,) = torch.autograd.grad(f(), t)
        (again,) = torch.autograd.grad(f(), t, create_graph=True)
        assert torch.equal(first, again)
        with pytest.raises(RuntimeError):  # (a gradient of the gradient: there is none, and none is made up)
            again.sum().backward()


@gpu
def test_forward_mode_is_refused():
    """A dual tensor's tangent would be lost without a word."""
    lp = torch.zeros(3, 4, device="cuda")
    u = torch.zeros(3, 4, 2, device="cuda")
    ones = torch.ones(3, device="cuda")
    with fwad.dual_level():
        x, w = fwad.make_dual(lp, torch.ones_like(lp)), fwad.make_dual(u, torch.ones_like(u))
        for f in (lambda: P.policy_loss(x, ones), lambda: P.preference_loss(x, lp), lambda: P.preference_loss(lp, x),
                  lambda: P.step_log_ratio(w, None, u, ones), lambda: P.policy_loss(x.t(), torch.ones(4, device="cuda"))):
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(NotImplementedError, match="forward"):
                    f()
        P.policy_loss(lp, ones)
        P.step_log_ratio(u, None, u, ones)


@gpu
@pytest.mark.parametrize("how", ["save_on_cpu", "checkpoint"])
def test_saved_tensors_may_go_away(how):
    """Saved tensors that were moved to the host, or made anew, in between: the backward pass reads what it is given, not where they were."""
    import torch.utils.checkpoint as cp

    lp, old, ref, adv, m = _policy_case(64, 300, torch.float32, "random", "rows")
    m = m.cuda()

    def run(x, away):
        def loss(x):
            y = x * 1.0
            a = P.policy_loss(y, adv.cuda(), old.cuda(), ref.cuda(), m.clone(), kl_coef=0.1, reduction="rows")[0]
            b = P.preference_loss(y[:32], y[32:], None, None, m[:32].clone(), m[32:].clone())[0]
            b = b + P.policy_loss(y, adv.cuda(), mask=m[:1].clone().expand(64, -1))[0]  # (a broadcast mask comes back as a whole one)
            c = P.step_log_ratio(y.view(64, 50, 6), None, old.cuda().view(64, 50, 6), torch.ones(64, device="cuda")).sum()
            return a + b + 1e-3 * c

        if away == "save_on_cpu":
            with torch.autograd.graph.save_on_cpu():
                value = loss(x)
        else:
            value = cp.checkpoint(loss, x, use_reentrant=False) if away else loss(x)
        junk = [torch.full((64, 300), float("nan"), device="cuda") for _ in range(40)]  # (what was freed is written over)
        value.backward()
        del junk
        return value.detach(), x.grad

    want = run(lp.cuda().requires_grad_(), None)
    got = run(lp.cuda().requires_grad_(), how)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


BIG = (1 << 31) + 4099  # elements, odd


def _room(gib):
    free, _ = torch.cuda.mem_get_info()
    if free < gib << 30:
        pytest.skip(f"needs {gib} GiB of device memory")


@gpu
@pytest.mark.parametrize("rows", [1, 3])
def test_policy_loss_past_32_bit_offsets(rows):
    """More than 2^31 entries: what lies behind them is read and written where it is.  All entries alike but the last few and one at 2^31."""
    _room(24)
    T = -(-BIG // rows)
    if rows == 1:
        T = (1 << 31) - 1  # the most steps a row may have; the second row's entries lie past 2^31
        rows = 2
    x = torch.full((rows, T), -0.125, device="cuda", dtype=torch.bfloat16)
    spots = [(0, 0), (rows - 1, T - 1), (rows - 1, T - 700), (rows - 1, 5)]
    for k, (r, c) in enumerate(spots):
        x[r, c] = 0.25 + 0.125 * k  # beyond the upper border
    mask = torch.ones(rows, T, device="cuda", dtype=torch.bool)
    mask[rows - 1, T - 2] = False
    loss, info, grad = P.policy_loss_and_grad(x, torch.ones(rows, device="cuda"), mask=mask, reduction="sum")
    n = rows * T - 1
    want = -((n - 4) * math.exp(-0.125) + 4 * 1.2)
    assert abs(float(loss) - want) <= 12 * H * abs(want)
    assert float(info["clip_fraction"]) == pytest.approx(4 / n, rel=1e-6)
    assert all(float(grad[s]) == 0.0 for s in spots) and float(grad[rows - 1, T - 2]) == 0.0
    flat = grad.view(-1)
    usual = float(torch.tensor(-math.exp(-0.125)).bfloat16())
    assert int((flat[-1000:] == usual).sum()) == 1000 - 3 and int((flat != usual).sum()) == 5


@gpu
def test_preference_loss_past_32_bit_offsets():
    _room(24)
    x = torch.zeros(1, BIG, device="cuda", dtype=torch.bfloat16)
    y = torch.zeros(1, 3, device="cuda", dtype=torch.bfloat16)
    x[0, -1], x[0, 1 << 31] = 2.0, 3.0
    loss, info, gx, gy = P.preference_loss_and_grad(x, y, beta=1.0)
    assert float(info["chosen_rewards"]) == 5.0 and abs(float(loss) - math.log1p(math.exp(-5.0))) < 1e-8
    assert bool((gx == gx[0, 0]).all()) and float(gx[0, 0]) == -float(gy[0, 0]) != 0.0


@gpu
def test_step_log_ratio_past_32_bit_offsets():
    _room(48)
    T, d = 3, 7
    B = -(-BIG // (T * d))
    u = torch.zeros(T, B, d, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    dw = torch.full((T, B, d), 0.5, device="cuda", dtype=torch.bfloat16)
    dt = torch.tensor([0.1, 0.2, 0.5], device="cuda")
    with torch.no_grad():
        u[-1, -1], u[-1, -2, 0] = 2.0, 1.0
    y = P.step_log_ratio(u, None, dw, dt)
    y.backward(torch.ones_like(y))
    y = y.detach()
    assert float(y[-1, -1]) == 7 * (2.0 * 0.5 - 0.25 * 4.0) and float(y[-1, -2]) == 0.25 and int((y != 0).sum()) == 1
    assert bool((u.grad[-1, -1] == -0.5).all()) and float(u.grad[-1, -2, 0]) == 0.0 and int((u.grad != 0.5).sum()) == 8


MANY = (1 << 24) + 99  # workgroups of 256 threads: more than a launch holds


@gpu
def test_step_log_ratio_of_more_rows_than_a_launch_holds():
    """A workgroup a row (dim > 512): forward and backward, the rows around the first launch's end and the last ones."""
    _room(80)
    T, d = 7, 513
    B = -(-MANY // T)
    u = torch.zeros(T, B, d, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    dw = torch.full((T, B, d), 0.5, device="cuda", dtype=torch.bfloat16)
    dt = torch.arange(1, T + 1, device="cuda") * 0.125
    rows = [0, (1 << 24) - 2, (1 << 24) - 1, 1 << 24, T * B - 1]
    with torch.no_grad():
        u.view(-1, d)[rows, 512] = 1.0
    y = P.step_log_ratio(u, None, dw, dt)
    y.backward(torch.ones_like(y))
    y = y.detach().view(-1)
    assert y[rows].cpu().tolist() == [0.5 - 0.5 * 0.125 * (r // B + 1) for r in rows] and int((y != 0).sum()) == len(rows)
    g = u.grad.view(-1, d)
    assert g[rows, 512].cpu().tolist() == [0.5 - 0.125 * (r // B + 1) for r in rows]
    assert int((g != 0.5).sum()) == len(rows)


@gpu
def test_preference_loss_of_more_rows_than_a_launch_holds():
    _room(64)
    pairs = MANY // 2 + 1  # two rows of a pair, a workgroup each
    x = torch.zeros(pairs, 1025, device="cuda", dtype=torch.bfloat16)
    y = torch.zeros(pairs, 1, device="cuda", dtype=torch.bfloat16)
    x[0, 0], x[-1, -1], y[-1, 0], y[-50, 0] = 2.0, 3.0, 1.0, 4.0
    loss, info, gx, gy = P.preference_loss_and_grad(x, y, beta=1.0, kind="hinge", grad_scale=float(pairs))
    c, r = info["chosen_rewards"], info["rejected_rewards"]
    assert float(c[0]) == 2.0 and float(c[-1]) == 3.0 and int((c != 0).sum()) == 2
    assert float(r[-1]) == 1.0 and float(r[-50]) == 4.0 and int((r != 0).sum()) == 2
    # losses: 0 for the first and the last pair, 5 for the 50th from the end, 1 for every other; slopes -1 where the loss is not 0
    assert abs(float(loss) * pairs - (pairs - 3 + 5)) <= 2 * H * pairs
    flat = gx.sum(1, dtype=torch.float32)
    assert float(flat[0]) == float(flat[-1]) == 0.0 and int((flat != -1025).sum()) == 2 and int((gy != 1).sum()) == 2
