"""AdamW over many tensors (sde_sampler_amd/utils/optim.py; include/sdeh.h: sdeh_adamw_step) against the formulas: 32-bit moments in 64 bits, 8-bit
moments bit for bit.

Tolerances: h = 2^-24 is half a step of fp32 relative to the value; n roundings of terms of absolute sum S are off by at most n h S (a last-digit
difference of sqrt and division counted as two).  Every step is checked from the state that the kernel itself left, so errors do not add up."""
import copy
import io
import math
import pickle

import numpy as np
import pytest
import torch

from sde_sampler_amd import _lib as L
from sde_sampler_amd import problems
from sde_sampler_amd.losses import policy as P
from sde_sampler_amd.utils.graphs import GraphedTrainStep
from sde_sampler_amd.utils.optim import AdamW

H = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
gpu = pytest.mark.gpu


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


# -- the 8-bit format in numpy -------------------------------------------------------------------------------------------------------------
def np_random(place, seed, step):
    with np.errstate(over="ignore"):
        key = np.uint32((seed * 0x3C6EF373 + step * 0xBB67AE85) & 0xFFFFFFFF)
        x = place.astype(np.uint32) * np.uint32(0x9E3779B1) + key
        x ^= x >> np.uint32(16)
        x *= np.uint32(0x6A09E667)
        x ^= x >> np.uint32(15)
        x *= np.uint32(0xBB67AE85)
        return x ^ (x >> np.uint32(16))


def np_encode(x, r16, signed):
    """codes and tops of one tensor (its last block may be short)"""
    depth, most = (15, 127) if signed else (31, 255)
    n, nb = x.size, -(-x.size // 256)
    bits = x.astype(np.float32).view(np.uint32).astype(np.int64)
    q = ((bits & 0x7FFFFFFF) + r16.astype(np.int64) * 16 + 8) >> 20
    pad = np.zeros(nb * 256, np.int64)
    pad[:n] = q
    top = np.clip(pad.reshape(nb, 256).max(1) >> 3, depth + 1, 255)
    c = q - 8 * (np.repeat(top, 256)[:n] - depth)
    if signed:
        c = np.clip(np.where(c < 1, 0, c), 0, most) | ((bits >> 24) & 128)
    else:
        c = np.where((bits & 0x7FFFFFFF) == 0, 0, np.clip(c, 1, most))
    return c.astype(np.uint8), top.astype(np.uint8)


def np_decode(c, top, signed):
    depth = 15 if signed else 31
    mag = (c & 127 if signed else c).astype(np.int64)
    t = np.repeat(top.astype(np.int64), 256)[:c.size]
    x = np.ldexp(1.0 + (mag % 8) / 8.0, t - 127 - depth + mag // 8)
    x = np.where(mag == 0, 0.0, x)
    return (np.where(c >= 128, -x, x) if signed else x).astype(np.float32)


def test_format_rounds_without_bias_and_keeps_its_own_values():
    """What is representable is kept for any random bits; anything else goes to one of its two neighbours, on average to itself."""
    rng = np.random.default_rng(0)
    x = (rng.standard_normal(256 * 40) * np.exp(rng.uniform(-3, 3, 256 * 40))).astype(np.float32)
    for signed in (True, False):
        y = x if signed else np.square(x)
        r = rng.integers(0, 1 << 16, y.size)
        c, top = np_encode(y, r, signed)
        v = np_decode(c, top, signed)
        for r2 in (0 * r, r, 0 * r + 65535):
            c2, top2 = np_encode(v, r2, signed)
            assert np.array_equal(np_decode(c2, top2, signed), v)
        big = np.abs(y) > np.repeat(np.abs(y).reshape(-1, 256).max(1), 256) * 2.0 ** -14
        assert (np.abs(v - y)[big] <= np.abs(y)[big] / 8).all()  # (three mantissa bits: neighbours are 1/8 of a power of two apart)
        mean = np.mean([np_decode(*np_encode(y, np_random(np.arange(y.size), 3, t) & 0xFFFF, signed), signed) for t in range(400)], 0, dtype=np.float64)
        # a neighbour is at most |y| / 8 away: standard deviation below |y| / 16; 400 draws, 6 deviations
        assert (np.abs(mean - y)[big] <= np.abs(y)[big] / 16 / 20 * 6).all()
    assert (np_encode(np.float32([1.0, 1e-30, 0.0]), np.zeros(3, int), False)[0] == [31 * 8, 1, 0]).all()


# -- one step in 64 bits ---------------------------------------------------------------------------------------------------------------------
def _want(p, g, m, v, t, scale, lr, b1, b2, eps, wd):
    p, g, m, v = (x.double() for x in (p, g, m, v))
    g = g * scale
    s_m = b1 * m.abs() + (1 - b1) * g.abs()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    denom = v.sqrt() / math.sqrt(1 - b2 ** t) + eps
    size = lr / (1 - b1 ** t)
    new = p * (1 - lr * wd) - size * m / denom
    e_m, e_v = 6 * H * s_m, 9 * H * v  # (clipped gradient, product, coefficient, sum; squared: twice)
    # sqrt halves v's relative error; its own digits, the bias correction's, eps, division, step size, products, sum
    e_p = size * (e_m / denom + m.abs() / denom * 16 * H) + 4 * H * (p.abs() + (size * m / denom).abs())
    return new, m, v, e_p, e_m, e_v


def _params(sizes, dtype, seed=0, unaligned=False):
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in sizes:
        x = (0.3 * torch.randn(n, generator=g)).to(dtype)
        if unaligned:
            x = torch.cat([x.new_zeros(1), x]).cuda()[1:]
        out.append(torch.nn.Parameter(x.cuda() if not unaligned else x))
    return out


def _set_grads(params, seed, unaligned=False):
    g = torch.Generator().manual_seed(100 + seed)
    for i, p in enumerate(params):
        x = (torch.randn(p.shape, generator=g) * 10.0 ** (-(i % 3))).to(p.dtype)
        x[torch.rand(p.shape, generator=g) < 0.1] = 0
        p.grad = torch.cat([x.new_zeros(1), x.reshape(-1)]).cuda()[1:].view(p.shape) if unaligned else x.cuda()


def _snapshot(opt, params):
    return [(p.detach().cpu().clone(), p.grad.cpu().clone(), {k: t.cpu().clone() for k, t in opt.state[p].items()} if p in opt.state else None) for p in params]


def _scale(grads, clip):
    if clip is None:
        return 1.0, None
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    return min(1.0, clip / (norm + 1e-6)), norm


SIZES = [1, 3, 255, 256, 257, 4095, 4096, 4097, 20001, 8192, 2]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("clip", [None, 0.5, 1e6])
@pytest.mark.parametrize("unaligned", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_step(dtype, clip, unaligned, bits):
    params = _params(SIZES, dtype, unaligned=unaligned)
    hyper = dict(lr=2e-2, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1)
    opt = AdamW(params, **hyper, state_bits=bits, max_grad_norm=clip, seed=11)
    first = 0
    for step in range(1, 5):
        _set_grads(params, step, unaligned)
        opt._plan()
        before = _snapshot(opt, params)
        opt.step()
        scale, norm = _scale([b[1] for b in before], clip)
        if clip is not None:
            assert abs(float(opt.grad_norm) - norm) <= 2 * H * norm
        first = 0
        for p, (p0, g0, s0) in zip(params, before):
            n, s = p.numel(), {k: t.cpu() for k, t in opt.state[p].items()}
            assert float(s["step"]) == step
            if bits == 8:
                m0 = torch.from_numpy(np_decode(s0["exp_avg"].numpy(), s0["exp_avg_top"].numpy(), True))
                v0 = torch.from_numpy(np_decode(s0["exp_avg_sq"].numpy(), s0["exp_avg_sq_top"].numpy(), False))
            else:
                m0, v0 = s0["exp_avg"], s0["exp_avg_sq"]
            new, m, v, e_p, e_m, e_v = _want(p0, g0, m0, v0, step, scale, hyper["lr"], *hyper["betas"], hyper["eps"], hyper["weight_decay"])
            err = (p.detach().cpu().double() - new).abs()
            assert (err <= e_p + 1.001 * half(dtype) * (new.abs() + e_p) + tiny(dtype)).all(), float(err.max())
            if bits == 32:
                assert ((s["exp_avg"].double() - m).abs() <= e_m + 1e-45).all() and ((s["exp_avg_sq"].double() - v).abs() <= e_v + 1e-38).all()
            else:
                f32 = np.float32
                g = g0.float().numpy() * f32(scale) if clip is not None else g0.float().numpy()
                b1, b2 = hyper["betas"]
                mm = m0.numpy() * f32(b1) + g * f32(1 - b1)
                vv = v0.numpy() * f32(b2) + g * g * f32(1 - b2)
                r = np_random(first * 256 + np.arange(n), 11, step)
                for name, x, r16, signed in (("exp_avg", mm, r & 0xFFFF, True), ("exp_avg_sq", vv, r >> 16, False)):
                    c, top = np_encode(x, r16, signed)
                    assert np.array_equal(s[name + "_top"].numpy(), top) and np.array_equal(s[name].numpy(), c), (name, n)
            first += -(-n // 256)


@gpu
@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-12, 1e-8])
def test_tiny_gradients(eps):
    """Second moments down to the subnormal numbers: sqrt(v) counts beside whatever eps there is."""
    p = torch.nn.Parameter(torch.ones(4096, device="cuda"))
    g = torch.full((4096,), 10.0).pow(torch.linspace(-24, -3, 4096))
    opt = AdamW([p], lr=0.5, eps=eps, weight_decay=0.0)
    p.grad = g.cuda()
    opt.step()
    s = {k: t.cpu() for k, t in opt.state[p].items()}
    # from the moments as they are held (g^2 below 1e-38 has few digits left, below 1e-45 none)
    denom = s["exp_avg_sq"].double().sqrt() / math.sqrt(1 - 0.999) + eps
    want = 1.0 - 0.5 / (1 - 0.9) * s["exp_avg"].double() / denom
    some = denom > 0
    assert some.sum() > 3000
    # sqrt, reciprocal, three products, two coefficients and two sums: below 20 roundings; a root taken for 0 is below 2^-63, 2^-58 with its bias correction
    tol = 20 * H * (1.0 + (want - 1.0).abs()) + ((want - 1.0).abs() * 2.0 ** -58 / eps if eps >= 1e-11 else 0.0)
    assert ((p.detach().cpu().double() - want).abs() <= tol)[some].all()


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_moments_are_the_states_values(bits):
    params = _params(SIZES, torch.float32)
    opt = AdamW([{"params": params[:4]}, {"params": params[4:], "lr": 0.1}], state_bits=bits)
    _set_grads(params, 0)
    opt.step()
    m, v = opt.moments()
    at = 0
    for p in params:
        s = {k: t.cpu() for k, t in opt.state[p].items()}
        n = p.numel()
        for flat, name, signed in ((m, "exp_avg", True), (v, "exp_avg_sq", False)):
            want = s[name] if bits == 32 else torch.from_numpy(np_decode(s[name].numpy(), s[name + "_top"].numpy(), signed))
            assert torch.equal(flat[at:at + n].cpu(), want)
        at += -(-n // 256) * 256
    assert at == m.numel() == v.numel()


@gpu
def test_agrees_with_torch_over_steps():
    """The same trajectory as clip_grad_norm_ + torch.optim.AdamW, two groups, a schedule on one, parameters of several shapes and two types."""
    mk = lambda: [torch.nn.Parameter(p.detach().view(s)) for p, s in zip(_params([6, 60, 1, 900], torch.float32), [(2, 3), (3, 4, 5), (), (30, 30)])]  # noqa: E731
    a, b = mk(), mk()
    groups = lambda ps: [{"params": ps[:2], "lr": 1e-2}, {"params": ps[2:], "weight_decay": 0.3}]  # noqa: E731
    ours, theirs = AdamW(groups(a), lr=3e-3, max_grad_norm=0.7), torch.optim.AdamW(groups(b), lr=3e-3)
    sched = [torch.optim.lr_scheduler.StepLR(o, step_size=3, gamma=0.5) for o in (ours, theirs)]
    for step in range(10):
        _set_grads(a, step)
        for x, y in zip(a, b):
            y.grad = x.grad.clone()
        norm = torch.nn.utils.clip_grad_norm_(b, 0.7)
        kept = [x.grad.clone() for x in a]
        ours.step()
        theirs.step()
        assert all(torch.equal(x.grad, k) for x, k in zip(a, kept))
        torch.testing.assert_close(ours.grad_norm, norm, rtol=1e-6, atol=0)
        for s in sched:
            s.step()
    for x, y in zip(a, b):  # (10 steps, each 20 roundings of a step of at most 1e-2 and 4 of the value)
        torch.testing.assert_close(x, y, rtol=10 * 8 * H, atol=10 * 1e-2 * 40 * H)


@gpu
def test_many_tensors_and_missing_gradients():
    """More tensors than one launch's arguments hold, some without entries, some without a gradient: those stay as they are."""
    sizes = [(37 * i) % 700 for i in range(130)]
    params = _params(sizes, torch.float32)
    extra = _params([300, 5000], torch.bfloat16, seed=5)
    opt = AdamW([{"params": params + extra}], lr=1e-2, max_grad_norm=0.5, weight_decay=0.0)
    _set_grads(params + extra, 1)
    idle = params[::7]
    for p in idle:
        p.grad = None
    live = [p for p in params + extra if p.grad is not None]
    before = _snapshot(opt, live)
    kept = [p.detach().clone() for p in idle]
    opt.step()
    scale, norm = _scale([b[1] for b in before], 0.5)
    assert abs(float(opt.grad_norm) - norm) <= 2 * H * norm
    for p, (p0, g0, _) in zip(live, before):
        new, m, v, e_p, _, _ = _want(p0, g0, 0 * g0, 0 * g0, 1, scale, 1e-2, 0.9, 0.999, 1e-8, 0.0)
        assert ((p.detach().cpu().double() - new).abs() <= e_p + 1.001 * half(p.dtype) * (new.abs() + e_p)).all()
    assert all(torch.equal(p, k) and float(opt.state[p]["step"]) == 0.0 for p, k in zip(idle, kept))
    for p in params + extra:
        p.grad = None
    opt.step()  # nothing to do


@gpu
def test_ok_decides_on_the_device():
    for bits in (32, 8):
        params = _params([1000, 7], torch.float32)
        opt = AdamW(params, max_grad_norm=1.0, state_bits=bits)
        _set_grads(params, 0)
        opt.step()
        before = _snapshot(opt, params)
        params[0].grad[3] = math.nan
        opt.step(ok=torch.zeros(1, dtype=torch.bool, device="cuda"))
        for p, (p0, _, s0) in zip(params, before):
            assert torch.equal(p.detach().cpu(), p0) and all(torch.equal(opt.state[p][k].cpu(), s0[k]) for k in s0)
        opt.step(ok=torch.ones(1, dtype=torch.bool, device="cuda"))
        assert float(opt.state[params[0]]["step"]) == 2.0
        assert bool(torch.isnan(opt.grad_norm)) and bool(torch.isnan(params[1]).all())  # (as clip_grad_norm_ would)
        m, v = opt.moments()
        assert bool(torch.isnan(m[:1000]).all()) and bool(torch.isnan(v[:1000]).all())


@gpu
def test_past_32_bit_offsets():
    """More than 2^31 entries in one tensor: its end is updated like its beginning."""
    free, _ = torch.cuda.mem_get_info()
    if free < 48 << 30:
        pytest.skip("needs 48 GiB of device memory")
    n = (1 << 31) + 4099
    p = torch.nn.Parameter(torch.ones(n, device="cuda", dtype=torch.bfloat16))
    p.grad = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    spots = [0, 255, (1 << 31) - 1, 1 << 31, (1 << 31) + 257, n - 1]
    p.grad[spots] = 1.0
    opt = AdamW([p], lr=0.5, weight_decay=0.0, state_bits=8, max_grad_norm=0.25)
    opt.step()
    assert abs(float(opt.grad_norm) - math.sqrt(6)) <= 4 * H
    p = p.detach()
    assert int((p != 1.0).sum()) == len(spots) and bool((p[spots] == 0.5).all())  # (a first step moves by lr, whatever the gradient's size)


@gpu
def test_learning_rate_on_the_device_and_closure():
    a, b = _params([500], torch.float32), _params([500], torch.float32)
    lr = torch.tensor(0.01, device="cuda")
    oa, ob = AdamW(a, lr=lr), AdamW(b, lr=0.01)
    for k in range(3):
        _set_grads(a, k)
        b[0].grad = a[0].grad.clone()
        lr.fill_(0.01 / (k + 1))
        ob.param_groups[0]["lr"] = float(lr)
        assert oa.step(lambda: 3.0) == 3.0
        ob.step()
    assert torch.equal(a[0], b[0])


@gpu
def test_step_hooks_and_the_profiler():
    from torch.optim.optimizer import register_optimizer_step_post_hook

    p = _params([10], torch.float32)
    opt, seen = AdamW(p), []
    _set_grads(p, 0)
    handles = [opt.register_step_pre_hook(lambda *a: seen.append("pre")), opt.register_step_post_hook(lambda *a: seen.append("post"))]
    opt.step()
    for h in handles:
        h.remove()
    assert seen == ["pre", "post"]
    h = register_optimizer_step_post_hook(lambda *a: seen.append("all"))
    opt.step()
    h.remove()
    opt.step()
    assert seen == ["pre", "post", "all"] and float(opt.state[p[0]]["step"]) == 3.0
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        opt.step(ok=torch.ones(1, dtype=torch.bool, device="cuda"))
    assert any("AdamW.step" in e.key for e in prof.key_averages()) and float(opt.state[p[0]]["step"]) == 4.0


@gpu
def test_second_moment_in_8_bits_decays_as_it_should():
    """2000 steps without gradients: rounding to the nearest would never leave the first code.  A step's rounding moves an entry by a code (at most 1/8)
    with probability at most 0.001 x 16: relative variance below 0.016 / 64 a step, 0.5 in all; the mean of 65536 entries is off by less than
    6 sqrt(0.5 / 65536) of itself."""
    p = torch.nn.Parameter(torch.zeros(65536, device="cuda"))
    opt = AdamW([p], lr=0.0, betas=(0.0, 0.999), state_bits=8)
    p.grad = torch.ones_like(p)
    opt.step()
    start = float(opt.moments()[1].mean(dtype=torch.float64))
    p.grad = torch.zeros_like(p)
    for _ in range(2000):
        opt.step()
    want = start * 0.999 ** 2000
    assert abs(float(opt.moments()[1].mean(dtype=torch.float64)) - want) <= want * 6 * math.sqrt(0.5 / 65536)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_is_seen_by_autograd(bits):
    """As with torch's optimizers: a graph whose forward pass saved a parameter before the step refuses its backward pass after it."""
    for make in (lambda ps: torch.optim.AdamW(ps), lambda ps: AdamW(ps, state_bits=bits, max_grad_norm=1.0)):
        p, idle = _params([12, 5], torch.float32)
        opt = make([p, idle])
        p.grad = torch.ones_like(p)
        opt.step()
        loss = (p * p).sum()
        versions = p._version, idle._version
        opt.step()
        assert p._version > versions[0] and idle._version == versions[1]
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    version = p._version
    norm = opt.grad_norm._version
    opt.step(ok=torch.ones(1, dtype=torch.bool, device="cuda"))
    assert p._version > version and opt.grad_norm._version > norm


@gpu
def test_steps_in_inference_mode():
    """Tensors made there have no version to move; a parameter without a gradient keeps its version, so that graphs that saved it go backward."""
    p, frozen = _params([12, 12], torch.float32)
    frozen.requires_grad_(False)
    opt = AdamW([p, frozen], max_grad_norm=1.0, lr=0.5, weight_decay=0.0)
    p.grad = torch.ones_like(p)
    x = torch.ones(12, device="cuda", requires_grad=True)
    loss = (frozen * x).sum()
    start = p.detach().clone()
    with torch.inference_mode():
        opt.step()
    opt.step()
    loss.backward()
    assert torch.equal(x.grad, frozen) and float(opt.state[p]["step"]) == 2.0
    assert ((start - p.detach()) - 1.0).abs().max() <= 2.0 ** -20  # (two steps of lr along a gradient that does not change, roundings of values below 2)


# -- state dicts ------------------------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_state_dict_round_trip(bits, dtype):
    """Resumed, deep-copied and unpickled optimizers go on bit for bit; loading keeps the buffers a captured step works on."""
    def after(opt, params, steps):
        for k in steps:
            _set_grads(params, k)
            opt.step()

    params = _params([700, 33], dtype)
    opt = AdamW(params, lr=1e-2, state_bits=bits, max_grad_norm=1.0, seed=4)
    after(opt, params, range(3))
    buf = io.BytesIO()
    torch.save(opt.state_dict(), buf)
    saved = torch.load(io.BytesIO(buf.getvalue()), weights_only=True)
    values = [p.detach().clone() for p in params]
    twin = copy.deepcopy((params, opt))
    third = pickle.loads(pickle.dumps((params, opt)))
    after(opt, params, range(3, 6))
    want = [p.detach().clone() for p in params]
    for ps, o in (twin, third):
        after(o, ps, range(3, 6))
        assert all(torch.equal(x, y) for x, y in zip(ps, want))
    fresh = [torch.nn.Parameter(v.clone()) for v in values]
    o = AdamW(fresh, lr=5.0, state_bits=bits, max_grad_norm=1.0, seed=4)
    o.load_state_dict(saved)
    assert o.param_groups[0]["lr"] == 1e-2
    after(o, fresh, range(3, 6))
    assert all(torch.equal(x, y) for x, y in zip(fresh, want))
    where = [t.data_ptr() for p in params for t in opt.state[p].values()]
    with torch.no_grad():
        for p, v in zip(params, values):
            p.copy_(v)
    opt.load_state_dict(saved)
    assert where == [t.data_ptr() for p in params for t in opt.state[p].values()]
    after(opt, params, range(3, 6))
    assert all(torch.equal(x, y) for x, y in zip(params, want))


@gpu
def test_loads_torch_state_and_refuses_other_formats():
    a, b = _params([50, 4], torch.float32), _params([50, 4], torch.float32)
    theirs = torch.optim.AdamW(b, lr=1e-2)
    for k in range(3):
        _set_grads(b, k)
        theirs.step()
    ours = AdamW(a, lr=1e-2)
    with torch.no_grad():
        for x, y in zip(a, b):
            x.copy_(y)
    ours.load_state_dict(theirs.state_dict())
    _set_grads(a, 9)
    _set_grads(b, 9)
    ours.step()
    theirs.step()
    for x, y in zip(a, b):
        torch.testing.assert_close(x, y, rtol=8 * H, atol=1e-2 * 40 * H)
    assert "capturable" not in ours.param_groups[0]
    back = torch.optim.AdamW(b, lr=1.0)
    back.load_state_dict(ours.state_dict())
    assert back.param_groups[0]["lr"] == 1e-2 and torch.equal(back.state[b[0]]["exp_avg"], ours.state[a[0]]["exp_avg"])
    for other in (torch.optim.AdamW(b, amsgrad=True), torch.optim.AdamW(b, maximize=True), torch.optim.Adam(b, weight_decay=0.1)):
        with pytest.raises(ValueError, match="amsgrad"):
            ours.load_state_dict(other.state_dict())
    with pytest.raises(ValueError, match="state_bits"):
        AdamW(_params([50, 4], torch.float32), state_bits=8).load_state_dict(ours.state_dict())
    with pytest.raises(ValueError):
        AdamW(_params([50, 5], torch.float32)).load_state_dict(ours.state_dict())
    ours.add_param_group({"params": _params([9], torch.float32), "lr": 0.5})
    kept = ours.state[a[0]]["exp_avg"].clone()
    ours._plan()
    assert torch.equal(ours.state[a[0]]["exp_avg"], kept)


@gpu
def test_loading_keeps_the_learning_rate_on_the_device():
    """`lr` on the device stays the tensor that the caller and a captured step hold; what is loaded -- from the device, the host or a number -- is its value."""
    p, q = _params([40], torch.float32), _params([40], torch.float32)
    lr = torch.tensor(0.5, device="cuda")
    opt = AdamW(p, lr=lr, weight_decay=0.0)
    _set_grads(p, 0)
    opt.step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        opt.step()
    saved = copy.deepcopy(opt.state_dict())  # (a state dict refers to the optimizer's own tensors)
    buf = io.BytesIO()
    torch.save(saved, buf)
    other = AdamW(q, lr=0.25, weight_decay=0.0)
    for state, value in ((saved, 0.5), (torch.load(io.BytesIO(buf.getvalue()), map_location="cpu", weights_only=True), 0.5), (other.state_dict(), 0.25)):
        lr.fill_(9.0)
        opt.load_state_dict(state)
        assert opt.param_groups[0]["lr"] is lr and float(lr) == value
    other.load_state_dict(opt.state_dict())
    with torch.no_grad():
        q[0].copy_(p[0])
    q[0].grad = p[0].grad.clone()
    lr.fill_(0.125)
    other.param_groups[0]["lr"] = 0.125
    g.replay()
    other.step()
    assert torch.equal(p[0], q[0])


@gpu
def test_a_state_dict_with_its_rate_on_the_host():
    a, b = _params([40], torch.float32), _params([40], torch.float32)
    opt = AdamW(a, lr=torch.tensor(0.5, device="cuda"))
    _set_grads(a, 0)
    opt.step()
    saved = opt.state_dict()
    saved["param_groups"][0]["lr"] = saved["param_groups"][0]["lr"].cpu()
    other = AdamW(b, lr=0.1)
    other.load_state_dict(saved)
    _set_grads(b, 0)
    other.step()
    assert float(other.param_groups[0]["lr"]) == 0.5 and float(other.state[b[0]]["step"]) == 2.0


@gpu
def test_load_hooks_see_and_change_the_state():
    """A pre-hook is given the whole state dict and may change it; a post-hook finds the state loaded."""
    params = _params([8], torch.float32)
    opt, seen = AdamW(params), []
    _set_grads(params, 0)
    opt.step()
    saved = opt.state_dict()
    moments = saved["state"][0]["exp_avg"].clone()

    def double(o, s):
        seen.append(len(s["state"]))
        return {**s, "state": {0: {**s["state"][0], "exp_avg": 2 * moments}}}

    opt.register_load_state_dict_pre_hook(double)
    opt.register_load_state_dict_post_hook(lambda o: seen.append(o.state[params[0]]["exp_avg"].clone()))
    opt.load_state_dict(saved)
    assert seen[0] == 1 and torch.equal(seen[1], 2 * moments)


def _all(opt, params):
    return [t.detach().cpu().clone() for p in params for t in (p, *opt.state[p].values())]


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_refused_load_changes_nothing(bits):
    params = _params([700, 33], torch.float32)
    opt = AdamW([{"params": params[:1]}, {"params": params[1:], "lr": 0.5}], state_bits=bits, max_grad_norm=1.0)
    for k in range(2):
        _set_grads(params, k)
        opt.step()
    before, where = _all(opt, params), [t.data_ptr() for p in params for t in opt.state[p].values()]
    groups = copy.deepcopy([{k: v for k, v in g.items() if k != "params"} for g in opt.param_groups])

    def broken():
        for change in (lambda s: s["state"][1].pop("exp_avg"), lambda s: s["state"][1].update(exp_avg=torch.zeros(5)),
                       lambda s: s["state"][1].update(more=torch.zeros(33)), lambda s: s["param_groups"][1].update(lr=-1.0),
                       lambda s: s["param_groups"][1].update(betas=(0.9, 1.0)), lambda s: s["param_groups"][1].update(amsgrad=True),
                       lambda s: s["param_groups"][1].pop("eps"),
                       lambda s: s["param_groups"].pop(), lambda s: s["param_groups"][1]["params"].append(2)):
            s = copy.deepcopy(opt.state_dict())
            s["state"][0]["step"] += 5
            s["param_groups"][0]["lr"] = 7.0
            change(s)
            yield s

    for s in broken():
        with pytest.raises(ValueError):
            opt.load_state_dict(s)
        assert [{k: v for k, v in g.items() if k != "params"} for g in opt.param_groups] == groups
        assert all(torch.equal(x, y) for x, y in zip(_all(opt, params), before))
        assert where == [t.data_ptr() for p in params for t in opt.state[p].values()] and opt.grad_norm is not None
    opt.step()
    assert float(opt.state[params[0]]["step"]) == 3.0


@gpu
def test_the_seed_travels_with_the_state():
    a, b = _params([3000], torch.float32), _params([3000], torch.float32)
    x, y = AdamW(a, state_bits=8, seed=5), AdamW(b, state_bits=8)
    for k in range(2):
        _set_grads(a, k)
        x.step()
    y.load_state_dict(x.state_dict())
    with torch.no_grad():
        b[0].copy_(a[0])
    for k in range(2, 6):
        _set_grads(a, k)
        _set_grads(b, k)
        x.step()
        y.step()
    assert torch.equal(a[0], b[0]) and all(torch.equal(x.state[a[0]][k], y.state[b[0]][k]) for k in x.state[a[0]])


# -- graphs, streams ----------------------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_replays_the_eager_one(bits):
    params = _params([5000, 64, 3], torch.float32)
    opt = AdamW(params, lr=1e-2, state_bits=bits, max_grad_norm=0.3)
    twin = _params([5000, 64, 3], torch.float32)
    eager = AdamW(twin, lr=1e-2, state_bits=bits, max_grad_norm=0.3)
    _set_grads(params, 0)
    _set_grads(twin, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    eager.step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        opt.step()
    for k in range(1, 6):
        _set_grads(twin, k)
        for p, q in zip(params, twin):
            p.grad.copy_(q.grad)
        eager.step()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(params, twin)) and torch.equal(opt.grad_norm, eager.grad_norm)


@gpu
def test_a_first_step_inside_a_capture_is_refused():
    """The state's zeros would be part of the graph."""
    params = _params([50], torch.float32)
    opt = AdamW(params)
    _set_grads(params, 0)
    spare = torch.zeros(4, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        spare += 1
        with pytest.raises(RuntimeError, match="captur"):
            opt.step()
    opt.step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        opt.step()
    for _ in range(3):
        g.replay()
    assert float(opt.state[params[0]]["step"]) == 4.0


def _problem(seed=0):
    spec = problems.baseline_spec("cfg1_dw_dis_lv")
    torch.manual_seed(seed)
    return problems.build(spec, device="cuda:0")


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_graphed_train_step_skips_on_the_device(bits):
    """GraphedTrainStep with this optimizer: the eager steps' parameters bit for bit, and a step whose loss is not finite changes nothing."""
    def build():
        prob = _problem()
        params = [p for p in prob.ctrl.parameters() if p.requires_grad]
        return prob, params, AdamW(params, lr=1e-3, weight_decay=0.0, state_bits=bits, max_grad_norm=1.0)

    prob, params, opt = build()
    torch.manual_seed(1)
    x = prob.prior.sample((512,))
    poison = torch.zeros((), device="cuda")
    step = GraphedTrainStep(lambda: prob.loss(prob.ts, x, prob.target.unnorm_log_prob, prob.second_log_prob)[0] + poison, [prob.loss], opt, warmup=2)
    for _ in range(3):
        step()
    torch.cuda.synchronize()
    assert int(step.n_skipped) == 0 and float(opt.state[params[0]]["step"]) == 5.0
    before = _snapshot(opt, params)
    poison.fill_(math.nan)
    step()
    torch.cuda.synchronize()
    assert int(step.n_skipped) == 1
    for p, (p0, _, s0) in zip(params, before):
        assert torch.equal(p.detach().cpu(), p0) and all(torch.equal(opt.state[p][k].cpu(), s0[k]) for k in s0)
    poison.zero_()
    step()
    torch.cuda.synchronize()
    assert int(step.n_skipped) == 1 and float(opt.state[params[0]]["step"]) == 6.0
    assert any(not torch.equal(p.detach().cpu(), p0) for p, (p0, _, _) in zip(params, before))


# -- the operators together ------------------------------------------------------------------------------------------------------------------------
@gpu
def test_policy_steps_on_stored_trajectories():
    """Trajectories of the engine, several policy steps on them: the log-ratios of the unchanged control are 0, the loss's gradient reaches every parameter
    of the network and is the one of the same formulas in torch's own operations; a preference step on the same paths runs."""
    prob = _problem()
    T, B = prob.ts.numel() - 1, 256
    x0 = prob.prior.sample((B,))
    noise = torch.randn(T, B, x0.shape[1], device="cuda")
    res = prob.eval(x0, compute_weights=True, return_traj=True, noise=noise)
    dt = prob.ts.diff()
    dw = noise * dt.sqrt()[:, None, None]
    xs, net = res.xs[:-1].detach(), prob.ctrl.base_model
    control = lambda: torch.stack([net(prob.ts[t], xs[t]) for t in range(0, T, 10)])  # noqa: E731  (every tenth step)
    dt, dw = dt[::10].contiguous(), dw[::10].contiguous()
    with torch.no_grad():
        behaviour = control()
    score = res.weights.reshape(-1)
    adv = (score - score.mean()) / score.std()
    mask = torch.rand(B, dt.numel(), device="cuda") < 0.9
    params = [p for p in net.parameters() if p.requires_grad]
    opt = AdamW(params, lr=1e-3, max_grad_norm=1.0)
    start = [p.detach().clone() for p in params]
    for k in range(3):
        u = control()
        ratio = P.step_log_ratio(u, behaviour, dw, dt)
        assert k or not ratio.any()
        loss, info = P.policy_loss(ratio.t(), adv, ref_log_prob=torch.zeros_like(ratio.t()), mask=mask, kl_coef=0.1)
        opt.zero_grad()
        loss.backward()
        with torch.enable_grad():
            e = (v := control()) - behaviour
            r = (e * dw - 0.5 * dt[:, None, None] * e * e).sum(-1).t()
            want = torch.maximum(-adv[:, None] * r.exp(), -adv[:, None] * r.exp().clamp(0.8, 1.2)) + 0.1 * (torch.exp(-r) - 1 + r)
            grads = torch.autograd.grad((want * mask).sum() / mask.sum(), params, allow_unused=True)
        del v
        for p, g in zip(params, grads):
            assert (p.grad is None) == (g is None)
            if g is not None:  # (both sides sum 2560 rows' contributions in fp32, in different orders)
                assert (p.grad - g).abs().max() <= 2e-5 * g.abs().max() + 1e-7
        opt.step()
        assert float(info["n_valid"]) == float(mask.sum())
    assert all(not torch.equal(p, s) for p, s in zip(params, start) if p.grad is not None and p.grad.any())
    better, worse = score.sort(descending=True).indices.split(B // 2)
    ratio = P.step_log_ratio(control(), behaviour, dw, dt).t()
    loss, info = P.preference_loss(ratio[better], ratio[worse], chosen_mask=mask[better], rejected_mask=mask[worse])
    opt.zero_grad()
    loss.backward()
    opt.step()
    assert torch.isfinite(loss) and info["chosen_rewards"].shape == (B // 2,) and float(opt.grad_norm) > 0.0


@gpu
@pytest.mark.parametrize("name", ["cfg1_dw_dis_lv", "gmm50_pis_headline"])
def test_documented_steps_on_stored_trajectories(name):
    """The documentation's example: the control called along the paths is the one that drove them, and its gradients are those of the formulas."""
    prob = problems.build(problems.baseline_spec(name), device="cuda:0")  # (its own grid: in 20 steps some paths of the double well reach |x| = 4000, where
    torch.manual_seed(3)                                                  # the k3 term of a moved control overflows in the formula itself)
    x0 = prob.prior.sample((128,))

    def control(xs):
        return torch.stack([prob.ctrl(t, x) for t, x in zip(prob.ts, xs)])

    opt = AdamW(prob.ctrl.parameters(), lr=1e-3, weight_decay=0.0, max_grad_norm=1.0)
    dt = prob.ts.diff()
    noise = torch.randn(dt.numel(), *x0.shape, device="cuda")
    res = prob.eval(x0, compute_weights=True, return_traj=True, noise=noise)
    dw = noise * dt.sqrt()[:, None, None]
    weight = res.weights.squeeze(-1)
    advantage = (weight - weight.mean()) / weight.std()
    with torch.no_grad():
        v = control(res.xs[:-1])
        # x + (drift + diff u) dt + diff dW; three layers of 64 products in fp32 are right to 1e-4 of their size, 1e-3 is asked for
        for k, (t, x) in enumerate(zip(prob.ts, res.xs[:-1])):
            diff = prob.sde.diff(t, x)
            want = x + (prob.sde.drift(t, x) + diff * v[k]) * dt[k] + diff * dw[k]
            tol = 1e-3 * diff * dt[k] * (1 + v[k].abs()) + 16 * H * (x.abs() + want.abs() + 1)
            assert ((res.xs[k + 1] - want).abs() <= tol).all()
    params = [p for p in prob.ctrl.parameters() if p.requires_grad]
    for k in range(3):
        u = control(res.xs[:-1])
        ratio = P.step_log_ratio(u, v, dw, dt).t()
        assert k or not ratio.any()
        loss, info = P.policy_loss(ratio, advantage, ref_log_prob=torch.zeros_like(ratio), kl_coef=0.05)
        opt.zero_grad()
        loss.backward()
        e = control(res.xs[:-1]) - v
        r = (e * dw - 0.5 * dt[:, None, None] * e * e).sum(-1).t()
        want = torch.maximum(-advantage[:, None] * r.exp(), -advantage[:, None] * r.exp().clamp(0.8, 1.2)) + 0.05 * (torch.exp(-r) - 1 + r)
        for p, g in zip(params, torch.autograd.grad(want.mean(), params, allow_unused=True)):
            assert (p.grad is None) == (g is None)
            if g is not None:  # (both sides sum 12 800 rows' contributions in fp32, in different orders)
                assert (p.grad - g).abs().max() <= 2e-5 * g.abs().max() + 1e-7
        opt.step()
        assert torch.isfinite(loss) and float(info["n_valid"]) == ratio.numel()


# -- refusals ----------------------------------------------------------------------------------------------------------------------------------
def test_constructor_refuses():
    p = [torch.nn.Parameter(torch.zeros(3))]
    for kw in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1.0), dict(weight_decay=-1.0), dict(state_bits=16),
               dict(max_grad_norm=0.0), dict(lr=torch.tensor(0.1))):
        with pytest.raises(ValueError):
            AdamW(p, **kw)
    p[0].grad = torch.zeros(3)
    with pytest.raises(RuntimeError, match="HIP device only"):
        AdamW(p).step()


def test_a_refused_group_is_not_added():
    p, q = torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.zeros(3))
    opt = AdamW([p])
    for bad in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0)):
        with pytest.raises(ValueError):
            opt.add_param_group({"params": [q], **bad})
        assert len(opt.param_groups) == 1
    opt.add_param_group({"params": [q], "lr": 0.1})
    assert len(opt.param_groups) == 2


def test_c_entry_refuses_bad_arguments():
    lib = L.load()
    head = lambda **k: L.ADAMW.pack(k.get("clip", 1.0), 0, 0, 1, k.get("groups", 1))  # noqa: E731
    group = lambda **k: L.ADAMW_GROUP.pack(k.get("lr", 0.1), k.get("b1", 0.9), k.get("b2", 0.99), k.get("eps", 0.0), k.get("wd", 0.0), 0, k.get("n", 1),  # noqa: E731
                                           k.get("dtype", 0), k.get("bits", 32), 0)
    table = lambda *row: np.array(row or (64, 64, 64, 64, 0, 0, 64, 5, 0), dtype=np.int64)  # noqa: E731
    call = lambda h, g, t=table(), s=64: lib.sdeh_adamw_step(h, g, None if t is None else t.ctypes.data, s, None)  # noqa: E731
    for bad in (dict(clip=-1.0), dict(clip=math.nan), dict(groups=-1)):
        assert call(head(**bad), group()) == -1, bad
    for bad in (dict(lr=-1.0), dict(lr=math.nan), dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0), dict(wd=-1.0), dict(n=-1), dict(dtype=3), dict(dtype=-1),
                dict(bits=16), dict(bits=8)):
        assert call(head(), group(**bad)) == -1, bad
    for row in ((0, 64, 64, 64, 0, 0, 64, 5, 0), (64, 0, 64, 64, 0, 0, 64, 5, 0), (64, 64, 64, 64, 0, 0, 0, 5, 0), (64, 64, 64, 64, 0, 0, 64, -5, 0),
                (64, 64, 64, 64, 0, 0, 64, 5, -1)):
        assert call(head(), group(), table(*row)) == -1, row
    assert call(None, group()) == call(head(), None) == call(head(), group(), None) == call(head(), group(), s=None) == call(head(), group(), s=72) == -1
    assert call(head(), group(), table(64, 64, 64, 64, 0, 0, 64, 1 << 60, 0)) == -2
    assert call(head(groups=0), group()) == call(head(), group(n=0), None) == 0
    assert lib.sdeh_adamw_moments(64, 64, 64, None, 1, 64, 64, None) == lib.sdeh_adamw_moments(66, 64, 64, 64, 1, 64, 64, None) == -1
    assert lib.sdeh_adamw_moments(None, None, None, None, 0, None, None, None) == 0


@gpu
def test_step_refuses():
    q = torch.nn.Parameter(torch.zeros(5, device="cuda"))
    q.grad = torch.ones_like(q)
    with pytest.warns(UserWarning, match="duplicate"), pytest.raises(ValueError, match="twice"):
        AdamW([q, q]).step()
    p = torch.nn.Parameter(torch.zeros(4, 6, device="cuda"))
    opt = AdamW([p])
    p.grad = torch.ones_like(p)
    opt.step()
    with pytest.raises(ValueError, match="ok must be"):
        opt.step(ok=torch.ones(1, dtype=torch.bool))
    p.data = torch.zeros(6, 4, device="cuda").t()
    with pytest.raises(RuntimeError, match="contiguous"):
        opt.step()
    p.grad = None
    p.data = torch.zeros(5, 6, device="cuda")
    p.grad = torch.ones_like(p)
    with pytest.raises(RuntimeError, match="30 entries"):
        opt.step()
    with pytest.raises(L.SdehUnsupported):
        q = torch.nn.Parameter(torch.zeros(3, device="cuda", dtype=torch.float64))
        q.grad = torch.ones_like(q)
        AdamW([q]).step()
    q = torch.nn.Parameter(torch.zeros(4, 6, device="cuda"))  # a gradient of another layout is laid out like its parameter
    q.grad = torch.arange(24.0, device="cuda").view(6, 4).t()
    AdamW([q], lr=1.0, weight_decay=0.0).step()
    assert float(q[0, 0]) == 0.0 and bool((q.view(-1)[1:] + 1.0).abs().max() < 1e-3)
