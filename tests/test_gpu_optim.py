"""Gradient norm, clipping and ClippedAdamW on the GPU against the formulas in 64 bits.

Tolerances.  E = 2^-24 is half a step of float32, relative.  The norms' sums run in fp64, so a norm is off by its one
rounding to float32 and the conversion of a double of some 1e-13 relative: 1.01 E.  A clipped value is compared bit for
bit with the product by the factor made of the returned norm.  Those of AdamW are written beside `_reference`.
"""
import copy
import math

import pytest
import torch

from torch.optim.optimizer import register_optimizer_step_post_hook

import pde_amd

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
E = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
INF = math.inf

# empty tensors first, last and between; one element; around a unit of 4096 and around a thread's 4 and 8 elements
SIZES = [0, 1, 4096, 4095, 0, 4097, 3, 8, 65536 + 5, 2, 131072, 12289, 0]


def _rand(shape, dtype=F32, seed=0, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _packed(sizes, dtype, seed=0):
    """tensors side by side in one buffer, the first one element off its start, with a guard value at either end"""
    flat = torch.cat([torch.full((1,), 7.0, device=DEV, dtype=dtype), _rand(sum(sizes), dtype, seed), torch.full((1,), 7.0, device=DEV, dtype=dtype)])
    out, at = [], 1
    for n in sizes:
        out.append(flat[at:at + n])
        at += n
    return flat, out


def _exact_norm(ts, p):
    each = torch.stack([torch.linalg.vector_norm(t.double().reshape(-1), p) if t.numel() else torch.zeros((), dtype=torch.float64, device=t.device) for t in ts])
    return torch.linalg.vector_norm(each, p), each


def _near(got, want, tol=1.01 * E):
    assert got.dtype == F32 and got.shape == want.shape
    assert bool(((got.double() - want).abs() <= tol * want.abs()).all()), (got, want)


def _leaves(grads):
    out = []
    for g in grads:
        p = torch.zeros_like(g).requires_grad_(True)
        p.grad = g
        out.append(p)
    return out


@pytest.mark.parametrize("p", [1, 2, INF])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_norm(dtype, p):
    _, ts = _packed(SIZES, dtype)
    want, each = _exact_norm(ts, p)
    total, got = pde_amd.get_total_norm(ts, p, per_tensor=True)
    _near(total, want)
    _near(got, each)
    _near(pde_amd.get_total_norm(ts, p), want)
    for t, w in zip(ts, each):
        _near(pde_amd.get_total_norm(t, p), w)
    assert torch.equal(pde_amd.get_total_norm(iter(ts), p), pde_amd.get_total_norm(ts, p))      # the same bits at every call


@pytest.mark.parametrize("count", [191, 192, 193, 500])
def test_norm_of_lists_longer_than_a_launch(count):
    ts = [_rand(1 + (i * 37) % 300, (F32, BF16, F16)[i % 3], seed=i, scale=2.0 ** (i % 7)) for i in range(count)]
    for p in (1, 2, INF):
        want, each = _exact_norm(ts, p)
        total, got = pde_amd.get_total_norm(ts, p, per_tensor=True)
        _near(total, want)
        _near(got, each)
        _near(pde_amd.get_total_norm(ts, p), want)


def test_norm_over_many_units_per_workgroup():
    # 9.6e6 elements = 2344 units: two for most workgroups, so that tensors begin and end inside a workgroup's run
    sizes = [1000003, 5, 3000001, 4096, 0, 8192, 5555555, 12287, 1]
    _, ts = _packed(sizes, F32, seed=3)
    want, each = _exact_norm(ts, 2)
    total, got = pde_amd.get_total_norm(ts, per_tensor=True)
    _near(total, want)
    _near(got, each)
    _near(pde_amd.get_total_norm(ts), want)


def test_norm_range():
    """squares of the largest and the smallest float32 values stay inside the sum's range"""
    big = torch.full((5,), 1e38, device=DEV)
    _near(pde_amd.get_total_norm([big]), torch.linalg.vector_norm(big.double()))
    tiny = torch.full((4097,), 1e-42, device=DEV)      # subnormal; the norm is 6.4e-41
    got, want = pde_amd.get_total_norm([tiny]).double(), torch.linalg.vector_norm(tiny.double())
    assert abs(float(got - want)) <= 2.0 ** -150      # half a step of the subnormals
    assert float(pde_amd.get_total_norm([torch.full((2,), 3e38, device=DEV)])) == INF      # beyond float32
    assert float(pde_amd.get_total_norm([torch.zeros(9, device=DEV), -torch.zeros(3, device=DEV)])) == 0.0


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("p", [1, 2, INF])
def test_norm_of_values_that_are_not_finite(dtype, p):
    for at in (0, 5000, 70000):
        _, ts = _packed([4097, 70001, 3], dtype, seed=1)
        ts[1][at] = -INF
        total, each = pde_amd.get_total_norm(ts, p, per_tensor=True)
        assert float(total) == INF and float(each[1]) == INF and math.isfinite(float(each[0])) and math.isfinite(float(each[2]))
        ts[1][at] = math.nan
        ts[0][1] = INF
        total, each = pde_amd.get_total_norm(ts, p, per_tensor=True)
        assert math.isnan(float(total)) and math.isnan(float(each[1])) and float(each[0]) == INF
        assert math.isnan(float(pde_amd.get_total_norm(ts, p)))
        with pytest.raises(RuntimeError, match="not finite"):
            pde_amd.get_total_norm(ts, p, error_if_nonfinite=True)


def test_norm_of_other_layouts():
    x = _rand((33, 70, 5), seed=2)
    for t in (x.permute(2, 0, 1), x[:, ::3], x[1:, 2:, :3], torch.randn((), device=DEV), x[:1].expand(8, 70, 5), x.to(memory_format=torch.contiguous_format)):
        _near(pde_amd.get_total_norm([t]), torch.linalg.vector_norm(t.double()))


def test_norm_beyond_32_bit_offsets():
    n = (1 << 31) + 4099
    t = torch.zeros(n, dtype=BF16, device=DEV)
    for i, v in ((0, 3.0), ((1 << 31) - 1, -4.0), (1 << 31, 12.0), (n - 1, 84.0)):
        t[i] = v
    assert float(pde_amd.get_total_norm([t])) == 85.0      # 9 + 16 + 144 + 7056 = 85^2
    assert float(pde_amd.get_total_norm([t], INF)) == 84.0
    p = _leaves([t])
    assert float(pde_amd.clip_grad_norm_(p, 42.5)) == 85.0
    c = torch.tensor(42.5) / (torch.tensor(85.0) + 1e-6)      # float32
    got = torch.stack([t[0], t[(1 << 31) - 1], t[1 << 31], t[n - 1]]).cpu()
    assert torch.equal(got, (torch.tensor([3.0, -4.0, 12.0, 84.0]) * c).to(BF16))


def _clipped(g, total, max_norm):
    """what clipping makes of g, given the float32 norm: the factor and the product in float32, one rounding"""
    c = (torch.full_like(total, max_norm) / (total + 1e-6)).clamp(max=1.0)      # scalar / tensor would round the reciprocal first
    return (g.float() * c).to(g.dtype)


@pytest.mark.parametrize("max_norm", [0.0, 1e-3, 1.0, 100.0])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_clip(dtype, max_norm):
    flat, ts = _packed(SIZES, dtype, seed=4)
    before = flat.clone()
    params = _leaves(ts)
    params.insert(3, torch.zeros(5, device=DEV, requires_grad=True))      # no gradient
    versions = [t._version for t in ts]
    total = pde_amd.clip_grad_norm_(params, max_norm)
    _near(total, _exact_norm([before[1:-1]], 2)[0])
    assert torch.equal(flat[1:-1], _clipped(before[1:-1], total, max_norm))
    assert float(flat[0]) == 7.0 and float(flat[-1]) == 7.0      # the neighbours
    assert all(t._version > v for t, v in zip(ts, versions))     # autograd is told
    assert params[3].grad is None


@pytest.mark.parametrize("p", [1, INF])
def test_clip_by_other_norms(p):
    flat, ts = _packed(SIZES, F32, seed=5)
    before = flat[1:-1].clone()
    total = pde_amd.clip_grad_norm_(_leaves(ts), 0.5, p)
    _near(total, _exact_norm([before], p)[0])
    assert torch.equal(flat[1:-1], _clipped(before, total, 0.5))


def test_clip_above_the_norm_changes_nothing():
    flat, ts = _packed(SIZES, F32, seed=6)
    flat[3], flat[4] = -0.0, 1e-42
    before = flat.clone()
    pde_amd.clip_grad_norm_(_leaves(ts), 1e6)
    assert torch.equal(flat.view(torch.int32), before.view(torch.int32))
    pde_amd.clip_grad_norm_(_leaves(ts), INF)
    assert torch.equal(flat.view(torch.int32), before.view(torch.int32))


def test_clip_of_a_norm_that_is_not_finite():
    _, ts = _packed([70000, 3], F32, seed=7)
    ts[0][66000] = INF
    before = [t.clone() for t in ts]
    with pytest.raises(RuntimeError, match="not finite"):
        pde_amd.clip_grad_norm_(_leaves(ts), 1.0, error_if_nonfinite=True)
    assert all(torch.equal(a, b) for a, b in zip(ts, before))      # raised before anything was scaled
    assert float(pde_amd.clip_grad_norm_(_leaves(ts), 1.0)) == INF      # factor 0, as in torch: inf * 0 is NaN
    assert int(torch.isnan(ts[0]).sum()) == 1 and float(ts[0].nan_to_num().abs().max()) == 0.0 and float(ts[1].abs().max()) == 0.0
    ts[1][0] = math.nan
    assert math.isnan(float(pde_amd.clip_grad_norm_(_leaves(ts), 1.0)))
    assert all(bool(torch.isnan(t).all()) for t in ts)


def test_clip_finite_with_error_check():
    _, ts = _packed([70000, 3], F32, seed=8)
    want = [t.clone() for t in ts]
    total = pde_amd.clip_grad_norm_(_leaves(ts), 1.0, error_if_nonfinite=True)
    other = pde_amd.clip_grad_norm_(_leaves(want), 1.0)
    assert torch.equal(total, other) and all(torch.equal(a, b) for a, b in zip(ts, want))


def test_clip_with_given_norm():
    for make in (lambda x: torch.tensor(x, device=DEV), lambda x: torch.tensor([x], dtype=torch.float64, device=DEV), lambda x: torch.tensor(x)):
        flat, ts = _packed(SIZES, BF16, seed=9)
        before = flat[1:-1].clone()
        pde_amd.clip_grads_with_norm_(_leaves(ts), 1.0, make(4.0))
        assert torch.equal(flat[1:-1], _clipped(before, torch.tensor(4.0, device=DEV), 1.0))
    with pytest.raises(ValueError, match="one value"):
        pde_amd.clip_grads_with_norm_(_leaves(ts), 1.0, torch.ones(2, device=DEV))
    with pytest.raises(TypeError, match="floating point"):
        pde_amd.clip_grads_with_norm_(_leaves(ts), 1.0, torch.ones((), dtype=torch.int64, device=DEV))


def test_clip_with_a_norm_that_lies_in_a_gradient():
    g = _rand(70000, seed=11)
    g[123] = 5.0
    before = g.clone()
    pde_amd.clip_grads_with_norm_(_leaves([g]), 1.0, g[123])
    assert torch.equal(g, _clipped(before, before[123], 1.0))


def test_clip_in_other_layouts_and_long_lists():
    grads = [_rand((7, 11, 3), seed=1).permute(2, 0, 1), _rand((4, 5, 6, 7), seed=2).to(memory_format=torch.channels_last), _rand((), seed=3)]
    grads += [_rand(1 + i % 50, (F32, BF16)[i % 2], seed=i) for i in range(400)]
    before = [g.clone() for g in grads]
    total = pde_amd.clip_grad_norm_(_leaves(grads), 2.0)
    _near(total, _exact_norm(before, 2)[0])
    for g, b in zip(grads, before):
        assert torch.equal(g, _clipped(b, total, 2.0))


# ----------------------------------------------------------------------------------------------------------------------
# AdamW
# ----------------------------------------------------------------------------------------------------------------------
def _reference(w, g, m, v, t, c=1.0, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2):
    """One step in 64 bits from float32 inputs: (w, m, v) and the bounds of a float32 computation's distance from them.

    Counted in E, relative, to first order, with a little over for products of errors and the constants' own roundings:
      g' = c g: 4 (norm, + 1e-6, quotient, product; the norm's own error within the first)
      m: its two products carry 2 (constant, product) and 4 + 2, the sum 1        -> 8 (b1 |m| + (1 - b1) |g'|)
      v: likewise with g' squared: 2 * 4 + 1 + 2, the sum 1                       -> 12 v, a sum of positive terms
      denominator: half of v's 12, square root 1, bias factor 2, + eps 2          -> 11
      update u = s m / d: s 1, quotient 1, product 1, d 11, m as above            -> 14 |u| + 8 s (b1 |m| + (1 - b1) |g'|) / d
      w: decay constant 1, product 1, final difference 1 (of |w| + |u|)           -> 3 |w| + 15 |u| + ...
    """
    w, g, m, v = (x.double() for x in (w, g, m, v))
    b1, b2 = betas
    g = c * g
    size = b1 * m.abs() + (1 - b1) * g.abs()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    s, d = lr / (1 - b1 ** t), v.sqrt() / math.sqrt(1 - b2 ** t) + eps
    u = s * m / d
    new = (1 - lr * weight_decay) * w - u
    floor = 2.0 ** -149      # a step of the subnormals, for sums that end there
    return (new, m, v), (E * (3 * w.abs() + 15 * u.abs() + 8 * s * size / d) + floor, 8 * E * size + floor, 12 * E * v + floor)


def _within(got, want, tol, what):
    worst = float(((got.double() - want).abs() / tol).max()) if got.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.2f} times the bound"


def _optimizer(sizes, dtype, seed, state_step=0, **kw):
    """(optimizer, parameters) with gradients and, where state_step > 0, the state of a run that is under way"""
    params = []
    for i, n in enumerate(sizes):
        p = _rand(n, dtype, seed + i, 0.1).requires_grad_(True)
        p.grad = _rand(n, dtype, seed + 100 + i, 10.0 ** (-(i % 4)))
        params.append(p)
    opt = pde_amd.ClippedAdamW(params, **kw)
    if state_step:
        for i, p in enumerate(params):
            opt.state[p] = dict(step=torch.tensor(float(state_step), device=DEV), exp_avg=_rand(sizes[i], F32, seed + 200 + i, 0.1),
                                exp_avg_sq=_rand(sizes[i], F32, seed + 300 + i, 0.3).square())
            if dtype is BF16:
                opt.state[p]["master"] = _rand(sizes[i], F32, seed + i, 0.1)
    return opt, params


def _snapshot(opt, params):
    """per parameter (value in float32, exp_avg, exp_avg_sq, step) before a step"""
    out = []
    for p in params:
        s = opt.state.get(p) or {}
        z = torch.zeros_like(p, dtype=F32, requires_grad=False)
        w = s["master"] if "master" in s else p.detach().float()
        out.append([x.clone() for x in (w, s.get("exp_avg", z), s.get("exp_avg_sq", z))] + [float(s.get("step", 0.0))])
    return out


def _check_step(opt, params, before, c=1.0, **kw):
    for p, (w, m, v, t) in zip(params, before):
        s = opt.state[p]
        assert float(s["step"]) == t + 1
        want, tol = _reference(w, p.grad, m, v, t + 1, c, **kw)
        _within(s["exp_avg"], want[1], tol[1], "exp_avg")
        _within(s["exp_avg_sq"], want[2], tol[2], "exp_avg_sq")
        if p.dtype is BF16:
            _within(s["master"], want[0], tol[0], "master")
            assert torch.equal(p.detach(), s["master"].to(BF16))      # one rounding, to nearest even
        else:
            _within(p.detach(), want[0], tol[0], "parameter")


@pytest.mark.parametrize("state_step", [0, 1, 1000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_adamw_step(dtype, state_step):
    kw = dict(lr=3e-3, betas=(0.85, 0.99), eps=1e-7, weight_decay=0.05)
    opt, params = _optimizer([n for n in SIZES if n], dtype, seed=10, state_step=state_step, **kw)
    for _ in range(3):
        before = _snapshot(opt, params)
        versions = [p._version for p in params]
        opt.step()
        _check_step(opt, params, before, **kw)
        assert opt.total_norm is None and all(p._version > v for p, v in zip(params, versions))
        for i, p in enumerate(params):
            p.grad = _rand(p.shape, dtype, 1000 + i, 0.01)


@pytest.mark.parametrize("max_norm", [0.0, 0.5, 1e6])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_adamw_clips(dtype, max_norm):
    opt, params = _optimizer([n for n in SIZES if n], dtype, seed=20, state_step=7, max_norm=max_norm)
    before = _snapshot(opt, params)
    grads = [p.grad.clone() for p in params]
    opt.step()
    norm = _exact_norm(grads, 2)[0]
    _near(opt.total_norm, norm)
    _check_step(opt, params, before, c=min(1.0, max_norm / (float(norm) + 1e-6)))
    assert all(torch.equal(p.grad, g) for p, g in zip(params, grads))      # gradients stay as they are


def test_adamw_equals_clip_then_step():
    """clipping inside the step, or ahead of it with the gradients written: the same bits"""
    a, pa = _optimizer([5000, 3, 70001], F32, seed=30, max_norm=0.25)
    b, pb = _optimizer([5000, 3, 70001], F32, seed=30)
    for _ in range(3):
        a.step()
        total = pde_amd.clip_grad_norm_(pb, 0.25)
        b.step()
        assert torch.equal(total, a.total_norm)
        for x, y in zip(pa, pb):
            assert torch.equal(x, y) and torch.equal(a.state[x]["exp_avg_sq"], b.state[y]["exp_avg_sq"])
            x.grad = _rand(x.shape, F32, x.numel(), 2.0)
            y.grad = x.grad.clone()


def test_adamw_unaligned_and_packed():
    sizes = [4097, 3, 1, 20001, 4096, 7]
    flats = [_packed(sizes, F32, seed=40 + i) for i in range(4)]
    (pf, ps), (gf, gs), (mf, ms), (vf, vs) = flats
    vf[1:-1].square_()
    opt = pde_amd.ClippedAdamW([p.requires_grad_(True) for p in ps], max_norm=1.0)
    for p, g, m, v in zip(ps, gs, ms, vs):
        p.grad = g
        opt.state[p] = dict(step=torch.tensor(4.0, device=DEV), exp_avg=m, exp_avg_sq=v)
    before = _snapshot(opt, ps)
    opt.step()
    _check_step(opt, ps, before, c=1.0 / (float(_exact_norm(gs, 2)[0]) + 1e-6))
    assert all(float(f[0]) == 7.0 and float(f[-1]) == 7.0 for f in (pf, gf, mf, vf))


def test_adamw_beyond_32_bit_offsets():
    n = (1 << 31) + 4099
    p = torch.zeros(n, device=DEV).requires_grad_(True)
    p.grad = torch.zeros(n, device=DEV)
    places = [0, (1 << 31) - 1, 1 << 31, n - 1]
    for i in places:
        p.grad[i] = 2.0
    opt = pde_amd.ClippedAdamW([p], lr=0.125, weight_decay=0.0, eps=0.5, max_norm=2.0)
    opt.step()
    assert float(opt.total_norm) == 4.0 and float(opt.state[p]["step"]) == 1.0
    # g' = 2 * 2 / (4 + 1e-6); first step: -lr g' / (|g'| + eps)
    c = 2.0 / (4.0 + 1e-6)
    got = torch.stack([p.detach()[i] for i in places]).double()
    want = -0.125 * (2 * c) / (2 * c + 0.5)
    assert bool(((got - want).abs() <= 40 * E * abs(want)).all())      # the bound of _reference at m = v = w = 0: 15 + 8 + 3, and some
    assert int(torch.count_nonzero(p.detach())) == 4 and int(torch.count_nonzero(opt.state[p]["exp_avg_sq"])) == 4
    del p, opt
    torch.cuda.empty_cache()


def test_adamw_long_lists_groups_and_missing_gradients():
    n = 500
    params = [_rand(1 + (i * 91) % 700, (F32, BF16)[i % 3 == 0], i, 0.1).requires_grad_(True) for i in range(n)]
    params.append(_rand(0, F32).requires_grad_(True))
    groups = [dict(params=params[0::2], lr=1e-2), dict(params=params[1::2], weight_decay=0.0, betas=(0.5, 0.9), eps=1e-4)]
    opt = pde_amd.ClippedAdamW(groups, lr=1e-3, weight_decay=0.1, max_norm=3.0)
    hyper = {}
    for g in opt.param_groups:
        for p in g["params"]:
            hyper[p] = {k: g[k] for k in ("lr", "betas", "eps", "weight_decay")}
    counts = [0] * len(params)
    for step in range(3):
        for i, p in enumerate(params):
            p.grad = None if (i + step) % 5 == 0 else _rand(p.shape, p.dtype, 7000 * (step + 1) + i)
        have = [i for i, p in enumerate(params) if p.grad is not None and p.numel()]
        before = dict(zip(have, _snapshot(opt, [params[i] for i in have])))
        idle = [(i, params[i].detach().clone(), copy.deepcopy(dict(opt.state.get(params[i], {})))) for i in range(n) if params[i].grad is None]
        opt.step()
        c = min(1.0, 3.0 / (float(_exact_norm([params[i].grad for i in have], 2)[0]) + 1e-6))
        for i in have:
            counts[i] += 1
            assert before[i][3] + 1 == counts[i]
            _check_step(opt, [params[i]], [before[i]], c, **hyper[params[i]])
        for i, value, state in idle:      # neither the value nor the state of a parameter without gradient moves
            assert torch.equal(params[i].detach(), value)
            assert all(torch.equal(opt.state[params[i]][k], v) for k, v in state.items())


def test_adamw_zero_gradients_and_extreme_values():
    p = torch.tensor([1.0, -2.0, 0.5, 3.0, 0.0], device=DEV, requires_grad=True)
    p.grad = torch.tensor([0.0, -0.0, 1e-30, 1e15, 1e-42], device=DEV)
    opt = pde_amd.ClippedAdamW([p], lr=0.1, weight_decay=0.0)
    opt.step()
    # first step: m / sqrt(v) is 1 up to eps, 0 / eps is 0, and (1e-30)^2 vanishes beside eps
    assert torch.allclose(p.detach(), torch.tensor([1.0, -2.0, 0.5, 2.9, 0.0], device=DEV), rtol=1e-6, atol=1e-12)
    p.grad = torch.full((5,), math.nan, device=DEV)
    opt.step()
    assert bool(torch.isnan(p).all())


@pytest.mark.parametrize("max_norm", [None, 1.0])
def test_adamw_skips_steps_whose_norm_is_not_finite(max_norm):
    opt, params = _optimizer([5000, 17, 300], F32, seed=50, max_norm=max_norm, skip_nonfinite=True)
    opt.step()
    good = [p.grad for p in params]
    for bad in (INF, math.nan):
        before, values = _snapshot(opt, params), [p.detach().clone() for p in params]
        params[1].grad = params[1].grad.clone()
        params[1].grad[16] = bad
        opt.step()
        assert not math.isfinite(float(opt.total_norm))
        for p, x, (w, m, v, t) in zip(params, values, before):
            s = opt.state[p]
            assert torch.equal(p.detach(), x) and torch.equal(s["exp_avg"], m) and torch.equal(s["exp_avg_sq"], v) and float(s["step"]) == t
        params[1].grad = good[1]
    before = _snapshot(opt, params)
    opt.step()
    c = 1.0 if max_norm is None else min(1.0, max_norm / (float(_exact_norm(good, 2)[0]) + 1e-6))
    _check_step(opt, params, before, c)


def test_adamw_with_given_norm():
    opt, params = _optimizer([5000, 17], F32, seed=60, max_norm=1.0)
    before = _snapshot(opt, params)
    norm = torch.tensor(8.0, device=DEV)
    opt.step(total_norm=norm)      # e.g. the norm over all ranks' shards
    assert opt.total_norm is norm
    _check_step(opt, params, before, 1.0 / (8.0 + 1e-6))
    opt.skip_nonfinite = True
    before = _snapshot(opt, params)
    opt.step(total_norm=torch.tensor(math.nan))
    assert all(float(opt.state[p]["step"]) == b[3] and torch.equal(p.detach(), b[0]) for p, b in zip(params, before))


def test_adamw_layouts():
    """parameters in other dense layouts, and gradients in another layout than their parameter's"""
    a = _rand((6, 5, 40), seed=1).permute(2, 0, 1).requires_grad_(True)
    b = _rand((3, 4, 5, 6), seed=2).to(memory_format=torch.channels_last).requires_grad_(True)
    c = _rand((64, 65), seed=3).requires_grad_(True)
    d = _rand((), seed=4).requires_grad_(True)
    a.grad, b.grad, d.grad = torch.empty_like(a).copy_(_rand(a.shape, seed=5)), _rand(b.shape, seed=6), _rand((), seed=7)
    c.grad = _rand((65, 64), seed=8).t()
    params = [a, b, c, d]
    assert a.grad.stride() == a.stride() and b.grad.stride() != b.stride()
    opt = pde_amd.ClippedAdamW(params, max_norm=0.5)
    for _ in range(2):
        before = _snapshot(opt, params)
        opt.step()
        _check_step(opt, params, before, 0.5 / (float(_exact_norm([p.grad for p in params], 2)[0]) + 1e-6))


def test_adamw_refuses_gradients_of_another_type():
    p = torch.zeros(4, device=DEV, requires_grad=True)
    p.grad = torch.eye(4, device=DEV)[0].to_sparse()
    with pytest.raises(TypeError, match="dense"):
        opt = pde_amd.ClippedAdamW([p])
        opt.step()
    with pytest.raises(ValueError, match="learning rate on the device"):
        p.grad = torch.ones(4, device=DEV)
        pde_amd.ClippedAdamW([p], lr=torch.tensor(1e-3, dtype=torch.float64, device=DEV)).step()


def test_adamw_state_dict_resumes():
    for dtype in (F32, BF16):
        a, pa = _optimizer([5000, 3, 70001], dtype, seed=70, lr=1e-2, max_norm=1.0)
        a.step()
        a.step()
        pb = [p.detach().clone().requires_grad_(True) for p in pa]
        b = pde_amd.ClippedAdamW(pb, max_norm=1.0)
        b.load_state_dict(a.state_dict())
        c = copy.deepcopy(a)      # shares nothing with a
        pc = [p for g in c.param_groups for p in g["params"]]
        for x, y, z in zip(pa, pb, pc):
            x.grad = _rand(x.shape, dtype, x.numel())
            y.grad, z.grad = x.grad.clone(), x.grad.clone()
        for opt in (a, b, c):
            opt.step()
        for x, y, z in zip(pa, pb, pc):
            assert torch.equal(x, y) and torch.equal(x, z) and x.data_ptr() != z.data_ptr()
            for k in a.state[x]:
                assert torch.equal(a.state[x][k], b.state[y][k]) and torch.equal(a.state[x][k], c.state[z][k])


def test_adamw_follows_parameters_that_move():
    """a parameter whose storage is replaced between steps, a parameter group added later, masters taken again"""
    opt, params = _optimizer([5000, 3], F32, seed=80)
    opt.step()
    old = params[0].detach()
    params[0].data = params[0].detach().clone()
    kept, before = old.clone(), _snapshot(opt, params)
    opt.step()
    _check_step(opt, params, before)
    assert torch.equal(old, kept)      # the old storage is left alone
    late = _rand(77, BF16, seed=81).requires_grad_(True)
    late.grad = _rand(77, BF16, seed=82)
    opt.add_param_group(dict(params=[late], lr=0.1))
    before = _snapshot(opt, params)
    opt.step()
    _check_step(opt, params, before)
    assert float(opt.state[late]["step"]) == 1.0
    with torch.no_grad():
        late.copy_(_rand(77, BF16, seed=83))
    opt.reload_masters()
    before = _snapshot(opt, [late])
    assert torch.equal(before[0][0], late.detach().float())
    opt.step()
    _check_step(opt, [late], before, lr=0.1)


def test_adamw_parameters_that_change_otherwise():
    """a parameter that leaves the device or changes its type or shape between steps is found before anything is launched"""
    def change(p, other):
        p.data = other
        p.grad = torch.zeros(other.shape, dtype=other.dtype, device=other.device)

    for other, error, match in ((torch.zeros(50), ValueError, "one device|on its device"), (torch.zeros(50, dtype=F16, device=DEV), TypeError, "float32 or bfloat16"),
                                (torch.zeros(50, dtype=BF16, device=DEV), ValueError, "must hold"), (torch.zeros(51, device=DEV), ValueError, "laid out"),
                                (torch.zeros(100, device=DEV)[::2], ValueError, "dense")):
        opt, params = _optimizer([7, 50], F32, seed=86)
        opt.step()
        before, value = _snapshot(opt, params), params[0].detach().clone()
        params[1].grad = None
        change(params[1], other)
        for _ in range(2):
            with pytest.raises(error, match=match):
                opt.step()
        assert torch.equal(params[0].detach(), value) and float(opt.state[params[0]]["step"]) == before[0][3]


def test_adamw_parameters_that_come_to_share_memory():
    opt, params = _optimizer([50, 50], F32, seed=87)
    opt.step()
    own, shared = params[1].detach(), params[0].detach()
    params[1].data = shared
    for _ in range(2):
        with pytest.raises(ValueError, match="share memory"):
            opt.step()
    params[1].data = own
    before = _snapshot(opt, params)
    opt.step()
    _check_step(opt, params, before)


def test_adamw_gradients_in_written_memory():
    """a gradient that is a view of a parameter's memory is refused; gradients that share memory among themselves are not"""
    flat = _rand(300, seed=98)
    p, q = flat[:100].requires_grad_(True), flat[100:200].requires_grad_(True)
    opt = pde_amd.ClippedAdamW([p, q], max_norm=1.0)
    both = _rand(120, seed=99)
    p.grad, q.grad = both[:100], both[20:]
    before = _snapshot(opt, [p, q])
    opt.step()
    norm = _exact_norm([p.grad, q.grad], 2)[0]
    _check_step(opt, [p, q], before, min(1.0, 1.0 / (float(norm) + 1e-6)))
    kept = flat.clone()
    for bad in (flat[50:150], flat[101:201], flat[:100], flat[199:299]):
        p.grad = bad
        for _ in range(2):
            with pytest.raises(ValueError, match="shares memory"):
                opt.step()
    assert torch.equal(flat, kept)
    p.grad = flat[200:]      # next to them, but apart
    opt.step()
    assert torch.equal(flat[200:], kept[200:]) and float(opt.state[p]["step"]) == 2.0


def test_adamw_takes_over_the_state_of_torch():
    pa = [_rand(n, F32, 88 + n, 0.1).requires_grad_(True) for n in (5000, 17)]
    theirs = torch.optim.AdamW(pa, lr=1e-2, weight_decay=0.1)
    for k in range(2):
        for p in pa:
            p.grad = _rand(p.shape, F32, 89 + k)
        theirs.step()
    pb = [p.detach().clone().requires_grad_(True) for p in pa]
    ours = pde_amd.ClippedAdamW(pb, max_norm=0.5)
    ours.load_state_dict(theirs.state_dict())
    for p in pb:
        p.grad = _rand(p.shape, F32, 95)
    before = _snapshot(ours, pb)
    assert [b[3] for b in before] == [2.0, 2.0] and torch.equal(before[0][1], theirs.state[pa[0]]["exp_avg"])
    ours.step()
    _check_step(ours, pb, before, 0.5 / (float(_exact_norm([p.grad for p in pb], 2)[0]) + 1e-6), lr=1e-2, weight_decay=0.1)
    other = torch.optim.AdamW(pa, amsgrad=True)
    ours.load_state_dict({**theirs.state_dict(), "param_groups": other.state_dict()["param_groups"]})
    with pytest.raises(ValueError, match="amsgrad"):
        ours.step()


def test_adamw_with_nothing_to_update():
    p = torch.zeros(3, device=DEV, requires_grad=True)
    q = torch.zeros(0, device=DEV, requires_grad=True)
    opt = pde_amd.ClippedAdamW([p, q], max_norm=1.0)
    opt.step()
    assert float(opt.total_norm) == 0.0
    q.grad = torch.zeros_like(q)
    opt.step()
    assert float(opt.total_norm) == 0.0
    p.grad = torch.ones_like(p)
    opt.step()
    assert float(opt.state[p]["step"]) == 1.0 and abs(float(opt.total_norm) - math.sqrt(3)) < 1e-6


def test_adamw_changed_settings():
    """settings of a group that change between steps"""
    opt, params = _optimizer([5000, 17], F32, seed=97)
    for kw in (dict(), dict(betas=(0.5, 0.9)), dict(eps=1e-2, lr=0.5), dict(weight_decay=0.25), dict()):
        opt.param_groups[0].update({**dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2), **kw})
        before = _snapshot(opt, params)
        opt.step()
        _check_step(opt, params, before, **kw)
    opt.param_groups[0]["betas"] = (1.5, 0.9)
    with pytest.raises(ValueError, match="betas"):
        opt.step()


def test_adamw_closure_and_scheduler():
    w = _rand((64, 64), seed=1).requires_grad_(True)
    x = _rand((8, 64), seed=2)
    opt = pde_amd.ClippedAdamW([w], lr=1e-2, max_norm=1.0)
    sched = torch.optim.lr_scheduler.StepLR(opt, step_size=1, gamma=0.5)

    def closure():
        opt.zero_grad()
        loss = (x @ w).square().mean()
        loss.backward()
        return loss

    for k in range(3):
        before = _snapshot(opt, [w])
        loss = opt.step(closure)
        assert loss.requires_grad is True or loss.grad_fn is not None
        c = min(1.0, 1.0 / (float(_exact_norm([w.grad], 2)[0]) + 1e-6))
        _check_step(opt, [w], before, c, lr=1e-2 * 0.5 ** k)
        sched.step()


def test_adamw_step_hooks():
    opt, params = _optimizer([50, 3], F32, seed=85)
    seen = []
    remove = [opt.register_step_pre_hook(lambda o, args, kwargs: seen.append(("pre", o is opt, len(o.state)))),
              opt.register_step_post_hook(lambda o, args, kwargs: seen.append(("post", o is opt, len(o.state)))),
              register_optimizer_step_post_hook(lambda o, args, kwargs: seen.append(("all", o is opt, len(o.state))))]
    before = _snapshot(opt, params)
    opt.state.clear()
    assert opt.step() is None
    for r in remove:
        r.remove()
    assert seen == [("pre", True, 0), ("post", True, 2), ("all", True, 2)]
    _check_step(opt, params, before)
    before = _snapshot(opt, params)
    opt.step()
    _check_step(opt, params, before)
    assert len(seen) == 3


# ----------------------------------------------------------------------------------------------------------------------
# graphs and streams
# ----------------------------------------------------------------------------------------------------------------------
def test_adamw_captured():
    """a captured step counts on, reads a learning rate that changes, and equals the eager one at every replay"""
    lr = torch.tensor(1e-2, device=DEV)
    a, pa = _optimizer([5000, 3, 70001], BF16, seed=90, lr=lr, max_norm=1.0)
    b, pb = _optimizer([5000, 3, 70001], BF16, seed=90, lr=lr, max_norm=1.0)
    a.step()
    b.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    norm = a.total_norm
    for k in range(4):
        lr.fill_(1e-2 / (k + 1))
        for x, y in zip(pa, pb):
            g = _rand(x.shape, BF16, 900 + k + x.numel(), 10.0 ** (k - 2))
            x.grad.copy_(g)
            y.grad.copy_(g)
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        assert torch.equal(norm, b.total_norm)
        for x, y in zip(pa, pb):
            assert torch.equal(x, y) and float(a.state[x]["step"]) == k + 2
            assert all(torch.equal(a.state[x][n], b.state[y][n]) for n in a.state[x])


def test_adamw_captured_step_outlives_its_plan():
    """a group added, settings changed and state loaded after a capture: the graph goes on with the parameters, the settings
    and the (loaded) state it was captured with"""
    opt, params = _optimizer([5000, 17], F32, seed=190, max_norm=1.0, lr=torch.tensor(1e-3, device=DEV))
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    late = _rand(70001, F32, seed=191).requires_grad_(True)
    late.grad = _rand(70001, F32, seed=192)
    opt.add_param_group(dict(params=[late], lr=0.1))
    opt.param_groups[0].update(betas=(0.5, 0.5), lr=7.0)
    opt.step()
    saved = copy.deepcopy(opt.state_dict())
    opt.step()
    opt.load_state_dict(saved)
    opt.step()
    filler = [torch.full((4096,), math.nan, device=DEV) for _ in range(64)]      # takes whatever memory was given back
    for _ in range(3):
        before, other = _snapshot(opt, params), late.detach().clone()
        graph.replay()
        torch.cuda.synchronize()
        _check_step(opt, params, before, min(1.0, 1.0 / (float(_exact_norm([p.grad for p in params], 2)[0]) + 1e-6)))
        assert torch.equal(late.detach(), other)
    del filler


def test_first_step_cannot_be_captured():
    opt, params = _optimizer([50], F32, seed=91)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="run one step before"):
        with torch.cuda.graph(graph):
            opt.step()
    before = _snapshot(opt, params)
    opt.step()
    _check_step(opt, params, before)


def test_clip_and_norm_captured():
    _, ts = _packed([5000, 3, 70001], F32, seed=92)
    params = _leaves(ts)
    src = [t.clone() for t in ts]
    pde_amd.clip_grad_norm_(params, 1.0)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        total = pde_amd.clip_grad_norm_(params, 1.0)
    with torch.cuda.graph(other):      # a second graph, replayed in between
        norms = pde_amd.get_total_norm(src, per_tensor=True)
    for k in range(3):
        for t, s in zip(ts, src):
            s.copy_(_rand(s.shape, F32, 920 + k + s.numel(), 3.0 ** k))
            t.copy_(s)
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        want = pde_amd.get_total_norm(src, per_tensor=True)
        assert torch.equal(total, want[0]) and torch.equal(norms[0], want[0]) and torch.equal(norms[1], want[1])
        for t, s in zip(ts, src):
            assert torch.equal(t, _clipped(s, total, 1.0))


def test_calls_on_two_streams_at_once():
    sets = [[_rand(n, F32, 930 + 10 * k + i) for i, n in enumerate([70001, 5, 300000])] for k in range(2)]
    kept = [[t.clone() for t in ts] for ts in sets]
    opts = [_optimizer([70001, 5, 300000], F32, seed=950 + 10 * k, max_norm=1.0) for k in range(2)]
    befores = [_snapshot(o, p) for o, p in opts]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    totals = [None, None]
    for k, s in enumerate(streams):
        with torch.cuda.stream(s):
            totals[k] = pde_amd.clip_grad_norm_(_leaves(sets[k]), 1.0)
            opts[k][0].step()
    torch.cuda.synchronize()
    for k in range(2):
        _near(totals[k], _exact_norm(kept[k], 2)[0])
        assert all(torch.equal(a, _clipped(b, totals[k], 1.0)) for a, b in zip(sets[k], kept[k]))
        opt, params = opts[k]
        _check_step(opt, params, befores[k], min(1.0, 1.0 / (float(_exact_norm([p.grad for p in params], 2)[0]) + 1e-6)))


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs a second GPU")
def test_tensors_on_another_device_than_the_current_one():
    other = torch.device("cuda:1")
    t = torch.randn(70001, device=other)
    p = torch.zeros_like(t).requires_grad_(True)
    p.grad = t
    with torch.cuda.device(0):
        _near(pde_amd.get_total_norm([t]), torch.linalg.vector_norm(t.double()))
        opt = pde_amd.ClippedAdamW([p], max_norm=1.0)
        opt.step()
        assert p.device == other and float(opt.state[p]["step"]) == 1.0
        with pytest.raises(ValueError, match="one device"):
            pde_amd.get_total_norm([t, torch.zeros(3, device="cuda:0")])


# ----------------------------------------------------------------------------------------------------------------------
# together: a loss of this package, its backward pass, the clipped update
# ----------------------------------------------------------------------------------------------------------------------
def _surrogate(seed):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Conv2d(3, 9, 3, padding=1), torch.nn.Tanh(), torch.nn.Conv2d(9, 15, 3, padding=1)).to(DEV)


def test_physics_training_steps():
    model = _surrogate(1)
    params = list(model.parameters())
    fn = pde_amd.TaylorGreen2DPDELoss(nx=32, ny=16, dt=0.05).to(DEV)
    opt = pde_amd.ClippedAdamW([dict(params=params[:2]), dict(params=params[2:], weight_decay=0.0)], lr=2e-3, max_norm=0.1)
    x = _rand((2, 3, 16, 32), seed=2)
    nu = torch.tensor([0.02, 0.05], device=DEV)
    for k in range(3):
        opt.zero_grad()
        out = model(x).reshape(2, 3, 5, 16, 32)
        total, _ = fn(out[:, 0], out[:, 1], out[:, 2], nu=nu)
        total.backward()
        before = _snapshot(opt, params)
        norm = _exact_norm([p.grad for p in params], 2)[0]
        opt.step()
        _near(opt.total_norm, norm)
        c = min(1.0, 0.1 / (float(norm) + 1e-6))
        _check_step(opt, params[:2], before[:2], c, lr=2e-3)
        _check_step(opt, params[2:], before[2:], c, lr=2e-3, weight_decay=0.0)


def test_norm_over_shards():
    """gradients in shards: squares added up by the packed reduction, the norm handed to clipping and update"""
    from pde_amd import dist
    shards = [[_rand(5001, seed=1), _rand(3, seed=2)], [_rand(70001, seed=3)]]
    squares = sum(dist.reduce_scalars({"n": pde_amd.get_total_norm(g) ** 2}, "sum")["n"] for g in shards)
    norm = squares.double().sqrt()
    want = _exact_norm(shards[0] + shards[1], 2)[0]
    assert abs(float(norm) / float(want) - 1) < 4 * E      # two norms and their squares
    before = [t.clone() for t in shards[1]]
    pde_amd.clip_grads_with_norm_(_leaves(shards[1]), 1.0, norm)
    assert torch.equal(shards[1][0], _clipped(before[0], norm.float(), 1.0))
    opt = pde_amd.ClippedAdamW(_leaves(shards[0]), max_norm=1.0)
    params = opt.param_groups[0]["params"]
    before = _snapshot(opt, params)
    opt.step(total_norm=norm)
    _check_step(opt, params, before, 1.0 / (float(norm) + 1e-6))


def test_captured_loss_step_feeds_the_update():
    """loss_fn.capture's gradients go through the model's backward pass into a clipped update; the per-field gradient norms
    come from the captured buffers"""
    model = _surrogate(3)
    params = list(model.parameters())
    fn = pde_amd.TaylorGreen2DPDELoss(nx=32, ny=16, dt=0.05).to(DEV)
    x = _rand((2, 3, 16, 32), seed=4)
    nu = torch.tensor([0.02, 0.05], device=DEV)
    fields = [torch.zeros(2, 5, 16, 32, device=DEV, requires_grad=True) for _ in range(3)]
    step = fn.capture(*fields, nu=nu)
    opt = pde_amd.ClippedAdamW(params, lr=1e-3, max_norm=0.1)
    for k in range(3):
        opt.zero_grad()
        out = model(x).reshape(2, 3, 5, 16, 32)
        with torch.no_grad():
            for f, o in zip(fields, out.unbind(1)):
                f.copy_(o)
        step()
        norm, each = pde_amd.get_total_norm(step.grads, per_tensor=True)
        want, want_each = _exact_norm(step.grads, 2)
        _near(norm, want)
        _near(each, want_each)
        out.backward(gradient=torch.stack(list(step.grads), 1))
        direct, _ = fn(*[o.detach().requires_grad_(True) for o in out.unbind(1)], nu=nu)
        assert torch.equal(direct.detach(), step.total)
        before = _snapshot(opt, params)
        opt.step()
        _check_step(opt, params, before, min(1.0, 0.1 / (float(_exact_norm([p.grad for p in params], 2)[0]) + 1e-6)), lr=1e-3)


def test_adamw_settings_that_it_has_not_are_refused_at_every_step():
    for bad in (dict(amsgrad=True), dict(maximize=True), dict(decoupled_weight_decay=False)):
        opt, params = _optimizer([50, 3], F32, seed=200)
        opt.step()
        before = _snapshot(opt, params)
        opt.param_groups[0].update(bad)
        for _ in range(2):
            with pytest.raises(ValueError, match="ClippedAdamW has no"):
                opt.step()
        assert all(torch.equal(p.detach(), b[0]) and float(opt.state[p]["step"]) == b[3] for p, b in zip(params, before))
        opt.param_groups[0].update(amsgrad=False, maximize=False, decoupled_weight_decay=True)
        opt.step()
        _check_step(opt, params, before)


@pytest.mark.parametrize("drop", ["group", "state", "optimizer"])
def test_adamw_description_stays_for_steps_on_other_streams(drop):
    """described on one stream, a step queued on another, the description dropped: its memory is not handed on before the
    step has run"""
    opt, params = _optimizer([5000, 3, 70001], F32, seed=230, max_norm=1.0)
    side, main = torch.cuda.Stream(), torch.cuda.current_stream()
    decoy = torch.zeros(1 << 20, device=DEV)
    late = _rand(5, F32, seed=231).requires_grad_(True)
    late.grad = _rand(5, F32, seed=232)
    busy = _rand((8192, 8192), seed=233)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        opt.step()
    main.wait_stream(side)
    saved = copy.deepcopy(opt.state_dict())
    before, states = _snapshot(opt, params), [opt.state[p] for p in params]
    torch.cuda.synchronize()
    for _ in range(4):
        busy @ busy      # some 30 ms ahead of the step
    opt.step()
    if drop == "group":
        opt.add_param_group(dict(params=[late]))
    elif drop == "state":
        opt.load_state_dict(saved)
    else:
        del opt
    with torch.cuda.stream(side):      # does not wait for the step
        blocks = [torch.full((64,), decoy.data_ptr(), dtype=torch.int64, device=DEV) for _ in range(64)]
    torch.cuda.synchronize()
    assert int(torch.count_nonzero(decoy)) == 0 and all(bool((b == decoy.data_ptr()).all()) for b in blocks)
    c = min(1.0, 1.0 / (float(_exact_norm([p.grad for p in params], 2)[0]) + 1e-6))
    for p, (w, m, v, t), state in zip(params, before, states):
        want, tol = _reference(w, p.grad, m, v, t + 1, c)
        assert float(state["step"]) == t + 1
        for got, x, bound, what in ((p.detach(), want[0], tol[0], "parameter"), (state["exp_avg"], want[1], tol[1], "exp_avg"),
                                    (state["exp_avg_sq"], want[2], tol[2], "exp_avg_sq")):
            _within(got, x, bound, what)


@pytest.mark.parametrize("what", ["betas", "rate tensor", "parameters"])
def test_adamw_memory_does_not_grow(what):
    """settings, a learning rate's tensor and parameters' memory that change at every step"""
    opt, params = _optimizer([5000, 3, 70001], F32, seed=210, max_norm=1.0, lr=torch.tensor(1e-3, device=DEV))
    used = []
    for k in range(40):
        group, kw = opt.param_groups[0], {}
        if what == "betas":
            group["betas"] = kw["betas"] = (0.95 - 0.001 * k, 0.999 - 0.001 * k)
        elif what == "rate tensor":
            kw["lr"] = 1e-3 / (1 + k)
            group["lr"] = torch.tensor(kw["lr"], device=DEV)
        else:
            for p in params:
                p.data = p.detach().clone()
        before = _snapshot(opt, params)
        opt.step()
        _check_step(opt, params, before, min(1.0, 1.0 / (float(_exact_norm([p.grad for p in params], 2)[0]) + 1e-6)), **kw)
        del before
        used.append(torch.cuda.memory_allocated())
    assert used[-1] == used[3], used


def test_adamw_one_cycle_schedule():
    """a schedule that moves lr and betas at every step"""
    opt, params = _optimizer([5000, 3], F32, seed=220, max_norm=1.0)
    schedule = torch.optim.lr_scheduler.OneCycleLR(opt, max_lr=1e-2, total_steps=20)
    seen = set()
    for _ in range(12):
        group = opt.param_groups[0]
        seen.add(group["betas"])
        before = _snapshot(opt, params)
        opt.step()
        _check_step(opt, params, before, min(1.0, 1.0 / (float(_exact_norm([p.grad for p in params], 2)[0]) + 1e-6)),
                    **{k: group[k] for k in ("lr", "betas", "eps", "weight_decay")})
        schedule.step()
    assert len(seen) == 12


def test_adamw_changed_settings_do_not_wait():
    """betas and a learning rate's tensor that change while the GPU is busy: the step returns before the GPU is done"""
    opt, params = _optimizer([5000, 3], F32, seed=240, max_norm=1.0, lr=torch.tensor(1e-3, device=DEV))
    rate = torch.tensor(2e-3, device=DEV)
    busy = _rand((8192, 8192), seed=241)
    busy @ busy
    opt.step()
    before = _snapshot(opt, params)
    done = torch.cuda.Event()
    torch.cuda.synchronize()
    for _ in range(20):
        busy @ busy      # some 150 ms
    done.record()
    opt.param_groups[0].update(betas=(0.5, 0.75), lr=rate)
    opt.step()
    assert not done.query()
    torch.cuda.synchronize()
    _check_step(opt, params, before, min(1.0, 1.0 / (float(_exact_norm([p.grad for p in params], 2)[0]) + 1e-6)), betas=(0.5, 0.75), lr=2e-3)


def test_adamw_captured_with_changed_settings():
    """settings that changed ahead of a capture: each graph keeps those it was captured with, eager steps have their own"""
    opt, params = _optimizer([5000, 17], F32, seed=250)
    opt.step()
    graphs = []
    for kw in (dict(betas=(0.5, 0.75)), dict(betas=(0.6, 0.8), eps=1e-3), dict(betas=(0.5, 0.75), lr=0.25)):
        kw = {**dict(lr=1e-3, eps=1e-8), **kw}
        opt.param_groups[0].update(kw)
        graphs.append((torch.cuda.CUDAGraph(), kw))
        with torch.cuda.graph(graphs[-1][0]):
            opt.step()
    eager = dict(betas=(0.7, 0.9), lr=1e-2)
    opt.param_groups[0].update(eager, eps=1e-8)
    opt.step()
    for _ in range(3):
        for graph, kw in graphs:
            before = _snapshot(opt, params)
            graph.replay()
            torch.cuda.synchronize()
            _check_step(opt, params, before, **kw)
            before = _snapshot(opt, params)
            opt.step()
            _check_step(opt, params, before, **eager)


def test_adamw_64_groups():
    params = [_rand(5 + i, F32, 260 + i, 0.1).requires_grad_(True) for i in range(64)]
    for i, p in enumerate(params):
        p.grad = _rand(p.shape, F32, 400 + i)
    hyper = [dict(lr=1e-3 * (i + 1), betas=(0.5 + 0.005 * i, 0.9 + 0.001 * i), eps=10.0 ** (-4 - i % 5), weight_decay=0.01 * i) for i in range(64)]
    opt = pde_amd.ClippedAdamW([dict(params=[p], **kw) for p, kw in zip(params, hyper)])
    for _ in range(2):
        before = _snapshot(opt, params)
        opt.step()
        for p, b, kw in zip(params, before, hyper):
            _check_step(opt, [p], [b], **kw)
        hyper = hyper[::-1]
        for g, kw in zip(opt.param_groups, hyper):
            g.update(kw)


def test_adamw_state_that_is_cleared_or_replaced():
    """whatever is in `state` at a step is used and written"""
    for dtype in (F32, BF16):
        opt, params = _optimizer([5000, 3, 70001], dtype, seed=270, max_norm=1.0)
        c = min(1.0, 1.0 / (float(_exact_norm([p.grad for p in params], 2)[0]) + 1e-6))

        def step():
            before = _snapshot(opt, params)
            opt.step()
            _check_step(opt, params, before, c)
            return [b[3] for b in before]

        step()
        old = dict(opt.state[params[1]])
        kept = {k: v.clone() for k, v in old.items()}
        opt.state.clear()
        assert step() == [0.0] * 3 and step() == [1.0] * 3      # starts again
        for name in old:      # one tensor of one parameter
            opt.state[params[2]][name] = opt.state[params[2]][name].clone().abs_()
            step()
        opt.state[params[0]] = {k: torch.zeros_like(v) if k != "master" else v for k, v in opt.state[params[0]].items()}
        assert step()[0] == 0.0
        opt.state[params[0]] = dict(opt.state[params[0]])      # another dictionary with the same tensors
        step()
        del opt.state[params[1]]
        assert step()[1] == 0.0
        opt.state = type(opt.state)(dict, {p: copy.deepcopy(opt.state[p]) for p in params})
        step()
        opt.state[params[1]]["note"] = 5      # an entry of the user's
        step()
        assert opt.state[params[1]]["note"] == 5
        assert all(torch.equal(old[k], kept[k]) for k in old)      # what was taken out is left alone
        del opt.state[params[0]]["exp_avg"]
        for _ in range(2):
            with pytest.raises(ValueError, match="must hold"):
                opt.step()


def test_adamw_entries_of_the_user_cost_no_new_description():
    """an entry that changes at every step: no description is copied to the device, so a step does not wait"""
    opt, params = _optimizer([5000, 3], F32, seed=280)
    opt.step()
    busy = _rand((8192, 8192), seed=281)
    busy @ busy
    done = torch.cuda.Event()
    torch.cuda.synchronize()
    for _ in range(20):
        busy @ busy      # some 150 ms
    done.record()
    for k in range(3):
        opt.state[params[0]]["note"] = k
        opt.step()
    assert not done.query()
    torch.cuda.synchronize()
    assert float(opt.state[params[0]]["step"]) == 4.0


def test_adamw_captured_step_keeps_state_that_is_replaced():
    """the graph goes on with the tensors it was captured with, eager steps take those that are in `state` now"""
    opt, params = _optimizer([5000, 17], F32, seed=290)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    theirs = [dict(opt.state[p]) for p in params]
    opt.state.clear()
    opt.step()
    filler = [torch.full((4096,), math.nan, device=DEV) for _ in range(64)]      # takes whatever memory was given back
    mine = [dict(opt.state[p]) for p in params]
    for k in range(3):
        for p, s in zip(params, theirs):
            opt.state[p] = s
        before = _snapshot(opt, params)
        graph.replay()
        torch.cuda.synchronize()
        _check_step(opt, params, before)
        for p, s in zip(params, mine):
            opt.state[p] = s
        before = _snapshot(opt, params)
        assert [b[3] for b in before] == [k + 1.0] * 2
        opt.step()
        _check_step(opt, params, before)
    del filler


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradients_of_negative_views_and_known_zeros(dtype):
    """memory that holds the negated values (the imaginary part of a conjugate), or nothing"""
    neg, zero = torch._neg_view, torch._efficientzerotensor
    values = [_rand(5000, dtype, 300), _rand(300, dtype, 301)]
    grads = lambda: [neg(-values[0]), values[1].clone(), zero(70, dtype=dtype, device=DEV)]      # noqa: E731
    opt, params = _optimizer([5000, 300, 70], dtype, seed=302, max_norm=0.5)
    for p, g in zip(params, grads()):
        p.grad = g
    assert params[0].grad.is_neg()
    norm = _exact_norm(values, 2)[0]
    for _ in range(2):
        before = _snapshot(opt, params)
        opt.step()
        for p, g in zip(params, values + [torch.zeros(70, dtype=dtype, device=DEV)]):
            p.grad = g
        _near(opt.total_norm, norm)
        _check_step(opt, params, before, 0.5 / (float(norm) + 1e-6))
        for p, g in zip(params, grads()):
            p.grad = g
    total, each = pde_amd.get_total_norm(grads(), per_tensor=True)
    _near(total, norm)
    _near(each, torch.cat([_exact_norm(values, 2)[1], torch.zeros(1, dtype=torch.float64, device=DEV)]))
    clipped = grads()[:2]
    pde_amd.clip_grad_norm_(_leaves(clipped), 0.5)
    assert all(torch.equal(c.resolve_neg(), _clipped(v, total, 0.5)) for c, v in zip(clipped, values))
    clipped = [v.clone() for v in values]
    pde_amd.clip_grads_with_norm_(_leaves(clipped), 1.0, neg(torch.tensor(-4.0, device=DEV)))
    assert all(torch.equal(c, _clipped(v, torch.tensor(4.0, device=DEV), 1.0)) for c, v in zip(clipped, values))
    opt.param_groups[0]["lr"] = neg(torch.tensor(-1e-3, device=DEV))
    with pytest.raises(ValueError, match="learning rate on the device"):
        opt.step()


def test_lazy_clones_keep_their_values():
    """what is written leaves clones that were made lazily, before or between calls, as they are"""
    g = _rand(5000, seed=310)
    kept, clone = g.clone(), torch._lazy_clone(g)
    total = pde_amd.clip_grad_norm_(_leaves([clone]), 0.5)
    assert torch.equal(g, kept) and torch.equal(clone, _clipped(kept, total, 0.5))
    opt, params = _optimizer([5000, 300], F32, seed=311)
    for _ in range(2):
        before = _snapshot(opt, params)
        clones = [torch._lazy_clone(p.detach()) for p in params] + [torch._lazy_clone(t) for p in params for t in opt.state.get(p, {}).values()]
        kept = [c.clone() for c in clones]
        opt.step()
        _check_step(opt, params, before)
        assert all(torch.equal(a, b) for a, b in zip(clones, kept))


@pytest.mark.parametrize("total", [1061.81005859375, 958.9559326171875, 3.0, 1.5258789, 65537.5])
def test_clip_of_every_float16(total):
    """the factor and the product in float32, then one rounding: at the first two norms some products lie on the middle
    between two float16 values, and the exact ones beside it"""
    values = torch.arange(-32768, 32768, dtype=torch.int32, device=DEV).to(torch.int16).view(F16)
    values = values[torch.isfinite(values)]
    norm = torch.tensor(total, device=DEV)
    for n in (values.numel(), 8, 7, 1):      # loads of 8, and the last elements one by one
        parts = [t.clone() for t in values.split(n)] if n > 8 else [t.clone() for t in values[20000:20840].split(n)]
        want = [_clipped(t, norm, 1.0) for t in parts]
        pde_amd.clip_grads_with_norm_(_leaves(parts), 1.0, norm)
        assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(parts, want))


# ----------------------------------------------------------------------------------------------------------------------
# the borders of a launch's list, and sizes from which on the kernels go other ways, on values that are all different
# ----------------------------------------------------------------------------------------------------------------------
# 255 tensors to a launch of the norm, the scaling and the norm ahead of an update, 319 to one of the update
LIST_LENGTHS = [254, 255, 256, 319, 320, 511, 640]


def _many(count, dtypes, seed):
    """`count` tensors of 0 to 300 values, and one of 9000; those beside the borders of a list are empty, or not, in turn"""
    sizes = [0 if i % 64 == 63 and i % 128 == 63 else 9000 if i == count // 2 else 1 + (i * 37) % 300 for i in range(count)]
    return [_rand(n, dtypes[i % len(dtypes)], seed + i, 2.0 ** (i % 7 - 3)) for i, n in enumerate(sizes)]


@pytest.mark.parametrize("count", LIST_LENGTHS)
def test_lists_around_a_launch(count):
    ts = _many(count, (F32, BF16, F16), 1000)
    for p in (1, 2, INF):
        want, each = _exact_norm(ts, p)
        total, got = pde_amd.get_total_norm(ts, p, per_tensor=True)
        _near(total, want)
        _near(got, each)
        _near(pde_amd.get_total_norm(ts, p), want)
    before = [t.clone() for t in ts]
    total = pde_amd.clip_grad_norm_(_leaves(ts), 1.0)
    _near(total, _exact_norm(before, 2)[0])
    assert all(torch.equal(t, _clipped(b, total, 1.0)) for t, b in zip(ts, before))
    ts = [b.clone() for b in before]
    pde_amd.clip_grads_with_norm_(_leaves(ts), 1.0, total)
    assert all(torch.equal(t, _clipped(b, total, 1.0)) for t, b in zip(ts, before))


@pytest.mark.parametrize("count", LIST_LENGTHS)
def test_adamw_lists_around_a_launch(count):
    params = [t.requires_grad_(True) for t in _many(count, (F32, BF16), 2000)]
    opt = pde_amd.ClippedAdamW(params, max_norm=1.0)
    for step in range(2):
        for i, p in enumerate(params):
            p.grad = None if i % 5 == step else _rand(p.shape, p.dtype, 3000 * (step + 1) + i)
        have = [p for p in params if p.grad is not None and p.numel()]
        before = _snapshot(opt, have)
        idle = [(p, p.detach().clone()) for p in params if p.grad is None]
        opt.step()
        norm = _exact_norm([p.grad for p in have], 2)[0]
        _near(opt.total_norm, norm)
        _check_step(opt, have, before, min(1.0, 1.0 / (float(norm) + 1e-6)))
        assert all(torch.equal(p.detach(), value) for p, value in idle)


# millions of elements: below and above 64 MB, from where on norm and scaling read past the cache, and more than one unit
# (16 KB) for each of 1024 workgroups either way
def _large(dtype, above):
    total = (66 << 20 if above else 40 << 20) // (4 if dtype is F32 else 2)
    return [total // 3, 5, total // 2 + 1, 4096, 0, 8192, total // 6, 12287, 1]


@pytest.mark.parametrize("above", [False, True])
@pytest.mark.parametrize("p", [1, 2, INF])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_norm_of_large_tensors(dtype, p, above):
    _, ts = _packed(_large(dtype, above), dtype, seed=3)
    want, each = _exact_norm(ts, p)
    total, got = pde_amd.get_total_norm(ts, p, per_tensor=True)
    _near(total, want)
    _near(got, each)
    _near(pde_amd.get_total_norm(ts, p), want)


@pytest.mark.parametrize("above", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_clip_of_large_tensors(dtype, above):
    flat, ts = _packed(_large(dtype, above), dtype, seed=4)
    before = flat.clone()
    total = pde_amd.clip_grad_norm_(_leaves(ts), 3.0)
    _near(total, _exact_norm([before[1:-1]], 2)[0])
    assert torch.equal(flat[1:-1], _clipped(before[1:-1], total, 3.0))
    assert float(flat[0]) == 7.0 and float(flat[-1]) == 7.0
    pde_amd.clip_grads_with_norm_(_leaves(ts), 1.0, torch.tensor(4.0, device=DEV))
    assert torch.equal(flat[1:-1], _clipped(_clipped(before[1:-1], total, 3.0), torch.tensor(4.0, device=DEV), 1.0))


# units of 1024 elements; from 512 on the update deals them out over the XCDs
@pytest.mark.parametrize("units", [511, 512, 513, 1024, 1029, 5000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_adamw_of_large_tensors(dtype, units):
    sizes = [7 * 1024, (units - 110) * 1024, 1, 99 * 1024 + 5, 1023, 1021]      # 7 + (units - 110) + 1 + 100 + 1 + 1
    opt, params = _optimizer(sizes, dtype, seed=500, state_step=3, max_norm=1.0)
    before = _snapshot(opt, params)
    opt.step()
    norm = _exact_norm([p.grad for p in params], 2)[0]
    _near(opt.total_norm, norm)
    _check_step(opt, params, before, min(1.0, 1.0 / (float(norm) + 1e-6)))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_adamw_beyond_the_cache(dtype):
    """gradients of more than 224 MB: the first of them are read past the cache for the norm"""
    n = (240 << 20) // (4 if dtype is F32 else 2)
    opt, params = _optimizer([n // 2 + 3, n // 2], dtype, seed=510, state_step=3, max_norm=1.0)
    before = _snapshot(opt, params)
    opt.step()
    norm = _exact_norm([p.grad for p in params], 2)[0]
    _near(opt.total_norm, norm)
    _check_step(opt, params, before, min(1.0, 1.0 / (float(norm) + 1e-6)))
    del opt, params, before
    torch.cuda.empty_cache()


@pytest.mark.parametrize("name", ["exp_avg", "exp_avg_sq", "master"])
def test_adamw_state_whose_layout_changes(name):
    """a state tensor that is transposed in place no longer lies as its parameter does"""
    p = _rand((64, 64), BF16, seed=600).requires_grad_(True)
    p.grad = _rand((64, 64), BF16, seed=601)
    opt = pde_amd.ClippedAdamW([p])
    opt.step()
    opt.state[p][name].t_()
    before = _snapshot(opt, [p])
    for _ in range(2):
        with pytest.raises(ValueError, match="laid out"):
            opt.step()
    opt.state[p][name] = opt.state[p][name].contiguous()
    opt.step()
    _check_step(opt, [p], before)
