"""AdamW's 8-bit states over runs of steps: codes rounded up or down at random so that the moments are right
on average (what optim.AdamW keeps, and adamw_step with rounding="stochastic")."""
import copy
import importlib

import pytest
import torch

from test_optim_gpu import BF, DEV, F32, HYPER, SIZES, _call, _exact, _lists, _values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def opt():
    return importlib.import_module("rwkv-megatron_amd").optim


def _gap(value, unit):
    """The distance of the two e4m3 numbers (times unit) around value: 2^-3 of its power of two, 2^-9 below 2^-6."""
    e = (value.abs() / unit).clamp(min=2.0 ** -6).log2().floor()
    return torch.exp2(e - 3) * unit


# A stored value is one of the two numbers next to the formula's (which 32 bits evaluate to 2^-20 of its terms).
# The errors of m and of v are independent with mean zero, up to that evaluation; the deviation of one is at most half
# the distance of its two values, so a sum stays within six times the root of the sum of their squares.
@pytest.mark.parametrize("ptype", [F32, BF])
def test_codes_are_right_on_average(opt, ptype):
    t = _lists([1 << 20, *SIZES], ptype, F32, True, seed=3)
    m0 = _values(t)[0]
    exact, _ = _exact(t)
    near, twin, later = (copy.deepcopy(t) for _ in range(3))
    later["step"] += 1
    for u in (t, twin, later):
        _call(opt, u, rounding="stochastic")
    _call(opt, near)
    code = lambda u, n, i=0: u[n][i].view(torch.uint8)
    for i in range(len(exact)):
        assert all(torch.equal(code(t, n, i), code(twin, n, i)) for n in "pmv")
        assert torch.equal(code(t, "p", i), code(near, "p", i))          # the update takes the unrounded moments
        assert all(torch.equal(t["scales"][k][i], near["scales"][k][i]) for k in (0, 1))
    assert 0.02 < float((code(t, "v") != code(later, "v")).float().mean()) < 0.5     # another step, other choices
    now = _values(t)
    for i, (_, m, v, _) in enumerate(exact):
        if not m.numel():
            continue
        wide = [t["scales"][k][i].double().repeat_interleave(256)[:m.numel()] for k in (0, 1)]
        em = 2.0 ** -20 * (m0[i].abs() + t["g"][i].double().abs())
        for got, want, unit, slack in ((now[0][i], m, wide[0], em), (now[1][i].sqrt(), v.sqrt(), wide[1], 2.0 ** -20 * v.sqrt())):
            off = (got - want).abs()
            assert bool((off <= 1.001 * _gap(want, unit) + slack + 2.0 ** -20 * unit).all()), i
        if i == 0:
            gm, gv = _gap(m, wide[0]), _gap(v.sqrt(), wide[1])
            gv = gv * 2 * (v.sqrt() + gv)
            assert abs(float((now[0][i] - m).sum())) <= 3 * float(gm.square().sum().sqrt()) + float(em.sum())
            assert abs(float((now[1][i] - v).sum())) <= 3 * float(gv.square().sum().sqrt()) + float(v.sum()) * 2.0 ** -20


# Gradients N(0, 1) of which half of every block falls to a tenth, or rises threefold, after 1000 steps.  The recursion
# of v is linear and the rounding has mean zero, so the mean of v over that in 32 bits is 1.  A step's rounding moves
# v by no more than its change does on average: variance at most |change| times the distance of the codes' squares,
# |change| at most 4 (1 - b2) v on average (its decay and g^2, and the same of the block's largest, which moves the scale)
# and the distance 0.27 v.  Over the steps that v remembers that adds up to a variance s / (1 - s), s = 0.54, a
# deviation of 1.1: of the mean of 8192 elements 0.012, six of which are 0.08.  For m: the codes' distance is at most
# 2^-3 of four deviations of m, half of it a step's deviation, over the steps remembered 1 / sqrt(1 - b1^2) of that,
# 0.57: 0.0063 of the projection on m, six of which are 0.04.
@pytest.mark.parametrize("b2", [0.995, 0.98])
def test_moments_follow_their_gradients(opt, b2):
    n, steps = 64 * 256, 3000
    ps = [torch.nn.Parameter(torch.zeros(n, device=DEV)) for _ in range(4)]
    kw = dict(lr=1e-3, betas=(0.9, b2), weight_decay=0.0)
    eight, wide = opt.AdamW(ps[:2], **kw, state_bits=8), opt.AdamW(ps[2:], **kw)
    half = (torch.arange(n, device=DEV) % 256 < 128)
    g = torch.Generator(device=DEV).manual_seed(1)
    for k in range(steps):
        grad = torch.randn(n, generator=g, device=DEV)
        for i, factor in enumerate((0.1, 3.0)):
            ps[i].grad = ps[i + 2].grad = torch.where(half, factor, 1.0) * grad if k >= 1000 else grad
        eight.step()
        wide.step()
    for p, q in zip(ps[:2], ps[2:]):
        (m, v), (m32, v32) = eight.moments(p), wide.moments(q)
        for part in (half, ~half):
            mean = float((v[part].double() / v32[part].double()).mean())
            assert abs(mean - 1) <= 0.08, mean
            a, b = m[part].double(), m32[part].double()
            assert abs(float(((a - b) * b).sum() / b.square().sum())) <= 0.04


def test_values_that_are_not_finite_and_zero_blocks(opt):
    t, u = _lists([600], F32, F32, True), _lists([600], F32, F32, True)
    t["g"][0][5], t["g"][0][300] = float("inf"), float("nan")
    _call(opt, t, rounding="stochastic")
    _call(opt, u, rounding="stochastic")
    bad = torch.zeros(600, dtype=torch.bool, device=DEV)
    bad[5] = bad[300] = True
    assert bool(t["p"][0][bad].isnan().all()) and torch.equal(t["p"][0][~bad], u["p"][0][~bad])
    m, v = _values(t)
    assert not bool(m[0][bad].isfinite().any()) and bool(m[0][~bad].isfinite().all()) and bool(v[0][~bad].isfinite().all())
    z = _lists([512], F32, F32, True)
    for n in ("m", "v"):
        z[n][0] = torch.zeros(512, device=DEV).to(torch.float8_e4m3fn)
    z["g"][0].zero_()
    z["g"][0][300] = 1e-37
    _call(opt, z, rounding="stochastic")
    m, v = _values(z)
    assert not bool(m[0].any()) and not bool(v[0].any()) and bool(z["p"][0].isfinite().all())


def test_states_of_32_bits_and_refusals(opt):
    t, u = _lists([300], F32, F32, False), _lists([300], F32, F32, False)
    _call(opt, t, rounding="stochastic")
    _call(opt, u)
    assert all(torch.equal(t[n][0], u[n][0]) for n in "pmv")
    with pytest.raises(ValueError, match="rounding"):
        _call(opt, t, rounding="up")
    assert float(t["step"]) == 7


# Step by step: every step of the optimizer is the formula's from the moments that it holds, so that a moment lost, negated
# or scaled between two steps shows (each would move p by a good part of lr; the bound is 2^-20 of the step, as in
# test_optim_gpu.py, and a rounding of p).
@pytest.mark.parametrize("bits", [8, 32])
def test_every_step_is_the_formula_of_the_moments_held(opt, bits):
    g = torch.Generator(device=DEV).manual_seed(4)
    ps = [torch.nn.Parameter(torch.randn(n, generator=g, device=DEV) * 0.1) for n in (5000, 100, 4096)]
    o = opt.AdamW(ps, **HYPER, state_bits=bits)
    lr, (b1, b2), eps, wd = HYPER["lr"], HYPER["betas"], HYPER["eps"], HYPER["weight_decay"]
    held = [(torch.zeros_like(p, dtype=torch.float64),) * 2 for p in ps]
    for k in range(1, 6):
        for p in ps:
            p.grad = torch.randn(p.shape, generator=g, device=DEV) * 0.02
        before = [p.detach().double() for p in ps]
        o.step()
        for i, p in enumerate(ps):
            m, v = held[i]
            gr = p.grad.double()
            m, v = b1 * m + (1 - b1) * gr, b2 * v + (1 - b2) * gr * gr
            u = lr / (1 - b1 ** k) * m / ((v / (1 - b2 ** k)).sqrt() + eps)
            want = before[i] * (1 - lr * wd) - u
            # m itself takes roundings of its two terms, which may cancel
            slack = lr / (1 - b1 ** k) * 2.0 ** -22 * (held[i][0].abs() + gr.abs()) / ((v / (1 - b2 ** k)).sqrt() + eps)
            assert bool(((p.detach().double() - want).abs() <= 2.0 ** -20 * u.abs() + 2.0 ** -22 * want.abs() + slack).all()), (k, i)
            now = [t.double() for t in o.moments(p)]
            if bits == 8 and p.numel() >= 4096:
                for got, exact, name in ((now[0], m, "exp_avg_scale"), (now[1].sqrt(), v.sqrt(), "exp_avg_sq_scale")):
                    unit = o.state[p][name].double().repeat_interleave(256)[:p.numel()]
                    assert bool(((got - exact).abs() <= 1.001 * _gap(exact, unit) + 2.0 ** -18 * unit).all()), (k, i, name)
            held[i] = now
