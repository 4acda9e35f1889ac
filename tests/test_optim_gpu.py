"""optim.AdamW and optim.adamw_step: steps against the formula in float64, 8-bit states, clipping,
parameters of every form, groups, state dicts, captured steps."""
import copy
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32, F8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
HYPER = dict(lr=1e-2, betas=(0.9, 0.995), eps=1e-8, weight_decay=0.1)
# sizes at the edges of a lane's 8, a scale's 256 and a block's 2048 elements, more tensors than a launch
# takes, an empty one and one of several blocks
SIZES = [1, 7, 8, 9, 255, 256, 257, 2047, 2048, 2049, 0, 5, 70001] + [33] * 60


@pytest.fixture(scope="module")
def opt():
    return importlib.import_module("rwkv-megatron_amd").optim


def _lists(sizes, ptype, gtype, eight, seed=0):
    g = torch.Generator().manual_seed(seed)
    mk = lambda n, s=1.0: (torch.randn(n, generator=g) * s).to(DEV)
    t = {"p": [mk(n).to(ptype) for n in sizes], "g": [mk(n, 0.01).to(gtype) for n in sizes],
         "step": torch.full((), 6.0, device=DEV), "scales": None}
    m, v = [mk(n, 0.01) for n in sizes], [mk(n, 0.01).square() + 1e-6 for n in sizes]
    if eight:
        blocks = [-(-n // 256) for n in sizes]
        t["m"] = [mk(n, 100.0).clamp(-448, 448).to(F8) for n in sizes]
        t["v"] = [mk(n, 100.0).abs().clamp(0.5, 448).to(F8) for n in sizes]
        t["scales"] = ([mk(b, 1e-4).abs() for b in blocks], [mk(b, 1e-4).abs() + 1e-5 for b in blocks])
    else:
        t["m"], t["v"] = m, v
    return t


def _values(t):
    """The states as numbers in float64."""
    if t["scales"] is None:
        return [m.double() for m in t["m"]], [v.double() for v in t["v"]]
    wide = lambda c, s: c.reshape(-1).double() * s.double().repeat_interleave(256)[:c.numel()]
    return ([wide(c, s) for c, s in zip(t["m"], t["scales"][0])],
            [wide(c, s) ** 2 for c, s in zip(t["v"], t["scales"][1])])


def _exact(t, max_norm=None, lr=1e-2, betas=(0.9, 0.995), eps=1e-8, weight_decay=0.1):
    g = [x.double() for x in t["g"]]
    norm = torch.stack([x.square().sum() for x in g]).sum().sqrt()
    c = 1.0 if max_norm is None else min(1.0, max_norm / (float(norm) + 1e-6))
    k = float(t["step"]) + 1
    out = []
    for p, x, m, v in zip(t["p"], g, *_values(t)):
        m = betas[0] * m + (1 - betas[0]) * c * x.reshape(m.shape)
        v = betas[1] * v + (1 - betas[1]) * (c * x.reshape(v.shape)) ** 2
        u = lr / (1 - betas[0] ** k) * m / ((v / (1 - betas[1] ** k)).sqrt() + eps)
        out.append((p.double().reshape(m.shape) * (1 - lr * weight_decay) - u, m, v, u))
    return out, norm


def _call(opt, t, **kw):
    return opt.adamw_step(t["p"], t["g"], t["m"], t["v"], t["step"], scales=t["scales"], **{**HYPER, **kw})


# Bounds: p is rounded once by half a step of its type, and the step's 32-bit evaluation (a dozen roundings
# of 2^-24 and a reciprocal, 2^-20 of the step and 2^-23 of p); a moment takes four roundings of its terms,
# which have one sign for v and for m up to |m| + |g| / 10.
@pytest.mark.parametrize("ptype,gtype", [(F32, F32), (BF, BF), (F32, BF), (BF, F32)])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("max_norm", [None, 0.5, 1e6])
def test_step_matches_float64(opt, ptype, gtype, eight, max_norm):
    t = _lists(SIZES, ptype, gtype, eight)
    m0 = _values(t)[0]
    exact, norm = _exact(t, max_norm)
    twin = copy.deepcopy(t)
    got = _call(opt, t, max_norm=max_norm)
    again = _call(opt, twin, max_norm=max_norm)
    if max_norm is None:
        assert got is None
    else:
        assert torch.equal(got, again) and got.shape == () and abs(float(got) - float(norm)) <= 2.0 ** -23 * float(norm)
    assert float(t["step"]) == 7
    now = _values(t)
    for i, (p, m, v, u) in enumerate(exact):
        for n in ("p", "m", "v"):
            assert torch.equal(t[n][i].view(torch.uint8), twin[n][i].view(torch.uint8))
        half = torch.finfo(ptype).eps / 2 * 1.01
        assert bool(((t["p"][i].double() - p).abs() <= half * p.abs() + 2.0 ** -20 * u.abs() + 2.0 ** -22 * p.abs()).all()), i
        em = 2.0 ** -21 * (m0[i].abs() + t["g"][i].double().abs())
        if not eight:
            assert bool(((now[0][i] - m).abs() <= em).all()) and bool(((now[1][i] - v).abs() <= 2.0 ** -21 * v).all())
            continue
        # a code is off by half a step: 2^-4 of its value, or 2^-10 of a scale's unit below 2^-6
        for value, want, scale, slack in ((now[0][i], m, t["scales"][0][i], em), (now[1][i].sqrt(), v.sqrt(), t["scales"][1][i], 0)):
            unit = scale.double().repeat_interleave(256)[:want.numel()]
            assert bool(((value - want).abs() <= 2.0 ** -4 * 1.001 * want.abs() + 2.0 ** -10 * 1.001 * unit + slack).all()), i
            if want.numel():
                top = torch.stack([b.abs().max() for b in want.split(256)])
                assert bool(((scale.double() * 448 - top).abs() <= 2.0 ** -19 * top + (em.max() if slack is em else 0)).all())


def test_grad_norm(opt):
    t = _lists(SIZES, F32, BF, False)
    want = torch.stack([g.double().square().sum() for g in t["g"]]).sum().sqrt()
    assert abs(float(opt.grad_norm(t["g"])) - float(want)) <= 2.0 ** -23 * float(want)
    big = torch.full((3_000_001,), 1e19, device=DEV)                 # a square past the range of 32 bits
    assert abs(float(opt.grad_norm([big])) / (1e19 * 3_000_001 ** 0.5) - 1) <= 2.0 ** -22


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("off", [0, 1])
def test_views_off_the_16_byte_grid_and_their_neighbours(opt, eight, off):
    t = _lists([4099], BF, BF, eight)
    u = copy.deepcopy(t)
    wides = []
    for n in ("p", "g", "m", "v"):
        x = u[n][0]
        wide = torch.full((x.numel() + 16,), 3, dtype=torch.float32, device=DEV).to(x.dtype)
        wide[off:off + 4099].copy_(x)
        u[n][0] = wide[off:off + 4099]
        wides.append(wide)
    _call(opt, t, max_norm=0.1)
    _call(opt, u, max_norm=0.1)
    for wide in wides:
        assert bool((wide[:off].float() == 3).all()) and bool((wide[off + 4099:].float() == 3).all())
    for n in ("p", "m", "v"):
        assert torch.equal(t[n][0].view(torch.uint8), u[n][0].contiguous().view(torch.uint8))


def test_strides_of_parameters_and_gradients(opt):
    """A parameter in another order of memory, and gradients that are expanded or transposed."""
    g = torch.Generator().manual_seed(2)
    p = torch.randn(40, 30, generator=g).to(DEV)
    gr = torch.randn(40, 30, generator=g).to(DEV)
    base, turned = torch.nn.Parameter(p.clone()), torch.nn.Parameter(p.t().contiguous().t())
    for param, grads in ((base, [gr, gr[:1].expand(40, 30)]), (turned, [gr, gr[:1].expand(40, 30)])):
        o = opt.AdamW([param], **HYPER, state_bits=32, max_norm=1.0)
        for x in grads:
            param.grad = x
            o.step()
    assert torch.equal(base, turned) and turned.stride() == (1, 40)
    with pytest.raises(ValueError, match="dense"):
        opt.adamw_step([p[:, ::2]], [gr[:, ::2]], [p[:, ::2].float()], [p[:, ::2].float()], torch.zeros((), device=DEV), lr=1.0)


def _params(dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter((torch.randn(*s, generator=g) * 0.1).to(dtype).to(DEV)) for s in [(64, 65), (5000,), (3,), (100, 100)]]


def _grads(ps, seed):
    g = torch.Generator().manual_seed(100 + seed)
    for p in ps:
        p.grad = (torch.randn(*p.shape, generator=g) * 0.02).to(p.dtype).to(DEV)


# Four steps beside torch's AdamW in float64 with the same clipping.  Each 32-bit step adds at most 2^-20 of
# its length (lr) and roundings of p, 2^-23.
def test_optimizer_follows_torch(opt):
    ps = _params(F32)
    qs = [torch.nn.Parameter(p.detach().double()) for p in ps]
    a, b = opt.AdamW(ps, **HYPER, max_norm=0.7), torch.optim.AdamW(qs, **HYPER)
    for k in range(4):
        _grads(ps, k)
        for p, q in zip(ps, qs):
            q.grad = p.grad.double()
        torch.nn.utils.clip_grad_norm_(qs, 0.7)
        a.step()
        b.step()
    for p, q in zip(ps, qs):
        assert float((p.double() - q).detach().abs().max()) <= 4 * (2.0 ** -17 * HYPER["lr"] + 2.0 ** -22 * float(q.detach().abs().max()))
    assert a.grad_norm.shape == ()


def test_8_bit_states_of_the_large_tensors_alone(opt):
    ps = _params(F32)
    o = opt.AdamW(ps, **HYPER, state_bits=8)
    for k in range(3):
        _grads(ps, k)
        o.step()
    kinds = ["exp_avg_scale" in o.state[p] for p in ps]
    assert kinds == [True, True, False, True]
    assert all(float(o.state[p]["step"]) == 3 for p in ps)
    ref = _params(F32)
    r = opt.AdamW(ref, **HYPER)
    for k in range(3):
        _grads(ref, k)
        r.step()
    assert torch.equal(ps[2], ref[2])
    for p, q in zip(ps, ref):
        # m and the root of v each off by 2^-4 at most a step: a step by a factor within (1 +- 2^-4)^2 / (1 -+ 2^-4)
        # of the first moments' |terms|; three steps of at most lr / (1 - b1) each
        assert float((p - q).detach().abs().max()) <= 3 * HYPER["lr"] * 3
        m, v = o.moments(p)
        m2, v2 = r.moments(q)
        assert float((m - m2).norm() / m2.norm()) <= 3 * 2.0 ** -4 and float((v.sqrt() - v2.sqrt()).norm() / v2.sqrt().norm()) <= 3 * 2.0 ** -4


def test_parameters_without_a_gradient_make_no_step(opt):
    ps, qs = _params(F32), _params(F32)
    a, b = opt.AdamW(ps, **HYPER), torch.optim.AdamW(qs, **HYPER, foreach=False, fused=False)
    for k, live in enumerate([(0, 1, 2, 3), (0, 2), (1,), (0, 1, 2, 3), (3,)]):
        _grads(ps, k)
        _grads(qs, k)
        for i in range(4):
            if i not in live:
                ps[i].grad = qs[i].grad = None
        a.step()
        b.step()
    assert [float(a.state[p]["step"]) for p in ps] == [3, 3, 3, 3] == [float(b.state[q]["step"]) for q in qs]
    for p, q in zip(ps, qs):
        # both in 32 bits: a few roundings a step
        assert float((p - q).detach().abs().max()) <= 5 * (2.0 ** -16 * HYPER["lr"] + 2.0 ** -22)
    ps2 = _params(F32)
    o = opt.AdamW(ps2, **HYPER)
    o.step()
    assert not o.state and all(torch.equal(p, q) for p, q in zip(ps2, _params(F32)))


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_state_dict_round_trip(opt, bits, dtype):
    ps, qs = _params(dtype), _params(dtype)
    make = lambda p: opt.AdamW([{"params": p[:2]}, {"params": p[2:], "lr": 1e-3}], **HYPER, state_bits=bits, max_norm=1.0)
    a, b = make(ps), make(qs)
    for k in range(2):
        _grads(ps, k)
        if k:
            ps[1].grad = None
        a.step()
    sd = copy.deepcopy(a.state_dict())
    with torch.no_grad():
        for p, q in zip(ps, qs):
            q.copy_(p)
    b.load_state_dict(sd)
    assert [float(b.state[q]["step"]) for q in qs] == [2, 1, 2, 2]
    for k in range(2, 4):
        _grads(ps, k)
        _grads(qs, k)
        a.step()
        b.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q)
        for n, s in a.state[p].items():
            assert s.dtype == b.state[q][n].dtype and torch.equal(s.view(torch.uint8) if s.dim() else s, b.state[q][n].view(torch.uint8) if s.dim() else b.state[q][n])


@pytest.mark.parametrize("bits", [8, 32])
def test_loads_a_state_dict_of_torch_and_of_the_other_kind(opt, bits):
    ps, qs = _params(F32), _params(F32)
    a = torch.optim.AdamW(ps, **HYPER)
    _grads(ps, 0)
    a.step()
    o = opt.AdamW(qs, **HYPER, state_bits=bits)
    o.load_state_dict(a.state_dict())
    for p, q in zip(ps, qs):
        m, v = o.moments(q)
        s = a.state[p]
        half = 2.0 ** -4 * 1.001 if bits == 8 and p.numel() >= 4096 else 0
        top = float(s["exp_avg"].abs().max()), float(s["exp_avg_sq"].sqrt().max())
        assert bool(((m - s["exp_avg"]).abs() <= half * s["exp_avg"].abs() + (2.0 ** -10 / 448 * 1.01 * top[0] if half else 0)).all())
        assert bool(((v.sqrt() - s["exp_avg_sq"].sqrt()).abs() <= half * s["exp_avg_sq"].sqrt() + (2.0 ** -10 / 448 * 1.01 * top[1] if half else 2.0 ** -22 * top[1])).all())
        assert float(o.state[q]["step"]) == 1
    back = opt.AdamW(_params(F32), **HYPER, state_bits=40 - bits)
    back.load_state_dict(o.state_dict())
    _grads(back.param_groups[0]["params"], 1)
    back.step()


# Values that are not finite stay where they are: in their element, in 8 bits too.
@pytest.mark.parametrize("eight", [False, True])
def test_gradients_that_are_not_finite(opt, eight):
    t, u = _lists([600], F32, F32, eight), _lists([600], F32, F32, eight)
    t["g"][0][5], t["g"][0][300] = float("inf"), float("nan")
    _call(opt, t)
    _call(opt, u)
    bad = torch.zeros(600, dtype=torch.bool, device=DEV)
    bad[5] = bad[300] = True
    assert bool(t["p"][0][bad].isnan().all()) and torch.equal(t["p"][0][~bad], u["p"][0][~bad])
    m, v = _values(t)
    assert not bool(m[0][bad].isfinite().any()) and bool(m[0][~bad].isfinite().all()) and bool(v[0][~bad].isfinite().all())
    # with clipping the norm is not finite either, as after torch.nn.utils.clip_grad_norm_
    w = _lists([600], F32, F32, eight)
    w["g"][0][300] = float("nan")
    assert bool(_call(opt, w, max_norm=1.0).isnan()) and bool(w["p"][0].isnan().all())


def test_zero_and_tiny_blocks_in_8_bits(opt):
    t = _lists([512], F32, F32, True)
    for n in ("m", "v"):
        t[n][0] = torch.zeros(512, device=DEV).to(F8)
    t["g"][0].zero_()
    t["g"][0][300] = 1e-37
    _call(opt, t)
    m, v = _values(t)
    assert not bool(m[0].any()) and not bool(v[0].any()) and bool(t["p"][0].isfinite().all())


def test_learning_rate_on_the_device_and_captured_steps(opt):
    ps, qs = _params(F32), _params(F32)
    lr = torch.full((), HYPER["lr"], device=DEV)
    for group in (ps, qs):
        _grads(group, 0)
    a = opt.AdamW(ps, **{**HYPER, "lr": lr}, state_bits=8, max_norm=0.5)
    b = opt.AdamW(qs, **HYPER, state_bits=8, max_norm=0.5)
    a.step()                                                 # the states are made before the capture
    b.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for k in range(1, 4):
        g = torch.Generator().manual_seed(k)
        for p, q in zip(ps, qs):
            q.grad = (torch.randn(*p.shape, generator=g) * 0.02).to(DEV)
            p.grad.copy_(q.grad)
        lr.fill_(HYPER["lr"] / k)
        b.param_groups[0]["lr"] = HYPER["lr"] / k
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        # the learning rate is 32 bits there and 64 here
        for p, q in zip(ps, qs):
            assert float((p - q).detach().abs().max()) <= k * 2.0 ** -20 * HYPER["lr"] * 8
        assert torch.equal(a.grad_norm, b.grad_norm)
    assert all(float(a.state[p]["step"]) == 4 for p in ps)


def test_a_first_step_is_not_captured(opt, monkeypatch):
    """States made inside a capture would be made again, as zeros, by every replay."""
    ps = _params(F32)
    o = opt.AdamW(ps, **HYPER)
    _grads(ps, 0)
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="captured"):
            o.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, _params(F32)))
    o.step()
    ps[1].grad = None
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="captured"):
            o.step()
    o.step()
    assert [float(o.state[p]["step"]) for p in ps] == [2, 1, 2, 2]


def test_updates_are_seen_by_autograd_and_other_streams(opt):
    p = torch.nn.Parameter(torch.ones(100, device=DEV))
    o = opt.AdamW([p], **HYPER)
    loss = (p * p).sum()
    p.grad = torch.ones_like(p)
    o.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    q = torch.nn.Parameter(torch.ones(100, device=DEV))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        r = opt.AdamW([q], **HYPER)
        q.grad = torch.ones_like(q)
        r.step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(p, q)


def test_a_tensor_past_32_bits(opt):
    """Elements past 2^31 (and bytes past 2^32) of one tensor, 8-bit states, with a small one behind it."""
    n = (1 << 31) + 3 * 2048 + 77
    t = _lists([777], BF, BF, True)
    big = {"p": torch.zeros(n, dtype=BF, device=DEV), "g": torch.zeros(n, dtype=BF, device=DEV),
           "m": torch.zeros(n, dtype=torch.uint8, device=DEV).view(F8), "v": torch.zeros(n, dtype=torch.uint8, device=DEV).view(F8)}
    scales = [torch.zeros(-(-n // 256), device=DEV) for _ in range(2)]
    at = n - 77 - 700                                      # the last whole blocks and the ragged end, in a copy
    at -= at % 256
    small = _lists([n - at], BF, BF, True, seed=4)
    for k in "pgmv":
        big[k][at:].copy_(small[k][0])
    for s, part in zip(scales, small["scales"]):
        s[at // 256:] = part[0]
    both = {k: [big[k], t[k][0].clone()] for k in "pgmv"}
    opt.adamw_step(both["p"], both["g"], both["m"], both["v"], torch.full((), 6.0, device=DEV),
                   scales=([scales[0], t["scales"][0][0].clone()], [scales[1], t["scales"][1][0].clone()]), **HYPER)
    _call(opt, small)
    _call(opt, t)
    for k in "pmv":
        assert torch.equal(big[k][at:].view(torch.uint8), small[k][0].view(torch.uint8))
        assert torch.equal(both[k][1].view(torch.uint8), t[k][0].view(torch.uint8))
    # the rest is 0 / (0 + eps) = 0 of a parameter of zero
    assert not bool(big["p"][:at].any()) and not bool(scales[0][:at // 256].any())
    norm = opt.grad_norm(both["g"])
    want = sum(float(g.double().square().sum()) for g in (small["g"][0], t["g"][0])) ** 0.5
    assert abs(float(norm) - want) <= 2.0 ** -23 * want


@pytest.mark.parametrize("bits", [8, 32])
def test_a_copy_of_the_optimizer_goes_on_by_itself(opt, bits):
    ps = _params(F32)
    a = opt.AdamW(ps, **HYPER, state_bits=bits, max_norm=0.3, min_8bit_numel=100)
    _grads(ps, 0)
    a.step()
    b = copy.deepcopy(a)
    qs = [q for g in b.param_groups for q in g["params"]]
    assert (b.state_bits, b.max_norm, b.min_8bit_numel) == (bits, 0.3, 100) and qs[0] is not ps[0]
    for k in (1, 2):
        _grads(ps, k)
        _grads(qs, k)
        a.step()
        if k == 1:
            assert float(b.state[qs[0]]["step"]) == 1
        b.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs)) and float(b.state[qs[3]]["step"]) == 3


def test_a_scheduler_and_a_learning_rate_on_the_cpu(opt):
    ps, qs = _params(F32), _params(F32)
    a = opt.AdamW(ps, **{**HYPER, "lr": torch.tensor(1e-2)})
    b = opt.AdamW(qs, **HYPER)
    for o in (a, b):
        s = torch.optim.lr_scheduler.LambdaLR(o, lambda k: 0.5 ** k)
        group = [p for g in o.param_groups for p in g["params"]]
        for k in range(3):
            _grads(group, k)
            o.step()
            s.step()
    # 0.01 in 32 bits and in 64
    assert all(float((p - q).detach().abs().max()) <= 3 * 2.0 ** -18 * 1e-2 + 2.0 ** -24 for p, q in zip(ps, qs))


def test_refusals(opt):
    t = _lists([64, 64], F32, F32, False)
    before = [x.clone() for x in t["p"]]

    def refused(err, **kw):
        a = {**t, **kw}
        with pytest.raises(err):
            opt.adamw_step(a["p"], a["g"], a["m"], a["v"], a["step"], scales=a["scales"], **HYPER)

    refused(ValueError, p=[t["p"][0], t["p"][0]])                     # the same tensor twice
    refused(ValueError, m=[t["m"][0], t["m"][0]])
    refused(ValueError, p=[t["p"][0], t["g"][1]])                     # a parameter that is also a gradient
    refused(ValueError, g=t["g"][:1])
    refused(ValueError, g=[t["g"][0], t["g"][1][:32]])
    refused(TypeError, p=[x.half() for x in t["p"]])
    refused(TypeError, m=[x.to(BF) for x in t["m"]])
    refused(TypeError, p=[])
    refused(ValueError, p=[x.cpu() for x in t["p"]])
    refused(ValueError, step=torch.zeros(2, device=DEV))
    refused(ValueError, step=torch.zeros(()))
    refused(ValueError, m=[x.to(F8) for x in t["m"]], v=[x.to(F8) for x in t["v"]],
            scales=([torch.zeros(2, device=DEV)] * 2, [torch.zeros(1, device=DEV)] * 2))
    refused(TypeError, scales=([torch.zeros(1, device=DEV) for _ in range(2)], [torch.zeros(1, device=DEV) for _ in range(2)]))
    assert float(t["step"]) == 6 and all(torch.equal(a, b) for a, b in zip(before, t["p"]))
    for kw in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-1.0), dict(max_norm=0.0), dict(state_bits=16)):
        with pytest.raises(ValueError):
            opt.AdamW(_params(F32), **{**HYPER, **kw})
    with pytest.raises(TypeError):
        opt.AdamW([torch.nn.Parameter(torch.zeros(4, device=DEV, dtype=torch.float16))])
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.zeros(4)
    with pytest.raises(ValueError):
        opt.AdamW([p]).step()
