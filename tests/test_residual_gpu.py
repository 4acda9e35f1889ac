"""residual.residual_norm: values and gradients against the formula in float64 and against
differences, the forms an input can have, and the layer and model that call it."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32, F16 = torch.bfloat16, torch.float32, torch.float16
EPS = 1e-5


@pytest.fixture(scope="module")
def rn():
    return importlib.import_module("rwkv-megatron_amd").residual.residual_norm


def _inputs(shape, C, stream, param, gate, cbias, seed=0):
    g = torch.Generator().manual_seed(seed + 131 * C + shape[0])
    mk = lambda *s: torch.randn(*s, generator=g)
    t = {"x": (mk(*shape, C) * 2 + 0.5).to(stream), "branch": mk(*shape, C).to(BF),
         "weight": (mk(C) * 0.3 + 1).to(param), "bias": mk(C).to(param)}
    if gate:
        t["gate"] = (2 * mk(*shape, C)).to(BF)
    if cbias:
        t["branch_bias"] = (0.5 * mk(C)).to(param)
    t = {n: v.to(DEV).requires_grad_(True) for n, v in t.items()}
    return t, mk(*shape, C).to(stream).to(DEV), mk(*shape, C).to(BF).to(DEV)


def _formula(t, scale):
    d = {n: v.detach().double().requires_grad_(True) for n, v in t.items()}
    f = d["branch"] + (d["branch_bias"] if "branch_bias" in d else 0)
    s = d["x"] + scale * (f * torch.sigmoid(d["gate"]) if "gate" in d else f)
    m = s.mean(-1, keepdim=True)
    r = ((s - m).square().mean(-1, keepdim=True) + EPS).rsqrt()
    return d, s, (s - m) * r, r


# Rows at the edges of a wave's 512 channels, of one to eight waves a row (of 1024 channels each above
# 4096), of the row groups of a block (four, two, one) and of the backward's ranges; every mix of types.
CASES = [
    ((1,), 8, BF, BF, True, True, 1.0), ((3,), 64, F32, F32, False, False, 1.0), ((5, 1), 512, BF, F32, True, False, 0.5),
    ((9,), 520, F32, BF, True, True, 2.0), ((2, 4), 1000, BF, BF, False, True, 1.0), ((33,), 1024, F32, F32, True, True, 1.0),
    ((7,), 1032, BF, F32, False, False, 1.0), ((777, 1), 2048, BF, BF, True, False, 1.0), ((6,), 2056, F32, F32, False, True, 0.1),
    ((17,), 4096, BF, BF, False, False, 1.0), ((5,), 4104, F32, F32, True, True, 1.0), ((3,), 8192, BF, F32, True, False, 1.0),
    ((4099,), 64, BF, F32, True, True, 1.0), ((2500,), 1024, BF, F16, False, False, -0.25)]


# Bounds: one rounding of the output's type (half a step: eps / 2 of the value), and the 32-bit
# evaluation's.  That evaluates s with a few roundings of |s| and its parts (2^-22 of them), a mean over C
# values with an error below 2^-18 of their largest (at most 2^4 additions a lane and 8 levels, and the
# reciprocal root), and sums over the rows below 2^-17 of the sum of the magnitudes.
@pytest.mark.parametrize("shape,C,stream,param,gate,cbias,scale", CASES)
def test_matches_float64(rn, shape, C, stream, param, gate, cbias, scale):
    t, ds, dy = _inputs(shape, C, stream, param, gate, cbias)
    call = lambda: rn(t["x"], t["branch"], t["weight"], t["bias"], EPS, gate=t.get("gate"),
                      branch_bias=t.get("branch_bias"), scale=scale)
    s, y = call()
    got = dict(zip(t, torch.autograd.grad((s, y), list(t.values()), (ds, dy))))
    s2, y2 = call()
    again = torch.autograd.grad((s2, y2), list(t.values()), (ds, dy))
    assert torch.equal(s, s2) and torch.equal(y, y2) and all(torch.equal(a, b) for a, b in zip(got.values(), again))
    assert s.dtype == stream and y.dtype == BF

    d, S, xh, r = _formula(t, scale)
    Y = xh * d["weight"] + d["bias"]
    want = dict(zip(d, torch.autograd.grad((S, Y), list(d.values()), (ds.double(), dy.double()))))
    half = lambda v: torch.finfo(v.dtype).eps / 2 * 1.01
    top = S.detach().abs().max()
    parts = (d["x"].abs() + abs(scale) * (d["branch"].abs() + (d["branch_bias"].abs() if cbias else 0))).detach()
    near = lambda v, w, slack: bool(((v.double() - w).abs() <= half(v) * w.abs() + slack).all())
    assert near(s.detach(), S.detach(), 2.0 ** -22 * parts)
    exh = 2.0 ** -17 * float(top * r.detach().max())                        # of xh
    assert near(y.detach(), Y.detach(), exh * float(d["weight"].detach().abs().max()) + 2.0 ** -22 * float(d["bias"].detach().abs().max()))
    g = float((dy.double() * d["weight"]).detach().abs().max())
    xm = float(xh.detach().abs().max())
    eds = 2.0 ** -17 * (float(ds.abs().max()) + float(r.detach().max()) * g * (1 + xm)) + float(r.detach().max()) * g * 4 * exh
    fm = float((d["branch"].abs() + (d["branch_bias"].abs() if cbias else 0)).detach().max())
    rows = tuple(range(len(shape)))
    slack = {"x": eds, "branch": abs(scale) * eds, "gate": abs(scale) * fm * eds,
             "weight": 2.0 ** -17 * (dy.double().abs() * xh.detach().abs()).sum(rows) + exh * dy.double().abs().sum(rows),
             "bias": 2.0 ** -17 * dy.double().abs().sum(rows),
             "branch_bias": 2.0 ** -17 * want["branch"].abs().sum(rows) + abs(scale) * eds * (len(S) if len(shape) == 1 else S.shape[0] * S.shape[1])}
    for n in t:
        assert got[n].dtype == t[n].dtype and got[n].shape == t[n].shape
        assert near(got[n], want[n], slack[n]), (n, float((got[n].double() - want[n]).abs().max()))


# Stepwise: the stream bit for bit that of the separate operators (a gate's sigmoid is the same function in
# both); y up to the order of a row's sums, which moves a value by 2^-20 of the row's largest at most and so
# over a rounding's edge now and then: one step of bf16 (2^-7 of it).  The gradients likewise: for a row in one
# wave the order is the same, and the compiler's choice of fused multiply-adds may move a value by 2^-23
# before its rounding, over an edge once in 2^15 values or so; the parameters' are sums in other orders.
@pytest.mark.parametrize("C", [64, 512, 1024, 2056])
@pytest.mark.parametrize("gate,cbias", [(False, False), (True, False), (False, True), (True, True)])
def test_stepwise_is_the_operators_one_by_one(rn, C, gate, cbias):
    pkg = importlib.import_module("rwkv-megatron_amd")
    t, ds, dy = _inputs((37,), C, BF, F32, gate, cbias, seed=5)
    if cbias:
        t["branch_bias"] = t["branch_bias"].detach().to(BF).requires_grad_(True)
    norm = pkg.modules.LayerNorm(C, eps=EPS, device=DEV)
    norm.weight, norm.bias = torch.nn.Parameter(t["weight"].detach()), torch.nn.Parameter(t["bias"].detach())
    f = t["branch"] + t["branch_bias"] if cbias else t["branch"]
    s1 = t["x"] + (pkg.channelmix.sigmoid_gate(f, t["gate"]) if gate else f)
    y1 = norm(s1)
    names = [n for n in t if n not in ("weight", "bias")]
    want = dict(zip([*names, "weight", "bias"], torch.autograd.grad((s1, y1), [*[t[n] for n in names], norm.weight, norm.bias], (ds, dy))))
    s2, y2 = _call(rn, t, stepwise=True)
    assert torch.equal(s1, s2)
    a, b = y1.detach().double(), y2.detach().double()
    assert bool(((a - b).abs() <= 2.0 ** -7 * a.abs() + 2.0 ** -18 * float(a.abs().max())).all())
    assert C > 512 or torch.equal(y1, y2)                    # one wave a row in both
    got = dict(zip(t, torch.autograd.grad((s2, y2), list(t.values()), (ds, dy))))
    for n in ("x", "branch", *(["gate"] if gate else [])):
        a, b = want[n].double(), got[n].double()
        assert float((a != b).double().mean()) <= 2.0 ** -8, n
        assert bool(((a - b).abs() <= 2.0 ** -6 * a.abs() + 2.0 ** -16 * float(a.abs().max())).all()), n
    for n in ("weight", "bias", *(["branch_bias"] if cbias else [])):
        half = 2.0 ** -7 if got[n].dtype == BF else 0
        assert bool(((got[n].double() - want[n].double()).abs() <= half * want[n].double().abs() + 2.0 ** -12).all()), n


# L = <s, ds> + <y, dy> between two points along the gradient.  An output's rounding, half a step of bf16
# (2^-9 of it on average), enters L at random: sqrt(N C) 2^-9 |y dy| at most, against a difference of 2 h
# |grad|, |grad| >= sqrt(N C) / 2 here and h = 2: below 2^-8; the third derivative adds less than that.
@pytest.mark.parametrize("name", ["x", "branch", "gate", "weight", "bias", "branch_bias"])
def test_gradient_against_differences(rn, name):
    t, ds, dy = _inputs((40,), 256, F32, F32, True, True, seed=3)

    def value(v):
        a = {**{n: p.detach() for n, p in t.items()}, name: v}
        s, y = rn(a["x"], a["branch"], a["weight"], a["bias"], EPS, gate=a["gate"], branch_bias=a["branch_bias"])
        return float((s.double() * ds.double()).sum() + (y.double() * dy.double()).sum())

    s, y = rn(t["x"], t["branch"], t["weight"], t["bias"], EPS, gate=t["gate"], branch_bias=t["branch_bias"])
    grad = torch.autograd.grad((s, y), t[name], (ds, dy))[0].double()
    p = t[name].detach()
    move = 2 * grad / grad.norm()
    hi, lo = (p + move).to(p.dtype), (p - move).to(p.dtype)           # bf16 points: the step as it was taken
    want = float((grad * (hi.double() - lo.double())).sum())
    assert abs(value(hi) - value(lo) - want) <= 2.0 ** -6 * abs(want)


def _call(rn, t, **kw):
    return rn(t["x"], t["branch"], t["weight"], t["bias"], EPS, gate=t.get("gate"), branch_bias=t.get("branch_bias"), **kw)


@pytest.mark.parametrize("form", ["transposed", "shifted", "expanded"])
def test_inputs_that_need_a_copy(rn, form):
    t, ds, dy = _inputs((6, 5), 64, BF, F32, True, True)
    base = torch.autograd.grad(_call(rn, t), list(t.values()), (ds, dy))

    def as_form(v):
        v = v.detach()
        if v.dim() < 3:
            return v.clone().requires_grad_(True)
        if form == "transposed":
            v = v.transpose(0, 1).contiguous().transpose(0, 1)
        elif form == "shifted":
            v = torch.cat([v.reshape(-1)[:1], v.reshape(-1)])[1:].view(v.shape)
        return v.requires_grad_(True)

    u = {n: as_form(v) for n, v in t.items()}
    if form == "expanded":
        row = t["gate"].detach()[:1, :1].clone().requires_grad_(True)
        full = row.detach().expand(6, 5, 64).contiguous().requires_grad_(True)
        a = torch.autograd.grad(_call(rn, {**u, "gate": row.expand(6, 5, 64)}), row, (ds, dy))[0]
        b = torch.autograd.grad(_call(rn, {**u, "gate": full}), full, (ds, dy))[0]
        # torch adds the 30 gradients in 32 bits and rounds once
        want = b.double().sum((0, 1), keepdim=True)
        assert bool(((a.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18 * b.double().abs().sum((0, 1))).all())
        return
    got = torch.autograd.grad(_call(rn, u), list(u.values()), (ds.transpose(0, 1).contiguous().transpose(0, 1), dy))
    assert all(torch.equal(a, b) for a, b in zip(base, got))


# Rows enough for the backward's blocks to take them in turn (6144 steps of a block's four, two or one rows
# and more), the last run cut short: a row's gradients are those that it has among few rows, bit for bit, and
# the parameters' are the sums, each in 32 bits below 2^-17 of the magnitudes' sum (as above).
@pytest.mark.parametrize("N,C", [(24578, 64), (12291, 1024), (6150, 2048), (6144, 4104)])
@pytest.mark.parametrize("cbias", [False, True])
def test_rows_in_turn(rn, N, C, cbias):
    t, ds, dy = _inputs((N,), C, BF, F32, False, cbias)
    rows, params = [n for n in t if t[n].dim() > 1], [n for n in t if t[n].dim() == 1]
    got = dict(zip(t, torch.autograd.grad(_call(rn, t), list(t.values()), (ds, dy))))
    for i in range(0, N, 1500):
        u = {n: (v.detach()[i:i + 1500].requires_grad_(True) if n in rows else v) for n, v in t.items()}
        part = torch.autograd.grad(_call(rn, u), [u[n] for n in rows], (ds[i:i + 1500], dy[i:i + 1500]))
        assert all(torch.equal(a, got[n][i:i + 1500]) for a, n in zip(part, rows))
    d, _, xh, _ = _formula(t, 1.0)
    sums = {"weight": dy.double() * xh.detach(), "bias": dy.double(), "branch_bias": got["branch"].double()}
    for n in params:
        # xh itself is off by 2^-17 of the largest s / std at most, d_branch by half a step of bf16 a row
        w = sums[n]
        slack = 2.0 ** -17 * w.abs().sum(0)
        if n == "weight":
            slack = slack + 2.0 ** -17 * float(xh.detach().abs().max() + 1) * dy.double().abs().sum(0)
        if n == "branch_bias":
            slack = slack + 2.0 ** -9 * 1.01 * w.abs().sum(0)
        assert bool(((got[n].double() - w.sum(0)).abs() <= slack).all()), n


@pytest.mark.parametrize("used", ["s", "y"])
@pytest.mark.parametrize("gate", [False, True])
def test_an_output_no_loss_uses(rn, used, gate):
    t, ds, dy = _inputs((21,), 128, BF, BF, gate, False)
    zero_s, zero_y = torch.zeros_like(ds), torch.zeros_like(dy)
    s, y = _call(rn, t)
    want = torch.autograd.grad((s, y), list(t.values()), (ds, zero_y) if used == "s" else (zero_s, dy))
    s, y = _call(rn, t)
    got = torch.autograd.grad(s if used == "s" else y, list(t.values()), ds if used == "s" else dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_frozen_parameters_and_no_grad(rn):
    t, ds, dy = _inputs((21,), 1024, BF, F32, True, True)
    s, y = _call(rn, t)
    base = torch.autograd.grad((s, y), (t["x"], t["branch"], t["gate"]), (ds, dy))
    u = {n: (v if n in ("x", "branch", "gate") else v.detach()) for n, v in t.items()}
    out = _call(rn, u)
    assert all(torch.equal(a, b) for a, b in zip(base, torch.autograd.grad(out, (u["x"], u["branch"], u["gate"]), (ds, dy))))
    only = {n: v.detach() for n, v in t.items()}
    only["branch_bias"].requires_grad_(True)
    full = torch.autograd.grad(_call(rn, t), t["branch_bias"], (ds, dy))[0]
    assert torch.equal(torch.autograd.grad(_call(rn, only), only["branch_bias"], (ds, dy))[0], full)
    with torch.no_grad():
        s1, y1 = _call(rn, t)
    assert torch.equal(s1, s) and torch.equal(y1, y) and not s1.requires_grad


def test_empty(rn):
    t, ds, dy = _inputs((2,), 64, BF, F32, True, True)
    u = {n: (v.detach()[:0].requires_grad_(True) if v.dim() > 1 else v) for n, v in t.items()}
    s, y = _call(rn, u)
    assert s.shape == (0, 64)
    g = torch.autograd.grad((s, y), list(u.values()), (ds[:0], dy[:0]))
    assert all(a.shape == v.shape and not bool(a.any()) for a, v in zip(g, u.values()))


# A row of the lowest numbers, a gate of minus or plus infinity, and a NaN: they stay in their rows.
def test_values_at_the_edge(rn):
    t, ds, dy = _inputs((6,), 128, BF, F32, True, False)
    clean = [v.detach() for v in _call(rn, t)]
    with torch.no_grad():
        t["gate"][1] = float("-inf")
        t["gate"][2] = float("inf")
        t["x"][4, 3] = float("nan")
    s, y = _call(rn, t)
    assert torch.equal(s[1], t["x"][1]) and torch.equal(s[2], (t["x"][2].float() + t["branch"][2].float()).to(BF))
    assert bool(y[4].isnan().all()) and int(s[4].isnan().sum()) == 1
    for i in (0, 3, 5):
        assert torch.equal(s[i], clean[0][i]) and torch.equal(y[i], clean[1][i])
    gx, gg = torch.autograd.grad((s, y), (t["x"], t["gate"]), (ds, dy))
    assert not bool(gg[1].any()) and not bool(gg[2].any())            # sg (1 - sg) = 0
    assert bool(gx[[0, 1, 2, 3, 5]].isfinite().all()) and bool(gx[4].isnan().all())


# Second derivatives run through torch's operators in 32 bits: against float64, with the bf16 roundings
# of the first gradients (2^-8 each) between the two passes.
def test_second_derivative(rn):
    t, ds, dy = _inputs((6,), 64, F32, F32, True, True)
    names = list(t)

    def second(fn, u, a, b):
        first = torch.autograd.grad(fn(u), [u[n] for n in names], (a, b), create_graph=True)
        return torch.autograd.grad(sum(v.to(torch.promote_types(v.dtype, F32)).square().sum() for v in first), [u[n] for n in names],
                                   materialize_grads=True, allow_unused=True)

    def exact(u):
        f = u["branch"] + u["branch_bias"]
        s = u["x"] + f * torch.sigmoid(u["gate"])
        return s, torch.nn.functional.layer_norm(s, (64,), u["weight"], u["bias"], EPS)

    got = second(lambda u: _call(rn, u), t, ds, dy)
    want = second(exact, {n: v.detach().double().requires_grad_(True) for n, v in t.items()}, ds.double(), dy.double())
    for n, a, b in zip(names, got, want):
        assert float((a.double() - b).abs().max()) <= 2.0 ** -5 * float(b.abs().max()), n


def test_saved_tensors_and_transforms(rn):
    t, ds, dy = _inputs((7,), 64, BF, F32, True, True)
    base = torch.autograd.grad(_call(rn, t), list(t.values()), (ds, dy))
    with torch.autograd.graph.saved_tensors_hooks(lambda v: v.cpu(), lambda v: v.to(DEV)):
        out = _call(rn, t)
    assert all(torch.equal(a, b) for a, b in zip(base, torch.autograd.grad(out, list(t.values()), (ds, dy))))
    out = _call(rn, t)
    with torch.no_grad():
        t["gate"].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, list(t.values()), (ds, dy))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda x: rn(x, t["branch"][0], t["weight"], t["bias"], EPS)[1])(t["x"])
    x, branch, w, b = (t[n].detach() for n in ("x", "branch", "weight", "bias"))
    with torch.autograd.forward_ad.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        rn(torch.autograd.forward_ad.make_dual(x, x), branch, w, b, EPS)


def test_graph_replays_and_another_stream(rn):
    t, ds, dy = _inputs((130,), 512, BF, F32, True, True)
    step = lambda: [v.detach() for v in _call(rn, t)] + list(torch.autograd.grad(_call(rn, t), list(t.values()), (ds, dy)))
    want = [v.clone() for v in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for rep in range(3):
        with torch.no_grad():
            for v in out:
                v.zero_()
        torch.randn(512, 512, device=DEV).sum().item()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, out)), rep


def test_a_single_row_without_batch_and_two_streams_at_once(rn):
    t, ds, dy = _inputs((1,), 256, BF, F32, True, True)
    a = _call(rn, t)
    u = {n: (v.detach()[0] if v.dim() > 1 else v.detach()).requires_grad_(True) for n, v in t.items()}
    b = _call(rn, u)
    assert b[0].shape == (256,) and torch.equal(a[0][0], b[0]) and torch.equal(a[1][0], b[1])
    ga = torch.autograd.grad(a, list(t.values()), (ds, dy))
    gb = torch.autograd.grad(b, list(u.values()), (ds[0], dy[0]))
    assert all(torch.equal(p.reshape(q.shape), q) for p, q in zip(ga, gb))

    sets = [_inputs((3000,), 512, BF, F32, True, True, seed=k) for k in (11, 12)]
    run = lambda t, ds, dy: torch.autograd.grad(_call(rn, t), list(t.values()), (ds, dy))
    want = [run(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [None, None]
    for _ in range(3):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k] = run(*sets[k])
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(a, b) for a, b in zip(w, g))


def test_offsets_past_32_bits(rn):
    """Rows further than 2^31 elements (and 2^32 bytes) into the tensors."""
    N, C = 540_000, 4096
    x, branch, dy = (torch.zeros(N, C, device=DEV, dtype=BF) for _ in range(3))
    rows = [0, 1, 262_143, 262_144, 524_287, 524_288, 539_999]
    t, ds, g = _inputs((len(rows),), C, BF, F32, False, False)
    with torch.no_grad():
        for k, r in enumerate(rows):
            x[r], branch[r], dy[r] = t["x"][k], t["branch"][k], g[k]
    x.requires_grad_(True)
    s, y = rn(x, branch, t["weight"].detach(), t["bias"].detach(), EPS)
    small = rn(t["x"].detach().requires_grad_(True), t["branch"].detach(), t["weight"].detach(), t["bias"].detach(), EPS)
    assert torch.equal(s[rows], small[0]) and torch.equal(y[rows], small[1])
    assert not bool(s.detach().view(-1)[C * 2:C * 262_143].any())
    xs = t["x"].detach().requires_grad_(True)
    want = torch.autograd.grad(rn(xs, t["branch"].detach(), t["weight"].detach(), t["bias"].detach(), EPS)[1], xs, g)[0]
    got = torch.autograd.grad(y, x, dy)[0]
    assert torch.equal(got[rows], want) and not bool(got[2:262_143].any())


def test_refusals(rn):
    t, _, _ = _inputs((4,), 64, BF, F32, True, True)
    a = {n: v.detach() for n, v in t.items()}
    call = lambda **kw: _call(rn, {**a, **kw})
    with pytest.raises(TypeError):
        call(branch=a["branch"].float())
    with pytest.raises(TypeError):
        call(x=a["x"].half())
    with pytest.raises(TypeError):
        call(weight=a["weight"].double())
    with pytest.raises(ValueError):
        call(gate=a["gate"][:3])
    with pytest.raises(ValueError):
        call(branch_bias=a["branch_bias"][:32])
    with pytest.raises(ValueError):
        call(weight=a["weight"].cpu())
    with pytest.raises(ValueError):
        call(x=a["x"].cpu())
    for C in (12, 8200):
        z = torch.zeros(2, C, device=DEV, dtype=BF)
        with pytest.raises(NotImplementedError):
            rn(z, z, z[0], z[0], EPS)
