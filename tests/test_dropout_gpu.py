"""residual_norm with dropout against the formulas in 64 bits, with the mask drawn on the host, and the layers
that call it.

Tolerances: outputs of one rounding, half a step (2^-8 in bf16, 2^-24 in fp32) of themselves, and the 32-bit
arithmetic before it: 2^-19 of the tensor's largest (a norm of up to 8192 terms and a dozen operations)."""
import copy

import pytest
import torch

from tests import philox

gpu = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
EPS = 1e-5


def test_known_numbers():
    """The generator's published vectors: counter 0 and key 0, and all bits set."""
    assert [hex(x) for x in philox.philox4x32([0], 0)[0]] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]


def make(N, C, gate, cbias, xt, pt, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)
    d = {"x": (2 * n(N, C)).to(xt), "branch": n(N, C).to(BF), "weight": (1 + 0.3 * n(C)).to(pt), "bias": (0.1 * n(C)).to(pt)}
    if gate:
        d["gate"] = n(N, C).to(BF)
    if cbias:
        d["branch_bias"] = (0.5 * n(C)).to(pt)
    return d, n(N, C).to(xt), n(N, C).to(BF)


def definition(d, mask, scale):
    f = d["branch"] + d["branch_bias"] if "branch_bias" in d else d["branch"]
    if "gate" in d:
        f = f * torch.sigmoid(d["gate"])
    s = d["x"] + scale * f * mask
    var, mean = torch.var_mean(s, -1, unbiased=False, keepdim=True)
    return s, (s - mean) / (var + EPS).sqrt() * d["weight"] + d["bias"]


def near(name, got, ref):
    got, ref = got.detach().double().cpu(), ref.detach()
    half = 2.0 ** -8 if got.dtype == BF else 2.0 ** -24
    return (got - ref).abs() - half * ref.abs()


@gpu
@pytest.mark.parametrize("N,C", [(1, 8), (3, 64), (5, 520), (33, 512), (64, 2048), (7, 4104), (17, 8192)])
@pytest.mark.parametrize("gate,cbias,xt,pt,p,scale", [(False, False, BF, BF, 0.1, 1.0), (True, True, F32, F32, 0.5, 0.5),
                                                      (True, False, BF, F32, 0.25, 1.0), (False, True, F32, BF, 0.9, 2.0)])
def test_against_the_formulas(pkg, N, C, gate, cbias, xt, pt, p, scale):
    d, ds, dy = make(N, C, gate, cbias, xt, pt, N + C)
    seed = 0x1234567 * C + (1 << 61) - N
    keep, factor = philox.kept(N * C, p, seed)
    mask = torch.from_numpy(keep).view(N, C).double() * factor
    u = {k: t.cuda().requires_grad_(True) for k, t in d.items()}
    r = {k: t.double().requires_grad_(True) for k, t in d.items()}
    kw = {k: u[k] for k in ("gate", "branch_bias") if k in u}
    key = torch.tensor([seed], device="cuda")
    s, y = pkg.residual.residual_norm(u["x"], u["branch"], u["weight"], u["bias"], EPS, scale=scale, dropout=p, seed=key, **kw)
    key.add_(1)                                             # the backward draws with the value that was read
    rs, ry = definition(r, mask, scale)
    got = torch.autograd.grad((s, y), list(u.values()), (ds.cuda(), dy.cuda()))
    want = torch.autograd.grad((rs, ry), list(r.values()), (ds.double(), dy.double()))
    for name, a, b in [("s", s, rs), ("y", y, ry)] + list(zip(u, got, want)):
        half = 2.0 ** -8 if a.dtype == BF else 2.0 ** -24
        b = b.detach()
        wide = 2.0 ** -19 * max(1.0, N ** 0.5 if b.dim() == 1 else 1.0)
        assert ((a.detach().double().cpu() - b).abs() <= half * b.abs() + wide * b.abs().max().clamp(min=1e-6)).all(), name
    dropped = mask == 0
    assert (got[list(u).index("branch")].cpu()[dropped] == 0).all()
    with torch.no_grad():
        s2, y2 = pkg.residual.residual_norm(u["x"], u["branch"], u["weight"], u["bias"], EPS, scale=scale, dropout=p,
                                            seed=torch.tensor([seed], device="cuda"), **kw)
    assert torch.equal(s, s2) and torch.equal(y, y2)


@gpu
def test_a_dropped_infinity_is_dropped(pkg):
    d, ds, dy = make(16, 64, False, False, BF, BF)
    keep, _ = philox.kept(16 * 64, 0.5, 9)
    d["branch"] = torch.where(torch.from_numpy(keep).view(16, 64), d["branch"], torch.tensor(float("inf"), dtype=BF))
    s, y = pkg.residual.residual_norm(*[d[k].cuda() for k in ("x", "branch", "weight", "bias")], EPS, dropout=0.5,
                                      seed=torch.tensor([9], device="cuda"))
    assert s.isfinite().all() and y.isfinite().all()


@gpu
@pytest.mark.parametrize("gate,cbias", [(False, False), (True, True)])
def test_stepwise_is_the_operators_one_by_one(pkg, gate, cbias):
    d, ds, dy = make(40, 512, gate, cbias, BF, BF, 5)
    u = {k: t.cuda() for k, t in d.items()}
    keep, factor = philox.kept(40 * 512, 0.25, 77)
    mask = torch.from_numpy(keep).view(40, 512).cuda()
    f = u["branch"] + u["branch_bias"] if cbias else u["branch"]
    if gate:
        f = (f.double() * torch.sigmoid(u["gate"].double())).to(BF)
    s = u["x"] + (f * mask * factor)
    kw = {k: u[k] for k in ("gate", "branch_bias") if k in u}
    s2, _ = pkg.residual.residual_norm(u["x"], u["branch"], u["weight"], u["bias"], EPS, stepwise=True, dropout=0.25,
                                       seed=torch.tensor([77], device="cuda"), **kw)
    if gate:                                                # a sigmoid in 32 bits may round the product the other way
        assert (s != s2).float().mean() < 1e-3
    else:
        assert torch.equal(s, s2)


@gpu
def test_a_backward_that_is_differentiated(pkg):
    d, ds, dy = make(4, 64, True, False, F32, F32, 3)
    keep, factor = philox.kept(4 * 64, 0.3, 5)
    mask = torch.from_numpy(keep).view(4, 64).double() * factor
    u = {k: t.cuda().requires_grad_(True) for k, t in d.items()}
    r = {k: t.double().requires_grad_(True) for k, t in d.items()}
    s, y = pkg.residual.residual_norm(u["x"], u["branch"], u["weight"], u["bias"], EPS, gate=u["gate"], dropout=0.3,
                                      seed=torch.tensor([5], device="cuda"))
    rs, ry = definition(r, mask, 1.0)
    second = []
    for outs, t, dd, yy in (((s, y), u, ds.cuda(), dy.cuda()), ((rs, ry), r, ds.double(), dy.double())):
        gx, = torch.autograd.grad(outs, t["x"], (dd, yy), create_graph=True)
        second.append(torch.autograd.grad(gx.square().sum(), t["branch"])[0].double().cpu())
    assert float((second[0] - second[1]).norm() / second[1].norm()) <= 2.0 ** -7


@gpu
def test_no_dropout_is_the_call_without(pkg):
    d, ds, dy = make(9, 256, True, True, BF, BF)
    u = {k: t.cuda() for k, t in d.items()}
    a = pkg.residual.residual_norm(*[u[k] for k in ("x", "branch", "weight", "bias")], EPS, gate=u["gate"], branch_bias=u["branch_bias"])
    b = pkg.residual.residual_norm(*[u[k] for k in ("x", "branch", "weight", "bias")], EPS, gate=u["gate"], branch_bias=u["branch_bias"],
                                   dropout=2.0 ** -18, seed=torch.tensor([1], device="cuda"))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@gpu
def test_refusals(pkg):
    d, _, _ = make(4, 64, False, False, BF, BF)
    a = [d[k].cuda() for k in ("x", "branch", "weight", "bias")]
    call = lambda **kw: pkg.residual.residual_norm(*a, EPS, **kw)
    for p in (-0.1, 1.0, 1.5, float("nan")):
        with pytest.raises(ValueError):
            call(dropout=p, seed=torch.zeros(1, dtype=torch.long, device="cuda"))
    with pytest.raises(TypeError):
        call(dropout=0.1)
    with pytest.raises(TypeError):
        call(dropout=0.1, seed=torch.zeros(2, dtype=torch.long, device="cuda"))
    with pytest.raises(TypeError):
        call(dropout=0.1, seed=torch.zeros(1, device="cuda"))
    with pytest.raises(ValueError):
        call(dropout=0.1, seed=torch.zeros(1, dtype=torch.long))


def _model(pkg, p, **kw):
    torch.manual_seed(0)
    cfg = pkg.modules.TransformerConfig(hidden_size=128, num_attention_heads=2, ffn_hidden_size=256, num_layers=2, hidden_dropout=p, **kw)
    return pkg.modules.RWKV6Model(cfg, 97, device="cuda")


@gpu
def test_the_model_drops_in_training_only(pkg):
    plain, drop = _model(pkg, 0.0), _model(pkg, 0.3)
    drop.load_state_dict(plain.state_dict())
    tokens = torch.randint(0, 97, (2, 50), device="cuda")
    assert torch.equal(plain.eval()(tokens), drop.eval()(tokens))
    plain.train(), drop.train()
    assert not torch.equal(plain(tokens), drop(tokens))
    runs = []
    for _ in range(2):                                      # the same generator state, the same masks
        torch.manual_seed(11)
        drop.zero_grad()
        loss = drop(tokens, tokens).mean()
        loss.backward()
        runs.append([loss.detach()] + [q.grad.clone() for q in drop.parameters() if q.grad is not None])
    assert all(torch.equal(a, b) for a, b in zip(*runs)) and all(x.isfinite().all() for x in runs[0])


@gpu
def test_a_layer_of_other_norms_drops_too(pkg):
    """The path of the separate operators (a hook on the norm): the same expectation, other random numbers."""
    m = _model(pkg, 0.5).train()
    n = copy.deepcopy(m)
    for layer in n.layers:
        layer.pre_mlp_layernorm.register_forward_hook(lambda *a: None)
        layer.input_layernorm.register_forward_hook(lambda *a: None)
    x = torch.randn(64, 2, 128, device="cuda").to(BF)
    with torch.no_grad():
        a = torch.stack([m.layers[0](x).float() for _ in range(200)]).mean(0)
        b = torch.stack([n.layers[0](x).float() for _ in range(200)]).mean(0)
        e = m.layers[0].eval()(x).float()
    # a mean of 200 draws of a variable of deviation |f| (p = 0.5): 0.07 |f| and the layer's own curvature
    spread = (e - x.float()).abs().mean()
    assert (a - b).abs().mean() <= 0.3 * spread


@gpu
def test_a_captured_step_draws_anew_on_each_replay(pkg):
    d, ds, dy = make(32, 256, False, False, BF, BF, 8)
    u = {k: t.cuda() for k, t in d.items()}
    branch = u["branch"].clone().requires_grad_(True)
    key = torch.tensor([41], device="cuda")
    dsc, dyc = ds.cuda(), dy.cuda()

    def step():
        s, y = pkg.residual.residual_norm(u["x"], branch, u["weight"], u["bias"], EPS, dropout=0.4, seed=key)
        g, = torch.autograd.grad((s, y), branch, (dsc, dyc))
        return s, y, g

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
        key.add_(1)
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        keep, _ = philox.kept(32 * 256, 0.4, 41 + i)
        assert ((got[2] == 0).cpu() == ~torch.from_numpy(keep).view(32, 256)).float().mean() > 0.999
        eager = key.clone()
        key.fill_(41 + i)
        want = step()
        key.copy_(eager)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
