"""Dropout in the layers: the kernels' stepwise gradients, what stands for a call that they do not take, and which
numbers either draws."""
import pytest
import torch

from tests import philox

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _norm(pkg, C=128):
    return pkg.modules.LayerNorm(C, eps=1e-5, device="cuda", dtype=BF)


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("cbias", [False, True])
def test_the_separate_operators_draw_once(pkg, gate, cbias):
    """Under autocast the kernel is not called: the numbers are those of one F.dropout from the generator's state."""
    G = torch.Generator(device="cuda").manual_seed(1)
    n = lambda *s: torch.randn(*s, generator=G, device="cuda").to(BF)
    x, f, b, g, norm = n(30, 2, 128), n(30, 2, 128), n(128), n(30, 2, 128), _norm(pkg)
    with torch.no_grad():
        torch.manual_seed(3)
        with torch.autocast("cuda", dtype=BF):
            s, y = pkg.modules._add_norm(norm, x, f, b if cbias else None, g if gate else None, dropout=0.5)
        after = torch.cuda.get_rng_state()
        whole = f + b if cbias else f
        if gate:
            whole = pkg.channelmix.sigmoid_gate(whole, g)
        torch.manual_seed(3)
        assert torch.equal(s, x + torch.nn.functional.dropout(whole, 0.5))
        assert torch.equal(after, torch.cuda.get_rng_state())


def test_the_fused_call_draws_one_number(pkg):
    """The mask is that of a seed from torch.randint at the generator's state."""
    x, f, norm = torch.zeros(40, 2, 128, device="cuda", dtype=BF), torch.ones(40, 2, 128, device="cuda", dtype=BF), _norm(pkg)
    with torch.no_grad():
        torch.manual_seed(4)
        s, _ = pkg.modules._add_norm(norm, x, f, dropout=0.25)
        after = torch.cuda.get_rng_state()
        torch.manual_seed(4)
        seed = torch.randint(2 ** 63 - 1, (1,), device="cuda")
        assert torch.equal(after, torch.cuda.get_rng_state())
        want, _ = pkg.residual.residual_norm(x, f, norm.weight, norm.bias, 1e-5, stepwise=True, dropout=0.25, seed=seed)
    assert torch.equal(s, want)


# The layers' call (its backward reads the stored sum where there is no gate) and the public one, against the operators
# one by one under the same mask, which round at the same places: a value differs where the norm's 32-bit sums, taken in
# another order, put it on the other side of a rounding, once in 2^8 values at most, and then by a step there, 2^-7 of the value.
# In a bf16 stream d_x is ds and the norm's part e, each sum rounded: a step of e, |e| <= |d_x| + |ds|, and one of d_x.  With the
# factor 1 / (1 - p) the branch's takes a step of the scaled and one of the dropped-out gradient more, and with a gate one of
# the product (d_gate: sigmoid' <= 1/4).  In 32 bits the sums' other order is 2^-16 of the largest at most; the
# parameters' gradients are such sums.
@pytest.mark.parametrize("N,C", [(37, 64), (37, 512), (37, 2056), (700, 128)])
@pytest.mark.parametrize("stream", [BF, torch.float32])
@pytest.mark.parametrize("layers", [True, False])
@pytest.mark.parametrize("gate,cbias", [(False, False), (False, True), (True, False), (True, True)])
def test_stepwise_gradients_are_the_operators(pkg, N, C, stream, layers, gate, cbias):
    p, key = 0.3, 1234567 + C
    G = torch.Generator().manual_seed(N + C)
    n = lambda *s: torch.randn(*s, generator=G)
    t = {"x": (2 * n(N, C)).to(stream), "branch": n(N, C).to(BF), "weight": 1 + 0.3 * n(C), "bias": 0.1 * n(C)}
    if gate:
        t["gate"] = n(N, C).to(BF)
    if cbias:
        t["branch_bias"] = (0.5 * n(C)).to(BF)
    t = {k: v.cuda().requires_grad_(True) for k, v in t.items()}
    ds, dy = n(N, C).to(stream).cuda(), n(N, C).to(BF).cuda()
    keep, factor = philox.kept(N * C, p, key)
    mask = torch.from_numpy(keep).view(N, C).cuda()
    norm = pkg.modules.LayerNorm(C, eps=1e-5, device="cuda")
    norm.weight, norm.bias = torch.nn.Parameter(t["weight"].detach()), torch.nn.Parameter(t["bias"].detach())
    f = t["branch"] + t["branch_bias"] if cbias else t["branch"]
    if gate:
        f = pkg.channelmix.sigmoid_gate(f, t["gate"])
    s1 = t["x"] + f * mask * factor
    y1 = norm(s1)
    names = [k for k in t if k not in ("weight", "bias")]
    want = dict(zip([*names, "weight", "bias"], torch.autograd.grad((s1, y1), [*[t[k] for k in names], norm.weight, norm.bias], (ds, dy))))
    s2, y2 = pkg._lib.native().residual_norm_dropout(t["x"], t["branch"], t["weight"], t["bias"], 1e-5, t.get("gate"), t.get("branch_bias"), 1.0,
                                                     True, layers, p, torch.tensor([key], device="cuda"))
    assert torch.equal(s1, s2)
    got = dict(zip(t, torch.autograd.grad((s2, y2), list(t.values()), (ds, dy))))
    step = 2.0 ** -7
    dx = want["x"].double().abs()
    off = {"x": 2 * step * dx + step * ds.double().abs() if stream == BF else torch.zeros_like(dx)}
    through = factor * (off["x"] + 2 * step * dx)
    off["branch"] = through + step * want["branch"].double().abs()
    if gate:
        whole = t["branch"].double() + (t["branch_bias"].double() if cbias else 0)
        off["gate"] = through * whole.abs() / 4 + step * want["gate"].double().abs()
    for k, limit in off.items():
        a, b = want[k].double(), got[k].double()
        if got[k].dtype == BF:
            assert float((a != b).double().mean()) <= 2.0 ** -8, k
        assert bool(((a - b).abs() <= limit + 2.0 ** -16 * float(a.abs().max())).all()), k
    assert (got["branch"][~mask] == 0).all()
    for k in ("weight", "bias", *(["branch_bias"] if cbias else [])):
        a, b = want[k].double(), got[k].double()
        # sums of N values of size 1 in 32 bits; d_branch_bias of values rounded to bf16, one in 2^8 of them another way
        wide = 2.0 ** -20 * N + (2.0 ** -8 * (N * 2.0 ** -8) ** 0.5 * 8 if k == "branch_bias" else 0)
        assert bool(((a - b).abs() <= (2.0 ** -8 if got[k].dtype == BF else 0) * 2 * a.abs() + wide).all()), k


# Second derivatives through the stored sum; bounds as in test_residual_gpu.py.
@pytest.mark.parametrize("cbias", [False, True])
def test_second_derivative_through_the_stored_sum(pkg, cbias):
    p, key, N, C = 0.3, 99, 6, 64
    G = torch.Generator().manual_seed(2)
    n = lambda *s: torch.randn(*s, generator=G)
    t = {"x": 2 * n(N, C), "branch": n(N, C).to(BF), "weight": 1 + 0.3 * n(C), "bias": 0.1 * n(C)}
    if cbias:
        t["branch_bias"] = 0.5 * n(C)
    t = {k: v.cuda().requires_grad_(True) for k, v in t.items()}
    ds, dy = n(N, C).cuda(), n(N, C).to(BF).cuda()
    keep, factor = philox.kept(N * C, p, key)
    mask = torch.from_numpy(keep).view(N, C).cuda().double() * factor

    def second(fn, u, a, b):
        first = torch.autograd.grad(fn(u), list(u.values()), (a, b), create_graph=True)
        return torch.autograd.grad(sum(v.to(torch.promote_types(v.dtype, torch.float32)).square().sum() for v in first), list(u.values()),
                                   materialize_grads=True, allow_unused=True)

    def exact(u):
        s = u["x"] + (u["branch"] + u["branch_bias"] if cbias else u["branch"]) * mask
        return s, torch.nn.functional.layer_norm(s, (C,), u["weight"], u["bias"], 1e-5)

    def fused(u):
        return pkg._lib.native().residual_norm_dropout(u["x"], u["branch"], u["weight"], u["bias"], 1e-5, None, u.get("branch_bias"), 1.0, True,
                                                       True, p, torch.tensor([key], device="cuda"))

    got = second(fused, t, ds, dy)
    want = second(exact, {k: v.detach().double().requires_grad_(True) for k, v in t.items()}, ds.double(), dy.double())
    for k, a, b in zip(t, got, want):
        assert float((a.double() - b).abs().max()) <= 2.0 ** -5 * float(b.abs().max()), k


def _dropped(added, whole, p):
    """added is whole with a share p of its elements dropped and the others times 1 / (1 - p), up to a rounding of the sum
    that it was taken out of."""
    kept = added != 0
    n = whole.numel()
    assert abs(float(kept.double().mean()) - (1 - p)) <= 5 * (p * (1 - p) / n) ** 0.5 + 1e-3
    return kept


@pytest.mark.parametrize("gate", [False, True])
def test_the_separate_operators_drop(pkg, gate):
    G = torch.Generator(device="cuda").manual_seed(5)
    n = lambda *s: torch.randn(*s, generator=G, device="cuda").to(BF)
    x, f, g, norm = torch.zeros(300, 2, 128, device="cuda", dtype=BF), n(300, 2, 128), n(300, 2, 128), _norm(pkg)
    norm.register_forward_hook(lambda *a: None)

    def call(seed, p=0.25):
        torch.manual_seed(seed)
        with torch.no_grad():
            return pkg.modules._add_norm(norm, x, f, gate=g if gate else None, dropout=p)[0]

    whole = call(0, 0.0)
    s = call(1)
    kept = _dropped(s, whole, 0.25)
    assert torch.equal(s, torch.where(kept, (whole.float() / 0.75).to(BF), torch.zeros_like(s)))
    assert torch.equal(s, call(1)) and not torch.equal(s, call(2))


def test_a_layer_by_itself_drops_the_channel_mix(pkg):
    p = 0.5
    cfg = pkg.modules.TransformerConfig(hidden_size=128, num_attention_heads=2, ffn_hidden_size=256, num_layers=2, hidden_dropout=p)
    torch.manual_seed(0)
    layer = pkg.modules.RWKV6Layer(cfg, device="cuda")
    mixed, stream = [], []
    layer.mlp.register_forward_hook(lambda m, i, o: mixed.append(o[0]))
    layer.pre_mlp_layernorm.register_forward_pre_hook(lambda m, i: stream.append(i[0]))
    x = torch.randn(300, 2, 128, device="cuda").to(BF)

    def call(seed):
        torch.manual_seed(seed)
        with torch.no_grad():
            out = layer(x)
        return out, mixed.pop(), stream.pop()

    layer.train()
    out, m, s = call(1)
    again, other = call(1)[0], call(2)[0]
    assert torch.equal(out, again) and not torch.equal(out, other)
    twice = s + (2 * m.float()).to(BF)
    assert bool(((out == s) | (out == twice)).all())
    seen = twice != s                                      # where adding it shows
    assert abs(float((out[seen] == s[seen]).double().mean()) - p) <= 5 * (p * (1 - p) / int(seen.sum())) ** 0.5
    layer.eval()
    out, m, s = call(1)
    assert torch.equal(out, s + m) and torch.equal(out, call(2)[0])


def test_a_captured_call_of_the_layers_draws_anew(pkg):
    """Each replay has the mask of the next number of the generator, as eager calls one after another."""
    x, f, norm = torch.zeros(40, 2, 128, device="cuda", dtype=BF), torch.ones(40, 2, 128, device="cuda", dtype=BF), _norm(pkg)
    call = lambda: pkg.modules._add_norm(norm, x, f, dropout=0.5)
    with torch.no_grad():
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        for rep in range(3):
            torch.manual_seed(7)
            got = []
            for _ in range(3):
                graph.replay()
                got.append([t.clone() for t in out])
            torch.cuda.synchronize()
            torch.manual_seed(7)
            for a in got:
                assert all(torch.equal(u, v) for u, v in zip(a, call())), rep
        assert not torch.equal(got[0][0], got[1][0])
