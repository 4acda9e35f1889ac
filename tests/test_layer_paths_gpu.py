"""What a program may do around the layers' fused path: replace a class's forward, change a norm's parameters
between forward and backward, and count on the memory that the separate operators held."""
import importlib

import pytest
import torch
import torch.utils.checkpoint

from test_residual_gpu import EPS, _inputs
from test_train_step_gpu import _batch, _grads, _model

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16


@pytest.fixture(scope="module")
def pkg():
    return importlib.import_module("rwkv-megatron_amd")


# A forward that a program puts in the class's place is the one that runs, in every module of the class.
@pytest.mark.parametrize("name,calls", [("RWKV6Layer", 3), ("RWKV6ChannelMix", 3), ("LayerNorm", 8)])
def test_a_forward_replaced_on_the_class_runs(pkg, monkeypatch, name, calls):
    M = pkg.modules
    model, (tokens, _) = _model(pkg), _batch()
    want = model(tokens).detach()
    cls, seen = getattr(M, name), []
    own = cls.forward

    def forward(self, *args):
        seen.append(self)
        return own(self, *args)

    monkeypatch.setattr(cls, "forward", forward)
    assert torch.equal(model(tokens), want) and len(seen) == calls


def test_a_call_replaced_on_the_class_runs(pkg, monkeypatch):
    M = pkg.modules
    model, (tokens, _) = _model(pkg), _batch()
    want = model(tokens).detach()
    seen = []

    def call(self, *args):
        seen.append(type(self))
        return torch.nn.Module._call_impl(self, *args)

    monkeypatch.setattr(M.RWKV6Layer, "__call__", call, raising=False)
    assert torch.equal(model(tokens), want) and len(seen) == 3
    monkeypatch.undo()
    monkeypatch.setattr(torch.nn.Module, "__call__", call)
    seen.clear()
    assert torch.equal(model(tokens), want) and seen.count(M.RWKV6Layer) == 3 and seen.count(M.LayerNorm) == 8


def _layer(pkg, bias):
    layer = _model(pkg, bias=bias).layers[1]
    x = torch.randn(70, 2, 128, generator=torch.Generator().manual_seed(3)).to(BF).to(DEV).requires_grad_(True)
    return layer, x


# The separate operators, x + (a + bias) and the norm, keep the sum for the backward and neither x nor a.
@pytest.mark.parametrize("bias", [False, True])
def test_the_time_mix_output_is_not_held_for_the_backward(pkg, bias):
    layer, x = _layer(pkg, bias)
    out, held = [], []
    layer.self_attention.register_forward_hook(lambda m, i, o: out.append(o[0]))

    def pack(t):
        held.append(t)
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        layer(x)
    assert out[0].data_ptr() not in {t.data_ptr() for t in held}


def _call_of_the_layers(pkg, t):
    return pkg._lib.native().residual_norm(t["x"], t["branch"], t["weight"], t["bias"], EPS, t.get("gate"), t.get("branch_bias"), 1.0, True, True)


# The layers' call, whose backward reads the sum as it was stored, beside the public one, whose backward forms it
# again from the inputs: that gives the same bits, so all that follows does.  Widths of one wave, several, two pieces a
# lane; enough rows for the backward's blocks to take them in turn.
@pytest.mark.parametrize("N,C", [(1, 8), (37, 512), (33, 1000), (5, 4104), (3, 8192), (24578, 64), (6150, 2048)])
@pytest.mark.parametrize("stream", [BF, torch.float32])
@pytest.mark.parametrize("cbias", [False, True])
def test_the_stored_sum_gives_the_same_gradients(pkg, N, C, stream, cbias):
    t, ds, dy = _inputs((N,), C, stream, torch.float32, False, cbias, seed=9)
    s, y = pkg.residual.residual_norm(t["x"], t["branch"], t["weight"], t["bias"], EPS, branch_bias=t.get("branch_bias"), stepwise=True)
    s2, y2 = _call_of_the_layers(pkg, t)
    assert torch.equal(s, s2) and torch.equal(y, y2)
    for used in ((s, y), (s,), (y,)):
        other = tuple(s2 if o is s else y2 for o in used)
        grads = tuple(ds if o is s else dy for o in used)
        a = torch.autograd.grad(used, list(t.values()), grads, retain_graph=True, allow_unused=True)
        b = torch.autograd.grad(other, list(t.values()), grads, retain_graph=True, allow_unused=True)
        assert all(torch.equal(u, v) for u, v in zip(a, b))


# Second derivatives go through the saved sum to the inputs; bounds as in test_residual_gpu.py.
@pytest.mark.parametrize("cbias", [False, True])
def test_second_derivative_through_the_stored_sum(pkg, cbias):
    t, ds, dy = _inputs((6,), 64, torch.float32, torch.float32, False, cbias)
    names = list(t)

    def second(fn, u, a, b):
        first = torch.autograd.grad(fn(u), [u[n] for n in names], (a, b), create_graph=True)
        return torch.autograd.grad(sum(v.to(torch.promote_types(v.dtype, torch.float32)).square().sum() for v in first), [u[n] for n in names],
                                   materialize_grads=True, allow_unused=True)

    def exact(u):
        s = u["x"] + (u["branch"] + u["branch_bias"] if cbias else u["branch"])
        return s, torch.nn.functional.layer_norm(s, (64,), u["weight"], u["bias"], EPS)

    got = second(lambda u: _call_of_the_layers(pkg, u), t, ds, dy)
    want = second(exact, {n: v.detach().double().requires_grad_(True) for n, v in t.items()}, ds.double(), dy.double())
    for n, a, b in zip(names, got, want):
        assert float((a.double() - b).abs().max()) <= 2.0 ** -5 * float(b.abs().max()), n


# Of the public call s may be changed in place, whatever the form.
def test_the_sum_of_a_public_call_may_be_changed_in_place(pkg):
    t, ds, dy = _inputs((6,), 64, BF, torch.float32, False, False)
    for stepwise in (False, True):
        call = lambda: pkg.residual.residual_norm(t["x"], t["branch"], t["weight"], t["bias"], EPS, stepwise=stepwise)
        want = torch.autograd.grad(call(), list(t.values()), (ds, dy))
        s, y = call()
        s.add_(1)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad((s, y), list(t.values()), (ds, dy)), want))


# A norm's backward uses the parameters that its forward saw; one of them changed in between (fp32, so the
# kernels of the separate norm worked on a copy) is not an error.
@pytest.mark.parametrize("bias", [False, True])
def test_a_norm_changed_between_forward_and_backward(pkg, bias):
    model, (tokens, labels) = _model(pkg, bias=bias), _batch()
    norms = [m for m in model.modules() if isinstance(m, pkg.modules.LayerNorm)]
    want = _grads(model, model(tokens, labels).mean())
    loss = model(tokens, labels).mean()
    with torch.no_grad():
        for n in norms:
            n.weight.mul_(2)
            n.bias.add_(1)
    for (n, a), b in zip(_grads(model, loss).items(), want.values()):
        assert torch.equal(a, b), n


# The same of the public call, in every type of a norm's parameters; a bf16 weight is held itself, as LayerNorm holds it.
@pytest.mark.parametrize("param", [torch.float32, torch.float16, BF])
@pytest.mark.parametrize("N,C", [(5, 64), (3, 2056), (2, 8192), (700, 512)])
def test_the_public_norm_changed_between_forward_and_backward(pkg, param, N, C):
    t, ds, dy = _inputs((N,), C, BF, param, True, False)
    call = lambda: pkg.residual.residual_norm(t["x"], t["branch"], t["weight"], t["bias"], EPS, gate=t["gate"])
    want = torch.autograd.grad(call(), list(t.values()), (ds, dy))
    out = call()
    with torch.no_grad():
        t["bias"].add_(1)
        if param != BF:
            t["weight"].mul_(2)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, list(t.values()), (ds, dy)), want))
    out = call()
    with torch.no_grad():
        t["weight"].mul_(2)
    if param == BF:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(out, list(t.values()), (ds, dy))


# The saved sum is an output of its own node: offloaded, checkpointed, used twice, and freed with the graph.
def test_offloading_checkpoints_and_two_backwards(pkg):
    layer, x = _layer(pkg, True)
    leaves = [x, *layer.parameters()]
    grads = lambda y, **kw: torch.autograd.grad(y.float().square().mean(), leaves, **kw)
    want = grads(layer(x))
    same = lambda got: all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(DEV)):
        y = layer(x)
    assert same(grads(y))
    assert same(grads(torch.utils.checkpoint.checkpoint(layer, x, use_reentrant=False)))
    y = layer(x)
    assert same(grads(y, retain_graph=True)) and same(grads(y))
    with pytest.raises(RuntimeError, match="second time"):
        grads(y)


def test_a_graph_without_a_backward_is_freed(pkg):
    model, (tokens, labels) = _model(pkg), _batch()
    model(tokens, labels)
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated()
    for _ in range(3):
        loss = model(tokens, labels)
        assert torch.cuda.memory_allocated() > held
        del loss
        assert torch.cuda.memory_allocated() == held
    loss = model(tokens, labels).mean()
    loss.backward()
    model.zero_grad(set_to_none=True)
    del loss
    assert torch.cuda.memory_allocated() == held
