"""What is dropped is gone: an infinity or a NaN in a dropped place of the branch or of its gate leaves every output,
gradient and second derivative as a zero there does, bit for bit."""
import pytest
import torch

from tests import philox
from tests.test_dropout_gpu import BF, EPS, F32, make

pytestmark = pytest.mark.gpu
P, SEED = 0.5, 9


def both(N, C, gate, cbias, xt, pt):
    """The inputs with zeros in the dropped places, and with infinities and NaN there."""
    d, ds, dy = make(N, C, gate, cbias, xt, pt, N + C)
    keep = torch.from_numpy(philox.kept(N * C, P, SEED)[0]).view(N, C)
    at = torch.arange(N * C).view(N, C) % 3
    bad = torch.where(at == 0, float("inf"), torch.where(at == 1, float("-inf"), float("nan"))).to(BF)
    zeros, wild = dict(d), dict(d)
    for n in ("branch", "gate"):
        if n in d:
            zeros[n] = torch.where(keep, d[n], torch.zeros((), dtype=BF))
            wild[n] = torch.where(keep, d[n], bad if n == "branch" else bad.flip(0))
    return zeros, wild, ds.cuda(), dy.cuda()


def call(pkg, d, stepwise):
    u = {n: t.cuda().requires_grad_(True) for n, t in d.items()}
    s, y = pkg.residual.residual_norm(u["x"], u["branch"], u["weight"], u["bias"], EPS, gate=u.get("gate"), branch_bias=u.get("branch_bias"),
                                      scale=0.5, stepwise=stepwise, dropout=P, seed=torch.tensor([SEED], device="cuda"))
    return u, s, y


@pytest.mark.parametrize("N,C", [(5, 64), (33, 2048), (6, 8192)])
@pytest.mark.parametrize("gate,cbias,xt,pt", [(True, True, F32, F32), (True, False, BF, BF), (False, True, BF, BF), (False, False, F32, BF)])
@pytest.mark.parametrize("stepwise", [False, True])
def test_gradients(pkg, N, C, gate, cbias, xt, pt, stepwise):
    zeros, wild, ds, dy = both(N, C, gate, cbias, xt, pt)
    got = []
    for d in (zeros, wild):
        u, s, y = call(pkg, d, stepwise)
        got.append([s, y, *torch.autograd.grad((s, y), list(u.values()), (ds, dy))])
    assert all(t.isfinite().all() for t in got[0])
    for name, a, b in zip(["s", "y", *zeros], *got):
        assert torch.equal(a, b), name


@pytest.mark.parametrize("gate,cbias", [(True, True), (False, False)])
def test_second_derivatives(pkg, gate, cbias):
    zeros, wild, ds, dy = both(7, 64, gate, cbias, F32, F32)
    got = []
    for d in (zeros, wild):
        u, s, y = call(pkg, d, False)
        first = torch.autograd.grad((s, y), list(u.values()), (ds, dy), create_graph=True)
        got.append([*first, *torch.autograd.grad(sum(t.float().square().sum() for t in first), [t for n, t in u.items() if n != "bias"])])
    assert all(t.isfinite().all() for t in got[0])
    for a, b in zip(*got):
        assert torch.equal(a, b)
