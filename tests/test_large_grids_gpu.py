"""Calls of more rows than a launch has blocks for, so that the blocks stride over the rows: the rows of every trip
are those of a small call, bit for bit."""
import importlib
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def pkg():
    return importlib.import_module("rwkv-megatron_amd")


# 2^20 blocks of four rows (a wave each) and of two (two waves each, whose sums go through shared memory, in the two
# arrays that the trips use in turn).
@pytest.mark.parametrize("N,C", [((1 << 22) + 4099, 64), ((1 << 21) + 2051, 1024)])
def test_residual_norm(pkg, N, C):
    g = torch.Generator(device=DEV).manual_seed(C)
    x, branch = (torch.randn(N, C, generator=g, device=DEV, dtype=BF) for _ in range(2))
    w, b = (torch.randn(C, generator=g, device=DEV) for _ in range(2))
    s, y = pkg.residual.residual_norm(x, branch, w, b, 1e-5)
    for i in (0, N // 2, N - 8192, N - 100):
        s1, y1 = pkg.residual.residual_norm(x[i:i + 8192], branch[i:i + 8192], w, b, 1e-5)
        assert torch.equal(s[i:i + 8192], s1) and torch.equal(y[i:i + 8192], y1), i
    # no row is left out: a value of every row is the sum's
    assert torch.equal(s[:, C - 1], (x[:, C - 1].float() + branch[:, C - 1].float()).to(BF))


# 2^21 blocks of four rows (a wave each), and of one row, some of them ignored or out of range: those leave the loop's
# trip before its barriers, with the whole block.
@pytest.mark.parametrize("N,V", [((1 << 23) + 4099, 8), ((1 << 21) + 1025, 8192)])
def test_cross_entropy(pkg, N, V):
    logits = torch.zeros(N, V, device=DEV, dtype=BF)
    targets = torch.arange(N, device=DEV) % V
    g = torch.Generator(device=DEV).manual_seed(V)
    rows = torch.cat([torch.arange(a, a + 1000, device=DEV) for a in (0, N // 2, N - 1000)])
    logits[rows] = torch.randn(len(rows), V, generator=g, device=DEV, dtype=BF)
    targets[rows[::7]] = -100
    targets[rows[::13]] = V
    logits.requires_grad_(True)
    losses = pkg.loss.cross_entropy(logits, targets)
    small = logits.detach()[rows].requires_grad_(True)
    want = pkg.loss.cross_entropy(small, targets[rows])
    assert torch.equal(losses.detach()[rows].view(torch.int32), want.detach().view(torch.int32))
    rest = torch.ones(N, dtype=torch.bool, device=DEV)
    rest[rows] = False
    # V exponentials of 0 are V; its logarithm in 32 bits
    assert float((losses.detach()[rest] - math.log(V)).abs().max()) <= 2.0 ** -20
    weight = torch.rand(N, generator=g, device=DEV)
    got = torch.autograd.grad(losses, logits, weight)[0]
    assert torch.equal(got[rows].view(torch.int16), torch.autograd.grad(want, small, weight[rows])[0].view(torch.int16))
    # the last class of a row of zeros: weight / V less the weight where it is the target
    hit = (targets == V - 1)[rest]
    last = weight[rest] * torch.where(hit, 1 / V - 1, 1 / V)
    assert bool(((got[rest, V - 1].float() - last).abs() <= 2.0 ** -8 * last.abs()).all())
