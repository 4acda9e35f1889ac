"""Dropout in the layers where the fused kernel does not take the call, and which numbers it draws."""
import pytest
import torch

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
