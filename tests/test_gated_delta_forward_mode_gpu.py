"""Forward-mode derivatives: the gated delta rule and its token step have none and say so, whichever input carries a
tangent, with gradients recorded or not; a refused step leaves the state as it was."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu
NAMES = ("q", "k", "v", "g", "beta")


def tensors(T):
    G = torch.Generator(device="cuda").manual_seed(T)
    n = lambda *s: torch.randn(*s, generator=G, device="cuda")
    return {"q": n(2, 1, T, 64).mul_(0.1).bfloat16(), "k": n(2, 1, T, 64).mul_(0.1).bfloat16(), "v": n(2, 2, T, 64).bfloat16(),
            "g": -n(2, 2, T).abs(), "beta": n(2, 2, T).sigmoid(), "state": n(2, 2, 64, 64)}


@pytest.mark.parametrize("recording", [True, False])
@pytest.mark.parametrize("name", NAMES + ("state",))
def test_a_tangent_is_refused(pkg, name, recording):
    d = tensors(3)
    before = d["state"].clone()
    version = d["state"]._version
    with fwd.dual_level(), torch.set_grad_enabled(recording):
        u = dict(d, **{name: fwd.make_dual(d[name], torch.ones_like(d[name]))})
        with pytest.raises((RuntimeError, NotImplementedError)):
            pkg.gated_delta.gated_delta_rule(*[u[n] for n in NAMES], initial_state=u["state"], output_final_state=True)
        with pytest.raises(NotImplementedError, match="forward"):
            pkg.gated_delta.gated_delta_step(*[u[n] for n in NAMES], u["state"])
    assert torch.equal(d["state"], before) and d["state"]._version == version


def test_a_level_without_tangents_changes_nothing(pkg):
    d = tensors(2)
    with torch.no_grad():
        a, sa = d["state"].clone(), d["state"].clone()
        want = pkg.gated_delta.gated_delta_step(*[d[n] for n in NAMES], a)
        with fwd.dual_level():
            got = pkg.gated_delta.gated_delta_step(*[d[n] for n in NAMES], sa)
    assert torch.equal(want, got) and torch.equal(a, sa)
