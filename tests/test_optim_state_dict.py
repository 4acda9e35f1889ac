"""optim.AdamW.load_state_dict on the CPU: states that do not fit are refused and leave the optimizer as it was."""
import copy

import pytest
import torch


def _param(*shape):
    return torch.nn.Parameter(torch.ones(shape))


def _saved(pkg, shape, bits=None):
    """The state dict after a step of torch's AdamW on a parameter of `shape`, or one with 8-bit states."""
    q = _param(*shape)
    o = torch.optim.AdamW([q], lr=0.25)
    q.grad = torch.full(shape, 0.5)
    o.step()
    if bits is None:
        return o.state_dict()
    e = pkg.optim.AdamW([q], lr=0.25, state_bits=8, min_8bit_numel=1)
    e.load_state_dict(o.state_dict())
    return e.state_dict()


def _look(o):
    return (copy.deepcopy([{k: v for k, v in g.items() if k != "params"} for g in o.param_groups]),
            {id(p): {k: v.clone() for k, v in s.items()} for p, s in o.state.items()})


def _same(a, b):
    return a[0] == b[0] and a[1].keys() == b[1].keys() and all(
        s.keys() == b[1][i].keys() and all(torch.equal(v.float(), b[1][i][k].float()) for k, v in s.items()) for i, s in a[1].items())


def _loaded(pkg, p, bits):
    o = pkg.optim.AdamW([p], lr=0.5, state_bits=bits, min_8bit_numel=1)
    o.load_state_dict(_saved(pkg, tuple(p.shape)))
    o.param_groups[0]["lr"] = 0.125
    return o


# A state of another shape, one that torch's copying would repeat over the rows among them; codes with the wrong
# number of scales; a state that lacks one.
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("shape,other", [((3, 4), (4,)), ((3, 4), (1, 4)), ((3, 4), (4, 3)), ((3, 4), (12,)), ((100, 100), (100,)),
                                         ((4,), ()), ((5,), (6,))])
def test_a_state_of_another_shape_is_refused(pkg, bits, shape, other):
    o = _loaded(pkg, _param(*shape), bits)
    before = _look(o)
    for sd in (_saved(pkg, other), _saved(pkg, other, 8)):
        with pytest.raises(ValueError, match="shape"):
            o.load_state_dict(sd)
        assert _same(_look(o), before)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("name,n", [("exp_avg_scale", 1), ("exp_avg_sq_scale", 4), ("exp_avg_scale", 0)])
def test_a_wrong_number_of_scales_is_refused(pkg, bits, name, n):
    o = _loaded(pkg, _param(600), bits)
    before = _look(o)
    sd = _saved(pkg, (600,), 8)
    sd["state"][0][name] = torch.ones(n)
    with pytest.raises(ValueError, match="scale"):
        o.load_state_dict(sd)
    del sd["state"][0][name]
    with pytest.raises(ValueError):
        o.load_state_dict(sd)
    assert _same(_look(o), before)


def test_one_state_that_does_not_fit_leaves_all_as_they_were(pkg):
    ps = [_param(4), _param(2, 3)]
    o = pkg.optim.AdamW([{"params": ps[:1]}, {"params": ps[1:], "lr": 0.5}])
    qs = [_param(4), _param(3, 2)]
    a = torch.optim.AdamW([{"params": qs[:1]}, {"params": qs[1:]}], lr=0.25)
    for q in qs:
        q.grad = torch.ones_like(q)
    a.step()
    before = _look(o)
    with pytest.raises(ValueError):
        o.load_state_dict(a.state_dict())
    assert _same(_look(o), before) and not o.state
    for wrong in ([{"params": qs}], [{"params": qs[:1]}, {"params": qs[1:]}, {"params": [_param(1)]}], [{"params": qs[1:]}, {"params": [_param(1), _param(2)]}]):
        with pytest.raises(ValueError):
            o.load_state_dict(torch.optim.AdamW(wrong).state_dict())
    assert _same(_look(o), before)


def test_states_that_fit_load(pkg):
    for bits in (8, 32):
        p = _param(3, 100)
        o = pkg.optim.AdamW([p], state_bits=bits, min_8bit_numel=1)
        o.load_state_dict(_saved(pkg, (3, 100)))
        o.load_state_dict(_saved(pkg, (3, 100), 8))
        m, v = o.moments(p)
        # two codes: half a step of e4m3 each, of m and of the root of v
        assert bool(((m - 0.05).abs() <= 0.05 * 2.0 ** -3).all()) and bool(((v.sqrt() - 0.00025 ** 0.5).abs() <= 0.00025 ** 0.5 * 2.0 ** -3).all())
        assert float(o.state[p]["step"]) == 1 and o.param_groups[0]["lr"] == 0.25
        o.load_state_dict(pkg.optim.AdamW([_param(3, 100)], lr=0.75).state_dict())
        assert not o.state and o.param_groups[0]["lr"] == 0.75


# What a pre-hook returns is what is loaded; a post-hook sees the states; both stay registered, and nothing else does.
@pytest.mark.parametrize("bits", [8, 32])
def test_hooks_around_loading(pkg, bits):
    p = _param(300)
    o = pkg.optim.AdamW([p], state_bits=bits, min_8bit_numel=1)
    seen = []

    def twice(opt, sd):
        sd = copy.deepcopy(sd)
        sd["state"][0]["exp_avg"] *= 2
        sd["state"][0]["step"] += 4
        return sd

    o.register_load_state_dict_pre_hook(twice)
    o.register_load_state_dict_post_hook(lambda opt: seen.append({k: v.clone() for k, v in opt.state[p].items()}))
    for k in range(2):
        o.load_state_dict(_saved(pkg, (300,)))
        m, _ = o.moments(p)
        # 0.1 in 32 bits; the largest of its block, so exact in 8 bits up to the scale
        assert bool(((m - 0.1).abs() <= 2.0 ** -20).all()) and float(o.state[p]["step"]) == 5
        assert len(seen) == k + 1 and seen[k].keys() == o.state[p].keys() and all(torch.equal(v.float(), o.state[p][n].float()) for n, v in seen[k].items())
    before = _look(o)
    refuse = o.register_load_state_dict_pre_hook(lambda opt, sd: _saved(pkg, (4,)))
    with pytest.raises(ValueError, match="shape"):
        o.load_state_dict(_saved(pkg, (300,)))
    assert _same(_look(o), before) and len(seen) == 2
    refuse.remove()
    # a copy, which has no hooks, loads too
    other = copy.deepcopy(o)
    other.load_state_dict(_saved(pkg, (300,)))
    assert float(other.state[other.param_groups[0]["params"][0]]["step"]) == 1
