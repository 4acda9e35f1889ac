"""CPU checks of the C entries of residual_norm, cross entropy and AdamW: bad calls return an error code
before any launch (the pointers are fake, nothing is dereferenced), and the Python functions refuse
tensors that are not on the GPU."""
import ctypes

import pytest
import torch

OK, INVALID, UNSUPPORTED, ALIGNMENT = 0, 1, 2, 4
F32, BF16 = 0, 1


def _p(addr):
    return ctypes.c_void_p(addr)


A = [_p(0x10000000 * i) for i in range(1, 16)]        # 256 MB apart


def _fwd(L, **kw):
    a = dict(x=A[0], xt=BF16, branch=A[1], cb=None, cbt=F32, gate=None, scale=1.0, step=0, gamma=A[2], beta=A[3], pt=F32,
             eps=1e-5, s=A[4], y=A[5], mean=A[6], rstd=A[7], N=4, C=64, stream=None)
    a.update(kw)
    return L.rwkv6_residual_norm_fwd(*a.values())


def _bwd(L, **kw):
    a = dict(x=A[0], xt=BF16, branch=A[1], cb=None, cbt=F32, gate=None, scale=1.0, step=0, gamma=A[2], gt=F32, mean=A[3],
             rstd=A[4], ds=None, dy=A[5], dx=A[6], db=A[7], dg=None, dgamma=A[8], dbeta=A[9], pt=F32, dcb=None, ws=A[10],
             N=4, C=64, stream=None)
    a.update(kw)
    return L.rwkv6_residual_norm_bwd(*a.values())


def test_residual_norm_refuses_before_launch(pkg):
    L = pkg._lib.load()
    assert _fwd(L, N=0) == OK
    for kw in (dict(x=None), dict(branch=None), dict(y=None), dict(gamma=None), dict(mean=None), dict(xt=2), dict(pt=7), dict(N=-1),
               dict(C=0), dict(cb=A[8], cbt=9), dict(s=A[0]), dict(y=A[4]), dict(s=_p(0x10000000 + 16)), dict(rstd=A[6]), dict(gate=A[5])):
        assert _fwd(L, **kw) == INVALID, kw
    for kw in (dict(C=12), dict(C=8200), dict(N=1 << 38)):
        assert _fwd(L, **kw) == UNSUPPORTED == _bwd(L, **kw), kw
        assert L.rwkv6_residual_norm_bwd_workspace_bytes(kw.get("N", 4), kw.get("C", 64)) == 0
    for n in ("x", "branch", "s", "y", "gate", "gamma"):
        assert _fwd(L, **{n: _p(0x90000008)}) == ALIGNMENT, n
    for kw in (dict(x=None), dict(dy=None), dict(dx=None), dict(dgamma=None), dict(ws=None), dict(dg=A[11]), dict(gate=A[11]),
               dict(dcb=A[11]), dict(cb=A[11]), dict(db=None, scale=0.5), dict(db=None, xt=F32), dict(db=None, gate=A[11], dg=A[12]),
               dict(dx=A[5]), dict(db=A[6]), dict(dbeta=A[8]), dict(ws=A[0]), dict(gt=5), dict(ds=A[6])):
        assert _bwd(L, **kw) == INVALID, kw
    # the partial sums of the largest call: 1024 ranges of three rows of C
    assert 0 < L.rwkv6_residual_norm_bwd_workspace_bytes(1 << 20, 8192) <= 1024 * 3 * 8192 * 4
    assert L.rwkv6_residual_norm_bwd_workspace_bytes(1, 8) == 3 * 8 * 4 == L.rwkv6_residual_norm_bwd_workspace_bytes(0, 8)


def _ce(L, back=False, **kw):
    a = dict(logits=A[0], dt=BF16, ld=100, target=A[1], ignore=-100)
    a.update(dict(stats=A[2], dl=A[3], d=A[4]) if back else dict(loss=A[2], stats=A[3]))
    a.update(N=4, V=100, stream=None)
    a.update(kw)
    return (L.rwkv6_cross_entropy_bwd if back else L.rwkv6_cross_entropy_fwd)(*a.values())


def test_cross_entropy_refuses_before_launch(pkg):
    L = pkg._lib.load()
    for back in (False, True):
        assert _ce(L, back, N=0) == OK
        for kw in (dict(logits=None), dict(target=None), dict(stats=None), dict(dt=3), dict(V=0), dict(ld=99), dict(N=-1)):
            assert _ce(L, back, **kw) == INVALID, kw
        for kw in (dict(V=(1 << 30) + 1, ld=1 << 31), dict(N=1 << 60), dict(ld=1 << 41)):
            assert _ce(L, back, **kw) == UNSUPPORTED, kw
        assert _ce(L, back, logits=_p(0x10000001)) == ALIGNMENT == _ce(L, back, stats=_p(0x40000004))
    assert _ce(L, loss=A[0]) == INVALID == _ce(L, loss=_p(0x10000000 + 798)) and _ce(L, stats=A[2]) == INVALID
    assert _ce(L, True, d=A[0]) == INVALID == _ce(L, True, d=None) == _ce(L, True, dl=None)
    assert _ce(L, True, d=_p(0x50000001)) == ALIGNMENT


def _arr(kind, values):
    return (kind * len(values))(*values)


def _step(L, n=2, size=300, eight=True, **kw):
    vp = ctypes.c_void_p
    at = lambda base: _arr(vp, [base + 0x100000 * i for i in range(n)])
    a = dict(p=at(0x10000000), pt=_arr(ctypes.c_int, [F32] * n), g=at(0x20000000), gt=_arr(ctypes.c_int, [F32] * n),
             m=at(0x30000000), v=at(0x40000000), ms=at(0x50000000) if eight else None, vs=at(0x60000000) if eight else None,
             numel=_arr(ctypes.c_int64, [size] * n), count=n, step=_p(0x70000000), lr=1e-3, lr_dev=None, b1=0.9, b2=0.99,
             eps=1e-8, wd=0.1, partials=None, P=0, max_norm=1.0, norm=None, ws=_p(0x71000000), stream=None)
    a.update(kw)
    return L.rwkv6_adamw_step(*a.values())


def test_adamw_refuses_before_launch(pkg):
    L = pkg._lib.load()
    vp = ctypes.c_void_p
    two = lambda a, b: _arr(vp, [a, b])
    for kw in (dict(p=None), dict(g=None), dict(step=None), dict(ws=None), dict(numel=None), dict(count=-1), dict(b1=1.0), dict(b2=-0.1),
               dict(vs=None), dict(ms=None), dict(P=1), dict(P=-1), dict(pt=_arr(ctypes.c_int, [0, 4])), dict(gt=_arr(ctypes.c_int, [2, 0])),
               dict(p=two(0x10000000, 0)), dict(m=two(0, 0x30000000)), dict(ms=two(0, 0x50000000)),
               dict(numel=_arr(ctypes.c_int64, [300, -1]))):
        assert _step(L, **kw) == INVALID, kw
    # a tensor listed twice, one that begins inside another, a parameter that is a gradient or a state
    for kw in (dict(p=two(0x10000000, 0x10000000)), dict(p=two(0x10000000, 0x10000000 + 1196)), dict(p=two(0x10000000, 0x20000000)),
               dict(v=two(0x30000000, 0x40100000)), dict(ms=two(0x50000000, 0x50000004)), dict(ws=_p(0x10000000)), dict(step=_p(0x40000000)),
               dict(norm=_p(0x70000000)), dict(lr_dev=_p(0x70000000))):
        assert _step(L, **kw) == INVALID, kw
    for kw in (dict(p=two(0x10000002, 0x10100000)), dict(g=two(0x20000001, 0x20100000)), dict(ws=_p(0x71000008)), dict(ms=two(0x50000002, 0x50100000)),
               dict(step=_p(0x70000002)), dict(partials=_p(0x72000004), P=1)):
        assert _step(L, **kw) == ALIGNMENT, kw
    assert _step(L, eight=False, m=two(0x30000002, 0x30100000)) == ALIGNMENT
    assert _step(L, size=1 << 41) == UNSUPPORTED
    sizes = lambda *s: _arr(ctypes.c_int64, list(s))
    assert L.rwkv6_grad_norm_partials(sizes(1, 0, 2048, 2049), 4) == 1 + 1 + 2
    big = [1 << 20] * 500
    assert 4096 <= L.rwkv6_grad_norm_partials(sizes(*big), 500) <= 8192 + 500
    g1 = _arr(ctypes.c_int, [F32])
    assert L.rwkv6_grad_norm_sums(two(0, 0), g1, sizes(5), 1, _p(0x1000), None) == INVALID
    assert L.rwkv6_grad_norm_sums(two(0x1000, 0), g1, sizes(5), 1, _p(0x1000), None) == INVALID
    assert L.rwkv6_grad_norm_sums(two(0x2001, 0), g1, sizes(5), 1, _p(0x1000), None) == ALIGNMENT
    assert L.rwkv6_grad_norm(None, 3, _p(0x1000), None) == INVALID == L.rwkv6_grad_norm(_p(0x1000), 3, None, None)


def test_python_functions_refuse_cpu_tensors(pkg):
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    w = torch.zeros(64)
    with pytest.raises(ValueError, match="GPU"):
        pkg.residual.residual_norm(x, x, w, w, 1e-5)
    with pytest.raises(ValueError, match="GPU"):
        pkg.loss.cross_entropy(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="GPU"):
        pkg.optim.adamw_step([w], [w], [w], [w], torch.zeros(()), lr=1e-3)
    with pytest.raises(ValueError, match="GPU"):
        pkg.optim.grad_norm([w])
    with pytest.raises(TypeError):
        pkg.optim.grad_norm([])
    p = torch.nn.Parameter(torch.zeros(4))
    for kw in (dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1.0), dict(weight_decay=-0.1), dict(max_norm=0.0), dict(state_bits=4)):
        with pytest.raises(ValueError):
            pkg.optim.AdamW([p], **kw)
    o = pkg.optim.AdamW([p])
    with pytest.raises(TypeError):
        o.add_param_group({"params": [torch.nn.Parameter(torch.zeros(4, dtype=torch.float16))]})
    with pytest.raises(ValueError):
        o.add_param_group({"params": [torch.nn.Parameter(torch.zeros(4))], "lr": -1.0})
    assert len(o.param_groups) == 1
    o.step()                                              # nothing has a gradient
    p.grad = torch.zeros(4)
    with pytest.raises(ValueError, match="GPU"):
        o.step()


def test_state_dicts_of_other_steps_are_refused(pkg):
    p, q = (torch.nn.Parameter(torch.ones(4)) for _ in range(2))
    o = pkg.optim.AdamW([p], lr=0.5)
    q.grad = torch.ones(4)
    for make in (lambda: torch.optim.AdamW([q], amsgrad=True), lambda: torch.optim.AdamW([q], maximize=True),
                 lambda: torch.optim.Adam([q], weight_decay=0.1), lambda: torch.optim.SGD([q], momentum=0.9)):
        other = make()
        other.step()
        with pytest.raises(ValueError):
            o.load_state_dict(other.state_dict())
        assert o.param_groups[0]["lr"] == 0.5 and not o.state
    other = torch.optim.AdamW([q], lr=0.25)
    other.step()
    o.load_state_dict(other.state_dict())
    assert o.param_groups[0]["lr"] == 0.25 and torch.equal(o.moments(p)[0], other.state[q]["exp_avg"])


def test_the_stochastic_step_refuses_the_same_calls(pkg):
    L = pkg._lib.load()

    class Other:
        rwkv6_adamw_step = L.rwkv6_adamw_step_stochastic

    vp = ctypes.c_void_p
    for kw in (dict(p=None), dict(step=None), dict(ws=None), dict(count=-1), dict(b2=1.0), dict(vs=None), dict(P=1),
               dict(p=_arr(vp, [0x10000000, 0x10000000])), dict(step=_p(0x40000000))):
        assert _step(Other, **kw) == INVALID, kw
    assert _step(Other, ws=_p(0x71000008)) == ALIGNMENT and _step(Other, size=1 << 41) == UNSUPPORTED
    with pytest.raises(ValueError, match="rounding"):
        pkg.optim.adamw_step([torch.zeros(4)], [torch.zeros(4)], [torch.zeros(4)], [torch.zeros(4)], torch.zeros(()), lr=1.0, rounding="down")


def test_residual_norm_backward_without_a_branch(pkg):
    """Only where x can be the sum that the forward stored: stepwise, without a gate."""
    L = pkg._lib.load()
    for kw in (dict(step=0), dict(step=1, gate=A[11], dg=A[12]), dict(step=1, x=None), dict(step=1, N=0, ws=None)):
        assert _bwd(L, branch=None, **kw) == INVALID, kw


def test_residual_norm_for_training_refuses_a_bad_copy_of_gamma(pkg):
    L = pkg._lib.load()

    def call(used, **kw):
        a = dict(x=A[0], xt=BF16, branch=A[1], cb=None, cbt=F32, gate=None, scale=1.0, step=0, gamma=A[2], beta=A[3], pt=F32,
                 eps=1e-5, s=A[4], y=A[5], mean=A[6], rstd=A[7], used=used, N=4, C=64, stream=None)
        a.update(kw)
        return L.rwkv6_residual_norm_train_fwd(*a.values())

    assert call(A[8], N=0) == OK == call(None, N=0)
    for used in (A[2], A[5], _p(0x40000000 - 16), A[7]):
        assert call(used) == INVALID, used
    assert call(_p(0x90000008)) == ALIGNMENT and call(A[8], C=12) == UNSUPPORTED


def test_the_partial_sums_of_the_largest_call(pkg):
    """768 blocks' sums of three rows of C."""
    L = pkg._lib.load()
    for C in (1024, 2048, 4096, 8192):
        assert L.rwkv6_residual_norm_bwd_workspace_bytes(1 << 20, C) == 768 * 3 * C * 4 == L.rwkv6_residual_norm_bwd_workspace_bytes(1 << 27, C)
