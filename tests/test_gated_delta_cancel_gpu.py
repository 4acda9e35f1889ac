"""The gated delta rule where a bf16 output is the small difference of large terms, against the definition in 64 bits.

A read at a key that was just written is what the state held less what the correction took off: with beta 1 and a key
whose length differs from 1 by a rounding, 2^-9 or less of either is left.  So are the gradients here.

Tolerances.  The output is rounded once, 2.4e-3 of the 2-norm at most (half a step of bf16, 2^-8 / sqrt(3)).  The terms that
cancel are formed in 32 bits, of operands in 32 bits: the sums of two steps of 32 terms in up to six products each (12
roundings of 2^-24), the products that six of nine leave out (3), the triangle's inverse over its four blocks (4), exponentials
of two ulps and factors (8), and the subtractions (2), fewer than 32, which in the 2-norm of thousands of elements add as
independent ones: sqrt(32 / 3) 2^-24 of the terms.  Five times that, 2^-20, is allowed.  `cancelled` is the terms' 2-norm
over the output's.  An operand of 16 bits (2^-17 / sqrt(3) = 4.4e-6 of a term in the mean) is past these bounds."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def nearly_unit(K, seed):
    """A key in bf16 of 64 entries +-1/8, one of them 2^-7 of itself longer: its squared length is 1 + 2.4e-4."""
    G = torch.Generator().manual_seed(seed)
    k = torch.zeros(K)
    k[torch.randperm(K, generator=G)[:64]] = 0.125 * (2 * torch.randint(0, 2, (64,), generator=G).float() - 1)
    i = int(k.abs().argmax())
    k[i] *= 1 + 2.0 ** -7
    return k.to(BF)


def definition(d, do, scale):
    """(o, d_q, d_k, terms of each that cancel) of one head [T, ..], in 64 bits."""
    q, k, v, g, beta, S = (d[n].double() for n in ("q", "k", "v", "g", "beta", "h0"))
    do = do.double()
    before, after, n, o, to, tq = [], [], [], [], [], []
    for t in range(len(g)):
        S = S * g[t].exp()
        before.append(S)
        n.append(beta[t] * (v[t] - k[t] @ S))
        to.append(scale * (q[t] @ S))
        tq.append(scale * (S @ do[t]))
        S = S + k[t][:, None] * n[t][None]
        after.append(S)
        o.append(scale * (q[t] @ S))
    D, dq, dk, tk = torch.zeros_like(S), [], [], []
    for t in reversed(range(len(g))):
        dq.append(scale * (after[t] @ do[t]))
        D = D + scale * q[t][:, None] * do[t][None]
        dn = k[t] @ D
        tk.append(D @ n[t])
        dk.append(tk[-1] - beta[t] * (before[t] @ dn))
        D = (D - beta[t] * k[t][:, None] * dn[None]) * g[t].exp()
    s = torch.stack
    return {"o": (s(o), s(to)), "q": (s(dq[::-1]), s(tq)), "k": (s(dk[::-1]), s(tk[::-1]))}


def case(name, K, V, T, seed):
    G = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=G)
    one = nearly_unit(K, seed)
    d = {"k": one.expand(T, K).contiguous(), "beta": torch.ones(T), "g": -0.02 * torch.rand(T, generator=G), "v": torch.zeros(T, V, dtype=BF)}
    if name == "other keys":                             # each written key is read, of a state without structure
        k = n(T, K)
        d["k"] = (k / k.norm(dim=-1, keepdim=True)).to(BF)
        d["h0"] = n(K, V)
    elif name == "one key":                              # a value is written, and read as a zero takes its place
        clears = torch.arange(T) % 2 == 1
        d["v"] = torch.where(clears[:, None], torch.zeros(()), n(T, V)).to(BF)
        d["g"] = torch.where(clears, d["g"], torch.tensor(-4.0))
        d["h0"] = torch.zeros(K, V)
    else:                                                # the values are twice what a decay of 1/2 leaves: n = S'^T k
        u = n(V).to(BF)
        d["v"] = u.expand(T, V).contiguous()
        d["g"].fill_(-0.6931471805599453)
        d["h0"] = one.float()[:, None] * u.float()[None]
    d["q"], do = d["k"].clone(), n(T, V).to(BF)
    if name == "one key":                                # nothing else is read
        d["q"][::2] = 0
        do[::2] = 0
    return d, do


def run(pkg, name, K, V, T=64, heads=2):
    """The kernels' o, d_q, d_k of `heads` heads side by side, and the definition's of each."""
    ds = [case(name, K, V, T, 10 * K + V + i) for i in range(heads)]
    u = {n: torch.stack([d[n] for d, _ in ds])[None].cuda().requires_grad_(True) for n in ("q", "k", "v", "g", "beta", "h0")}
    o, _ = pkg.gated_delta.gated_delta_rule(*[u[n] for n in ("q", "k", "v", "g", "beta")], initial_state=u["h0"])
    dq, dk = torch.autograd.grad(o, (u["q"], u["k"]), torch.stack([w for _, w in ds])[None].cuda())
    want = [definition(d, w, K ** -0.5) for d, w in ds]
    return {"o": o, "q": dq, "k": dk}, want


def held(name, got, want, least):
    for i, w in enumerate(want):
        ref, terms = w[name]
        cancelled = float(terms.norm() / ref.norm())
        off = float((got[name][0, i].detach().double().cpu() - ref).norm() / ref.norm())
        print(f"{name}: cancelled {cancelled:.0f}, off {off:.1e}", flush=True)
        assert cancelled >= least
        assert off <= 2.4e-3 + 2.0 ** -20 * cancelled


SIZES = [(64, 64), (128, 64), (64, 192), (128, 128)]


@pytest.mark.parametrize("K,V", SIZES)
@pytest.mark.parametrize("name", ["other keys", "one key"])
def test_a_read_of_what_was_just_written(pkg, name, K, V):
    held("o", *run(pkg, name, K, V), least=300)


@pytest.mark.parametrize("K,V", SIZES)
def test_the_queries_gradient_of_such_reads(pkg, K, V):
    held("q", *run(pkg, "one key", K, V), least=300)


@pytest.mark.parametrize("K,V", SIZES)
def test_the_keys_gradient_where_a_write_doubles_what_was_kept(pkg, K, V):
    """d_k = D n - S' (D^T k) and both are k's direction times u d_o."""
    held("k", *run(pkg, "twice", K, V), least=300)
