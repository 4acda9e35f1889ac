"""The gated delta rule's kernels against the recurrence in 64 bits (token by token, gradients by autograd).

Tolerances.  A bf16 output is rounded once: half a step, at most 2^-8 of the value, an error of at most
2^-8 / sqrt(3) = 2.3e-3 of the tensor's 2-norm.  Computed operands enter the products as two bf16 numbers, at
most 2^-16 off (2^-16 / sqrt(3) = 8.8e-6 in the 2-norm); on the way to any output no more than six of them
follow one another (state, written values, triangle, their gradients, p or m, the sums): sqrt(6) of that is
2.2e-5, and 32-bit sums add less than 1e-6.  So 32-bit outputs are held to 2.5e-5 of the 2-norm and bf16 ones
to 2.4e-3; a single bf16 value to 2^-8 of itself and 1e-4 of the tensor's largest.

d_beta and d_g are sums of products (d_beta_t = sum_v dw_v e_v for the written w = beta e, d_g_t = sum over the
decayed state and its gradient), and a sum may be much smaller than its products: n products each off by
2.2e-5 of itself, independently, leave an error of 2.2e-5 sqrt(sum of their squares) in the mean.  Three times
that is allowed on top, the products taken from the definition in 64 bits.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def recurrence(q, k, v, g, beta, scale, h0=None, steps=None):
    """(o, state) of the definition, in the inputs' type.  steps: a list that gets each token's (w, e, S')."""
    group = v.shape[1] // q.shape[1]
    q, k = q.repeat_interleave(group, 1), k.repeat_interleave(group, 1)
    B, HV, T, V = v.shape
    S = h0 if h0 is not None else v.new_zeros(B, HV, q.shape[-1], V)
    o = []
    for t in range(T):
        S = S * g[:, :, t].exp()[..., None, None]
        e = v[:, :, t] - (k[:, :, t, None] @ S)[:, :, 0]
        w = beta[:, :, t, None] * e
        if steps is not None:
            w.retain_grad()
            if S.requires_grad:
                S.retain_grad()
            steps.append((w, e, S))
        S = S + k[:, :, t, :, None] * w[:, :, None]
        o.append(scale * (q[:, :, t, None] @ S)[:, :, 0])
    return (torch.stack(o, 2) if o else v.new_zeros(B, HV, 0, V)), S


def inputs(B, H, HV, T, K, V, seed=0, beta=F32, strong=False, h0=False, vt=BF):
    G = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=G)
    unit = lambda x: (x / x.norm(dim=-1, keepdim=True)).to(BF)
    d = {"q": unit(n(B, H, T, K)), "k": unit(n(B, H, T, K)), "v": n(B, HV, T, V).to(vt)}
    rate = torch.rand(1, HV, 1, generator=G) * (12 if strong else 1.5)
    d["g"] = -rate * torch.nn.functional.softplus(n(B, HV, T) - (0 if strong else 2))
    d["beta"] = torch.sigmoid(1.5 * n(B, HV, T)).to(beta)
    if h0:
        d["h0"] = 0.3 * n(B, HV, K, V)
    return d


def close(name, got, ref):
    got, ref = got.detach().double().cpu(), ref.detach().double().cpu()
    assert got.shape == ref.shape, name
    if not ref.numel():
        return
    rel = float((got - ref).norm() / ref.norm().clamp(min=1e-30))
    print(f"{name}: {rel:.2e}", end=" ")
    return rel


def check(name, got, ref, products=None):
    """products: the 2-norm of the products that the sums of a 32-bit output are taken of."""
    bf = got.dtype == BF
    rel = close(name, got, ref)
    if rel is None:
        return
    assert rel <= (2.4e-3 if bf else 2.5e-5) + (3 * 2.2e-5 * products / float(ref.norm()) if products else 0), (name, rel)
    if bf:
        a, b = got.detach().double().cpu(), ref.detach().double().cpu()
        assert ((a - b).abs() <= 2.0 ** -8 * b.abs() + 1e-4 * b.abs().max()).all(), name


def run_train(pkg, d, scale=None, final=False, wo=None, wh=None):
    """Outputs and gradients of sum(o wo) + sum(state wh), of the kernels and of the definition."""
    names = [n for n in ("q", "k", "v", "g", "beta", "h0") if n in d]
    gpu = {n: d[n].cuda().requires_grad_(True) for n in names}
    ref = {n: d[n].double().requires_grad_(True) for n in names}
    o, S = pkg.gated_delta.gated_delta_rule(*[gpu[n] for n in names[:5]], scale=scale, initial_state=gpu.get("h0"),
                                            output_final_state=final)
    steps = []
    ro, rS = recurrence(*[ref[n] for n in names[:5]], scale if scale is not None else d["q"].shape[-1] ** -0.5, ref.get("h0"), steps)
    outs, routs, gs, rgs = [o], [ro], [wo.cuda()], [wo.double()]
    if final:
        outs.append(S), routs.append(rS), gs.append(wh.cuda()), rgs.append(wh.double())
    got = torch.autograd.grad(outs, [gpu[n] for n in names], gs)
    torch.autograd.backward(routs, rgs)
    want = [ref[n].grad for n in names]
    norm = lambda pairs: float(sum((a * b).square().sum() for a, b in pairs)) ** 0.5
    products = {"beta": norm((w.grad, e.detach()) for w, e, _ in steps),
                "g": norm((S.grad, S.detach()) for _, _, S in steps if S.grad is not None)}
    check("o", o, ro)
    if final:
        check("state", S, rS)
    for n, a, b in zip(names, got, want):
        assert a.dtype == d[n].dtype
        check("d_" + n, a, b, products.get(n) if a.dtype == F32 else None)
    print()


SHAPES = [
    # B, H, HV, T, K, V
    (1, 1, 1, 1, 64, 64), (2, 1, 1, 2, 64, 64), (1, 2, 2, 17, 64, 64), (1, 1, 1, 63, 128, 64), (1, 2, 4, 64, 64, 128),
    (2, 1, 3, 65, 64, 64), (1, 2, 2, 128, 128, 128), (3, 1, 2, 129, 128, 64), (1, 1, 1, 300, 64, 192), (2, 3, 3, 200, 64, 64),
]

# more heads: a walk's block takes 16, 32 or 64 columns of the state by their number (up to 256, 512 and more tiles of 16)
MANY = [(4, 17, 17, 70, 64, 64), (5, 30, 30, 66, 64, 64), (3, 6, 12, 70, 128, 128), (3, 24, 24, 66, 128, 128), (2, 33, 33, 5, 128, 192)]


@pytest.mark.parametrize("shape", SHAPES + MANY, ids=str)
@pytest.mark.parametrize("strong", [False, True])
def test_training(pkg, shape, strong):
    B, H, HV, T, K, V = shape
    d = inputs(*shape, seed=sum(shape), strong=strong)
    run_train(pkg, d, wo=torch.randn(B, HV, T, V).to(BF))


@pytest.mark.parametrize("shape", SHAPES[::2], ids=str)
def test_training_with_states_on_both_ends(pkg, shape):
    B, H, HV, T, K, V = shape
    d = inputs(*shape, seed=1 + sum(shape), h0=True)
    run_train(pkg, d, scale=0.7, final=True, wo=torch.randn(B, HV, T, V).to(BF), wh=torch.randn(B, HV, K, V))


@pytest.mark.parametrize("shape", SHAPES + MANY, ids=str)
def test_prompt(pkg, shape):
    d = inputs(*shape, seed=2 + sum(shape), h0=True)
    with torch.no_grad():
        o, S = pkg.gated_delta.gated_delta_rule(*[d[n].cuda() for n in ("q", "k", "v", "g", "beta")], initial_state=d["h0"].cuda(),
                                                output_final_state=True)
    ro, rS = recurrence(*[d[n].double() for n in ("q", "k", "v", "g", "beta")], shape[4] ** -0.5, d["h0"].double())
    check("o", o, ro)
    check("state", S, rS)


@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 64, 64), (8, 2, 4, 1, 64, 64), (3, 1, 3, 1, 128, 128), (5, 2, 2, 4, 128, 64),
                                   (2, 1, 1, 9, 64, 128), (1, 1, 2, 3, 128, 320)], ids=str)
@pytest.mark.parametrize("beta", [BF, F32])
def test_step(pkg, shape, beta):
    d = inputs(*shape, seed=3 + sum(shape), h0=True, beta=beta)
    S = d["h0"].cuda()
    o = pkg.gated_delta.gated_delta_step(*[d[n].cuda() for n in ("q", "k", "v", "g", "beta")], S)
    ro, rS = recurrence(*[d[n].double() for n in ("q", "k", "v", "g", "beta")], shape[4] ** -0.5, d["h0"].double())
    check("o", o, ro)
    assert close("state", S, rS) <= 1e-6           # 32-bit arithmetic throughout: sums of 128 terms
