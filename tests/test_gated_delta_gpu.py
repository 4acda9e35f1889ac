"""The gated delta rule's kernels against the recurrence in 64 bits (token by token, gradients by autograd).

Tolerances.  A bf16 output is rounded once: half a step, at most 2^-8 of the value, an error of at most
2^-8 / sqrt(3) = 2.3e-3 of the tensor's 2-norm.  For a computed operand of two bf16 numbers, at most 2^-16 off
(2^-16 / sqrt(3) = 8.8e-6 in the 2-norm), and no more than six of them after one another on the way to any output
(state, written values, triangle, their gradients, p or m, the sums), sqrt(6) of that is 2.2e-5, and 32-bit sums
add less than 1e-6: 32-bit outputs are held to 2.5e-5 of the 2-norm (operands of three numbers, exact, stay far
below) and bf16 ones to 2.4e-3; a single bf16 value to 2^-8 of itself and 1e-4 of the tensor's largest.

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


def on_gpu(d):
    return {n: t.cuda() for n, t in d.items()}


NAMES = ("q", "k", "v", "g", "beta")


@pytest.mark.parametrize("T", [1000, 4097])
def test_a_long_sequence(pkg, T):
    """Errors of a chunk decay with the state: the bounds are those of a short sequence."""
    d = inputs(1, 2, 2, T, 64, 64, seed=T, h0=True)
    run_train(pkg, d, final=True, wo=torch.randn(1, 2, T, 64).to(BF), wh=torch.randn(1, 2, 64, 64))


# few heads: the chunks are walked in segments side by side (7 to 16 of them here), the last of them shorter
SEGMENTED = [(1, 1, 1, 1500, 64, 64), (1, 1, 2, 2049, 64, 128), (2, 1, 1, 1300, 128, 64), (1, 2, 2, 1999, 128, 128), (1, 1, 3, 1500, 128, 192)]


@pytest.mark.parametrize("shape", SEGMENTED, ids=str)
@pytest.mark.parametrize("states", [False, True])
def test_segments(pkg, shape, states):
    """A decay that leaves half of a state after 300 tokens: what a segment gets from the one before it counts."""
    B, H, HV, T, K, V = shape
    L = pkg._lib.load()
    chunks, one = B * HV * ((T + 63) // 64), B * HV * K * (K + V) * 4       # a map and a state for each segment but the last
    for back, rest in ((0, 10240 + 512 + 256), (1, 4 * K * V + 256 * V)):
        n = L.rwkv6_gated_delta_workspace_bytes(B, HV, T, K, V, back) - chunks * rest
        assert n % one == 0 and n >= 2 * one
    d = inputs(*shape, seed=sum(shape), h0=states)
    d["g"] = d["g"].clamp(min=-0.0023)
    d["g"][:, :, 700] = -float("inf") if not states else -0.1
    with torch.no_grad():                                 # without what a backward needs
        o, S = pkg.gated_delta.gated_delta_rule(*[d[n].cuda() for n in NAMES], initial_state=d["h0"].cuda() if states else None,
                                                output_final_state=True)
    ro, rS = recurrence(*[d[n].double() for n in NAMES], K ** -0.5, d["h0"].double() if states else None)
    check("o", o, ro)
    check("state", S, rS)
    if states:
        run_train(pkg, d, final=True, wo=torch.randn(B, HV, T, V).to(BF), wh=torch.randn(B, HV, K, V))


def test_segments_captured_and_on_other_streams(pkg):
    d = on_gpu(inputs(2, 2, 2, 2000, 64, 64, seed=15, h0=True))

    w = torch.randn(2, 2, 2000, 64, device="cuda").to(BF)
    leaves = [d[n].clone().requires_grad_(True) for n in NAMES]

    def prompt():
        with torch.no_grad():
            return pkg.gated_delta.gated_delta_rule(*[d[n] for n in NAMES], initial_state=d["h0"], output_final_state=True)

    def train():
        o, S = pkg.gated_delta.gated_delta_rule(*leaves, initial_state=d["h0"], output_final_state=True)
        return torch.autograd.grad((o, S), leaves, (w, d["h0"]))

    want = [prompt(), train()]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in streams * 2:
        with torch.cuda.stream(s):
            got.append([prompt(), train()])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for x, y in zip(g, want) for a, b in zip(x, y))
    graphs, outs = [], []
    for f in (prompt, prompt, train):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(f())
    for rep in range(3):
        d["h0"].mul_(2)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in o] for o in outs]
        want = [prompt(), prompt(), train()]
        assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y)), rep


def test_slow_decay_keeps_an_old_state(pkg):
    d = inputs(1, 1, 1, 2000, 64, 64, seed=4, h0=True)
    d["g"].fill_(-1e-6)
    d["beta"].mul_(0.01)
    run_train(pkg, d, final=True, wo=torch.randn(1, 1, 2000, 64).to(BF), wh=torch.randn(1, 1, 64, 64))


@pytest.mark.parametrize("case", ["forget", "closed", "open", "no_decay", "neighbours"])
def test_edges_of_decay_and_beta(pkg, case):
    d = inputs(1, 2, 2, 150, 64, 64, seed=6, h0=True)
    if case == "forget":                                # everything before tokens 3, 64 and 100 is forgotten
        d["g"][:, :, [3, 64, 100]] = torch.tensor([-float("inf"), -1e30, -2000.0])
    elif case == "closed":
        d["beta"].zero_()
    elif case == "open":
        d["beta"].fill_(1)
    elif case == "no_decay":
        d["g"].zero_()
    else:                                               # large sums of decays, small ones between neighbours
        d["g"].fill_(-30)
        d["g"][:, :, 1::2] = -0.1
    o, S = pkg.gated_delta.gated_delta_rule(*[d[n].cuda() for n in NAMES], initial_state=d["h0"].cuda(), output_final_state=True)
    ro, rS = recurrence(*[d[n].double() for n in NAMES], 64 ** -0.5, d["h0"].double())
    check("o", o, ro)
    check("state", S, rS)
    if case == "forget":                                # e^-inf has no derivative by autograd; its limit is 0
        u = [d[n].cuda().requires_grad_(True) for n in NAMES]
        o, _ = pkg.gated_delta.gated_delta_rule(*u, initial_state=d["h0"].cuda())
        grads = torch.autograd.grad(o, u, torch.ones_like(o))
        assert all(x.isfinite().all() for x in grads)
        # a difference of sums over the chunk: 64 terms of the largest's size, 2^-20 off at most
        assert grads[3][:, :, [3, 64, 100]].abs().max() <= 64 * 2.0 ** -20 * grads[3].abs().max()
    else:
        run_train(pkg, d, wo=torch.randn(1, 2, 150, 64).to(BF))


@pytest.mark.parametrize("T, h0", [(2, False), (5, False), (40, True), (130, True)])
def test_the_decay_s_gradient_where_little_is_kept(pkg, T, h0):
    """e^-18 = 1.5e-8 of a state is left after a token: what a token reads of itself, which no decay enters, is 10^8 times
    the gradient of g, and rounds none of it.  Bounds as everywhere, of the gradient's own norm."""
    d = inputs(2, 2, 2, T, 64, 64, seed=T, h0=h0)
    d["g"] = d["g"] * 0.01 - 18
    run_train(pkg, d, wo=torch.randn(2, 2, T, 64, generator=torch.Generator().manual_seed(T)).to(BF))


@pytest.mark.parametrize("K", [64, 128])
@pytest.mark.parametrize("period", [1, 3])
def test_the_same_keys_again(pkg, K, period):
    """Every correction taken whole and nothing forgotten: the chunk's triangle is as full as it gets."""
    d = inputs(1, 1, 1, 200, K, 64, seed=K + period, h0=True)
    d["k"] = d["k"][:, :, torch.arange(200) % period].contiguous()
    d["beta"].fill_(1)
    d["g"].zero_()
    G = torch.Generator().manual_seed(period)
    run_train(pkg, d, final=True, wo=torch.randn(1, 1, 200, 64, generator=G).to(BF), wh=torch.randn(1, 1, K, 64, generator=G))


@pytest.mark.parametrize("scale", [1e-12, 1e12])
def test_gradients_of_any_size(pkg, scale):
    """d_o is taken as it is: its size goes through to all gradients."""
    d = inputs(1, 1, 1, 100, 64, 64, seed=8)
    run_train(pkg, d, wo=(scale * torch.randn(1, 1, 100, 64)).to(BF))


def test_a_difference_of_losses(pkg):
    """The gradients of g and beta against central differences of the kernels' own final state."""
    d = inputs(1, 1, 1, 70, 64, 64, seed=9, h0=True)
    u = on_gpu(d)
    w = torch.randn(1, 1, 64, 64, generator=torch.Generator().manual_seed(1)).cuda()
    call = lambda g, b: (pkg.gated_delta.gated_delta_rule(u["q"], u["k"], u["v"], g, b, initial_state=u["h0"], output_final_state=True)[1].double()
                         * w).sum()
    g, b = u["g"].requires_grad_(True), u["beta"].requires_grad_(True)
    dg, db = torch.autograd.grad(call(g, b), (g, b))
    for t, grad in ((g, dg), (b, db)):
        step = torch.randn(t.shape, generator=torch.Generator().manual_seed(2)).cuda() * 1e-2
        with torch.no_grad():
            args = lambda s: (g + s * step, b) if t is g else (g, b + s * step)
            slope = float(call(*args(1)) - call(*args(-1))) / 2
        # the third derivative's part, 1e-4 of the slope, and 32-bit sums of 4096 products of the state
        assert abs(slope - float((grad * step).sum())) <= 2e-3 * float((grad * step).abs().sum()) + 1e-4


@pytest.mark.parametrize("T", [0, 1, 70])
def test_no_tokens_and_no_sequences(pkg, T):
    d = on_gpu(inputs(2, 1, 2, T, 64, 64, h0=True))
    for B in (0, 2):
        u = {n: t[:B].detach().requires_grad_(True) for n, t in d.items()}
        o, S = pkg.gated_delta.gated_delta_rule(*[u[n] for n in NAMES], initial_state=u["h0"], output_final_state=True)
        assert o.shape == (B, 2, T, 64) and S.shape == (B, 2, 64, 64)
        if T == 0:
            assert torch.equal(S, u["h0"])
        grads = torch.autograd.grad((o, S), list(u.values()), (torch.ones_like(o), torch.ones_like(S)))
        assert [x.shape for x in grads] == [x.shape for x in u.values()]
        if T == 0:
            assert (grads[-1] == 1).all()
        state = d["h0"][:B].clone()
        with torch.no_grad():
            assert pkg.gated_delta.gated_delta_step(*[u[n] for n in NAMES], state).shape == (B, 2, T, 64)
        if T == 0:
            assert torch.equal(state, d["h0"][:B])
    o, S = pkg.gated_delta.gated_delta_rule(*[d[n][:, :, :0] if n in ("g", "beta") else d[n][:, :, :0] for n in NAMES], output_final_state=True)
    assert (S == 0).all()


@pytest.mark.parametrize("dt", [F32, torch.float16])
def test_wider_inputs_are_rounded_on_entry(pkg, dt):
    d = on_gpu(inputs(1, 2, 4, 90, 64, 64, seed=11))
    u = {n: (t.to(dt) if n != "g" else t).requires_grad_(True) for n, t in d.items()}
    r = {n: t.detach().to(BF) if n in "qkv" else t.detach() for n, t in u.items()}
    r = {n: t.requires_grad_(True) for n, t in r.items()}
    o, _ = pkg.gated_delta.gated_delta_rule(*[u[n] for n in NAMES])
    p, _ = pkg.gated_delta.gated_delta_rule(*[r[n] for n in NAMES])
    assert o.dtype == dt and torch.equal(o, p.to(dt))
    w = torch.randn_like(p)
    for a, b in zip(torch.autograd.grad(o, list(u.values()), w.to(dt)), torch.autograd.grad(p, list(r.values()), w)):
        assert torch.equal(a, b.to(a.dtype))


def test_strided_inputs_are_read_where_they_lie(pkg):
    """Projections' outputs [T, B, heads * channels] seen as [B, heads, T, channels], a part of a wider row, one sequence
    spread over a batch, and strides that have to be copied."""
    B, H, HV, T, K, V = 2, 2, 4, 130, 64, 128
    d = on_gpu(inputs(B, H, HV, T, K, V, seed=12))
    want = pkg.gated_delta.gated_delta_rule(*[d[n] for n in NAMES])[0]
    wide = torch.full((T, B, (2 * H) * K + HV * V + 8), float("nan"), device="cuda", dtype=BF)
    views = {}
    for n, at, heads, C in (("q", 0, H, K), ("k", H * K, H, K), ("v", 2 * H * K, HV, V)):
        part = wide[:, :, at:at + heads * C]
        part.copy_(d[n].permute(2, 0, 1, 3).reshape(T, B, heads * C))
        views[n] = part.view(T, B, heads, C).permute(1, 2, 0, 3)
    for n in ("g", "beta"):
        views[n] = d[n].permute(2, 0, 1).contiguous().permute(1, 2, 0)
    u = {n: t.detach().requires_grad_(True) for n, t in views.items()}
    c = {n: t.detach().contiguous().requires_grad_(True) for n, t in d.items()}
    o = pkg.gated_delta.gated_delta_rule(*[u[n] for n in NAMES])[0]
    assert torch.equal(o, want)
    w = torch.randn(T, B, HV * V, device="cuda").to(BF).view(T, B, HV, V).permute(1, 2, 0, 3)
    p = pkg.gated_delta.gated_delta_rule(*[c[n] for n in NAMES])[0]
    for a, b in zip(torch.autograd.grad(o, [u[n] for n in NAMES], w), torch.autograd.grad(p, [c[n] for n in NAMES], w.contiguous())):
        assert torch.equal(a, b)
    same = d["k"][:1].expand(B, H, T, K)                 # the same keys for every sequence
    a = pkg.gated_delta.gated_delta_rule(d["q"], same, *[d[n] for n in NAMES[2:]])[0]
    b = pkg.gated_delta.gated_delta_rule(d["q"], same.contiguous(), *[d[n] for n in NAMES[2:]])[0]
    assert torch.equal(a, b)
    odd = torch.empty(B, H, T, K + 1, device="cuda", dtype=BF)[..., :K].copy_(d["q"])
    back = d["v"].flip(-1).flip(-1).transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(pkg.gated_delta.gated_delta_rule(odd, d["k"], back, d["g"], d["beta"])[0], want)


def test_the_same_bits_every_time_and_on_other_streams(pkg):
    d = on_gpu(inputs(2, 3, 6, 333, 128, 64, seed=13))
    w = torch.randn(2, 6, 333, 64, device="cuda").to(BF)

    def once():
        u = [d[n].detach().requires_grad_(True) for n in NAMES]
        o, S = pkg.gated_delta.gated_delta_rule(*u, output_final_state=True)
        return [o, S, *torch.autograd.grad((o, S), u, (w, torch.ones_like(S)))]

    want = once()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in streams * 2:
        with torch.cuda.stream(s):
            got.append(once())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_a_captured_pass_and_a_captured_step(pkg):
    """Forward and backward, and three token steps on a state, in one graph each; eager work between the replays."""
    d = on_gpu(inputs(2, 2, 2, 200, 64, 64, seed=14, h0=True))
    w = torch.randn(2, 2, 200, 64, device="cuda").to(BF)
    leaves = [d[n].clone().requires_grad_(True) for n in NAMES]
    state = d["h0"].clone()

    def train():
        o, _ = pkg.gated_delta.gated_delta_rule(*leaves, initial_state=d["h0"])
        return [o, *torch.autograd.grad(o, leaves, w)]

    def steps():
        with torch.no_grad():
            return [pkg.gated_delta.gated_delta_step(*[d[n][:, :, t:t + 1] for n in NAMES], state) for t in range(3)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train(), steps()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for f in (train, steps):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(f())
    for rep in range(4):
        for n, t in zip(NAMES, leaves):
            t.data.copy_(d[n])
            if n == "v":
                t.data.mul_(1 + rep)
        state.copy_(d["h0"] * (1 + rep))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs[0] + outs[1]] + [state.clone()]
        state.copy_(d["h0"] * (1 + rep))
        want = train() + steps() + [state]
        assert all(torch.equal(a, b) for a, b in zip(got, want)), rep


def test_a_step_on_a_slice_of_a_pool(pkg):
    """Every second state of a pool [slots, HV, K, V] with slots between, and heads outside sequences; the others stay."""
    B, H, HV, K, V = 3, 2, 2, 64, 64
    d = on_gpu(inputs(B, H, HV, 2, K, V, seed=15, h0=True))
    want = d["h0"].clone()
    o = pkg.gated_delta.gated_delta_step(*[d[n] for n in NAMES], want)
    pool = torch.full((2 * B, HV, K, V), 7.0, device="cuda")
    pool[::2] = d["h0"]
    version = pool._version
    p = pkg.gated_delta.gated_delta_step(*[d[n] for n in NAMES], pool[::2])
    assert torch.equal(o, p) and torch.equal(pool[::2], want) and (pool[1::2] == 7).all() and pool._version > version
    heads = d["h0"].transpose(0, 1).contiguous().transpose(0, 1)
    p = pkg.gated_delta.gated_delta_step(*[d[n] for n in NAMES], heads)
    assert torch.equal(o, p) and torch.equal(heads, want)
    with torch.inference_mode():
        s = d["h0"].clone()
        assert torch.equal(pkg.gated_delta.gated_delta_step(*[d[n].clone() for n in NAMES], s), o)


def test_tokens_one_by_one_are_the_sequence(pkg):
    """A prompt by the rule, then its continuation by steps, against the rule over both."""
    d = on_gpu(inputs(2, 2, 4, 75, 128, 64, seed=16))
    cut = 70
    with torch.no_grad():
        full, last = pkg.gated_delta.gated_delta_rule(*[d[n] for n in NAMES], output_final_state=True)
        o, S = pkg.gated_delta.gated_delta_rule(*[d[n][:, :, :cut] for n in NAMES], output_final_state=True)
        rest = [pkg.gated_delta.gated_delta_step(*[d[n][:, :, t:t + 1] for n in NAMES], S) for t in range(cut, 75)]
    assert torch.equal(o, full[:, :, :cut])
    assert close("state", S, last) <= 2e-6
    assert close("o", torch.cat(rest, 2), full[:, :, cut:]) <= 1e-3        # a few values on the other side of a rounding


def test_offsets_past_32_bits(pkg):
    """A state and values whose elements lie past 2^31: the last sequences against the same alone."""
    B, HV, K, V = 5000, 8, 64, 1 << 9
    g = torch.Generator(device="cuda").manual_seed(3)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")
    q, k, v = n(B, HV, 1, K).mul_(0.1).to(BF), n(B, HV, 1, K).mul_(0.1).to(BF), n(B, HV, 1, V).to(BF)
    gg, beta = -n(B, HV, 1).abs(), n(B, HV, 1).sigmoid()
    state = torch.zeros(B, HV, K, V, device="cuda")                          # 1.3 G elements, offsets in bytes past 2^32
    state[-3:] = n(3, HV, K, V)
    alone = state[-3:].clone()
    o = pkg.gated_delta.gated_delta_step(q, k, v, gg, beta, state)
    p = pkg.gated_delta.gated_delta_step(q[-3:], k[-3:], v[-3:], gg[-3:], beta[-3:], alone)
    assert torch.equal(o[-3:], p) and torch.equal(state[-3:], alone)
    a = pkg.gated_delta.gated_delta_rule(q, k, v, gg, beta, initial_state=state, output_final_state=True)
    b = pkg.gated_delta.gated_delta_rule(q[-3:], k[-3:], v[-3:], gg[-3:], beta[-3:], initial_state=alone, output_final_state=True)
    assert close("o", a[0][-3:], b[0]) <= 1e-3 and close("state", a[1][-3:], b[1]) <= 1e-6


def test_refusals(pkg):
    d = on_gpu(inputs(2, 2, 4, 9, 64, 64, h0=True))
    rule, step = pkg.gated_delta.gated_delta_rule, pkg.gated_delta.gated_delta_step
    args = lambda **kw: [{**d, **kw}[n] for n in NAMES]
    bad = [(ValueError, dict(k=d["k"][:, :1])), (ValueError, dict(v=d["v"][:, :3])), (ValueError, dict(v=d["v"][:, :, :8])),
           (ValueError, dict(g=d["g"][:, :, :8])), (ValueError, dict(beta=d["beta"].unsqueeze(-1))), (TypeError, dict(g=d["g"].double())),
           (TypeError, dict(q=d["q"].int())), (NotImplementedError, dict(q=d["q"][..., :32], k=d["k"][..., :32])),
           (NotImplementedError, dict(v=d["v"][..., :48])), (ValueError, dict(beta=d["beta"].cpu())), (ValueError, dict(q=d["q"][0])),
           (TypeError, dict(beta=0.5))]
    for kind, kw in bad:
        with pytest.raises(kind):
            rule(*args(**kw))
        with pytest.raises(kind):
            step(*args(**kw), d["h0"])
    for kind, h0 in ((ValueError, d["h0"][:, :2]), (TypeError, d["h0"].int()), (ValueError, d["h0"].cpu())):
        with pytest.raises(kind):
            rule(*args(), initial_state=h0)
        with pytest.raises((ValueError, TypeError)):
            step(*args(), h0)
    for state in (d["h0"].to(BF), d["h0"].transpose(2, 3), d["h0"][:1].expand(2, 4, 64, 64), d["h0"].clone().requires_grad_(True)):
        before = state.detach().clone()
        with pytest.raises((ValueError, TypeError)):
            step(*args(), state)
        assert torch.equal(before, state)
    with pytest.raises(ValueError, match="backward"):
        step(*args(v=d["v"].detach().requires_grad_(True)), d["h0"].clone())
    with pytest.raises(NotImplementedError):
        v = d["v"].detach().requires_grad_(True)
        torch.autograd.grad(rule(*args(v=v))[0].float().sum(), v, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda v: rule(*args(v=v))[0].float().sum())(d["v"])


def test_a_changed_input_is_an_error_in_the_backward(pkg):
    d = on_gpu(inputs(1, 1, 1, 66, 64, 64))
    v = d["v"].requires_grad_(True)
    k = d["k"].clone()
    o, _ = pkg.gated_delta.gated_delta_rule(d["q"], k, v, d["g"], d["beta"])
    k.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()


def test_only_the_final_state_is_used(pkg):
    d = inputs(1, 2, 2, 100, 64, 64, seed=18, h0=True)
    u = {n: t.cuda().requires_grad_(True) for n, t in d.items()}
    r = {n: t.double().requires_grad_(True) for n, t in d.items()}
    _, S = pkg.gated_delta.gated_delta_rule(*[u[n] for n in NAMES], initial_state=u["h0"], output_final_state=True)
    _, rS = recurrence(*[r[n] for n in NAMES], 0.125, r["h0"])
    w = torch.randn(1, 2, 64, 64)
    for n, a, b in zip(list(u)[1:], torch.autograd.grad(S, list(u.values()), w.cuda())[1:],
                       torch.autograd.grad(rS, [r[n] for n in list(u)[1:]], w.double())):
        assert close(n, a, b) <= (2.4e-3 if a.dtype == BF else 1e-4), n


def test_a_layer_of_the_operators_together(pkg):
    """Projections, the rule, GroupNorm with a gate, the output projection, and the dropped-out residual with the next
    norm: forward and backward in bf16 against the formulas in 64 bits with the same mask."""
    from tests import philox
    T, B, H, C, p, seed = 150, 2, 4, 256, 0.25, 99
    G = torch.Generator().manual_seed(20)
    n = lambda *s: torch.randn(*s, generator=G)
    w = {k: n(C, C) / 16 for k in ("wq", "wk", "wv", "wg", "wo")}
    w.update(wd=n(H, C) / 16, wb=n(H, C) / 16, gn=1 + 0.1 * n(C), gb=0.1 * n(C), ln=1 + 0.1 * n(C), lb=0.1 * n(C))
    w = {k: t.to(BF) for k, t in w.items()}
    x, h = n(T, B, C).to(BF), n(T, B, C).to(BF)
    keep, factor = philox.kept(T * B * C, p, seed)
    mask = torch.from_numpy(keep).view(T, B, C).double() * factor
    ws, wy = n(T, B, C).to(BF), n(T, B, C).to(BF)
    F = torch.nn.functional
    heads = lambda t: t.view(T, B, H, 64).permute(1, 2, 0, 3)
    gates = lambda t: t.permute(1, 2, 0)

    def kernels():
        u = {k: t.cuda().requires_grad_(True) for k, t in dict(w, x=x, h=h).items()}
        lin = lambda k: F.linear(u["h"], u[k])
        q, k = (F.normalize(heads(lin(m)).float(), dim=-1).to(BF) for m in ("wq", "wk"))
        o, _ = pkg.gated_delta.gated_delta_rule(q, k, heads(lin("wv")), -F.softplus(gates(lin("wd")).float()), gates(lin("wb")).float().sigmoid())
        y = pkg.timemix.group_norm_gate(o, lin("wg"), u["gn"], u["gb"], 1e-5, head_first=True)
        s, z = pkg.residual.residual_norm(u["x"], F.linear(y, u["wo"]), u["ln"], u["lb"], 1e-5, dropout=p,
                                          seed=torch.tensor([seed], device="cuda"))
        return (s, z), u, torch.autograd.grad((s, z), list(u.values()), (ws.cuda(), wy.cuda()))

    def formulas():
        u = {k: t.double().requires_grad_(True) for k, t in dict(w, x=x, h=h).items()}
        lin = lambda k: u["h"] @ u[k].t()
        q, k = (F.normalize(heads(lin(m)), dim=-1) for m in ("wq", "wk"))
        o, _ = recurrence(q, k, heads(lin("wv")), -F.softplus(gates(lin("wd"))), gates(lin("wb")).sigmoid(), 0.125)
        o = o.permute(2, 0, 1, 3).reshape(T * B, C)
        y = F.group_norm(o, H, u["gn"], u["gb"], 1e-5).view(T, B, C) * F.silu(lin("wg"))
        s = u["x"] + mask * (y @ u["wo"].t())
        z = F.layer_norm(s, (C,), u["ln"], u["lb"], 1e-5)
        return (s, z), u, torch.autograd.grad((s, z), list(u.values()), (ws.double(), wy.double()))

    (s, z), u, got = kernels()
    (rs, rz), _, want = formulas()
    # a dozen bf16 roundings on the way out and as many back, 2.3e-3 of the 2-norm each at most, the norms' derivatives
    # (factors of two or so) between them
    for name, a, b in [("s", s, rs), ("z", z, rz)] + list(zip(u, got, want)):
        assert close(name, a, b) <= 3e-2, name
