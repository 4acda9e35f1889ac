"""The gated delta rule's ways through its kernels that few sizes take, against the definition in 64 bits: beta in bf16,
wide values, segments whose walks have blocks of 64 columns, sequences in segments with and without states, arrays whose
elements lie past 2^31.  Tolerances as in test_gated_delta_gpu.py; the definition runs on the GPU in 64 bits."""
import pytest
import torch

from tests.test_gated_delta_gpu import BF, F32, MANY, NAMES, SHAPES, check, close, inputs, on_gpu, recurrence, run_train

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", SHAPES + MANY, ids=str)
def test_training_with_beta_in_bf16(pkg, shape):
    B, H, HV, T, K, V = shape
    d = inputs(*shape, seed=21 + sum(shape), beta=BF)
    run_train(pkg, d, wo=torch.randn(B, HV, T, V, generator=torch.Generator().manual_seed(T)).to(BF))


@pytest.mark.parametrize("shape", [(1, 1, 2, 130, 64, 256), (2, 1, 1, 65, 64, 448), (1, 1, 1, 70, 128, 512), (1, 9, 18, 129, 64, 512)], ids=str)
def test_training_with_wide_values(pkg, shape):
    B, H, HV, T, K, V = shape
    G = torch.Generator().manual_seed(sum(shape))
    d = inputs(*shape, seed=22 + sum(shape), h0=True)
    run_train(pkg, d, final=True, wo=torch.randn(B, HV, T, V, generator=G).to(BF), wh=torch.randn(B, HV, K, V, generator=G))


def against_the_definition(pkg, d, final):
    """run_train with the definition on the GPU; d lies there."""
    G = torch.Generator(device="cuda").manual_seed(5)
    names = [n for n in (*NAMES, "h0") if n in d]
    u = {n: d[n].detach().requires_grad_(True) for n in names}
    r = {n: d[n].detach().double().requires_grad_(True) for n in names}
    o, S = pkg.gated_delta.gated_delta_rule(*[u[n] for n in NAMES], initial_state=u.get("h0"), output_final_state=final)
    steps = []
    ro, rS = recurrence(*[r[n] for n in NAMES], d["q"].shape[-1] ** -0.5, r.get("h0"), steps)
    outs, routs, ws = [o], [ro], [torch.randn(o.shape, generator=G, device="cuda").to(BF)]
    if final:
        outs.append(S), routs.append(rS), ws.append(torch.randn(S.shape, generator=G, device="cuda"))
    got = torch.autograd.grad(outs, list(u.values()), ws)
    torch.autograd.backward(routs, [w.double() for w in ws])
    norm = lambda pairs: float(sum((a * b).square().sum() for a, b in pairs)) ** 0.5
    products = {"beta": norm((w.grad, e.detach()) for w, e, _ in steps),
                "g": norm((s.grad, s.detach()) for _, _, s in steps if s.grad is not None)}
    check("o", o, ro)
    if final:
        check("state", S, rS)
    for n, a in zip(names, got):
        check("d_" + n, a, r[n].grad, products.get(n) if a.dtype == F32 else None)
    print(flush=True)


def segments(pkg, B, HV, T, K, V):
    """Of the forward's and the backward's walks, by what their workspaces hold for each segment but the last."""
    L = pkg._lib.load()
    chunks, one = B * HV * ((T + 63) // 64), B * HV * K * (K + V) * 4
    return [1 + (L.rwkv6_gated_delta_workspace_bytes(B, HV, T, K, V, back) - chunks * rest) // one
            for back, rest in ((0, 10240 + 512 + 256), (1, 4 * K * V + 256 * V))]


# more than 512 tiles of 16 columns in the walks before the segments and in the segments, forward and backward
WIDE = [(1, 12, 12, 1500, 64, 128), (1, 12, 24, 1500, 128, 128), (1, 4, 4, 1480, 64, 512)]


@pytest.mark.parametrize("shape", WIDE, ids=str)
@pytest.mark.parametrize("states", [False, True])
def test_segments_in_blocks_of_64_columns(pkg, shape, states):
    B, H, HV, T, K, V = shape
    for p in segments(pkg, B, HV, T, K, V):
        assert p > 2 and B * HV * (V // 16) * p > 512
    d = on_gpu(inputs(*shape, seed=23 + sum(shape), h0=states))
    d["g"].clamp_(min=-0.0023)                             # half of a state is left after 300 tokens
    against_the_definition(pkg, d, states)


@pytest.mark.parametrize("shape", [(1, 1, 1, 1500, 64, 64), (1, 1, 2, 2049, 64, 128), (2, 1, 1, 1300, 128, 64), (1, 2, 4, 1000, 64, 256)], ids=str)
def test_training_in_segments_without_states(pkg, shape):
    B, H, HV, T, K, V = shape
    assert segments(pkg, B, HV, T, K, V)[1] > 2
    d = on_gpu(inputs(*shape, seed=24 + sum(shape)))
    d["g"].clamp_(min=-0.0023)
    against_the_definition(pkg, d, False)


def test_the_token_step_past_2_31_elements(pkg):
    """9000 x 8 states of 64 x 512, 2.4 G elements: the last sequences against the same alone."""
    B, HV, K, V = 9000, 8, 64, 512
    G = torch.Generator(device="cuda").manual_seed(3)
    n = lambda *s: torch.randn(*s, generator=G, device="cuda")
    u = {"q": n(B, HV, 1, K).mul_(0.1).to(BF), "k": n(B, HV, 1, K).mul_(0.1).to(BF), "v": n(B, HV, 1, V).to(BF), "g": -n(B, HV, 1).abs(),
         "beta": n(B, HV, 1).sigmoid()}
    state = torch.zeros(B, HV, K, V, device="cuda")
    state[-3:] = n(3, HV, K, V)
    state[:3] = n(3, HV, K, V)
    both = torch.cat([state[:3], state[-3:]])
    with torch.no_grad():
        _, last = pkg.gated_delta.gated_delta_rule(*[u[m] for m in NAMES], initial_state=state, output_final_state=True)
        o = pkg.gated_delta.gated_delta_step(*[u[m] for m in NAMES], state)
        p = pkg.gated_delta.gated_delta_step(*[torch.cat([u[m][:3], u[m][-3:]]) for m in NAMES], both)
    assert torch.equal(o[:3], p[:3]) and torch.equal(o[-3:], p[3:])
    assert torch.equal(state[:3], both[:3]) and torch.equal(state[-3:], both[3:])
    assert close("state", last[-3:], both[3:]) <= 2e-6 and close("state", last[:3], both[:3]) <= 2e-6


def test_training_past_2_31_elements(pkg):
    """64 x 8 heads of 8320 tokens, 64 x 512: values, outputs, kept states and written values of 2.2 G elements each.  The last
    two heads against the definition."""
    B, HV, T, K, V = 64, 8, 8320, 64, 512
    G = torch.Generator(device="cuda").manual_seed(4)
    n = lambda *s: torch.randn(*s, generator=G, device="cuda", dtype=BF)
    u = {"q": n(B, HV, T, K).mul_(0.125), "k": n(B, HV, T, K).mul_(0.125), "v": n(B, HV, T, V), "g": n(B, HV, T).float().abs().mul_(-0.02),
         "beta": n(B, HV, T).float().sigmoid()}
    u["k"][-1, -2:] = torch.nn.functional.normalize(u["k"][-1, -2:].float(), dim=-1).to(BF)
    w = n(B, HV, T, V)
    r = {m: t[-1:, -2:].double().requires_grad_(True) for m, t in u.items()}
    u = {m: t.requires_grad_(True) for m, t in u.items()}
    o, _ = pkg.gated_delta.gated_delta_rule(*[u[m] for m in NAMES])
    got = torch.autograd.grad(o, list(u.values()), w)
    steps = []
    ro, _ = recurrence(*[r[m] for m in NAMES], K ** -0.5, None, steps)
    ro.backward(w[-1:, -2:].double())
    norm = lambda pairs: float(sum((a * b).square().sum() for a, b in pairs)) ** 0.5
    products = {"beta": norm((x.grad, e.detach()) for x, e, _ in steps),
                "g": norm((s.grad, s.detach()) for _, _, s in steps if s.grad is not None)}
    check("o", o[-1:, -2:], ro)
    for m, a in zip(NAMES, got):
        check("d_" + m, a[-1:, -2:], r[m].grad, products.get(m) if a.dtype == F32 else None)
