"""The gated delta rule over sequences and over tokens, and dropout in the residual add: what is measured of
them, and their plain forms.

``listed()`` names the cases; ``draw(rng)`` gives further ones of the same ranges.  ``prepare`` makes
what a program holds before the call, ``run`` is one pass: the package's entry points where ``own`` is
true, else the operator's formula in elementary torch operations in 32 bits.  ``exact`` is the
operator's definition in 64 bits.

Kinds of case (the key ``kind``):
  rule  gated_delta.gated_delta_rule over whole sequences: forward and backward (``train``), or a prompt
        that starts from a state and leaves one
  step  gated_delta.gated_delta_step: a few tokens a sequence, the state updated where it lies
  drop  residual.residual_norm with dropout: a block's output, gated, dropped out and scaled, added to
        the stream, and the next LayerNorm; forward and backward
"""
import importlib

import numpy as np
import torch

own = False

DEV = "cuda"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
CHUNK = 64                                         # tokens of a chunk of the plain form
EPS = 1e-5
TYPES = {"bf16": BF16, "fp32": F32}


# ---------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------

def listed():
    return [
        # a small language model of width 512, batch 2 x 512: bound by launches and one chunk after another
        dict(name="rule_train_2x8x512", kind="rule", B=2, H=8, HV=8, T=512, K=64, V=64, beta="bf16", train=True),
        # the heads of a 1.6B-shape layer, batch 8 x 4096
        dict(name="rule_train_8x32x4096", kind="rule", B=8, H=32, HV=32, T=4096, K=64, V=64, beta="bf16", train=True),
        # heads of 128 channels, two value heads to a key head, batch 4 x 2048
        dict(name="rule_train_4x32x2048_128", kind="rule", B=4, H=16, HV=32, T=2048, K=128, V=128, beta="bf16",
             train=True),
        # an odd number of tokens, key and value heads of different sizes, beta kept in fp32
        dict(name="rule_train_3x10x1001", kind="rule", B=3, H=5, HV=10, T=1001, K=64, V=128, beta="fp32", train=True),
        # a long prompt of one conversation, continued from a state
        dict(name="rule_prompt_1x32x32768", kind="rule", B=1, H=32, HV=32, T=32768, K=64, V=64, beta="bf16",
             train=False),
        # a short question
        dict(name="rule_prompt_1x32x77_128", kind="rule", B=1, H=16, HV=32, T=77, K=128, V=128, beta="bf16",
             train=False),
        # one generated token for eight conversations
        dict(name="step_8x32", kind="step", B=8, H=32, HV=32, T=1, K=64, V=64, beta="bf16"),
        # and for 256, heads of 128 channels
        dict(name="step_256x32_128", kind="step", B=256, H=16, HV=32, T=1, K=128, V=128, beta="bf16"),
        # four drafted tokens, odd numbers of conversations and heads
        dict(name="step_33x21x4", kind="step", B=33, H=7, HV=21, T=4, K=128, V=64, beta="fp32"),
        # the small language model's time mix into the stream
        dict(name="drop_1024x512", kind="drop", N=1024, C=512, gate=False, cbias=False, scale=1.0, p=0.1,
             stream="bf16", param="bf16"),
        # the time mix's output into the channel mix's norm, 1.6B-shape training step
        dict(name="drop_16384x2048", kind="drop", N=16384, C=2048, gate=False, cbias=False, scale=1.0, p=0.1,
             stream="bf16", param="bf16"),
        # 7B width, an odd number of tokens, a gated output with a bias, a stream and parameters kept in fp32
        dict(name="drop_wide_2049x4096", kind="drop", N=2049, C=4096, gate=True, cbias=True, scale=0.5, p=0.2,
             stream="fp32", param="fp32"),
    ]


def _log_int(rng, lo, hi):
    """A whole number from lo to hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    """One more case; none costs more than the largest listed one of its kind."""
    kind = rng.choice(["rule", "rule", "rule", "prompt", "prompt", "step", "step", "drop", "drop"])
    if kind == "drop":
        C = 8 * _log_int(rng, 8, 1024)
        return dict(kind="drop", N=_log_int(rng, 1, 16384 * 2048 // C), C=C, gate=rng.random() < 0.5,
                    cbias=rng.random() < 0.3, scale=rng.choice([1.0, 1.0, 0.5, 0.2]),
                    p=rng.choice([0.05, 0.1, 0.2, 0.5]), stream=rng.choice(["bf16", "bf16", "fp32"]),
                    param=rng.choice(["bf16", "fp32"]))
    K, V = rng.choice([64, 64, 128]), rng.choice([64, 64, 128])
    H, group = rng.randint(1, 16), rng.choice([1, 1, 2, 3])
    c = dict(kind="step" if kind == "step" else "rule", B=1, H=H, HV=H * group, T=1, K=K, V=V,
             beta=rng.choice(["bf16", "fp32"]))
    if kind == "step":
        c["B"], c["T"] = _log_int(rng, 1, 256 * 32 * 128 * 128 // (K * V * c["HV"] * 4)), rng.choice([1, 1, 1, 2, 3, 5, 8])
        return c
    c["train"] = kind == "rule"
    c["B"] = rng.choice([1, 2, 3, 4, 8]) if c["train"] else rng.choice([1, 1, 2])
    c["T"] = _log_int(rng, 1, min(4096, 8 * 32 * 4096 * 64 * 64 // (c["B"] * c["HV"] * K * V)) if c["train"] else 16384)
    return c


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, std=1.0, dtype=BF16):
    return torch.randn(*shape, generator=g, device=DEV).mul_(std).to(dtype)


def _rand(g, *shape, lo=0.0, hi=1.0, dtype=F32):
    return torch.rand(*shape, generator=g, device=DEV).mul_(hi - lo).add_(lo).to(dtype)


def _unit(g, *shape):
    x = torch.randn(*shape, generator=g, device=DEV)
    return (x / x.square().sum(-1, keepdim=True).sqrt()).to(BF16)


def _delta_inputs(case, seed):
    """Queries and keys of length 1, as a layer normalises them; values N(0, 1); the decay of a head by
    its own rate (0 to 16) and step (0.001 to 0.1), the token's share through a softplus; beta a sigmoid."""
    g, c = _gen(seed), case
    B, H, HV, T, K, V = (c[n] for n in ("B", "H", "HV", "T", "K", "V"))
    s = {"q": _unit(g, B, H, T, K), "k": _unit(g, B, H, T, K), "v": _randn(g, B, HV, T, V)}
    rate = _rand(g, HV, 1, lo=0.02, hi=16.0)
    step = torch.exp(_rand(g, HV, 1, lo=-6.9, hi=-2.3))
    s["g"] = -rate * torch.log1p(torch.exp(_randn(g, B, HV, T, std=0.5, dtype=F32) + torch.log(torch.expm1(step))))
    s["beta"] = (1 / (1 + torch.exp(-_randn(g, B, HV, T, std=1.5, dtype=F32)))).to(TYPES[c["beta"]])
    if c["kind"] == "step" or not c["train"]:
        s["state"] = _randn(g, B, HV, K, V, std=0.3, dtype=F32)
    else:
        s["do"] = _randn(g, B, HV, T, V)
    return s


def _drop_inputs(case, seed):
    """The stream a few times the block's output, parameters at trained magnitudes, gradients N(0, 1)."""
    g, N, C = _gen(seed), case["N"], case["C"]
    xt, pt = TYPES[case["stream"]], TYPES[case["param"]]
    s = {"x": _randn(g, N, C, std=2.0, dtype=xt), "branch": _randn(g, N, C),
         "gate": _randn(g, N, C) if case["gate"] else None,
         "cbias": _randn(g, C, std=0.5, dtype=pt) if case["cbias"] else None,
         "weight": _rand(g, C, lo=0.5, hi=1.5, dtype=pt), "bias": _randn(g, C, std=0.1, dtype=pt)}
    s["ds"], s["dy"] = _randn(g, N, C, dtype=xt), _randn(g, N, C)
    s["seed"] = torch.randint(0, 2 ** 62, (1,), generator=g, device=DEV)
    return s


_INPUTS = {"rule": _delta_inputs, "step": _delta_inputs, "drop": _drop_inputs}


def prepare(case, seed):
    s = _INPUTS[case["kind"]](case, seed)
    s["case"] = case
    if case["kind"] == "drop" or case.get("train"):
        for n in _leaves(s):
            s[n].requires_grad_(True)
    return s


def _leaves(s):
    names = ("x", "branch", "gate", "cbias", "weight", "bias") if s["case"]["kind"] == "drop" else ("q", "k", "v", "g", "beta")
    return [n for n in names if s[n] is not None]


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------

def run(s):
    kind = s["case"]["kind"]
    if own:
        return _RUN_OWN[kind](s, importlib.import_module("rwkv-megatron_amd"))
    with torch.no_grad():
        return _RUN_PLAIN[kind](s)


def _rule_own(s, pkg):
    args = [s[n] for n in ("q", "k", "v", "g", "beta")]
    if not s["case"]["train"]:
        with torch.no_grad():
            o, state = pkg.gated_delta.gated_delta_rule(*args, initial_state=s["state"], output_final_state=True)
        return {"o": o, "state": state}
    o, _ = pkg.gated_delta.gated_delta_rule(*args)
    return {"o": o, **{"d_" + n: t for n, t in zip(_leaves(s), torch.autograd.grad(o, args, s["do"]))}}


def _step_own(s, pkg):
    o = pkg.gated_delta.gated_delta_step(*[s[n] for n in ("q", "k", "v", "g", "beta", "state")])
    return {"o": o, "state": s["state"]}


def _drop_own(s, pkg):
    c, names = s["case"], _leaves(s)
    st, y = pkg.residual.residual_norm(s["x"], s["branch"], s["weight"], s["bias"], EPS, gate=s["gate"],
                                       branch_bias=s["cbias"], scale=c["scale"], dropout=c["p"], seed=s["seed"])
    grads = torch.autograd.grad((st, y), [s[n] for n in names], (s["ds"], s["dy"]))
    return {"s": st, "y": y, **{"d_" + n: t for n, t in zip(names, grads)}}


# Plain forms: 32 bits, each output rounded once.

def _chunks(x, group=1):
    """[B, H, T, ...] as fp32 chunks [B * H * group, chunks, 64, ...], zeros behind the last token."""
    x = x.float().repeat_interleave(group, 1).flatten(0, 1)
    pad = -x.shape[1] % CHUNK
    if pad:
        x = torch.cat([x, x.new_zeros(x.shape[0], pad, *x.shape[2:])], 1)
    return x.view(x.shape[0], -1, CHUNK, *x.shape[2:])


def _tokens(x, like):
    """Chunks back to [B, H, T, ...] in the type and sizes of `like`, heads of a group summed."""
    B, H, T = like.shape[:3]
    x = x.flatten(1, 2)[:, :T]
    return x.reshape(B, H, -1, *x.shape[1:]).sum(2).to(like.dtype) if x.shape[0] != B * H else x.reshape(like.shape).to(like.dtype)


def _rule_forms(s):
    """What forward and backward share of a chunk: the decays, the inverse of the delta rule's triangle, the
    corrected values and the states entering the chunks, one chunk after another."""
    c = s["case"]
    group, scale = c["HV"] // c["H"], c["K"] ** -0.5
    q, k, v, g, beta = _chunks(s["q"], group), _chunks(s["k"], group), _chunks(s["v"]), _chunks(s["g"]), _chunks(s["beta"])
    G = g.double().cumsum(-1)
    lower = torch.ones(CHUNK, CHUNK, device=DEV, dtype=torch.bool).tril()
    decay = torch.exp(torch.where(lower, G[..., :, None] - G[..., None, :], -torch.inf)).float()
    eG, eL, eC = torch.exp(G).float()[..., None], torch.exp(G[..., -1:] - G).float()[..., None], torch.exp(G[..., -1]).float()
    kk = (k @ k.transpose(-1, -2)) * decay
    A = (kk * beta[..., None]).tril(-1)
    # (1 + A)^-1 = (1 - A)(1 + A^2)(1 + A^4) ...: A^64 = 0
    inv = torch.eye(CHUNK, device=DEV) - A
    for _ in range(5):
        A = A @ A
        inv = inv + inv @ A
    P = (q @ k.transpose(-1, -2)) * decay * scale
    U, W = inv @ (beta[..., None] * v), inv @ (beta[..., None] * eG * k)
    S = s["state"].flatten(0, 1) if "state" in s else v.new_zeros(v.shape[0], c["K"], c["V"])
    ke, ins, news = (k * eL).transpose(-1, -2), [], []
    for i in range(q.shape[1]):
        ins.append(S)
        news.append(U[:, i] - W[:, i] @ S)
        S = eC[:, i, None, None] * S + ke[:, i] @ news[-1]
    ins, news = torch.stack(ins, 1), torch.stack(news, 1)
    o = scale * eG * (q @ ins) + P @ news
    return dict(q=q, k=k, v=v, beta=beta, decay=decay, eG=eG, eL=eL, eC=eC, kk=kk, inv=inv, P=P, W=W, ins=ins, news=news,
                o=o, S=S, scale=scale)


def _rule_plain(s):
    f = _rule_forms(s)
    out = {"o": _tokens(f["o"], s["v"])}
    if not s["case"]["train"]:
        return {**out, "state": f["S"].reshape(s["state"].shape)}
    q, k, beta, eG, eL, ins, news, scale = (f[n] for n in ("q", "k", "beta", "eG", "eL", "ins", "news", "scale"))
    T = lambda x: x.transpose(-1, -2)
    do = _chunks(s["do"])
    local, from_o = T(f["P"]) @ do, scale * (T(q * eG) @ do)
    dS, outs, dnews = torch.zeros_like(ins[:, 0]), [], []
    for i in reversed(range(q.shape[1])):
        outs.append(dS)
        dnews.append(local[:, i] + (k[:, i] * eL[:, i]) @ dS)
        dS = f["eC"][:, i, None, None] * dS + from_o[:, i] - T(f["W"][:, i]) @ dnews[-1]
    outs, dnews = torch.stack(outs[::-1], 1), torch.stack(dnews[::-1], 1)
    r = T(f["inv"]) @ dnews
    dv = beta[..., None] * r
    dP, dM = (do @ T(news)).tril() * f["decay"] * scale, -(dv @ T(news)).tril(-1) * f["decay"]
    kS = k @ ins
    dq = scale * eG * (do @ T(ins)) + dP @ k
    k_out = eL * (news @ T(outs))                                # through the chunk's last state
    k_in = -eG * (dv @ T(ins))                                   # through the values' correction
    dk = k_out + k_in + T(dP) @ q + dM @ k + T(dM) @ k
    pairs = dM * (k @ T(k))
    dbeta = (r * (f["v"] - eG * kS)).sum(-1) - ((r @ T(news)).tril(-1) * f["kk"]).sum(-1)
    writes = dP * (q @ T(k))
    dG = scale * (eG * (do @ T(ins)) * q).sum(-1) + writes.sum(-1) - writes.sum(-2) + (k_in * k).sum(-1) + pairs.sum(-1) - pairs.sum(-2)
    kept = (k_out * k).sum(-1)
    dG = dG - kept
    dG[..., -1] += kept.sum(-1) + f["eC"] * (ins * outs).sum((-1, -2))
    dg = dG.flip(-1).cumsum(-1).flip(-1)
    for n, x in (("q", dq), ("k", dk), ("v", dv), ("g", dg), ("beta", dbeta)):
        out["d_" + n] = _tokens(x, s[n])
    return out


def _step_plain(s):
    c = s["case"]
    group = c["HV"] // c["H"]
    q, k = (s[n].float().repeat_interleave(group, 1) * f for n, f in (("q", c["K"] ** -0.5), ("k", 1.0)))
    v, a, beta, S, o = s["v"].float(), torch.exp(s["g"].float()), s["beta"].float(), s["state"], []
    for t in range(c["T"]):
        S = S * a[:, :, t, None, None]
        e = beta[:, :, t, None] * (v[:, :, t] - (S * k[:, :, t, :, None]).sum(-2))
        S = S + k[:, :, t, :, None] * e[:, :, None]
        o.append((S * q[:, :, t, :, None]).sum(-2))
    s["state"].copy_(S)
    return {"o": torch.stack(o, 2).to(BF16), "state": s["state"]}


def _philox(seed, n):
    """n numbers of 16 bits: Philox4x32-10 (Salmon et al. 2011) of the counters 0, 1, 2, ... under the key
    `seed`, eight from each, low halves first."""
    low = 0xFFFFFFFF
    c0 = torch.arange(-(-n // 8), device=DEV)
    c0, c1 = c0 & low, c0 >> 32
    c2, c3, k0, k1 = torch.zeros_like(c0), torch.zeros_like(c0), seed & low, (seed >> 32) & low
    product = lambda m, x: ((m * (x >> 16) + ((m * (x & 0xFFFF)) >> 16)) >> 16, (m * (x & 0xFFFF) + ((m * (x >> 16) & 0xFFFF) << 16)) & low)
    for _ in range(10):
        (h0, l0), (h1, l1) = product(0xD2511F53, c0), product(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([x for w in (c0, c1, c2, c3) for x in (w & 0xFFFF, w >> 16)], -1).view(-1)[:n]


def _drop_plain(s):
    c, C = s["case"], s["case"]["C"]
    cut = round(c["p"] * 65536)
    kept = (_philox(s["seed"], c["N"] * C) >= cut).view(c["N"], C).float() * (65536 / (65536 - cut))
    f = s["branch"].float()
    if c["cbias"]:
        f = f + s["cbias"].float()
    sg = 1 / (1 + torch.exp(-s["gate"].float())) if c["gate"] else None
    t = s["x"].float() + c["scale"] * (kept * (f * sg if c["gate"] else f))
    d = t - t.sum(-1, keepdim=True) / C
    rstd = 1 / torch.sqrt((d * d).sum(-1, keepdim=True) / C + EPS)
    xh = d * rstd
    out = {"s": t.to(s["x"].dtype), "y": (xh * s["weight"].float() + s["bias"].float()).to(BF16)}
    dy = s["dy"].float()
    g = dy * s["weight"].float()
    dt = s["ds"].float() + rstd * (g - g.sum(-1, keepdim=True) / C - xh * ((g * xh).sum(-1, keepdim=True) / C))
    df = c["scale"] * kept * dt
    db = df * sg if c["gate"] else df
    out["d_x"], out["d_branch"] = dt.to(s["x"].dtype), db.to(BF16)
    if c["gate"]:
        out["d_gate"] = (df * f * sg * (1 - sg)).to(BF16)
    if c["cbias"]:
        out["d_cbias"] = db.sum(0).to(s["cbias"].dtype)
    out["d_weight"] = (dy * xh).sum(0).to(s["weight"].dtype)
    out["d_bias"] = dy.sum(0).to(s["bias"].dtype)
    return out


_RUN_OWN = {"rule": _rule_own, "step": _step_own, "drop": _drop_own}
_RUN_PLAIN = {"rule": _rule_plain, "step": _step_plain, "drop": _drop_plain}


# ---------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------

def exact(case, seed):
    return {"rule": _rule_exact, "step": _rule_exact, "drop": _drop_exact}[case["kind"]](case, seed)


def _rule_exact(case, seed):
    """The recurrence, token by token:  S' = e^g S,  e = v - S'^T k,  S = S' + beta k e^T,  o = scale S^T q."""
    c, s = case, _delta_inputs(case, seed)
    B, H, HV, T, K, V = (c[n] for n in ("B", "H", "HV", "T", "K", "V"))
    if T > 40000:
        return None
    train = c.get("train", False)
    group, scale = HV // H, K ** -0.5
    first = lambda x: x.double().movedim(2, 0).contiguous()                      # token first
    q, k = (first(s[n].repeat_interleave(group, 1)) for n in ("q", "k"))
    v, a, beta = first(s["v"]), first(s["g"]).exp(), first(s["beta"])
    S = s["state"].double() if "state" in s else torch.zeros(B, HV, K, V, dtype=F64, device=DEV)
    states, e, o = [], torch.empty_like(v), torch.empty_like(v)
    for t in range(T):
        S = S * a[t, :, :, None, None]
        e[t] = v[t] - (k[t, :, :, None] @ S)[:, :, 0]
        if train:
            states.append(S)                                                     # decayed, before the token
        S = torch.addcmul(S, k[t, ..., None], (beta[t, :, :, None] * e[t])[:, :, None])
        o[t] = scale * (q[t, :, :, None] @ S)[:, :, 0]
    back = lambda x: x.movedim(0, 2)
    if not train:
        return {"o": back(o), "state": S}
    do, dS = first(s["do"]), torch.zeros_like(S)
    dq, dk, dv, dg, db = (torch.zeros_like(x) for x in (q, k, v, a, beta))
    for t in reversed(range(T)):
        dec = states.pop()
        S = torch.addcmul(dec, k[t, ..., None], (beta[t, :, :, None] * e[t])[:, :, None])
        dq[t] = scale * (S @ do[t, ..., None])[..., 0]
        dS = torch.addcmul(dS, q[t, ..., None], scale * do[t, :, :, None])
        into = (k[t, :, :, None] @ dS)[:, :, 0]                                  # gradient of beta e
        db[t] = (into * e[t]).sum(-1)
        dv[t] = beta[t, :, :, None] * into
        dk[t] = (dS @ (beta[t, :, :, None] * e[t])[..., None])[..., 0] - (dec @ dv[t, ..., None])[..., 0]
        dS = dS - k[t, ..., None] * dv[t, :, :, None]
        dg[t] = (dS * dec).sum((-1, -2))
        dS = dS * a[t, :, :, None, None]
    heads = lambda x: back(x).unflatten(1, (H, group)).sum(2)
    return {"o": back(o), "d_q": heads(dq), "d_k": heads(dk), "d_v": back(dv), "d_g": back(dg), "d_beta": back(db)}


def _drop_exact(case, seed):
    s, c = _drop_inputs(case, seed), case
    cut = round(c["p"] * 65536)
    # Philox4x32-10 on 64-bit words of the host
    n, key = c["N"] * c["C"], int(s["seed"])
    word = np.zeros((4, -(-n // 8)), np.uint64)
    word[0] = np.arange(word.shape[1]) & 0xFFFFFFFF
    word[1] = np.arange(word.shape[1]) >> 32
    for r in range(10):
        a, b = word[0] * np.uint64(0xD2511F53), word[2] * np.uint64(0xCD9E8D57)
        k0, k1 = (key + r * 0x9E3779B9) & 0xFFFFFFFF, ((key >> 32) + r * 0xBB67AE85) & 0xFFFFFFFF
        word = np.stack([(b >> np.uint64(32)) ^ word[1] ^ np.uint64(k0), b & np.uint64(0xFFFFFFFF),
                         (a >> np.uint64(32)) ^ word[3] ^ np.uint64(k1), a & np.uint64(0xFFFFFFFF)])
    bits = np.ascontiguousarray(word.T.astype("<u4")).view("<u2").reshape(-1)[:n]
    kept = torch.from_numpy((bits >= cut).reshape(c["N"], c["C"])).to(DEV).double() / (1 - cut / 65536)
    names = [m for m in ("x", "branch", "gate", "cbias", "weight", "bias") if s[m] is not None]
    p = {m: s[m].double().requires_grad_(True) for m in names}
    f = p["branch"] + p["cbias"] if c["cbias"] else p["branch"]
    st = p["x"] + c["scale"] * kept * (f * torch.sigmoid(p["gate"]) if c["gate"] else f)
    var, mean = torch.var_mean(st, -1, unbiased=False, keepdim=True)
    y = (st - mean) * (var + EPS).rsqrt() * p["weight"] + p["bias"]
    grads = torch.autograd.grad((st, y), [p[m] for m in names], (s["ds"].double(), s["dy"].double()))
    return {"s": st.detach(), "y": y.detach(), **{"d_" + m: t for m, t in zip(names, grads)}}


# ---------------------------------------------------------------------------------------
# work of one pass
# ---------------------------------------------------------------------------------------

def work(case):
    """Bytes: every input read once, every output written once.  Operations: those of the recurrence and of
    the formulas, one each, an exponential or root counted as one."""
    c, size = case, {"bf16": 2, "fp32": 4}
    if c["kind"] == "drop":
        n, xs = c["N"] * c["C"], size[c["stream"]]
        acts = 4 if c["gate"] else 2                                # branch, gate
        total = 2 * (acts + xs) + xs + 2 + xs + 2                   # x, branch, gate and their gradients; s, y, ds, dy
        return {"bytes": n * total + c["C"] * 4 * size[c["param"]], "flops": n * 40}
    B, H, HV, T, K, V = (c[n] for n in ("B", "H", "HV", "T", "K", "V"))
    qk, vo, gates = B * H * T * K * 4, B * HV * T * V * 4, B * HV * T * (4 + size[c["beta"]])
    if c.get("train"):
        return {"bytes": 2 * qk + 2 * vo + 2 * gates, "flops": B * HV * T * K * V * 21}
    return {"bytes": qk + vo + gates + 2 * B * HV * K * V * 4, "flops": B * HV * T * K * V * 7}
