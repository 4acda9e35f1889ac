"""The operators a training step runs around its products: what is measured of them, and their plain forms.

``listed()`` names the cases; ``draw(rng)`` gives further ones of the same ranges.  ``prepare`` makes
what a program holds before the call, ``run`` is one pass: the package's entry points where ``own`` is
true, else the operator's formula in elementary torch operations in 32 bits.  ``exact`` is the
operator's definition in 64 bits.

Kinds of case (the key ``kind``):
  norm   residual.residual_norm: a block's output, gated and scaled, added to the stream, and the
         next LayerNorm; forward and backward (``train``), or the forward of a few tokens
  loss   loss.cross_entropy over the vocabulary, forward and backward
  adamw  optim.adamw_step over the parameters of RWKV-6 layers, states of 32 or 8 bits, with or
         without clipping by the gradients' norm
"""
import importlib

import torch

own = False

DEV = "cuda"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
F8, F8_MAX, BLOCK = torch.float8_e4m3fn, 448.0, 256
TINY = 2.0 ** -118                                 # a block of smaller values stores zeros
EPS = 1e-5
LR, BETAS, ADAM_EPS, DECAY, MAX_NORM, STEP = 2.5e-4, (0.9, 0.995), 1e-8, 0.1, 1.0, 100.0
TYPES = {"bf16": BF16, "fp32": F32}


# ---------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------

def listed():
    return [
        # one generated token for eight conversations: after a channel mix, into the next layer
        dict(name="norm_decode_8x2048", kind="norm", N=8, C=2048, gate=True, cbias=False, scale=1.0,
             stream="bf16", param="bf16", train=False),
        # the time mix's output into the channel mix's norm, 1.6B-shape training step
        dict(name="norm_tmix_16384x2048", kind="norm", N=16384, C=2048, gate=False, cbias=False, scale=1.0,
             stream="bf16", param="bf16", train=True),
        # the channel mix's gated output into the next layer's norm, same step
        dict(name="norm_cmix_16384x2048", kind="norm", N=16384, C=2048, gate=True, cbias=False, scale=1.0,
             stream="bf16", param="bf16", train=True),
        # 7B width, an odd number of tokens, a stream and parameters kept in fp32, a scaled residual
        # and a projection with a bias
        dict(name="norm_wide_2049x4096", kind="norm", N=2049, C=4096, gate=True, cbias=True, scale=0.5,
             stream="fp32", param="fp32", train=True),
        # the tiny language model's loss: batch 2 x 512
        dict(name="loss_1024x65536", kind="loss", N=1024, V=65536, dtype="bf16"),
        # the 1.6B-shape training step's: batch 4 x 4096
        dict(name="loss_16384x65536", kind="loss", N=16384, V=65536, dtype="bf16"),
        # an odd vocabulary, logits in fp32: no row but the first starts on 16 bytes
        dict(name="loss_1001x50001_fp32", kind="loss", N=1001, V=50001, dtype="fp32"),
        # the layers of the tiny language model, fp32 parameters: bound by launches
        dict(name="adamw_2_layers_512", kind="adamw", C=512, F=1792, L=2, V=0, dtype="fp32", bits=32, clip=True),
        # four layers of the 1.6B shape, bf16 parameters
        dict(name="adamw_4_layers_2048", kind="adamw", C=2048, F=7168, L=4, V=0, dtype="bf16", bits=32, clip=True),
        # the same with states of 8 bits
        dict(name="adamw8_4_layers_2048", kind="adamw", C=2048, F=7168, L=4, V=0, dtype="bf16", bits=8, clip=True),
        # an odd vocabulary's embedding and head with one layer, fp32 parameters, no clipping
        dict(name="adamw8_vocab_50001x512", kind="adamw", C=512, F=1792, L=1, V=50001, dtype="fp32", bits=8,
             clip=False),
    ]


def _log_int(rng, lo, hi):
    """A whole number from lo to hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    """One more case; none costs more than the largest listed one of its kind."""
    kind = rng.choice(["norm", "norm", "norm", "norm_few", "loss", "loss", "loss_few", "adamw", "adamw", "adamw"])
    if kind in ("norm", "norm_few"):
        C = 8 * _log_int(rng, 8, 1024)
        few = kind == "norm_few"
        return dict(kind="norm", N=_log_int(rng, 1, 256) if few else _log_int(rng, 64, 16384 * 2048 // C), C=C,
                    gate=rng.random() < 0.5, cbias=rng.random() < 0.3, scale=rng.choice([1.0, 1.0, 0.5, 0.2]),
                    stream=rng.choice(["bf16", "bf16", "fp32"]), param=rng.choice(["bf16", "fp32"]),
                    train=not few)
    if kind in ("loss", "loss_few"):
        V = rng.choice([_log_int(rng, 200, 131072), 65536, 32000])
        N = _log_int(rng, 1, 64) if kind == "loss_few" else _log_int(rng, 32, min(65536, 16384 * 32768 // V))
        return dict(kind="loss", N=N, V=V, dtype=rng.choice(["bf16", "bf16", "fp32"]))
    C, L = rng.choice([256, 512, 768, 1024, 2048]), rng.choice([1, 2, 3])
    return dict(kind="adamw", C=C, F=8 * rng.randint(C // 4, C // 2), L=L,
                V=rng.choice([0, _log_int(rng, 200, 65536 if C < 2048 else 4096)]),
                dtype=rng.choice(["bf16", "fp32"]), bits=rng.choice([8, 32]), clip=rng.random() < 0.6)


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, std=1.0, dtype=BF16):
    return torch.randn(*shape, generator=g, device=DEV).mul_(std).to(dtype)


def _rand(g, *shape, lo=0.0, hi=1.0, dtype=F32):
    return torch.rand(*shape, generator=g, device=DEV).mul_(hi - lo).add_(lo).to(dtype)


def _norm_inputs(case, seed):
    """The stream a few times the block's output, parameters at trained magnitudes, gradients N(0, 1)."""
    g, N, C = _gen(seed), case["N"], case["C"]
    xt, pt = TYPES[case["stream"]], TYPES[case["param"]]
    s = {"x": _randn(g, N, C, std=2.0, dtype=xt), "branch": _randn(g, N, C),
         "gate": _randn(g, N, C) if case["gate"] else None,
         "cbias": _randn(g, C, std=0.5, dtype=pt) if case["cbias"] else None,
         "weight": _rand(g, C, lo=0.5, hi=1.5, dtype=pt), "bias": _randn(g, C, std=0.1, dtype=pt)}
    if case["train"]:
        s["ds"], s["dy"] = _randn(g, N, C, dtype=xt), _randn(g, N, C)
    return s


def _loss_inputs(case, seed):
    """Logits N(0, 2^2) with the target's raised by 4, a twentieth of the targets ignored (the last position
    of a document, padding), the gradient of a mean over the rest."""
    g, N, V = _gen(seed), case["N"], case["V"]
    logits = _randn(g, N, V, std=2.0, dtype=TYPES[case["dtype"]])
    targets = torch.randint(0, V, (N,), generator=g, device=DEV)
    rows = torch.arange(N, device=DEV)
    logits[rows, targets] += 4
    ignored = torch.rand(N, generator=g, device=DEV) < 0.05
    weight = (~ignored).float() / (~ignored).sum().clamp(min=1) * _rand(g, N, lo=0.5, hi=1.5)
    return {"logits": logits, "targets": torch.where(ignored, -100, targets), "dloss": weight}


def _shapes(case):
    """The parameter shapes of L RWKV-6 layers (and an embedding with its head for V > 0)."""
    C, Fh, V = case["C"], case["F"], case["V"]
    layer = [(C,)] * 4                                                          # the two LayerNorms
    layer += [(C, 5, 32), (5, 32, C), (5, C), (C, 1, 64), (1, 64, C), (1, C)]   # the two bottlenecks
    layer += [(C,)] * 4 + [(C, C)] * 5                                          # mixing, time_first, GroupNorm; projections
    layer += [(2, C), (Fh, C), (C, C), (C, Fh)]                                 # the channel mix
    return layer * case["L"] + ([(V, C), (V, C), (C,), (77,)] if V else [])


def _adamw_inputs(case, seed):
    """Parameters, gradients and states in the middle of training: one flat buffer each, a tensor's part
    starting at a multiple of 256 elements, the elements between parts zero."""
    g, shapes = _gen(seed), _shapes(case)
    sizes = [int(torch.Size(s).numel()) for s in shapes]
    starts, total = [], 0
    for n in sizes:
        starts.append(total)
        total += -(-n // BLOCK) * BLOCK
    live = torch.ones(total, device=DEV)
    for a, n in zip(starts, sizes):
        live[a + n:a + -(-n // BLOCK) * BLOCK] = 0
    dt = TYPES[case["dtype"]]
    s = {"p": (_randn(g, total, std=0.02, dtype=F32) * live).to(dt)}
    scale = torch.exp(_rand(g, total // BLOCK, lo=-14.0, hi=-7.0)).repeat_interleave(BLOCK) * live
    s["g"] = (_randn(g, total, dtype=F32) * scale).to(dt)
    m = _randn(g, total, std=0.3, dtype=F32) * scale
    v = (_randn(g, total, dtype=F32).square() * 0.2 + 0.8) * scale.square()
    if case["bits"] == 8:
        s["m"], s["ms"] = _quantised(m)
        s["v"], s["vs"] = _quantised(v.sqrt())
    else:
        s["m"], s["v"] = m, v
    s["step"] = torch.full((), STEP, device=DEV)
    cut = lambda t: [t[a:a + n].view(shape) for a, n, shape in zip(starts, sizes, shapes)]
    part = lambda t: [t[a // BLOCK:a // BLOCK + -(-n // BLOCK)] for a, n in zip(starts, sizes)]
    s["lists"] = {n: cut(s[n]) for n in ("p", "g", "m", "v")}
    if case["bits"] == 8:
        s["lists"]["scales"] = (part(s["ms"]), part(s["vs"]))
    return s


def prepare(case, seed):
    make = {"norm": _norm_inputs, "loss": _loss_inputs, "adamw": _adamw_inputs}[case["kind"]]
    s = make(case, seed)
    if case["kind"] == "norm" and case["train"]:
        for n in _leaves(s):
            s[n].requires_grad_(True)
    if case["kind"] == "loss":
        s["logits"].requires_grad_(True)
    s["case"] = case
    return s


def _leaves(s):
    return [n for n in ("x", "branch", "gate", "cbias", "weight", "bias") if s[n] is not None]


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------

def run(s):
    kind = s["case"]["kind"]
    if own:
        return _RUN_OWN[kind](s, importlib.import_module("rwkv-megatron_amd"))
    with torch.no_grad():
        return _RUN_PLAIN[kind](s)


def _norm_own(s, pkg):
    c = s["case"]
    call = lambda: pkg.residual.residual_norm(s["x"], s["branch"], s["weight"], s["bias"], EPS, gate=s["gate"],
                                              branch_bias=s["cbias"], scale=c["scale"])
    if not c["train"]:
        with torch.no_grad():
            y = call()
        return {"s": y[0], "y": y[1]}
    st, y = call()
    names = _leaves(s)
    grads = torch.autograd.grad((st, y), [s[n] for n in names], (s["ds"], s["dy"]))
    return {"s": st, "y": y, **{"d_" + n: t for n, t in zip(names, grads)}}


def _loss_own(s, pkg):
    losses = pkg.loss.cross_entropy(s["logits"], s["targets"])
    return {"losses": losses, "d_logits": torch.autograd.grad(losses, s["logits"], s["dloss"])[0]}


def _adamw_own(s, pkg):
    c, lists = s["case"], s["lists"]
    norm = pkg.optim.adamw_step(lists["p"], lists["g"], lists["m"], lists["v"], s["step"], lr=LR, betas=BETAS,
                                eps=ADAM_EPS, weight_decay=DECAY, max_norm=MAX_NORM if c["clip"] else None,
                                scales=lists.get("scales"))
    return _adamw_outputs(s, norm)


def _adamw_outputs(s, norm):
    """The updated parameters and states (8-bit states as float8 numbers and their blocks' scales)."""
    out = {n: s[n] for n in ("p", "m", "v", "ms", "vs", "step") if n in s}
    return {**out, "norm": norm} if s["case"]["clip"] else out


# Plain forms: 32 bits, each output rounded once.

def _norm_plain(s):
    c, C = s["case"], s["case"]["C"]
    f = s["branch"].float()
    if c["cbias"]:
        f = f + s["cbias"].float()
    sg = 1 / (1 + torch.exp(-s["gate"].float())) if c["gate"] else None
    t = s["x"].float() + c["scale"] * (f * sg if c["gate"] else f)
    d = t - t.sum(-1, keepdim=True) / C
    rstd = 1 / torch.sqrt((d * d).sum(-1, keepdim=True) / C + EPS)
    xh = d * rstd
    out = {"s": t.to(s["x"].dtype), "y": (xh * s["weight"].float() + s["bias"].float()).to(BF16)}
    if not c["train"]:
        return out
    dy = s["dy"].float()
    g = dy * s["weight"].float()
    dt = s["ds"].float() + rstd * (g - g.sum(-1, keepdim=True) / C - xh * ((g * xh).sum(-1, keepdim=True) / C))
    df = c["scale"] * dt
    db = df * sg if c["gate"] else df
    out["d_x"], out["d_branch"] = dt.to(s["x"].dtype), db.to(BF16)
    if c["gate"]:
        out["d_gate"] = (df * f * sg * (1 - sg)).to(BF16)
    if c["cbias"]:
        out["d_cbias"] = db.sum(0).to(s["cbias"].dtype)
    out["d_weight"] = (dy * xh).sum(0).to(s["weight"].dtype)
    out["d_bias"] = dy.sum(0).to(s["bias"].dtype)
    return out


def _loss_plain(s):
    l, t = s["logits"].float(), s["targets"]
    rows = torch.arange(l.shape[0], device=DEV)
    live = t != -100
    at = torch.where(live, t, 0)
    m = l.amax(-1, keepdim=True)
    e = torch.exp(l - m)
    z = e.sum(-1, keepdim=True)
    losses = torch.where(live, torch.log(z[:, 0]) + (m[:, 0] - l[rows, at]), 0.0)
    d = e / z
    d[rows, at] -= 1
    w = torch.where(live, s["dloss"], 0.0)
    return {"losses": losses, "d_logits": (d * w[:, None]).to(s["logits"].dtype)}


def _quantised(x):
    """x in blocks of 256 as float8 codes and a scale a block: code = x * (448 / max), scale = max / 448."""
    b = x.view(-1, BLOCK)
    top = b.abs().amax(-1, keepdim=True)
    top = torch.where(top < TINY, 0.0, top)
    inv = torch.where(top > 0, F8_MAX / top, 0.0)
    return (b * inv).to(F8).view(-1), (top / F8_MAX).view(-1)


def _values(code, scale):
    return (code.float().view(-1, BLOCK) * scale[:, None]).view(-1)


def _adamw_plain(s):
    c, (b1, b2) = s["case"], BETAS
    g, norm = s["g"].float(), None
    if c["clip"]:
        norm = s["g"].double().square().sum().sqrt().float()
        g = g * torch.clamp(MAX_NORM / (norm + 1e-6), max=1.0)
    s["step"] += 1
    t = s["step"].double()
    bc1, bc2 = 1 - b1 ** t, torch.sqrt(1 - b2 ** t)
    m = _values(s["m"], s["ms"]) if c["bits"] == 8 else s["m"]
    v = _values(s["v"], s["vs"]).square() if c["bits"] == 8 else s["v"]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    root = torch.sqrt(v)
    update = m / (root * (1 / bc2).float() + ADAM_EPS)
    s["p"].copy_(s["p"].float() * (1 - LR * DECAY) - (LR / bc1).float() * update)
    if c["bits"] == 8:
        (qm, sm), (qv, sv) = _quantised(m), _quantised(root)
        s["m"].copy_(qm), s["ms"].copy_(sm), s["v"].copy_(qv), s["vs"].copy_(sv)
    else:
        s["m"].copy_(m), s["v"].copy_(v)
    return _adamw_outputs(s, norm)


_RUN_OWN = {"norm": _norm_own, "loss": _loss_own, "adamw": _adamw_own}
_RUN_PLAIN = {"norm": _norm_plain, "loss": _loss_plain, "adamw": _adamw_plain}


# ---------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------

def exact(case, seed):
    return {"norm": _norm_exact, "loss": _loss_exact, "adamw": _adamw_exact}[case["kind"]](case, seed)


def _norm_exact(case, seed):
    s = _norm_inputs(case, seed)
    names = _leaves(s)
    p = {n: s[n].double().requires_grad_(case["train"]) for n in names}
    f = p["branch"] + p["cbias"] if case["cbias"] else p["branch"]
    st = p["x"] + case["scale"] * (f * torch.sigmoid(p["gate"]) if case["gate"] else f)
    var, mean = torch.var_mean(st, -1, unbiased=False, keepdim=True)
    y = (st - mean) * (var + EPS).rsqrt() * p["weight"] + p["bias"]
    out = {"s": st.detach(), "y": y.detach()}
    if case["train"]:
        grads = torch.autograd.grad((st, y), [p[n] for n in names], (s["ds"].double(), s["dy"].double()))
        out.update({"d_" + n: t for n, t in zip(names, grads)})
    return out


def _loss_exact(case, seed):
    s = _loss_inputs(case, seed)
    l = s["logits"].double()
    lse = torch.logsumexp(l, -1)
    hit = (s["targets"] >= 0) & (s["targets"] < case["V"])
    picked = l.gather(-1, s["targets"].clamp(min=0)[:, None])[:, 0]
    d = l.sub_(lse[:, None]).exp_()
    d.scatter_add_(-1, s["targets"].clamp(min=0)[:, None], -torch.ones_like(lse)[:, None])
    d *= torch.where(hit, s["dloss"].double(), 0)[:, None]
    return {"losses": torch.where(hit, lse - picked, 0), "d_logits": d}


def _adamw_exact(case, seed):
    """8-bit states as the numbers that the codes round: the moment (or its root) over the block's scale."""
    s, (b1, b2) = _adamw_inputs(case, seed), BETAS
    eight = case["bits"] == 8
    wide = lambda n: s[n].double() * s[n + "s"].double().repeat_interleave(BLOCK) if eight else s[n].double()
    g = s["g"].double()
    norm = g.norm()
    if case["clip"]:
        g = g * min(1.0, MAX_NORM / (float(norm) + 1e-6))
    m = b1 * wide("m") + (1 - b1) * g
    v = b2 * (wide("v") ** 2 if eight else wide("v")) + (1 - b2) * g ** 2
    t = STEP + 1
    step = LR / (1 - b1 ** t) * m / (v.sqrt() / (1 - b2 ** t) ** 0.5 + ADAM_EPS)
    out = {"p": s["p"].double() * (1 - LR * DECAY) - step, "step": torch.full((), t, dtype=F64)}
    for n, x in (("m", m), ("v", v.sqrt() if eight else v)):
        out[n] = x
        if eight:
            out[n + "s"] = x.view(-1, BLOCK).abs().amax(-1) / F8_MAX
            out[n] = torch.nan_to_num(x / out[n + "s"].repeat_interleave(BLOCK))
    return {**out, "norm": norm} if case["clip"] else out


# ---------------------------------------------------------------------------------------
# work of one pass
# ---------------------------------------------------------------------------------------

def work(case):
    """Bytes: every input read once, every output written once.  Operations: one an arithmetic operation
    of the formula, an exponential or root counted as one."""
    size = {"bf16": 2, "fp32": 4}
    if case["kind"] == "norm":
        n, xs = case["N"] * case["C"], size[case["stream"]]
        acts = 2 + (2 if case["gate"] else 0)                       # branch, gate
        total, ops = acts + xs + xs + 2, 14                         # x, s, y
        if case["train"]:
            same = not case["gate"] and case["scale"] == 1 and xs == 2      # d_branch is dx
            total += xs + 2 + xs + (0 if same else acts)            # ds, dy, dx, d_branch, d_gate
            ops += 22
        return {"bytes": n * total + case["C"] * 4 * size[case["param"]], "flops": n * ops}
    if case["kind"] == "loss":
        n = case["N"] * case["V"]
        return {"bytes": n * 2 * size[case["dtype"]] + case["N"] * 16, "flops": n * 8}
    n = sum(int(torch.Size(s).numel()) for s in _shapes(case))
    return {"bytes": n * (3 * size[case["dtype"]] + (4 * (1 + 4 / BLOCK) if case["bits"] == 8 else 16)),
            "flops": n * (30 if case["bits"] == 8 else 18)}
