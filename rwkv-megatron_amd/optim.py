"""AdamW over many tensors at once, with states in 32 or in 8 bits and clipping by the gradients' norm.

The reference trains with AdamW, decoupled weight decay and a gradient clip
(/root/reference/example_config.yaml:199-221; Megatron's training loop, pretrain_rwkv6.py:281-286).

    norm = sqrt(sum of all gradients' squares)        c = min(1, max_norm / (norm + 1e-6))
    g = c g;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;  t = step + 1
    p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)

* ``AdamW`` is the optimizer (a torch.optim.Optimizer); ``adamw_step`` the same step on lists of
  tensors; ``grad_norm`` the norm alone.
* Parameters are bf16 or fp32; the arithmetic and the moments are fp32, p is rounded once.  A bf16
  parameter has no wider copy: where that matters keep the parameters in fp32, as the modules here
  take them.
* 8-bit states: float8 (e4m3) codes and one fp32 scale for every 256 consecutive elements; the second
  moment by its root, which doubles the range that a code covers.  ``AdamW`` rounds codes up or down so
  that both moments are right on average, by less than 2^-3 of the value (the root's); over a run of steps the
  root of the second moment then scatters by about a sixth of its value around that of 32 bits.
  ``adamw_step`` alone rounds to the nearest code (2^-4 of the value at most) unless it is told otherwise:
  the nearest code of a second moment that moves by less than half a code a step is the old one, so over
  many such steps it follows its block's largest and not its own gradients.
* A step is a handful of launches whatever the number of tensors, nothing is copied to or read from
  the device, and the step count lives there: a captured step (HIP graph) counts on replay.
"""
from __future__ import annotations

import torch

from . import _lib

BLOCK = 256                    # elements under one scale of an 8-bit state


def grad_norm(grads):
    """The 2-norm of all elements of `grads` (bf16 or fp32 tensors on one GPU), a 0-dim fp32 tensor; the sum
    of squares in 64 bits, in a fixed order."""
    grads = _tensors("grads", grads)
    native = _lib.native()
    return native.grad_norm(native.grad_norm_sums(grads))


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, *, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
               max_norm=None, scales=None, rounding="nearest"):
    """One AdamW step over lists of tensors, in place.

    params, grads: bf16 or fp32, dense in memory; exp_avgs, exp_avg_sqs: fp32 of the parameters' shapes,
    or with scales = (exp_avg_scales, exp_avg_sq_scales) float8_e4m3fn codes, the scales fp32
    [ceil(numel / 256)] a tensor (exp_avg_sqs then stands for the roots: v = (code * scale)^2; rounding
    "nearest", or "stochastic" for a run of steps, module docstring).  step: one
    fp32 number on the GPU, the steps done before; it is counted up.  lr is a number or a one-element fp32
    tensor on the GPU.  With max_norm the gradients count times min(1, max_norm / (norm + 1e-6)), without
    being changed, and the norm over all of them is returned (0-dim fp32), else None."""
    params, grads = _tensors("params", params), _tensors("grads", grads)
    m, v = _tensors("exp_avgs", exp_avgs), _tensors("exp_avg_sqs", exp_avg_sqs)
    ms, vs = ([], []) if scales is None else (_tensors("scales", scales[0]), _tensors("scales", scales[1]))
    if scales is not None and not len(ms) == len(vs) == len(params):
        raise ValueError("lists of different lengths")
    if rounding not in ("nearest", "stochastic"):
        raise ValueError(f'rounding must be "nearest" or "stochastic", got {rounding!r}')
    _check_hyper(lr, betas, eps, weight_decay, max_norm)
    native = _lib.native()
    sums = None if max_norm is None else native.grad_norm_sums(grads)
    return _step(native, params, grads, m, v, ms, vs, step, lr, betas, eps, weight_decay, max_norm, sums,
                 rounding == "stochastic")


def _step(native, params, grads, m, v, ms, vs, step, lr, betas, eps, weight_decay, max_norm, sums, stochastic):
    tensor = isinstance(lr, torch.Tensor) and lr.is_cuda
    return native.adamw_step(params, grads, m, v, ms, vs, step, 0.0 if tensor else float(lr), lr if tensor else None,
                             betas[0], betas[1], eps, weight_decay, 0.0 if max_norm is None else max_norm, sums, stochastic)


def _tensors(name, ts):
    ts = list(ts)                               # the tensors themselves are looked at where they are read
    if not ts:
        raise TypeError(f"{name} must be tensors, one at least")
    return ts


def _check_hyper(lr, betas, eps, weight_decay, max_norm):
    if not isinstance(lr, torch.Tensor) and not lr >= 0:
        raise ValueError(f"invalid learning rate {lr}")
    if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
        raise ValueError(f"betas must lie in [0, 1), got {betas}")
    if not eps >= 0 or not weight_decay >= 0:
        raise ValueError(f"eps and weight_decay must not be negative, got {eps} and {weight_decay}")
    if max_norm is not None and not max_norm > 0:
        raise ValueError(f"max_norm must be positive, got {max_norm}")


def _not_captured(what):
    """Raises where a captured step would make tensors that every replay makes anew."""
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what}: run one such step before it is captured in a graph")


class AdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay over bf16 or fp32 parameters on one GPU.

    state_bits=8 keeps the moments in 8 bits (module docstring; rounded right on average, the same bits for
    the same step, gradient and state) for tensors of min_8bit_numel elements and more; smaller ones (norms,
    biases, mixing coefficients) keep 32 bits.  max_norm clips by the norm of all gradients of the step, in
    all groups (`grad_norm` holds it afterwards, a 0-dim tensor); the gradients themselves stay as they are.  lr may be a one-element fp32 tensor on the GPU, which a
    captured step reads on replay; a step is captured after one like it has run (the states exist then).

    State of a parameter: ``step`` (one tensor for all parameters that have made the same steps),
    ``exp_avg`` and ``exp_avg_sq`` (fp32), or in 8 bits ``exp_avg``, ``exp_avg_scale``, ``exp_avg_sq_root`` and
    ``exp_avg_sq_scale``.  A state dict of torch.optim.AdamW loads; states are converted to the kind
    that this optimizer keeps for the parameter."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32,
                 max_norm=None, min_8bit_numel=4096):
        _check_hyper(lr, betas, eps, weight_decay, max_norm)
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        self.state_bits, self.max_norm, self.min_8bit_numel = state_bits, max_norm, min_8bit_numel
        self.grad_norm = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def __getstate__(self):                        # torch's own holds the state and the groups alone
        own = dict(state_bits=self.state_bits, max_norm=self.max_norm, min_8bit_numel=self.min_8bit_numel, grad_norm=None)
        return {**super().__getstate__(), **own}

    def add_param_group(self, group):
        super().add_param_group(group)
        g = self.param_groups[-1]
        try:
            _check_hyper(g["lr"], g["betas"], g["eps"], g["weight_decay"], None)
            for p in g["params"]:
                if p.dtype not in (torch.bfloat16, torch.float32):
                    raise TypeError(f"parameters must be bfloat16 or float32, got {p.dtype}")
        except Exception:
            self.param_groups.pop()
            raise

    def _eight(self, p):
        return self.state_bits == 8 and p.numel() >= self.min_8bit_numel

    def _new_state(self, p):
        like = dict(memory_format=torch.preserve_format)
        if not self._eight(p):
            return {"exp_avg": torch.zeros_like(p, dtype=torch.float32, **like),
                    "exp_avg_sq": torch.zeros_like(p, dtype=torch.float32, **like)}
        scale = lambda: torch.zeros(-(-p.numel() // BLOCK), dtype=torch.float32, device=p.device)
        code = lambda: torch.zeros_like(p, dtype=torch.uint8, **like).view(torch.float8_e4m3fn)
        return {"exp_avg": code(), "exp_avg_scale": scale(), "exp_avg_sq_root": code(), "exp_avg_sq_scale": scale()}

    def _lists(self, group):
        """The group's parameters with gradients in lists that one call updates: those of one kind of state
        that have made the same steps, and so share the tensor that counts them."""
        lists, sharing, new = {}, {}, {}
        for p in group["params"]:
            if p.grad is not None:
                if p.grad.is_sparse:
                    raise RuntimeError("AdamW does not take sparse gradients")
                if p.device.type != "cuda":
                    raise ValueError("parameters must live on the GPU")
                if not self.state[p]:
                    _not_captured("the first step of a parameter makes its states")
                    key = (p.device, self._eight(p))
                    if key not in new:
                        new[key] = torch.zeros((), dtype=torch.float32, device=p.device)
                    self.state[p].update(step=new[key], **self._new_state(p))
            if self.state.get(p):
                key = id(self.state[p]["step"])
                sharing[key] = sharing.get(key, 0) + 1
                if p.grad is not None:
                    lists.setdefault(key, []).append(p)
        for key, ps in lists.items():
            if len(ps) < sharing[key]:             # the others make no step: these go on with a count of their own
                _not_captured("parameters that have made the same steps part")
                step = self.state[ps[0]]["step"].clone()
                for p in ps:
                    self.state[p]["step"] = step
        return list(lists.values())

    @torch.no_grad()
    def step(self, closure=None):
        """One step; returns the closure's loss, if there is one."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        work = [(group, ps) for group in self.param_groups for ps in self._lists(group)]
        if not work:
            return loss
        native, sums = _lib.native(), None
        if self.max_norm is not None:
            _check_hyper(0.0, (0, 0), 0, 0, self.max_norm)
            sums = native.grad_norm_sums([p.grad for _, ps in work for p in ps])
        for group, ps in work:
            states = [self.state[p] for p in ps]
            eight = "exp_avg_scale" in states[0]
            take = lambda name: [s[name] for s in states]
            norm = _step(native, ps, [p.grad for p in ps], take("exp_avg"),
                         take("exp_avg_sq_root" if eight else "exp_avg_sq"), take("exp_avg_scale") if eight else [],
                         take("exp_avg_sq_scale") if eight else [], states[0]["step"], group["lr"], group["betas"],
                         group["eps"], group["weight_decay"], self.max_norm, sums, True)
        self.grad_norm = norm
        return loss

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """Loads a state dict of this class or of torch.optim.AdamW; states keep their own types (torch's
        loading would cast them to the parameters').  A step of another kind (amsgrad, maximize, weight decay
        added to the gradient) is refused, and so is a state that does not have its parameter's shape; the
        optimizer is then as it was.  Pre-hooks may change the dict, post-hooks find the states loaded."""
        loaded = {}

        def take(_, sd):                           # the last pre-hook: sees what the others made of the dict
            loaded.update(self._loaded(sd))
            return {**sd, "state": {}}

        hooks = [self.register_load_state_dict_pre_hook(take),
                 self.register_load_state_dict_post_hook(lambda _: self.state.update(loaded), prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for h in hooks:
                h.remove()

    def _loaded(self, state_dict):
        """The states that a state dict stands for, a parameter, as this optimizer keeps them."""
        saved_groups = [g["params"] for g in state_dict["param_groups"]]
        groups = [g["params"] for g in self.param_groups]
        if [len(g) for g in saved_groups] != [len(g) for g in groups]:
            raise ValueError("the state dict has other parameter groups than the optimizer")
        for g in state_dict["param_groups"]:
            if g.get("amsgrad") or g.get("maximize") or (g.get("weight_decay") and not g.get("decoupled_weight_decay", True)):
                raise ValueError("the state dict is of a step with amsgrad, maximize or weight decay in the gradient")
        pairs = [[(p, state_dict["state"][i]) for i, p in zip(ids, ps) if state_dict["state"].get(i)]
                 for ids, ps in zip(saved_groups, groups)]
        for st in state_dict["state"].values():
            if st:
                _check_names(st)
        for p, st in (pair for group in pairs for pair in group):
            _check_shapes(p, st)
        loaded = {}
        for group in pairs:
            steps = {}                             # one tensor for equal counts, as a run would have made them
            for p, old in group:
                state = self._new_state(p)
                key = (float(old["step"]), p.device, "exp_avg_scale" in state)
                if key not in steps:
                    steps[key] = torch.full((), key[0], dtype=torch.float32, device=p.device)
                if ("exp_avg_scale" in state and "exp_avg_scale" in old
                        and state["exp_avg"].stride() == old["exp_avg"].stride()):
                    for name, t in state.items():
                        t.copy_(old[name])
                else:
                    m, v = _moments(old)
                    if "exp_avg_scale" in state:
                        _encode(state["exp_avg"], state["exp_avg_scale"], m.to(p.device))
                        _encode(state["exp_avg_sq_root"], state["exp_avg_sq_scale"], v.to(p.device).sqrt())
                    else:
                        state["exp_avg"].copy_(m)
                        state["exp_avg_sq"].copy_(v)
                loaded[p] = dict(step=steps[key], **state)
        return loaded

    def moments(self, p):
        """The fp32 values that a parameter's states stand for: (exp_avg, exp_avg_sq)."""
        return _moments(self.state[p])


def _check_names(state):
    """Raises for a state that is neither torch's AdamW's nor an 8-bit one of this class."""
    eight = {"exp_avg_scale", "exp_avg_sq_root", "exp_avg_sq_scale"}
    wanted = {"step", "exp_avg", *(eight if eight & set(state) else {"exp_avg_sq"})}
    if not wanted <= set(state):
        raise ValueError(f"the state dict is not of an AdamW step: a state holds {sorted(state)}")


def _check_shapes(p, state):
    for name in ("exp_avg", "exp_avg_sq", "exp_avg_sq_root"):
        if name in state and state[name].shape != p.shape:
            raise ValueError(f"a state's {name} has the shape {tuple(state[name].shape)}, its parameter {tuple(p.shape)}")
    for name in ("exp_avg_scale", "exp_avg_sq_scale"):
        blocks = -(-p.numel() // BLOCK)
        if name in state and tuple(state[name].shape) != (blocks,):
            raise ValueError(f"{name} must be a scale for {BLOCK} elements of a shape {tuple(p.shape)}, {blocks} in all, "
                             f"got {tuple(state[name].shape)}")


def _flat(t):
    """The elements of a dense tensor in the order they lie in memory."""
    return t.as_strided((t.numel(),), (1,))


def _decode(code, scale):
    out = torch.empty_like(code, dtype=torch.float32)
    s = scale.repeat_interleave(BLOCK)[:code.numel()]
    _flat(out).copy_(_flat(code).float() * s)
    return out


def _encode(code, scale, value):
    """value into code (of the same strides as the parameter) and scale, as the kernel rounds."""
    v = torch.empty_like(code, dtype=torch.float32).copy_(value)
    n = code.numel()
    b = torch.zeros(scale.numel() * BLOCK, dtype=torch.float32, device=code.device)
    b[:n] = _flat(v)
    b = b.view(-1, BLOCK)
    top = torch.where(b.isfinite(), b, 0).abs().amax(-1)
    top = torch.where(top < 2.0 ** -118, 0.0, top)
    inv = torch.where(top > 0, top.reciprocal() * 448.0, 0.0)
    _flat(code).copy_((b * inv[:, None]).to(torch.float8_e4m3fn).view(-1)[:n])
    scale.copy_(top * (1.0 / 448.0))


def _moments(state):
    if "exp_avg_scale" in state:
        return (_decode(state["exp_avg"], state["exp_avg_scale"]),
                _decode(state["exp_avg_sq_root"], state["exp_avg_sq_scale"]).square())
    return state["exp_avg"].float(), state["exp_avg_sq"].float()
