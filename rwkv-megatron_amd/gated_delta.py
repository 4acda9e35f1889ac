"""The gated delta rule, a recurrent mixer beside WKV6, on HIP kernels.

A head keeps a state S [K, V] that a token decays, corrects towards its value at its key, and reads:

    S' = e^g S        e = v - S'^T k        S = S' + beta k e^T        o = scale S^T q

``gated_delta_rule`` runs whole sequences in chunks of 64 tokens, with gradients;
``gated_delta_step`` runs a few tokens of each sequence on a state that it updates where it lies.
The reference has no such mixer; the layouts are those of ``chunk_rwkv6`` (head-first, a state in and
out), and o is laid out as ``timemix.group_norm_gate(..., head_first=True)`` reads it where V is 64.
The autograd function is csrc/autograd.cpp's; it raises if the HIP library is missing, there is no
fallback.
"""
from __future__ import annotations

import torch

from . import _lib

_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def gated_delta_rule(q, k, v, g, beta, scale=None, initial_state=None, output_final_state=False):
    """Returns ``(o, final_state or None)``.

    q, k [B,H,T,K] with K 64 or 128; v [B,HV,T,V] with V a multiple of 64 up to 512, HV a multiple of H:
    value head h reads key head h // (HV // H).  g [B,HV,T] is the log decay (at most 0 for a state that stays
    bounded; below -1024 it is -1024), beta [B,HV,T] the share of the correction.  Keys are expected at
    length 1 or less (longer ones make the correction overshoot, as the formula has it); nothing is normalised
    here.  scale None means K**-0.5.  initial_state [B,HV,K,V]; final_state is fp32.

    q, k, v are used as bf16 (fp32 and fp16 are rounded on entry), o [B,HV,T,V] has v's type.  g and the states
    are fp32, beta bf16 or fp32.  Inside, 32 bits: o and the gradients of q, k and v are rounded to bf16 once (then to
    their tensor's type), final_state and the gradients of g and initial_state not at all.  q, k, v may be strided (a projection's output seen as [B,H,T,K] is read where it lies).  Gradients for
    all inputs, also from final_state; the backward itself cannot be differentiated.  The same bits every time.

    Kept for the backward: about 680 bytes a token and value head at K = V = 64 (of each chunk of 64 tokens its
    triangle, the state that enters it and the values it writes, in 32 bits).  A chunk is one system of equations: a NaN
    or an infinity in a token may reach every token of its chunk, those before it too, so padding holds finite numbers."""
    scale = q.shape[-1] ** -0.5 if scale is None and isinstance(q, torch.Tensor) and q.dim() else scale
    try:
        out = _lib.native().gated_delta_rule(q, k, v, g, beta, initial_state, float(scale), bool(output_final_state))
    except TypeError:                       # not a tensor: say which; or raised on the way (a hook)
        _validate(q, k, v, g, beta)
        raise
    if out is None:
        _validate(q, k, v, g, beta)
        _validate_state("initial_state", initial_state, q, v)
        raise ValueError("gated_delta_rule's arguments do not fit together")
    return out


def gated_delta_step(q, k, v, g, beta, state, scale=None):
    """The rule over a few tokens (one of a conversation, or a handful of drafted ones): returns o [B,HV,T,V] in
    v's type and updates state [B,HV,K,V] in place.

    Shapes and types as gated_delta_rule's; state is fp32, each [K,V] of it dense, sequences and heads at any
    strides that are multiples of 4 (a slice of a larger pool is updated where it lies).  Arithmetic in 32 bits.  There is no backward: nothing
    that requires a gradient is taken while gradients are recorded, and no dual tensor of forward-mode derivatives."""
    scale = q.shape[-1] ** -0.5 if scale is None and isinstance(q, torch.Tensor) and q.dim() else scale
    try:
        out = _lib.native().gated_delta_step(q, k, v, g, beta, state, float(scale))
    except TypeError:
        _validate(q, k, v, g, beta)
        raise
    if out is None:
        _validate(q, k, v, g, beta)
        _validate_state("state", state, q, v)
        if state.dtype != torch.float32:
            raise TypeError(f"state must be float32, got {state.dtype}")
        if state.stride(3) != 1 or state.stride(2) != state.shape[3]:
            raise ValueError("state must have each [K,V] dense in memory")
        if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, g, beta, state)):
            raise ValueError("gated_delta_step has no backward: call it under torch.no_grad(), or gated_delta_rule")
        if state.requires_grad:
            raise ValueError("state is updated in place and cannot require a gradient")
        raise ValueError("gated_delta_step's arguments do not fit together")
    return out


def _validate(q, k, v, g, beta):
    named = (("q", q), ("k", k), ("v", v), ("g", g), ("beta", beta))
    for name, t in named:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if t.device.type != "cuda":
            raise ValueError(f"{name} must live on the GPU (got {t.device})")
        if t.dtype not in _TYPES:
            raise TypeError(f"{name}: unsupported dtype {t.dtype}")
        if t.layout != torch.strided:
            raise NotImplementedError(f"{name} must be a strided tensor")
    if q.dim() != 4:
        raise ValueError(f"q must be [B,H,T,K], got shape {tuple(q.shape)}")
    if k.shape != q.shape:
        raise ValueError(f"k must match q's shape {tuple(q.shape)}, got {tuple(k.shape)}")
    B, H, T, K = q.shape
    if v.dim() != 4 or v.shape[0] != B or v.shape[2] != T:
        raise ValueError(f"v must be [B,HV,T,V] with B, T of q, got {tuple(v.shape)}")
    HV, V = v.shape[1], v.shape[3]
    if H < 1 or HV < 1 or HV % H:
        raise ValueError(f"the value heads ({HV}) must be a multiple of the key heads ({H})")
    if K not in (64, 128) or V % 64 or not 64 <= V <= 512:
        raise NotImplementedError(f"K must be 64 or 128 and V a multiple of 64 up to 512, got K={K}, V={V}")
    for name, t in (("g", g), ("beta", beta)):
        if tuple(t.shape) != (B, HV, T):
            raise ValueError(f"{name} must be [B,HV,T] = {(B, HV, T)}, got {tuple(t.shape)}")
    if len({t.device for _, t in named}) != 1:
        raise ValueError("all tensors must be on the same device")


def _validate_state(name, t, q, v):
    if t is None and name == "initial_state":
        return
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.dtype.is_floating_point:
        raise TypeError(f"{name} must be of a floating type, got {t.dtype}")
    want = (q.shape[0], v.shape[1], q.shape[3], v.shape[3])
    if tuple(t.shape) != want:
        raise ValueError(f"{name} must be [B,HV,K,V] = {want}, got {tuple(t.shape)}")
    if t.device != q.device:
        raise ValueError("all tensors must be on the same device")
