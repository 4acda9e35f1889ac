"""A block's output into the residual stream, fused with the LayerNorm that the next block reads.

The reference's layer adds a block's output (and a skipped bias) to the stream and normalises the
sum for the next block (/root/reference/rwkv_megatron/rwkv6_layer_specs.py:543-548); the channel
mix's output is gated by a sigmoid before that (:533-536):

    f = (branch + branch_bias) * sigmoid(gate)
    s = x + scale * f
    y = LayerNorm(s) * weight + bias

``residual_norm`` is one kernel forward and two backward (the gradients of everything, and the sums
over the rows for the parameters') where torch runs an add, a product and a LayerNorm of which each
reads and writes the stream.  modules.RWKV6Layer and RWKV6Model call it.  The autograd function is
csrc/autograd.cpp's; it raises if the HIP library is missing, there is no fallback.
"""
from __future__ import annotations

import torch

from . import _lib

MAX_CHANNELS = 8192


def residual_norm(x, branch, weight, bias, eps, gate=None, branch_bias=None, scale=1.0, stepwise=False):
    """(s, y) = (x + scale (branch + branch_bias) sigmoid(gate), LayerNorm(s) weight + bias).

    x [..., C] bf16 or fp32 (s comes back in the same type); branch and gate [..., C] bf16;
    weight, bias, branch_bias [C] in any of fp32, bf16, fp16; y [..., C] bf16.  Without a gate the
    factor is 1, without a branch_bias the term 0; scale is a number.  C is a multiple of 8 up to
    8192.  s is rounded once, y is the norm of s before that rounding; inside, 32 bits.  With
    stepwise=True the numbers are those of separate operators: the sum with the bias, the product with
    the gate (bf16) and s (x's type) are rounded before they are used, y is the norm of s as returned,
    and the gradients are rounded at the same places.

    Gradients for x, branch, gate, weight, bias and branch_bias; sums over the rows run in a fixed
    order.  A backward that is differentiated again runs through torch's operators."""
    out = _lib.native().residual_norm(x, branch, weight, bias, eps, gate, branch_bias, scale, stepwise, False)
    return _refuse(x, branch, weight, bias, gate, branch_bias) if out is None else out


def _refuse(x, branch, weight, bias, gate, branch_bias):
    """Raises for a call that the kernels do not take, and says why."""
    for name, t in (("x", x), ("branch", branch), ("gate", gate)):
        if t is None:
            continue
        if t.device.type != "cuda":
            raise ValueError(f"{name} must live on the GPU")
        if t.shape != x.shape:
            raise ValueError(f"{name} must have x's shape {tuple(x.shape)}, got {tuple(t.shape)}")
        if t.dtype != torch.bfloat16 and not (t is x and t.dtype == torch.float32):
            raise TypeError(f"{name} must be bfloat16{' or float32' if t is x else ''}, got {t.dtype}")
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"x must be [..., C], got shape {tuple(x.shape)}")
    C = x.shape[-1]
    if C % 8 or C > MAX_CHANNELS:
        raise NotImplementedError(f"C must be a multiple of 8 up to {MAX_CHANNELS}, got {C}")
    for name, t in (("weight", weight), ("bias", bias), ("branch_bias", branch_bias)):
        if t is None:
            continue
        if t.dtype not in (torch.bfloat16, torch.float32, torch.float16):
            raise TypeError(f"{name} must be a bfloat16, float32 or float16 tensor")
        if tuple(t.shape) != (C,):
            raise ValueError(f"{name} must be [C] = {(C,)}, got {tuple(t.shape)}")
    if len({t.device for t in (x, branch, gate, weight, bias, branch_bias) if t is not None}) != 1:
        raise ValueError("all tensors must be on the same device")
    raise NotImplementedError("residual_norm takes dense (strided) tensors of at most 2^40 elements")
