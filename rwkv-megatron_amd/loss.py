"""Cross entropy of the language model's logits and its gradient, on HIP kernels.

The reference's model returns a loss a token when it is given labels (Megatron's GPTModel, which
/root/reference/rwkv_megatron/rwkv6_model.py:28-184 subclasses), and the training driver averages it
over the unmasked tokens (/root/reference/pretrain_rwkv6.py:144-179).

``cross_entropy`` reads the logits in their own type, once in the forward and once in the backward,
and writes their gradient; in torch the same loss starts with a 32-bit copy of the logits (4.3 GB for
16384 tokens of a 65536-way head).  modules.RWKV6Model.forward calls it when it is given labels.  The
autograd function is csrc/autograd.cpp's; it raises if the HIP library is missing, there is no
fallback.
"""
from __future__ import annotations

import torch

from . import _lib


def cross_entropy(logits, targets, ignore_index=-100):
    """losses[...] = log(sum_j exp(logits[..., j])) - logits[..., targets[...]] in fp32.

    logits [..., V] bf16 or fp32, targets [...] of integers.  Rows may lie apart in memory (a slice of a
    padded vocabulary is read where it is).  A target equal to ignore_index has loss 0 and a gradient
    of zeros, whatever its logits; any other outside 0 .. V - 1 gives NaN in both (it is not read).
    Sums in 32 bits, the same bits every time.  The gradient has the logits' type; a backward that is
    differentiated again runs through torch's operators."""
    for name, t in (("logits", logits), ("targets", targets)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if t.device.type != "cuda":
            raise ValueError(f"{name} must live on the GPU")
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"logits must be bfloat16 or float32, got {logits.dtype}")
    if targets.dtype not in (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8):
        raise TypeError(f"targets must be integers, got {targets.dtype}")
    if logits.dim() < 1 or logits.shape[-1] == 0 or logits.shape[:-1] != targets.shape:
        raise ValueError(f"logits [..., V] and targets [...] expected, got {tuple(logits.shape)} and {tuple(targets.shape)}")
    if logits.device != targets.device:
        raise ValueError("logits and targets must be on the same device")
    return _lib.native().cross_entropy(logits, targets, int(ignore_index))
