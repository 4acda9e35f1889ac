"""MI355X-native RWKV-6 time-mix hot path (drop-in for RWKV-Megatron's fla call).

The package directory name carries a dash, so load it with
``importlib.import_module("rwkv-megatron_amd")``.

Exports
  chunk_rwkv6, fused_recurrent_rwkv6   fla-compatible WKV6 ops (wkv.py, HIP kernels)
  wkv6_seqfirst                        WKV6 on the time-mix module's [T,B,H*64] layout
  gated_delta                          the gated delta rule over sequences and over tokens
  timemix                              fused token-shift/ddlerp and GroupNorm*gate ops
  channelmix                           fused channel-mix shift/lerp, relu^2, sigmoid gate
  residual                             residual add, gate and scale fused with the next LayerNorm
  loss                                 cross entropy over the vocabulary
  optim                                AdamW over many tensors, states in 32 or 8 bits
  modules                              RWKV6TimeMix / RWKV6ChannelMix / ... mirrors of
                                       rwkv_megatron/rwkv6_layer_specs.py
"""
from .wkv import chunk_rwkv6, fused_recurrent_rwkv6, wkv6_seqfirst  # noqa: F401
from . import _lib, channelmix, gated_delta, loss, optim, residual, timemix, modules  # noqa: F401

__all__ = ["chunk_rwkv6", "fused_recurrent_rwkv6", "wkv6_seqfirst", "gated_delta", "timemix", "channelmix", "residual", "loss", "optim",
           "modules"]
