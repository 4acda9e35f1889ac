"""Layers that were saved as whole objects before they had a dropout: they load and run as they did."""
import copy
import io

import pytest
import torch


def _layer(pkg, device):
    cfg = pkg.modules.TransformerConfig(hidden_size=128, num_attention_heads=2, ffn_hidden_size=256, num_layers=2)
    torch.manual_seed(0)
    return pkg.modules.RWKV6Layer(cfg, device=device)


def _old(layer):
    layer = copy.deepcopy(layer)
    del layer.__dict__["hidden_dropout"]
    f = io.BytesIO()
    torch.save(layer, f)
    f.seek(0)
    return torch.load(f, weights_only=False)


def test_no_dropout(pkg):
    layer = _old(_layer(pkg, "cpu"))
    assert layer.train()._dropout() == 0 and layer.eval()._dropout() == 0


@pytest.mark.gpu
def test_the_same_outputs(pkg):
    layer = _layer(pkg, "cuda")
    x = torch.randn(20, 2, 128, device="cuda").bfloat16()
    for train in (False, True):
        assert torch.equal(_old(layer).train(train)(x), layer.train(train)(x))
