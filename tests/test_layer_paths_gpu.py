"""What a program may do around the layers' fused path: replace a class's forward, change a norm's parameters
between forward and backward, and count on the memory that the separate operators held."""
import importlib

import pytest
import torch

from test_train_step_gpu import _batch, _grads, _model

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16


@pytest.fixture(scope="module")
def pkg():
    return importlib.import_module("rwkv-megatron_amd")


# A forward that a program puts in the class's place is the one that runs, in every module of the class.
@pytest.mark.parametrize("name,calls", [("RWKV6Layer", 3), ("RWKV6ChannelMix", 3), ("LayerNorm", 8)])
def test_a_forward_replaced_on_the_class_runs(pkg, monkeypatch, name, calls):
    M = pkg.modules
    model, (tokens, _) = _model(pkg), _batch()
    want = model(tokens).detach()
    cls, seen = getattr(M, name), []
    own = cls.forward

    def forward(self, *args):
        seen.append(self)
        return own(self, *args)

    monkeypatch.setattr(cls, "forward", forward)
    assert torch.equal(model(tokens), want) and len(seen) == calls


def test_a_call_replaced_on_the_class_runs(pkg, monkeypatch):
    M = pkg.modules
    model, (tokens, _) = _model(pkg), _batch()
    want = model(tokens).detach()
    seen = []

    def call(self, *args):
        seen.append(type(self))
        return torch.nn.Module._call_impl(self, *args)

    monkeypatch.setattr(M.RWKV6Layer, "__call__", call, raising=False)
    assert torch.equal(model(tokens), want) and len(seen) == 3
    monkeypatch.undo()
    monkeypatch.setattr(torch.nn.Module, "__call__", call)
    seen.clear()
    assert torch.equal(model(tokens), want) and seen.count(M.RWKV6Layer) == 3 and seen.count(M.LayerNorm) == 8
