"""The selection bias of set_routing() in the layers: kept in fp32, saved and loaded, checked."""

import pytest
import torch

from reframework_b200.moe import FusedMoE
from reframework_b200.parallel.ep import EPFusedMoE, _LayerCfg

E, TOPK, H, I = 8, 2, 64, 32


def _fused():
    moe = FusedMoE(E, TOPK, H, I, dtype=torch.float32)
    with torch.no_grad():
        for p in moe.parameters():
            p.normal_(0, 0.02)
    return moe


def _sharded():
    return EPFusedMoE.from_full(_fused(), 1, 0)


def _bias():
    return torch.tensor([0.0123456789, -0.1, 1e-7, 0.3, -0.05, 70000.0, float("-inf"), 0.7])


@pytest.mark.parametrize("cast", [lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.double(),
                                  lambda m: m.to("cpu", torch.float16), lambda m: torch.nn.Sequential(m).bfloat16()[0]])
def test_a_layer_cast_to_another_type_keeps_its_selection_bias(cast):
    moe = _fused()
    moe.set_routing(scoring="sigmoid", select_bias=_bias())
    ep = EPFusedMoE.from_full(moe, 1, 0)
    for layer in (moe, ep):
        layer = cast(layer)
        assert layer.gate.dtype != torch.float32
        assert layer.select_bias.dtype == torch.float32 and torch.equal(layer.select_bias, _bias())
    assert "select_bias" in dict(moe.named_buffers())
    assert moe.to("meta").select_bias.is_meta
