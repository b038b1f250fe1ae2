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


@pytest.mark.parametrize("make", [_fused, _sharded])
@pytest.mark.parametrize("prefix", ["", "layers.3.mlp"])
def test_the_bias_is_loaded_whatever_the_order(make, prefix, caplog):
    src = make()
    src.set_routing(scoring="sigmoid", select_bias=_bias())
    saved = {k: v.clone() for k, v in src.state_dict(prefix=prefix).items()}
    before, after = make(), make()
    before.set_routing(scoring="sigmoid")
    before.load_state_dict(saved, prefix=prefix)
    assert not caplog.records
    after.load_state_dict(saved, prefix=prefix)
    assert after.routing is None and "set_routing" in caplog.text  # loaded, not in use yet: said so
    after.set_routing(scoring="sigmoid")
    for layer in (before, after):
        assert layer.routing.scoring == "sigmoid" and torch.equal(layer.select_bias, _bias())
        assert layer.select_bias.dtype == torch.float32


@pytest.mark.parametrize("make", [_fused, _sharded])
def test_set_routing_keeps_replaces_and_clears_the_bias(make):
    layer, b = make(), _bias()
    layer.set_routing(select_bias=b)
    at = layer.select_bias.data_ptr()
    b.zero_()  # copied
    layer.set_routing(scoring="sigmoid", num_groups=2, topk_groups=1)
    assert torch.equal(layer.select_bias, _bias()) and layer.routing.num_groups == 2
    layer.set_routing(select_bias=b.double())
    assert torch.equal(layer.select_bias, b) and layer.select_bias.data_ptr() == at
    with pytest.raises(ValueError, match="select_bias"):
        layer.set_routing(select_bias="drop")
    assert layer.routing.scoring == "softmax"
    layer.set_routing(select_bias=None)
    assert layer.select_bias is None


@pytest.mark.parametrize("make", [_fused, _sharded])
@pytest.mark.parametrize("routed", [False, True])
def test_a_bias_of_another_length_is_refused(make, routed):
    layer = make()
    if routed:
        layer.set_routing(scoring="sigmoid", select_bias=_bias())
    with pytest.raises(ValueError, match="e_score_correction_bias must have 8 elements"):
        layer.load_state_dict({"gate.e_score_correction_bias": torch.zeros(E + 1)})
    assert (torch.equal(layer.select_bias, _bias()) if routed else layer.select_bias is None)


def test_a_sharded_layer_has_its_own_bias():
    moe = _fused()
    moe.set_routing(scoring="sigmoid", select_bias=_bias())
    ep = EPFusedMoE.from_full(moe, 1, 0)
    moe.select_bias.zero_()
    assert torch.equal(ep.select_bias, _bias())


def test_a_bias_set_in_inference_mode_can_be_replaced_outside():
    moe = _fused()
    with torch.inference_mode():
        moe.set_routing(scoring="sigmoid", select_bias=_bias())
        moe.set_routing(select_bias=_bias().flip(0))
    moe.load_state_dict({"gate.e_score_correction_bias": _bias()})
    assert torch.equal(moe.select_bias, _bias())
    with torch.inference_mode():
        moe.load_state_dict({"gate.e_score_correction_bias": _bias().flip(0)})
    assert torch.equal(moe.select_bias, _bias().flip(0))
