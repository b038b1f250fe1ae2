"""Refusals of grouped routing, 4-bit experts and the 8-bit RMSNorm: on the host, before any launch."""

import pytest
import torch

from reframework_b200 import _lib
from reframework_b200 import kernels as K
from reframework_b200.moe import FusedMoE

P = 1 << 20  # a 16-byte aligned address that no refused call touches


def _route(L, **kw):
    a = dict(x=P, xdt=0, gate=None, gdt=0, T=4, H=64, E=64, K=6, scoring=0, groups=8, keep=3, gs=0, scale=1.0, rd=-1,
             sg=None, ss=None, w=P, i32=P, ws=None, wsb=0)
    a.update(kw)
    return L.rf_moe_router_grouped_topk(a["x"], a["xdt"], a["gate"], a["gdt"], None, a["T"], a["H"], a["E"], a["K"],
                                        a["scoring"], None, a["groups"], a["keep"], a["gs"], 1, a["scale"], a["rd"], a["sg"],
                                        a["ss"], a["w"], a["i32"], None, None, a["ws"], a["wsb"], None)


@pytest.mark.parametrize("kw, needle", [
    (dict(xdt=5), "dtype"), (dict(rd=9), "round_dtype"), (dict(scoring=2), "scoring"), (dict(gs=2), "group_score"),
    (dict(T=-1), "sizes"), (dict(E=2048, H=2048, groups=1, keep=1), "1024"), (dict(groups=7), "num_groups"),
    (dict(groups=0), "num_groups"), (dict(groups=64), "num_groups"), (dict(keep=0), "topk_groups"), (dict(keep=9), "topk_groups"),
    (dict(groups=32, keep=32, E=32, H=32, gs=1), "two experts"), (dict(K=0), "K <="), (dict(K=17, keep=8), "K <="),
    (dict(K=10, keep=1), "K <="), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(H=32), "logits"), (dict(sg=P), "logits"), (dict(gate=P, H=60), "multiple of 8"), (dict(w=None), "outputs"),
    (dict(x=None), "null"), (dict(gate=P, sg=P), "shared_scale"), (dict(x=P + 4), "aligned"), (dict(gate=P), "workspace"),
])
def test_route_refusals(kw, needle):
    L = _lib.lib()
    assert _route(L, **kw) == 1
    assert needle in L.rf_moe_last_error().decode()


def test_empty_batches_do_nothing():
    L = _lib.lib()
    assert _route(L, T=0, x=None, w=None, i32=None) == 0
    assert L.rf_moe_add_rmsnorm_q8(None, None, 0, 64, 2, None, None, 1e-6, 0, None, None, None, None, None) == 0
    assert L.rf_moe_int4_experts(None, 2, P, P, 128, P, P, 128, None, None, 0, 2, 8, 128, 64, 0, None, None, None, None, None,
                                 0, None) == 0


def _norm(L, **kw):
    a = dict(x=P, r=None, T=4, H=256, dt=2, w=P, b=None, eps=1e-6, g=0, ro=None, n=None, q=2 * P, s=P)
    a.update(kw)
    return L.rf_moe_add_rmsnorm_q8(a["x"], a["r"], a["T"], a["H"], a["dt"], a["w"], a["b"], a["eps"], a["g"], a["ro"], a["n"],
                                   a["q"], a["s"], None)


@pytest.mark.parametrize("kw, needle, status", [
    (dict(dt=3), "dtype", 1), (dict(T=-1), "sizes", 1), (dict(H=0), "sizes", 1), (dict(H=252), "16 bytes", 1),
    (dict(eps=-1.0), "eps", 1), (dict(eps=float("nan")), "eps", 1), (dict(g=16), "group_size", 1), (dict(H=160, g=128), "group_size", 1),
    (dict(H=65536), "65536", 2), (dict(H=32768, dt=0), "65536", 2), (dict(x=None), "null", 1), (dict(w=None), "null", 1),
    (dict(q=None, s=None), "null", 1), (dict(s=None), "null", 1), (dict(q=None), "null", 1), (dict(r=P), "null", 1),
    (dict(x=P + 8), "aligned", 1), (dict(q=2 * P + 8), "aligned", 1), (dict(n=2 * P), "alias", 1),
    (dict(r=P, ro=3 * P, n=3 * P), "alias", 1), (dict(r=P, ro=2 * P), "alias", 1),
])
def test_norm_refusals(kw, needle, status):
    L = _lib.lib()
    assert _norm(L, **kw) == status
    assert needle in L.rf_moe_last_error().decode()


def _experts(L, **kw):
    a = dict(x=P, dt=2, w1=P, s1=P, g1=128, w2=P, s2=P, g2=128, w=P, ids=P, T=4, K=2, E=8, H=128, I=64, act=0, sy=None, ss=None,
             r=None, out=P, ws=P, wsb=1 << 30)
    a.update(kw)
    return L.rf_moe_int4_experts(*[a[k] for k in ("x", "dt", "w1", "s1", "g1", "w2", "s2", "g2", "w", "ids", "T", "K", "E", "H",
                                                  "I", "act", "sy", "ss", "r", "out", "ws", "wsb")], None)


@pytest.mark.parametrize("kw, needle", [
    (dict(dt=0), "bf16 and fp16"), (dict(dt=7), "bf16 and fp16"), (dict(act=3), "activation"), (dict(T=-1), "sizes"),
    (dict(K=17), "sizes"), (dict(K=0), "sizes"), (dict(E=0), "sizes"), (dict(E=1025), "sizes"), (dict(H=100), "sizes"),
    (dict(I=60), "sizes"), (dict(T=1 << 31), "sizes"), (dict(g1=16), "group"), (dict(g2=256), "group"), (dict(w1=None), "weights"),
    (dict(s2=None), "weights"), (dict(x=None), "null"), (dict(ids=None), "null"), (dict(out=None), "null"),
    (dict(x=P + 8), "aligned"), (dict(r=P + 2), "aligned"), (dict(ws=None), "workspace"), (dict(wsb=100), "workspace"),
    (dict(ws=P + 16), "workspace"),
])
def test_experts_refusals(kw, needle):
    L = _lib.lib()
    assert _experts(L, **kw) == 1
    assert needle in L.rf_moe_last_error().decode()


def test_int4_sizes_and_pack_refusals():
    L = _lib.lib()
    # 2 slots, 24 rows in each half -> 2 row blocks each, K 72 -> 2 k blocks: 2 * 4 * 2 * 512 bytes
    assert L.rf_moe_int4_data_size(2, 48, 72, 64, 1) == 2 * 4 * 2 * 512
    assert L.rf_moe_int4_scales_count(2, 48, 72, 64, 1) == 2 * 4 * 2 * 16
    for bad in ((0, 16, 64, 64, 0), (1, 12, 64, 64, 0), (1, 16, 60, 64, 0), (1, 16, 64, 16, 0), (1, 24, 64, 64, 1)):
        assert L.rf_moe_int4_data_size(*bad) == -1 and L.rf_moe_int4_scales_count(*bad) == -1
    assert L.rf_moe_int4_pack(P, P, 0, 1, 16, 64, 64, 0, P, P, None) == 1  # fp32 scales
    assert L.rf_moe_int4_pack(P, P, 2, 1, 16, 64, 48, 0, P, P, None) == 1
    assert L.rf_moe_int4_quantize(P, 5, 2, 1, 16, 64, 64, 0, P, P, None) == 1
    assert L.rf_moe_int4_dequantize(P, None, 2, 1, 16, 64, 64, 0, P, None) == 1


def test_wrappers_want_cuda_tensors():
    x = torch.zeros(4, 64)
    with pytest.raises(_lib.RfMoeError, match="CUDA"):
        K.router_grouped_topk(x, None, 2)
    with pytest.raises(_lib.RfMoeError, match="CUDA"):
        K.add_rmsnorm_q8(x, torch.ones(64))
    with pytest.raises(_lib.RfMoeError, match="CUDA"):
        K.int4_quantize(torch.zeros(1, 16, 64))


@pytest.mark.parametrize("kw, needle", [
    (dict(scoring="relu"), "scoring"), (dict(group_score="mean"), "group score"), (dict(num_groups=3), "num_groups"),
    (dict(num_groups=4, topk_groups=5), "topk_groups"), (dict(num_groups=8, topk_groups=1), "do not fit"),
    (dict(num_groups=8, topk_groups=8, group_score="top2"), "two experts"), (dict(scale=float("inf")), "scale"),
    (dict(select_bias=torch.zeros(7)), "select_bias"),
])
def test_layer_routing_refusals(kw, needle):
    moe = FusedMoE(8, 2, 64, 32, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match=needle):
        moe.set_routing(**kw)
    assert moe.routing is None and moe.select_bias is None


def test_layer_routing_state():
    moe = FusedMoE(8, 2, 64, 32, dtype=torch.bfloat16)
    assert "gate.e_score_correction_bias" not in moe.state_dict()
    b = torch.arange(8).double()
    moe.set_routing(scoring="sigmoid", select_bias=b, num_groups=4, topk_groups=2, group_score="top2", scale=2.5)
    assert torch.equal(moe.state_dict()["gate.e_score_correction_bias"], b.float())
    moe.load_state_dict({"m.gate.e_score_correction_bias": b.flip(0)}, prefix="m")
    assert torch.equal(moe.select_bias, b.flip(0).float())
    with pytest.raises(_lib.RfMoeError, match="CUDA"):
        moe.quantize_experts()
