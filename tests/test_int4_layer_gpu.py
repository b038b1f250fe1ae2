"""Grouped routing, 4-bit experts and the 8-bit norm as a decoder layer uses them: through FusedMoE, eager, captured into
a CUDA graph, with shared experts, residual and the following norm; and their refusals in the layer."""

import types

import pytest
import torch

import operator_refs as R
from reframework_b200 import _lib
from reframework_b200 import kernels as K
from reframework_b200._lib import RfMoeError
from reframework_b200.moe import FusedMoE
from reframework_b200.moe.graph import capture_forward
from reframework_b200.parallel.ep import EPFusedMoE

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
E, TOPK, H, I = 16, 4, 256, 192


@pytest.fixture(autouse=True)
def _device_clean(cuda_ok):
    yield
    assert _lib.device_status() == 0


def _layer(dtype=torch.bfloat16, shared=0, shared_gate=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    moe = FusedMoE(E, TOPK, H, I, dtype=dtype, router_dtype=torch.float32, num_shared_experts=shared,
                   shared_intermediate_size=I if shared else 0, shared_expert_gate=shared_gate)
    with torch.no_grad():
        for p in moe.parameters():
            p.copy_((torch.randn(p.shape, generator=g) * 0.05).to(dtype))
    moe = moe.to(DEV)
    moe.set_routing(scoring="sigmoid", select_bias=torch.randn(E, generator=g) * 0.05, num_groups=4, topk_groups=2,
                    group_score="top2", scale=2.5)
    return moe


def _x(T, seed, dtype=torch.bfloat16):
    return torch.randn(T, H, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def _reference(moe, w1, w2, x, residual=None, shared=False):
    """The layer from its routing on: (out fp64, bound) with the layer's own weights and ids."""
    w, ids = moe.route(x)
    kw = {}
    if shared:
        kw["shared_y"] = K.shared_experts(x, moe.shared_w1.detach(), moe.shared_w2.detach(), "silu")
        if moe.shared_gate is not None:
            kw["shared_scale"] = torch.sigmoid(x.double() @ moe.shared_gate.detach().double()).float()
    ref, bound = R.experts(x, w1.double(), w2.double(), w, ids, "silu", residual=residual, **kw)
    if shared and moe.shared_gate is not None:  # the gate's own fp32 sum and sigmoid, against the 64-bit one above
        mag = x.double().abs() @ moe.shared_gate.detach().double().abs()
        bound = bound + (H * 2.0 ** -23 * mag[:, None] + 2.0 ** -20) * kw["shared_y"].double().abs()
    return ref, bound


@pytest.mark.parametrize("T", [1, 5, 64, 400])
@pytest.mark.parametrize("shared,shared_gate", [(0, False), (1, True), (2, False)])
def test_forward(T, shared, shared_gate):
    moe = _layer(shared=shared, shared_gate=shared_gate, seed=T)
    x, res = _x(T, 1), _x(T, 2)
    moe.quantize_experts(64)
    assert moe.uses_int4 and len(moe.experts_w1) == 0
    w1, w2 = (K.int4_dequantize(q) for q in moe._int4)
    with torch.no_grad():
        out = moe(x, residual=res)
        ref, bound = _reference(moe, w1, w2, x, res, bool(shared))
    assert bool(((out.double() - ref).abs() <= bound).all())


def test_routing_of_the_layer():
    moe = _layer()
    x = _x(100, 3)
    w, ids = moe.route(x)
    lg = K.router_topk(x, moe.gate.detach(), TOPK, want_logits=True)[3]
    rw, rids = R.route(lg, TOPK, scoring="sigmoid", select_bias=moe.select_bias, num_groups=4, topk_groups=2,
                       group_score="top2", scale=2.5)
    assert torch.equal(ids, rids)
    torch.testing.assert_close(w.double(), rw, rtol=160 * 2.0 ** -24, atol=0)


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("T", [1, 33])
def test_decoder_step_with_norms(quantised, T):
    """moe(x) + residual, its norm in 16 bits and in e4m3: the three forms agree on the same residual."""
    moe = _layer(shared=1, seed=9)
    if quantised:
        moe.quantize_experts(32)
    norm = types.SimpleNamespace(weight=1 + 0.1 * torch.randn(H, device=DEV), eps=1e-6, bias=None)
    x, res = _x(T, 4), _x(T, 5)
    with torch.no_grad():
        plain = moe(x, residual=res)
        normed, r = moe.forward_add_residual(x, res, norm)
        q, scales, r8 = moe.forward_add_residual_q8(x, res, norm, group_size=128)
    assert torch.equal(r, plain) and torch.equal(r8, plain)
    _, z = R.norm(plain, norm.weight)
    zerr = 91 * 2.0 ** -24 * z.abs()
    assert bool(((normed.double() - z).abs() <= 2.0 ** -8 * 1.001 * z.abs() + zerr).all())
    sc = scales.double()[..., None]
    err = (q.double().view(T, -1, 128) * sc - z.view(T, -1, 128)).abs().view(T, H)
    most = torch.maximum(z.abs() * 2.0 ** -4, (sc * 2.0 ** -10).expand(T, H // 128, 128).reshape(T, H))
    assert bool((err <= most + 2.0 ** -20 * z.abs() + 2 * zerr).all())


@pytest.mark.parametrize("T", [1, 64, 300])
def test_captured_layers_share_nothing(T):
    """Two captured layers replayed in turn, and on two streams at once, equal their eager forwards."""
    moes = [_layer(seed=s) for s in (11, 12)]
    for m in moes:
        m.quantize_experts(128)
    graphs = [capture_forward(m, _x(T, 6)) for m in moes]
    x = _x(T, 7)
    with torch.no_grad():
        want = [m(x) for m in moes]
    for _ in range(2):
        for g, y in zip(graphs, want):
            assert torch.equal(g(x), y)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in moes]
    outs = []
    for g, s in zip(graphs, streams):
        with torch.cuda.stream(s):
            outs.append(g(x))
    torch.cuda.synchronize()
    assert all(torch.equal(o, y) for o, y in zip(outs, want))


def test_quantised_state_and_refusals():
    moe = _layer(seed=13)
    before = {k: v.clone() for k, v in moe.state_dict().items()}
    moe.quantize_experts(32)
    after = moe.state_dict()
    assert set(after) == set(before) and torch.equal(after["gate.weight"], before["gate.weight"])
    for k in before:
        if ".experts." in k or k.startswith("experts."):
            b, a = before[k].float(), after[k].float()
            top = torch.zeros(b.shape[0], -(-b.shape[1] // 32), 32, device=DEV)
            top.view(b.shape[0], -1)[:, : b.shape[1]] = b.abs()
            half = (top.amax(-1) / 7 * (1 + 1 / 32) / 2).repeat_interleave(32, 1)[:, : b.shape[1]]
            assert bool(((a - b).abs() <= half * (1 + 1e-5)).all())
    again = _layer(seed=14)
    again.load_state_dict(after)
    again.quantize_experts(32)  # codes of dequantised weights: the same codes where scales agree
    with torch.no_grad():
        assert torch.isfinite(again(_x(9, 8))).all()
    with pytest.raises(RfMoeError, match="already"):
        moe.quantize_experts()
    with pytest.raises(RfMoeError, match="4-bit"):
        moe.build_offload_cache(DEV, 2)
    with pytest.raises(RfMoeError, match="before quantize_experts"):
        moe.load_state_dict(before)
    with pytest.raises(RfMoeError, match="4-bit"):
        EPFusedMoE.from_full(moe, 1, 0)
    offloaded = _layer(seed=15)
    offloaded.build_offload_cache(DEV, 4)
    with pytest.raises(RfMoeError, match="offloaded"):
        offloaded.quantize_experts()
    wide = FusedMoE(E, TOPK, H, I, dtype=torch.float32, device=DEV)
    with pytest.raises(RfMoeError, match="bfloat16 and float16"):
        wide.quantize_experts()
    with pytest.raises(RfMoeError, match="groups of 48"):
        _layer().quantize_experts(48)
    entropy = _layer(seed=16)
    entropy.entropy_adaptive_k = True
    with pytest.raises(RfMoeError, match="entropy"):
        entropy(_x(2, 1))


def test_moves_with_the_layer_and_empty_batch():
    moe = _layer(seed=17, shared=1, shared_gate=True)
    moe.quantize_experts(64)
    x = _x(6, 9)
    with torch.no_grad():
        want = moe(x)
        back = moe.cpu().to(DEV)(x)
        assert torch.equal(want, back)
        assert moe(x[:0]).shape == (0, H)
        q, s, r = moe.forward_add_residual_q8(x[:0], x[:0], types.SimpleNamespace(weight=torch.ones(H, device=DEV), eps=1e-6))
    assert q.shape == (0, H) and s.shape == (0, 1) and r.shape == (0, H)


def test_offloaded_layer_routes_in_groups():
    moe = _layer(seed=18)
    x = _x(40, 10)
    with torch.no_grad():
        want = moe(x)
        ids = moe.route(x)[1]
        moe.build_offload_cache(DEV, 4)
        assert torch.equal(moe.route(x)[1], ids)
        got = moe(x)
    torch.testing.assert_close(got.float(), want.float(), rtol=2.0 ** -6, atol=2.0 ** -8 * float(want.abs().max()))


def test_a_captured_layer_routes_with_the_bias_set_or_loaded_later():
    moe = _layer(seed=21)
    graph = capture_forward(moe, _x(20, 1))
    x = _x(20, 2)
    for seed, loads in ((1, False), (2, True)):
        b = torch.randn(E, generator=torch.Generator().manual_seed(seed)) * 0.3
        before = graph(x).clone()
        if loads:
            moe.load_state_dict({"gate.e_score_correction_bias": b})
        else:
            moe.set_routing(scoring="sigmoid", select_bias=b, num_groups=4, topk_groups=2, group_score="top2", scale=2.5)
        with torch.no_grad():
            want = moe(x)
        assert torch.equal(graph(x), want) and not torch.equal(want, before)
