"""Grouped routing (kernels.router_grouped_topk) against its definition in 64 bits: the ids exactly (the order is
that of the exact scores), the weights to fp32."""

import math

import pytest
import torch

import operator_refs as R
from reframework_b200 import _lib
from reframework_b200 import kernels as K
from reframework_b200.moe import grouped_topk

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
# a score: an accurate exponential (2 ulp) over a sum of fast ones (each within 2 + 1.173 |l - max| ulp, 16 for
# |l - max| <= 12), the arguments' rounding (12 half ulps each), up to 37 additions, a division:
# 4 + 32 + 24 + 37 + 1 = 98 roundings; renormalised, the sum cancels: 2 * (4 + 12 + 1) and 16 + 3 more
W_TOL = 160 * 2.0 ** -24


@pytest.fixture(autouse=True)
def _device_clean(cuda_ok):
    yield
    assert _lib.device_status() == 0


def _logits(T, E, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, E, generator=g) * 1.5).to(dtype).to(DEV)


def _check(logits, top_k, **kw):
    w, ids, ids64, _, _ = K.router_grouped_topk(logits, None, top_k, ids64=True, **kw)
    rw, rids = R.route(logits, top_k, **kw)
    assert torch.equal(ids.long(), rids) and torch.equal(ids64, rids)
    torch.testing.assert_close(w.double(), rw, rtol=W_TOL, atol=1e-37, equal_nan=True)
    return w, ids


SHAPES = [  # T, E, K, groups, kept
    (1, 64, 6, 8, 3), (61, 60, 4, 1, 1), (333, 256, 8, 8, 4), (17, 8, 2, 1, 1), (5, 1, 1, 1, 1), (7, 4, 4, 2, 2),
    (129, 160, 6, 8, 3), (40, 60, 5, 4, 2), (33, 1024, 16, 32, 7), (65, 148, 8, 4, 2), (64, 64, 16, 32, 8),
    (2, 1000, 3, 1, 1), (1000, 20, 7, 4, 3),
]


@pytest.mark.parametrize("T,E,top_k,groups,keep", SHAPES)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("bias", [False, True])
def test_against_definition(T, E, top_k, groups, keep, scoring, group_score, bias):
    if group_score == "top2" and (groups == 1 or E // groups < 2):
        pytest.skip("no groups of two")
    g = torch.Generator().manual_seed(T + E)
    b = (torch.randn(E, generator=g) * 0.05).to(DEV) if bias else None
    for dtype, renorm, scale in ((torch.float32, True, 2.5), (torch.bfloat16, False, 1.0), (torch.float16, True, 1.0)):
        _check(_logits(T, E, dtype, E * top_k), top_k, scoring=scoring, select_bias=b, num_groups=groups,
               topk_groups=keep, group_score=group_score, renormalize=renorm, scale=scale)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("group_score", ["max", "top2"])
def test_scores_closer_than_fp32(scoring, group_score):
    """Neighbouring fp32 logits, and a bias that cancels their differences to within rounding."""
    T, E = 512, 64
    g = torch.Generator().manual_seed(3)
    l = torch.full((T, E), 0.75)
    l = (l.view(torch.int32) + torch.randint(-3, 4, (T, E), generator=g, dtype=torch.int32)).view(torch.float32).to(DEV)
    s = torch.softmax(l.double(), 1) if scoring == "softmax" else torch.sigmoid(l.double())
    b = (0.7 - s[0]).float()
    for bias in (None, b):
        _check(l, 8, scoring=scoring, select_bias=bias, num_groups=8, topk_groups=4, group_score=group_score)


@pytest.mark.parametrize("groups,keep", [(1, 1), (8, 3), (4, 2)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_ties_go_to_the_lower_id(groups, keep, scoring):
    l = torch.zeros(3, 148 if groups == 4 else 64, device=DEV)
    l[1, 10:20] = 1.0
    for b in (None, torch.zeros(l.shape[1], device=DEV)):
        for gs in ("max", "top2"):
            _check(l, 9, scoring=scoring, select_bias=b, num_groups=groups, topk_groups=keep, group_score=gs)


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("E,groups", [(64, 8), (148, 4)])
def test_infinite_and_nan_logits(bias, group_score, E, groups):
    """Rows of NaN, of -inf, with a few of them, with masks of the lowest value: ids stay valid and distinct."""
    l = _logits(9, E, torch.float32, 5)
    l[0] = math.nan
    l[1] = -math.inf
    l[2, ::2] = -math.inf
    l[3, :E - 3] = torch.finfo(torch.float32).min
    l[4, 7] = math.nan
    l[5, 1:] = -math.inf
    l[6, 9:12] = -math.inf
    b = torch.linspace(-0.1, 0.1, E, device=DEV) if bias else None
    for scoring in ("softmax", "sigmoid"):
        _, ids = _check(l, 8, scoring=scoring, select_bias=b, num_groups=groups, topk_groups=2, group_score=group_score)
        assert all(len(set(r)) == 8 for r in ids.tolist())


def test_closed_experts():
    """A bias of -inf closes an expert; when fewer than K stay open the lowest closed ids fill up."""
    l = _logits(50, 32, torch.float32, 8)
    b = torch.full((32,), -math.inf, device=DEV)
    b[[3, 30]] = 0.0
    _, ids = _check(l, 4, scoring="sigmoid", select_bias=b)
    assert bool((torch.sort(ids[:, :2], 1).values == torch.tensor([3, 30], device=DEV, dtype=torch.int32)).all())
    _check(l, 4, scoring="softmax", select_bias=b, num_groups=4, topk_groups=2, group_score="top2")
    _check(l, 4, scoring="softmax", select_bias=torch.full((32,), -math.inf, device=DEV), num_groups=4, topk_groups=2)


def test_strided_unaligned_and_empty_logits():
    wide = _logits(20, 130, torch.float32, 9)
    _check(wide[:, 1:61], 4, scoring="softmax")
    _check(wide.t()[:64], 4, scoring="softmax")
    flat = torch.randn(1 + 4 * 60, device=DEV)
    _check(flat[1:].view(4, 60), 4, scoring="sigmoid")  # a base that is not 16-byte aligned
    w, ids, _, _, _ = K.router_grouped_topk(wide[:0], None, 3)
    assert w.shape == (0, 3) and ids.shape == (0, 3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shared", [False, True])
def test_with_gate_equals_logits_form(dtype, shared):
    """From x and the gate: the same choice and weights as from the logits that the call itself returns."""
    g = torch.Generator().manual_seed(4)
    T, H, E = 77, 264, 64
    x = torch.randn(T, H, generator=g).to(dtype).to(DEV)
    cat = (torch.randn(E + 1, H, generator=g) * 0.1).to(dtype).to(DEV)
    gate, sg = cat[:E], cat[E] if shared else None
    b = (torch.randn(E, generator=g) * 0.05).to(DEV)
    kw = dict(scoring="sigmoid", select_bias=b, num_groups=8, topk_groups=4, group_score="top2", scale=2.5)
    w, ids, _, lg, ss = K.router_grouped_topk(x, gate, 8, shared_gate=sg, bias=b, want_logits=True, **kw)
    mag = x.double().abs() @ gate.double().abs().T
    ref = x.double() @ gate.double().T + b.double()
    assert bool(((lg.double() - ref).abs() <= H * 2.0 ** -23 * (mag + b.double().abs())).all())
    w2, ids2, _, _, _ = K.router_grouped_topk(lg, None, 8, **kw)
    assert torch.equal(ids, ids2) and torch.equal(w, w2)
    if shared:
        z = x.double() @ sg.double()
        torch.testing.assert_close(ss.double(), torch.sigmoid(z), rtol=1e-4, atol=0)
    rounded = K.router_grouped_topk(x, gate, 8, want_logits=True, round_dtype=torch.bfloat16, **kw)
    assert torch.equal(rounded[3], rounded[3].bfloat16().float())


def test_a_token_does_not_depend_on_the_batch():
    l = _logits(300, 256, torch.float32, 12)
    kw = dict(scoring="sigmoid", num_groups=8, topk_groups=4, group_score="top2",
              select_bias=torch.linspace(-0.1, 0.1, 256, device=DEV))
    w, ids, _, _, _ = K.router_grouped_topk(l, None, 8, **kw)
    w1, ids1, _, _, _ = K.router_grouped_topk(l[123:124], None, 8, **kw)
    assert torch.equal(ids[123:124], ids1) and torch.equal(w[123:124], w1)


def test_plain_softmax_routing_agrees_with_router_topk_and_grouped_topk():
    l = _logits(200, 60, torch.float32, 13)
    w, ids, _, _, _ = K.router_topk(l, None, 4)
    gw, gids, _, _, _ = K.router_grouped_topk(l, None, 4)
    assert torch.equal(ids, gids)
    torch.testing.assert_close(w, gw, rtol=W_TOL, atol=0)
    fw, fids = grouped_topk(l, 4, True, num_groups=4, topk_groups=2, scoring="sigmoid", scale=1.5)
    rw, rids = R.route(l, 4, scoring="sigmoid", num_groups=4, topk_groups=2, scale=1.5)
    assert torch.equal(fids, rids)
    torch.testing.assert_close(fw.double(), rw, rtol=W_TOL, atol=0)


def test_on_a_side_stream_and_in_a_graph():
    l = _logits(64, 64, torch.float32, 14)
    want = K.router_grouped_topk(l, None, 6, scoring="sigmoid")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = K.router_grouped_topk(l, None, 6, scoring="sigmoid")
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = K.router_grouped_topk(l, None, 6, scoring="sigmoid")
    l.copy_(_logits(64, 64, torch.float32, 15))
    graph.replay()
    want = K.router_grouped_topk(l, None, 6, scoring="sigmoid")
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


@pytest.mark.parametrize("T,E,top_k", [(300, 8, 2), (300, 64, 6), (500, 256, 8), (200, 1000, 16), (100, 1024, 16)])
@pytest.mark.parametrize("spread", [0.01, 1.5, 8.0])
@pytest.mark.parametrize("renormalize", [False, True])
def test_how_near_softmax_weights_come(T, E, top_k, spread, renormalize):
    """With d = max - l: a score e^-d / sum has an expf of at most 2 ulp (4 * 2^-24) whose argument is rounded (d * 2^-24)
    and a division; the sum is off by 2 + 1.673 * mean(d) ulp, mean(d) <= ln E over a softmax, and by its NV + 5
    additions, NV <= 32 the power of two from E / 32 on.  Renormalised, the sum cancels, and each of the two sides has
    d + 5, the second also four additions, a division and the scale's product."""
    l = _logits(T, E, torch.float32, E) * (spread / 1.5)
    w, ids, _, _, _ = K.router_grouped_topk(l, None, top_k, renormalize=renormalize)
    rw, rids = R.route(l, top_k, scoring="softmax", renormalize=renormalize)
    assert torch.equal(ids.long(), rids)
    d = (l.amax(1, keepdim=True) - torch.gather(l, 1, rids)).double()
    nv = 1
    while 32 * nv < E:
        nv *= 2
    of_sum = 2 * (2 + 1.673 * math.log(E)) + nv + 5
    steps = 2 * (d.amax(1, keepdim=True) + 5) + 6 if renormalize else of_sum + d + 5 + 1
    assert bool(((w.double() - rw).abs() <= steps * 2.0 ** -24 * rw + 2.0 ** -149).all())
