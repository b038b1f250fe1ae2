"""Grouped routing where a lane's experts are not a power of two (3, 5, 6, 7, 12, 14, 24 of them): the places past them
hold no expert, so they take no part in a group's score, whatever the bias.  Against the definition in 64 bits."""

import math

import pytest
import torch

import operator_refs as R
from reframework_b200 import _lib
from reframework_b200 import kernels as K

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
# weights: as derived in test_router_grouped_gpu.py
W_TOL = 160 * 2.0 ** -24
# E, groups: experts a lane 3, 5, 5, 3, 3, 3, 6, 12, 7, 14, 24
LAYOUTS = [(60, 4), (160, 8), (40, 8), (72, 8), (96, 8), (96, 32), (192, 8), (384, 8), (56, 8), (448, 32), (768, 8)]


@pytest.fixture(autouse=True)
def _device_clean(cuda_ok):
    yield
    assert _lib.device_status() == 0


def _check(logits, top_k, **kw):
    w, ids, _, _, _ = K.router_grouped_topk(logits, None, top_k, **kw)
    rw, rids = R.route(logits, top_k, **kw)
    assert torch.equal(ids.long(), rids), f"{int((ids.long() != rids).any(1).sum())} of {len(ids)} tokens"
    torch.testing.assert_close(w.double(), rw, rtol=W_TOL, atol=1e-37, equal_nan=True)
    return ids


def _logits(T, E, seed, dtype=torch.float32):
    return (torch.randn(T, E, generator=torch.Generator().manual_seed(seed)) * 1.5).to(dtype).to(DEV)


@pytest.mark.parametrize("E,groups", LAYOUTS)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("mean,spread", [(0.0, 0.05), (-0.05, 0.05), (-0.8, 0.1), (0.5, 0.1)])
def test_biased_groups(E, groups, scoring, group_score, mean, spread):
    b = (mean + spread * torch.randn(E, generator=torch.Generator().manual_seed(E + groups))).to(DEV)
    for dtype in (torch.float32, torch.bfloat16):
        for keep in (1, groups // 2):
            _check(_logits(257, E, E, dtype), min(6, keep * (E // groups)), scoring=scoring, select_bias=b, num_groups=groups,
                   topk_groups=keep, group_score=group_score)


@pytest.mark.parametrize("E,groups", LAYOUTS)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_groups_with_one_open_expert(E, groups, scoring):
    """Every second group has one open expert: its two largest sum to -inf, behind every group with two."""
    per = E // groups
    b = (-0.3 + 0.05 * torch.randn(E, generator=torch.Generator().manual_seed(E))).view(groups, per)
    b[::2, 1:] = -math.inf
    for row in (b, b.flip(1)):
        ids = _check(_logits(100, E, groups), min(6, per), scoring=scoring, select_bias=row.reshape(-1).to(DEV),
                     num_groups=groups, topk_groups=groups // 2, group_score="top2")
        assert bool((ids // per % 2 == 1).all())


def test_the_better_pair_wins():
    """Zero logits in 8 groups of 12: scores of 0.5, group 0 with 0.2 and -0.3, group 1 with 0.09 and 0.08."""
    b = torch.full((96,), -0.8)
    b[0], b[12], b[13] = -0.30, -0.41, -0.42
    ids = _check(torch.zeros(5, 96, device=DEV), 2, scoring="sigmoid", select_bias=b.to(DEV), num_groups=8, topk_groups=1,
                 group_score="top2")
    assert ids.tolist() == [[12, 13]] * 5


@pytest.mark.parametrize("E,groups", LAYOUTS)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("group_score", ["max", "top2"])
def test_infinite_and_nan_logits(E, groups, bias, group_score):
    l = _logits(8, E, 5)
    l[0] = math.nan
    l[1] = -math.inf
    l[2, ::2] = -math.inf
    l[3, : E - 3] = torch.finfo(torch.float32).min
    l[4, 7] = math.nan
    l[5, 1:] = -math.inf
    b = torch.linspace(-0.9, -0.7, E, device=DEV) if bias else None
    for scoring in ("softmax", "sigmoid"):
        ids = _check(l, 3, scoring=scoring, select_bias=b, num_groups=groups, topk_groups=2, group_score=group_score)
        assert all(len(set(r)) == 3 for r in ids.tolist())
