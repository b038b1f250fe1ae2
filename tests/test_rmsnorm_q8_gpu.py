"""Residual + RMSNorm with an e4m3 output (kernels.add_rmsnorm_q8) against its definition in 64 bits."""

import math

import pytest
import torch

import operator_refs as R
from reframework_b200 import _lib
from reframework_b200 import kernels as K

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


@pytest.fixture(autouse=True)
def _device_clean(cuda_ok):
    yield
    assert _lib.device_status() == 0


def _inputs(T, H, dtype, seed, residual, bias):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, generator=g)
    x[:, ::37] *= 20
    r = (torch.randn(T, H, generator=g) * 2).to(dtype).to(DEV) if residual else None
    w = (1 + 0.2 * torch.randn(H, generator=g)).to(DEV)
    b = (0.1 * torch.randn(H, generator=g)).to(DEV) if bias else None
    return x.to(dtype).to(DEV), w, r, b


def _check(x, w, residual, bias, group, normed=True, eps=1e-6):
    T, H = x.shape
    out = K.add_rmsnorm_q8(x, w, residual=residual, bias=bias, eps=eps, group_size=group, want_normed=normed)
    r, z = R.norm(x, w, residual=residual, bias=bias, eps=eps)
    assert torch.equal(out.residual, r)
    # z: the sum of H squares (at most 16 * 8 + 5 + 32 fp32 additions in a row: half their relative error after the
    # root), mean, root, division, two products, and the bias' addition
    fp32 = (165 / 2 + 8) * 2.0 ** -24
    zerr = fp32 * (z.abs() + (0 if bias is None else 2 * bias.double().abs()))
    g = group or H
    zg, eg = z.view(T, -1, g), zerr.view(T, -1, g)
    top = zg.abs().amax(-1)
    want = torch.where(top > 0, top / 448, 1.0)
    slack = eg.amax(-1) / 448 + 2.0 ** -22 * want
    assert out.scales.shape == (T, H // g) and out.q.dtype == torch.float8_e4m3fn
    assert bool(((out.scales.double() - want).abs() <= slack).all())
    # e4m3: half a step is 2^-4 of the value, or 2^-10 below the normal range; 2^-22: the quotient's own rounding
    sc = out.scales.double()[..., None]
    got = out.q.double().view(T, -1, g) * sc
    err = (got - zg).abs()
    assert bool((err <= (zg.abs() * 2.0 ** -4).clamp_min(sc.abs() * 2.0 ** -10) + 2.0 ** -22 * zg.abs() + 2 * eg).all())
    if normed:
        u = torch.finfo(x.dtype).eps / 2
        tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0
        assert bool(((out.normed.double() - z).abs() <= (u * (1 + 2.0 ** -10)) * z.abs() + zerr + tiny).all())
    return out


@pytest.mark.parametrize("T,H", [(1, 8), (3, 64), (5, 104), (2, 256), (33, 512), (7, 1000), (64, 1024), (9, 2048), (3, 4096),
                                 (2, 6144), (1, 11008), (3, 16384), (1, 32768), (700, 384)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rows(T, H, dtype):
    if H * dtype.itemsize > 65536:
        pytest.skip("past the longest row")
    for residual, bias in ((False, False), (True, False), (True, True)):
        _check(*_inputs(T, H, dtype, T + H, residual, bias), 0)


@pytest.mark.parametrize("H", [128, 384, 2048, 7168])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_groups(H, group, dtype):
    _check(*_inputs(21, H, dtype, H + group, True, False), group)
    _check(*_inputs(4, H, dtype, H - group, False, True), group, normed=False)


def test_many_rows_take_every_block_twice():
    _check(*_inputs(5000, 256, torch.bfloat16, 1, True, False), 0)
    _check(*_inputs(2500, 1024, torch.bfloat16, 2, True, False), 128)


def test_zero_rows_and_values_that_are_not_finite():
    x, w, _, _ = _inputs(6, 512, torch.bfloat16, 3, False, False)
    x[0] = 0
    x[1, 5] = math.nan
    x[2, 100] = math.inf
    x[3, 200] = -math.inf
    for group in (0, 128):
        out = K.add_rmsnorm_q8(x, w, group_size=group)
        g = group or 512
        assert bool((out.scales[0] == 1).all()) and bool((out.q[0].float() == 0).all())
        back = out.q.float().view(6, -1, g) * out.scales[..., None]
        assert bool(torch.isnan(back[1]).all())  # a NaN reaches every mean
        for t, col in ((2, 100), (3, 200)):      # an infinity makes its own group NaN, the others zero
            bad = torch.zeros(512 // g, dtype=torch.bool, device=DEV)
            bad[col // g] = True
            assert torch.equal(torch.isnan(back[t]).all(-1), bad) and bool((back[t][~bad] == 0).all())
        assert not bool(torch.isnan(out.q.float()).any())
        assert bool(torch.isfinite(back[4:]).all())


def test_tiny_and_huge_values():
    x, w, _, _ = _inputs(4, 512, torch.float32, 4, False, False)
    _check(x * 1e-18, w, None, None, 128)
    _check(x * 1e15, w, None, None, 128)
    out = K.add_rmsnorm_q8(x, w * 1e-38)  # scales at the end of the normal range
    assert bool(torch.isfinite(out.q.float()).all()) and bool((out.scales > 0).all())


def test_strided_unaligned_empty_and_norm_only():
    x, w, r, _ = _inputs(40, 640, torch.bfloat16, 5, True, False)
    _check(x[::2, :512], w[:512], r[::2, :512], None, 64)
    flat = torch.randn(3 + 4 * 256, device=DEV).bfloat16()
    _check(flat[3:].view(4, 256), w[:256], None, None, 0)
    out = K.add_rmsnorm_q8(x[:0], w, residual=r[:0])
    assert out.q.shape == (0, 640) and out.scales.shape == (0, 1)
    only = K.add_rmsnorm_q8(x, w, residual=r, want_q=False, want_normed=True)
    full = K.add_rmsnorm_q8(x, w, residual=r, want_normed=True)
    assert only.q is None and torch.equal(only.normed, full.normed) and torch.equal(only.residual, full.residual)


def test_inputs_stay_and_graph_replays():
    x, w, r, _ = _inputs(32, 1024, torch.bfloat16, 6, True, False)
    x0, r0 = x.clone(), r.clone()
    want = K.add_rmsnorm_q8(x, w, residual=r, group_size=128)
    assert torch.equal(x, x0) and torch.equal(r, r0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = K.add_rmsnorm_q8(x, w, residual=r, group_size=128)
    graph.replay()
    assert torch.equal(got.q.view(torch.uint8), want.q.view(torch.uint8)) and torch.equal(got.scales, want.scales)


@pytest.mark.parametrize("T,H", [(3, 64), (5, 512), (64, 4096), (700, 1024), (400, 6144)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("over", ["x", "residual"])
def test_the_sum_in_place_of_an_input(T, H, dtype, over):
    """The library call with residual_out = x or = residual: the same bits as with an output of its own."""
    x, w, r, _ = _inputs(T, H, dtype, T, True, False)
    want = K.add_rmsnorm_q8(x, w, residual=r, group_size=32, want_normed=True)
    q, scales, normed = torch.empty_like(want.q), torch.empty_like(want.scales), torch.empty_like(x)
    out = {"x": x, "residual": r}[over]
    rc = _lib.lib().rf_moe_add_rmsnorm_q8(x.data_ptr(), r.data_ptr(), T, H, _lib.dtype_code(dtype), w.data_ptr(), None, 1e-6, 32,
                                          out.data_ptr(), normed.data_ptr(), q.data_ptr(), scales.data_ptr(),
                                          _lib.stream_of(x.device))
    assert rc == 0
    assert torch.equal(out, want.residual) and torch.equal(normed, want.normed)
    assert torch.equal(q.view(torch.uint8), want.q.view(torch.uint8)) and torch.equal(scales, want.scales)
