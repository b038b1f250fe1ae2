"""4-bit expert weights: layout, quantiser, and the experts' products against their definition in 64 bits."""

import pytest
import torch

import operator_refs as R
from reframework_b200 import _lib
from reframework_b200 import kernels as K
from reframework_b200.moe import fused_experts_int4

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


@pytest.fixture(autouse=True)
def _device_clean(cuda_ok):
    yield
    _lib.set_gemm_impl(0)
    assert _lib.device_status() == 0


def _codes(S, N, Kd, group, dtype, gen, fine=False):
    """Random codes and scales; fine: scales with all of the dtype's bits, as from a checkpoint."""
    codes = torch.randint(0, 256, (S, N, Kd // 2), generator=gen, dtype=torch.uint8)
    ng = -(-Kd // group)
    s = 0.004 + 0.006 * torch.rand(S, N, ng, generator=gen)
    if not fine:
        m, ex = torch.frexp(s)
        s = torch.ldexp(torch.round(m * 32) / 32, ex)
    return codes.to(DEV), s.to(dtype).to(DEV)


@pytest.mark.parametrize("S,N,Kd,group,gated", [(1, 8, 8, 32, False), (3, 48, 72, 64, True), (2, 40, 136, 128, False),
                                                (2, 32, 256, 32, True), (1, 272, 200, 128, True), (5, 16, 64, 64, False)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_pack_and_back(S, N, Kd, group, gated, dtype):
    g = torch.Generator().manual_seed(N)
    codes, scales = _codes(S, N, Kd, group, dtype, g, fine=True)
    w = K.int4_pack(codes, scales, group_size=group, gated=gated)
    assert torch.equal(K.int4_dequantize(w), R.dequantise(codes, scales, group).to(dtype))


@pytest.mark.parametrize("N,Kd,group,gated", [(48, 72, 64, True), (16, 520, 128, False), (32, 256, 32, True)])
@pytest.mark.parametrize("src,dtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                       (torch.float32, torch.bfloat16), (torch.float32, torch.float16)])
def test_quantise(N, Kd, group, gated, src, dtype):
    g = torch.Generator().manual_seed(Kd)
    w = (torch.randn(2, N, Kd, generator=g) * 0.02).to(src).to(DEV)
    w[0, 3] = 0
    q = K.int4_quantize(w, group_size=group, gated=gated, dtype=dtype)
    back = K.int4_dequantize(q).double()
    ng = -(-Kd // group)
    pad = torch.zeros(2, N, ng * group, dtype=torch.float64, device=DEV)
    pad[..., :Kd] = w.double()
    m, ex = torch.frexp((pad.view(2, N, ng, group).abs().amax(-1) / 7).float())
    s = torch.ldexp(torch.round(m * 32) / 32, ex).double().repeat_interleave(group, -1)[..., :Kd]
    # the nearest multiple of s: half a step, a little more where |w| / s is clamped at 7 (s up to 1/33 short of max / 7)
    assert bool(((back - w.double()).abs() <= s * (0.5 + 1e-6)).all())
    mult = torch.where(s > 0, back / s, 0.0)
    assert bool((mult == torch.round(mult)).all()) and float(mult.max()) <= 7 and float(mult.min()) >= -8


CASES = [  # T, E, top_k, H, I, group1, group2
    (1, 4, 1, 64, 32, 32, 32), (1, 8, 2, 256, 384, 128, 128), (3, 8, 2, 264, 40, 128, 32), (8, 8, 2, 128, 136, 64, 64),
    (9, 1, 1, 512, 256, 128, 64), (17, 60, 4, 192, 88, 128, 128), (64, 16, 16, 128, 64, 32, 128), (130, 8, 3, 72, 56, 64, 32),
    (300, 4, 2, 256, 512, 128, 128), (700, 3, 1, 320, 200, 64, 128), (1025, 8, 2, 128, 96, 32, 64), (257, 2, 2, 640, 1152, 128, 32),
]


def _case(T, E, top_k, H, I, g1, g2, dtype, seed, skew=0.0, fine=False):
    g = torch.Generator().manual_seed(seed)
    c1, s1 = _codes(E, 2 * I, H, g1, dtype, g, fine)
    c2, s2 = _codes(E, H, I, g2, dtype, g, fine)
    x = torch.randn(T, H, generator=g).to(dtype).to(DEV)
    p = torch.arange(1, E + 1).double() ** -skew
    ids = torch.multinomial(p.expand(max(T, 1), E), top_k, generator=g)[:T].to(torch.int32).to(DEV)
    w = torch.softmax(torch.randn(T, top_k, generator=g), 1).to(DEV)
    return x, (c1, s1), (c2, s2), w, ids


def _check(x, q1, q2, w, ids, g1, g2, activation="silu", **kw):
    w1 = K.int4_pack(*q1, group_size=g1, gated=True)
    w2 = K.int4_pack(*q2, group_size=g2)
    out = K.moe_experts_int4(x, w1, w2, w, ids, activation=activation, **kw)
    ref, bound = R.experts(x, R.dequantise(*q1, g1), R.dequantise(*q2, g2), w, ids, activation, **kw)
    assert out.dtype == x.dtype and out.shape == x.shape
    err = (out.double() - ref).abs()
    assert bool((err <= bound).all()), f"{float((err / bound).nan_to_num().max()):.3f} of the bound"
    return out, w1, w2


@pytest.mark.parametrize("T,E,top_k,H,I,g1,g2", CASES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("impl", [0, 1, 5])  # automatic, few-row kernel, CTA pairs
def test_experts(T, E, top_k, H, I, g1, g2, dtype, impl):
    _lib.set_gemm_impl(impl)
    _check(*_case(T, E, top_k, H, I, g1, g2, dtype, T + I), g1, g2)


@pytest.mark.parametrize("T", [1, 12, 400])
@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh"])
def test_activations(T, activation):
    _check(*_case(T, 4, 2, 256, 192, 128, 64, torch.bfloat16, T, skew=2.0), 128, 64, activation)


@pytest.mark.parametrize("T", [1, 5, 333])
@pytest.mark.parametrize("gated_scale", [False, True])
def test_shared_output_and_residual(T, gated_scale):
    c = _case(T, 8, 2, 256, 128, 128, 128, torch.bfloat16, 7)
    g = torch.Generator().manual_seed(1)
    sy = torch.randn(T, 256, generator=g).bfloat16().to(DEV)
    res = torch.randn(T, 256, generator=g).bfloat16().to(DEV)
    ss = torch.rand(T, generator=g).to(DEV) if gated_scale else None
    out, w1, w2 = _check(*c, 128, 128, shared_y=sy, shared_scale=ss, residual=res)
    again = K.moe_experts_int4(c[0], w1, w2, c[3], c[4], shared_y=sy, shared_scale=ss, residual=res, out=res)
    assert again.data_ptr() == res.data_ptr() and torch.equal(again, out)


@pytest.mark.parametrize("T", [2, 40, 600])
@pytest.mark.parametrize("impl", [1, 5])
def test_uneven_routing(T, impl):
    """All tokens on one expert, the same expert twice in a token, and experts without tokens."""
    _lib.set_gemm_impl(impl)
    x, q1, q2, w, ids = _case(T, 16, 2, 128, 96, 64, 64, torch.bfloat16, 21)
    ids[:] = 5
    _check(x, q1, q2, w, ids, 64, 64)
    ids[:, 1] = 15
    _check(x, q1, q2, w, ids, 64, 64)


def test_ids_outside_are_dropped_and_reported():
    x, q1, q2, w, ids = _case(12, 8, 2, 128, 64, 64, 64, torch.bfloat16, 22)
    ids[3] = -1
    ids[7, 1] = 8
    ref_ids = torch.where((ids < 0) | (ids >= 8), -1, ids)
    _check(x, q1, q2, w, ref_ids, 64, 64)
    assert _lib.device_status() == 1  # RF_DEV_BAD_EXPERT_ID
    out = K.moe_experts_int4(x, K.int4_pack(*q1, group_size=64, gated=True), K.int4_pack(*q2, group_size=64), w, ids)
    assert bool((out[3] == 0).all())
    assert _lib.device_status() == 1


def test_empty_batch_strided_and_unaligned_inputs():
    x, q1, q2, w, ids = _case(24, 8, 2, 128, 64, 64, 64, torch.bfloat16, 23)
    _check(x[::2], q1, q2, w[::2], ids[::2], 64, 64)
    _check(x[:, :].t().contiguous().t(), q1, q2, w, ids, 64, 64)
    flat = torch.zeros(1 + 24 * 128, dtype=torch.bfloat16, device=DEV)
    flat[1:] = x.reshape(-1)
    out, w1, w2 = _check(flat[1:].view(24, 128), q1, q2, w, ids, 64, 64)
    assert K.moe_experts_int4(x[:0], w1, w2, w[:0], ids[:0]).shape == (0, 128)
    f = fused_experts_int4(x.float(), w1, w2, w.double(), ids.long())
    assert f.dtype == torch.float32 and torch.equal(f, out.float())


@pytest.mark.parametrize("T", [4, 300])
@pytest.mark.parametrize("impl", [1, 5])
def test_not_a_number_stays_in_its_token(T, impl):
    _lib.set_gemm_impl(impl)
    x, q1, q2, w, ids = _case(T, 4, 2, 128, 64, 64, 64, torch.bfloat16, 24)
    w1, w2 = K.int4_pack(*q1, group_size=64, gated=True), K.int4_pack(*q2, group_size=64)
    want = K.moe_experts_int4(x, w1, w2, w, ids)
    x[1] = float("nan")
    got = K.moe_experts_int4(x, w1, w2, w, ids)
    assert bool(torch.isnan(got[1]).all())
    keep = torch.arange(T, device=DEV) != 1
    assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("T", [1, 64, 500])
def test_repeats_bit_for_bit_and_two_streams(T):
    x, q1, q2, w, ids = _case(T, 8, 2, 512, 256, 128, 128, torch.bfloat16, 25, skew=1.0)
    w1, w2 = K.int4_pack(*q1, group_size=128, gated=True), K.int4_pack(*q2, group_size=128)
    want = K.moe_experts_int4(x, w1, w2, w, ids)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(3)], []
    for i in range(6):
        with torch.cuda.stream(streams[i % 3]):
            outs.append(K.moe_experts_int4(x, w1, w2, w, ids))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("T,E,top_k,H,I", [(2048, 16, 6, 2048, 1408), (1500, 8, 2, 4096, 2048)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompt_repeats_bit_for_bit(T, E, top_k, H, I, dtype):
    """Many tiles a CTA pair, the rings of codes and tokens always full: every run gives the same bits, and the right ones."""
    x, q1, q2, w, ids = _case(T, E, top_k, H, I, 128, 128, dtype, 30)
    want, w1, w2 = _check(x, q1, q2, w, ids, 128, 128)
    outs = [K.moe_experts_int4(x, w1, w2, w, ids) for _ in range(24)]
    assert [int((o != want).sum()) for o in outs] == [0] * 24


@pytest.mark.parametrize("T", [1, 64, 500])
def test_captured_and_replayed(T):
    x, q1, q2, w, ids = _case(T, 8, 2, 512, 256, 128, 128, torch.bfloat16, 26)
    w1, w2 = K.int4_pack(*q1, group_size=128, gated=True), K.int4_pack(*q2, group_size=128)
    K.moe_experts_int4(x, w1, w2, w, ids)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = K.moe_experts_int4(x, w1, w2, w, ids)
        graphs.append((g, out))
    x2, _, _, w_, ids2 = _case(T, 8, 2, 512, 256, 128, 128, torch.bfloat16, 27)
    x.copy_(x2), w.copy_(w_), ids.copy_(ids2)
    want = K.moe_experts_int4(x, w1, w2, w, ids)
    for g, _ in graphs:
        g.replay()
    assert all(torch.equal(o, want) for _, o in graphs)


def test_against_16_bit_experts():
    """The same weights through the 16-bit path: its three more roundings of h and y apart, the same numbers."""
    T, E, H, I = 200, 8, 512, 384
    x, q1, q2, w, ids = _case(T, E, 2, H, I, 128, 128, torch.bfloat16, 28)
    out, w1, w2 = _check(x, q1, q2, w, ids, 128, 128)
    ref = K.moe_experts(x, K.int4_dequantize(w1), K.int4_dequantize(w2), w, ids, precise=True)
    # each side is within its bound of the exact value; theirs rounds g, u, act and y too: five roundings of 2^-8
    # spread over sums of I terms, far below 5 * 2^-8 of the largest output
    assert float((out.float() - ref.float()).abs().max()) <= 5 * 2.0 ** -8 * float(ref.float().abs().max())


@pytest.mark.parametrize("T", [1, 64, 400])
@pytest.mark.parametrize("impl", [1, 5])
def test_scales_with_all_their_bits(T, impl):
    """Checkpoint scales: where scale * (code - 8) needs more than 16 bits holds, the operand may be rounded once
    (half a step, u = eps / 2 of each weight): both products' bounds grow by u of their magnitudes."""
    _lib.set_gemm_impl(impl)
    g1 = g2 = 64
    x, q1, q2, w, ids = _case(T, 4, 2, 256, 128, g1, g2, torch.bfloat16, 29, fine=True)
    w1, w2 = K.int4_pack(*q1, group_size=g1, gated=True), K.int4_pack(*q2, group_size=g2)
    out = K.moe_experts_int4(x, w1, w2, w, ids)
    d1, d2 = R.dequantise(*q1, g1), R.dequantise(*q2, g2)
    ref, bound = R.experts(x, d1, d2, w, ids, "silu")
    u = 2.0 ** -8
    extra = torch.zeros_like(ref)
    for e in range(4):
        t, k = torch.nonzero(ids == e, as_tuple=True)
        xe, wk = x[t].double(), w[t, k].double()[:, None]
        gu, mag = xe @ d1[e].T, xe.abs() @ d1[e].abs().T
        g, up = gu[:, :128], gu[:, 128:]
        a = R.act("silu", g)
        dh = u * (1.2 * mag[:, :128] * (up.abs() + u * mag[:, 128:]) + a.abs() * mag[:, 128:])
        extra.index_add_(0, t, wk * (((1 + 2 * u) * dh + u * (a * up).abs()) @ d2[e].abs().T))
    assert bool(((out.double() - ref).abs() <= bound + (1 + u) * extra).all())


@pytest.mark.parametrize("T", [1, 7, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("over", ["residual", "shared_y", "x"])
def test_the_output_in_place_of_an_input(T, dtype, over):
    """out may be one of the call's own rows: the same bits as with an output of its own."""
    x, q1, q2, w, ids = _case(T, 8, 2, 256, 128, 128, 64, dtype, 31)
    g = torch.Generator().manual_seed(2)
    sy, res = (torch.randn(T, 256, generator=g).to(dtype).to(DEV) for _ in range(2))
    w1, w2 = K.int4_pack(*q1, group_size=128, gated=True), K.int4_pack(*q2, group_size=64)
    want = K.moe_experts_int4(x, w1, w2, w, ids, shared_y=sy, residual=res)
    out = {"residual": res, "shared_y": sy, "x": x}[over]
    got = K.moe_experts_int4(x, w1, w2, w, ids, shared_y=sy, residual=res, out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(got, want)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind,size", [("codes near 8", 1.0), ("closed channels", 100.0), ("closed channels", 1000.0),
                                       ("closed channels", 50000.0)])
@pytest.mark.parametrize("impl", [1, 5])
def test_where_the_offset_of_the_codes_cancels_most(group, dtype, kind, size, impl):
    """x of one sign with codes 7..9, and huge channels whose codes are all 8, which add nothing.  The few-row kernel's
    codes carry an offset B: a group's sum is off by up to F = 4 * PER * 17 * 2^-23 * (B + 15) of scale * sum |x|
    beyond R.experts' bound (PER = group / 32; derived at the kernel); the CTA-pair kernel's codes carry none."""
    _lib.set_gemm_impl(impl)
    T, E, H, I = 6, 2, 512, 256
    x, (c1, s1), (c2, s2), w, ids = _case(T, E, 1, H, I, group, group, dtype, 33)
    if kind == "codes near 8":
        q = torch.randint(7, 10, (E, 2 * I, H), generator=torch.Generator().manual_seed(5), dtype=torch.uint8)
        c1 = (q[..., 0::2] | (q[..., 1::2] << 4)).to(DEV)
        x = x.abs()
    else:
        c1[:, :, 2] = (c1[:, :, 2] & 0x0f) | 0x80       # k = 5
        c1[:, :, 128] = (c1[:, :, 128] & 0xf0) | 0x08   # k = 256
        x[:, 5], x[:, 256] = size, -size
    w1, w2 = K.int4_pack(c1, s1, group_size=group, gated=True), K.int4_pack(c2, s2, group_size=group)
    out = K.moe_experts_int4(x, w1, w2, w, ids)
    d1, d2 = R.dequantise(c1, s1, group), R.dequantise(c2, s2, group)
    ref, bound = R.experts(x, d1, d2, w, ids, "silu")
    if impl == 1:
        f = 4 * (group // 32) * 17 * 2.0 ** -23 * ((16 if dtype == torch.float16 else 128) + 15)
        u = torch.finfo(dtype).eps / 2
        for t in range(T):
            e = int(ids[t, 0])
            g, up = (d1[e] @ x[t].double()).view(2, I)
            extra = f * (s1[e].double() @ x[t].double().abs().view(-1, group).sum(1)).view(2, I)
            h = R.act("silu", g) * up
            # |act'| < 1.2, as in R.experts; its own bounds of g and u, eg and eu, are below 2^-7 of |x||w|
            mag = (d1[e].abs() @ x[t].double().abs()).view(2, I) * H * 2.0 ** -23
            dh = 1.2 * extra[0] * (up.abs() + extra[1] + mag[1]) + (R.act("silu", g).abs() + 1.2 * mag[0]) * extra[1]
            most = h.abs() + dh * 2 + u
            bound[t] += (1 + 4 * u) * (d2[e].abs() @ dh + f * s2[e].double() @ most.view(-1, group).sum(1))
    assert bool(((out.double() - ref).abs() <= bound).all())
