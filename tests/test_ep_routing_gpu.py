"""set_routing() in the expert-parallel layer: a 1-rank NCCL group on one GPU, against the layer it was made from."""

import pytest
import torch

import operator_refs as R
from reframework_b200 import _lib
from reframework_b200 import kernels as K
from reframework_b200.moe import FusedMoE
from reframework_b200.parallel import dist as D
from reframework_b200.parallel.ep import EPFusedMoE
from test_ep_gpu import _free_port

pytestmark = pytest.mark.gpu
E, TOPK, H, I = 40, 4, 256, 128
OPTIONS = dict(scoring="sigmoid", num_groups=8, topk_groups=3, group_score="top2", scale=2.5)  # 5 experts a group


@pytest.fixture(scope="module")
def device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    dev = torch.device("cuda", 0)
    D.init(backend="nccl", init_method=f"tcp://127.0.0.1:{_free_port()}", rank=0, world_size=1, ep_size=1, timeout_s=60,
           device_id=dev)
    yield dev
    D.destroy()


@pytest.fixture(autouse=True)
def _device_clean(device):
    yield
    assert _lib.device_status() == 0


def _layer(dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    moe = FusedMoE(E, TOPK, H, I, dtype=torch.bfloat16, router_dtype=torch.float32)
    with torch.no_grad():
        for p in moe.parameters():
            p.copy_((torch.randn(p.shape, generator=g) * 0.05).bfloat16())
    return moe.to(dev)


def _bias(seed):
    return -0.7 + 0.1 * torch.randn(E, generator=torch.Generator().manual_seed(seed))


def _x(T, dev):
    return torch.randn(T, H, generator=torch.Generator().manual_seed(T)).bfloat16().to(dev)


def _routed_as_defined(layer, x):
    """The [T, E] counts of the definition, from the layer's own fp32 logits, against what the layer exchanged."""
    lg = K.router_topk(x, layer.gate.detach(), TOPK, want_logits=True)[3]
    _, ids = R.route(lg, TOPK, select_bias=layer.select_bias, **OPTIONS)
    return torch.bincount(ids.reshape(-1), minlength=E)


@pytest.mark.parametrize("p2p", [True, False])
@pytest.mark.parametrize("token_sharded", [True, False])
@pytest.mark.parametrize("T", [1, 37, 300])
def test_a_sharded_layer_routes_as_its_own(device, p2p, token_sharded, T):
    full = _layer(device)
    full.set_routing(select_bias=_bias(1), **OPTIONS)
    ep = EPFusedMoE.from_full(full, 1, 0, token_sharded=token_sharded)
    ep.p2p = p2p
    x = _x(T, device)
    try:
        with torch.no_grad():
            assert torch.equal(ep(x), full(x))
        if ep.last_counts_dev is not None:
            counts = ep.last_counts_dev.reshape(-1, E).sum(0)
        else:
            counts = torch.as_tensor(ep.last_counts).reshape(-1, E).sum(0)
        assert torch.equal(counts.long().cpu(), _routed_as_defined(full, x).cpu())
        plain = EPFusedMoE.from_full(_layer(device), 1, 0, token_sharded=token_sharded)
        plain.p2p = p2p
        with torch.no_grad():
            assert not torch.equal(plain(x), ep(x))  # softmax top-k chooses and weighs otherwise
        plain.close()
    finally:
        ep.close()


def test_its_own_options_and_a_loaded_bias(device):
    full = _layer(device)
    x = _x(64, device)
    ep = EPFusedMoE.from_full(full, 1, 0, token_sharded=True)
    try:
        full.set_routing(select_bias=_bias(2), **OPTIONS)
        ep.load_state_dict(full.state_dict())
        ep.set_routing(**OPTIONS)
        assert torch.equal(ep.select_bias, full.select_bias)
        with torch.no_grad():
            assert torch.equal(ep(x), full(x))
            full.set_routing(select_bias=_bias(3), **OPTIONS)
            assert not torch.equal(ep(x), full(x))
            ep.load_state_dict(full.state_dict())
            assert torch.equal(ep(x), full(x))
            assert ep(x[:0]).shape == (0, H)
    finally:
        ep.close()
    ep.entropy_adaptive_k = True
    with pytest.raises(_lib.RfMoeError, match="entropy"):
        ep(x)
