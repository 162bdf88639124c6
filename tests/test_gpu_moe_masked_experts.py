"""GPU: the MoE core with expert groups where masked experts leave slots empty (index -1): the empty slots add
nothing and are no error.  A core of a smaller top_k that has no empty slots gives the same outputs."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _core(H, dh, K, keep, de=256):
    from flash_mh_moe.moe import CoreMultiHeadMoE, CoreMultiHeadMoEConfig, init_moe_params_
    m = CoreMultiHeadMoE(CoreMultiHeadMoEConfig(
        hidden_size=H * dh, num_heads=H, num_experts=16, top_k=K, expert_intermediate_size=de, num_layers=1,
        params_dtype=torch.bfloat16, route_scale=2.5, num_expert_groups=4, topk_expert_groups=keep)).cuda()
    init_moe_params_(m, seed=0)
    bias = m.router.expert_bias.view(H, 16)
    bias.copy_(0.05 * torch.randn(bias.shape, generator=torch.Generator().manual_seed(1)))
    bias[:, ::4] = float("-inf")                          # one expert of each group of four
    return m


# head rows of the short and of the long quantiser
@pytest.mark.parametrize("H,dh", [(2, 256), (1, 512), (1, 768), (1, 2048)])
@pytest.mark.parametrize("S", [1, 77, 700])
def test_empty_slots(H, dh, S):
    from flash_mh_moe import _lib
    full, four = _core(H, dh, 3, 1), _core(H, dh, 4, 1)
    x = torch.randn(S, H * dh, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    _lib.check_device_status(x.device)
    want = full(x)
    w, idx = four._route(x.view(S, H, dh))
    assert (idx[..., 3] == -1).all() and (w[..., 3] == 0).all() and (idx[..., :3] >= 0).all()
    got = four(x)
    _lib.check_device_status(x.device)
    assert torch.equal(got, want)


def test_tokens_without_an_expert():
    from flash_mh_moe import _lib
    m = _core(1, 256, 2, 2)
    x = torch.randn(50, 256, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    m.router.expert_bias.fill_(float("-inf"))
    y = m(x)
    _lib.check_device_status(x.device)
    assert (y == 0).all()
