"""GPU: the MoE layer with MXFP4 linears has no derivatives, and says so: a gradient or a tangent that is asked
for is an error, never a missing term."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _layer(d=512, fmt="mxfp4"):
    from flash_mh_moe.layer import MLPActivationType, MoEConfig, MultiHeadMoELayer, MultiHeadMoELayerConfig
    from flash_mh_moe.moe import init_moe_params_
    mc = MoEConfig(num_experts=8, top_k=2, expert_intermediate_size=256, shared_expert_intermediate_size=256,
                   modality_specific_expert_intermediate_size=256, num_heads=2)
    layer = MultiHeadMoELayer(MultiHeadMoELayerConfig(d, 1, 1, MLPActivationType.SWIGLU7, torch.bfloat16, 256, 256,
                                                      torch.bfloat16, None, mc, linear_format=fmt)).cuda()
    g = torch.Generator(device="cuda").manual_seed(0)
    with torch.no_grad():
        for name, p in layer.named_parameters():
            if not name.startswith("moe_mlp."):
                p.copy_(torch.randn(p.shape, generator=g, device="cuda") * 0.02)
    init_moe_params_(layer.moe_mlp, seed=0)
    return layer


def test_no_silent_gradient():
    layer = _layer()
    x = torch.randn(20, 512, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").bfloat16()
    y = layer(x)
    assert y.requires_grad
    with pytest.raises(RuntimeError, match="backward"):
        y.float().sum().backward()
    y.add_(1.0)                                            # an ordinary result for the rest
    with torch.no_grad():
        z = layer(x)
    assert not z.requires_grad and torch.equal(y.detach(), z + 1.0)
    for p in layer.parameters():
        p.requires_grad_(False)
    assert not layer(x).requires_grad
    layer.merge_linear.weight.requires_grad_(True)
    assert layer(x).requires_grad


def test_no_silent_tangent():
    import torch.autograd.forward_ad as fwad
    layer = _layer()
    x = torch.randn(20, 512, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").bfloat16()
    with torch.no_grad(), fwad.dual_level():
        with pytest.raises(ValueError, match="forward-mode"):
            layer(fwad.make_dual(x, torch.ones_like(x)))
