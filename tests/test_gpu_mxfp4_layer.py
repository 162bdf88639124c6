"""GPU: the MoE core with expert groups and the MoE layer with MXFP4 linears run the operators they
say they run."""
import numpy as np
import pytest
import torch

from oracle import mxfp4_ref as mx
from oracle import route_experts_ref as rr

pytestmark = pytest.mark.gpu


def _core(groups, keep, E=32, H=2, K=4):
    from flash_mh_moe.moe import CoreMultiHeadMoE, CoreMultiHeadMoEConfig, init_moe_params_
    cfg = CoreMultiHeadMoEConfig(hidden_size=H * 256, num_heads=H, num_experts=E, top_k=K, expert_intermediate_size=256,
                                 num_layers=1, params_dtype=torch.bfloat16, route_scale=2.5,
                                 num_expert_groups=groups, topk_expert_groups=keep)
    m = CoreMultiHeadMoE(cfg).cuda()
    init_moe_params_(m, seed=0)
    m.router.expert_bias.copy_(0.05 * torch.randn(m.router.expert_bias.shape, generator=torch.Generator().manual_seed(1)))
    return m


def test_core_routes_within_groups():
    from flash_mh_moe.route import router_logits
    m = _core(8, 3)
    x = torch.randn(100, 512, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    xh = x.view(100, 2, 256)
    p, i = m._route(xh)
    logits = router_logits(xh, m.gate, 32).double().cpu().numpy()
    ref = rr.select(logits, 4, "sigmoid", m.router.expert_bias.view(2, 32).cpu().numpy(), 8, 3)
    assert np.array_equal(i.cpu().numpy(), ref)
    assert all(len(set(row // 4)) <= 3 for row in i.reshape(-1, 4).cpu().numpy())
    y = m(x)
    assert torch.equal(y, m._flash_forward(xh, p, i).reshape(100, 512))
    # one group: the path it had
    a, b = _core(1, 1), _core(8, 8)
    ya, yb = a(x), b(x)
    assert torch.equal(a._route(xh)[1], b._route(xh)[1])
    assert (ya - yb).float().norm() <= 1e-2 * ya.float().norm()      # weights differ in their last bits


def test_layer_with_mxfp4_linears():
    from flash_mh_moe.layer import MLPActivationType, MoEConfig, MultiHeadMoELayer, MultiHeadMoELayerConfig, group_layout
    from flash_mh_moe.moe import init_moe_params_
    from flash_mh_moe.mxfp4 import mxfp4_linear, mxfp4_quantize
    d, groups = 512, [60, 0, 41]
    mc = MoEConfig(num_experts=8, top_k=2, expert_intermediate_size=256, shared_expert_intermediate_size=256,
                   modality_specific_expert_intermediate_size=256, num_heads=2)

    def make(fmt):
        torch.manual_seed(0)
        layer = MultiHeadMoELayer(MultiHeadMoELayerConfig(
            d, 3, 1, MLPActivationType.SWIGLU7, torch.bfloat16, 256, 256, torch.bfloat16, None, mc, linear_format=fmt)).cuda()
        with torch.no_grad():
            for name, p in layer.named_parameters():
                if not name.startswith("moe_mlp."):
                    p.copy_(torch.randn(p.shape, generator=torch.Generator().manual_seed(len(name))) * 0.02)
        init_moe_params_(layer.moe_mlp, seed=0)
        return layer

    layer = make("mxfp4")
    x = torch.randn(sum(groups), d, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    y = layer(x, groups)
    sizes, cu = group_layout(groups, len(x), 3, x.device)
    norm = layer.pre_norm(x, cu_groups=cu)
    split = mxfp4_linear(norm, mxfp4_quantize(layer.split_linear.weight))
    merged = mxfp4_linear(layer.moe_mlp(split), mxfp4_quantize(layer.merge_linear.weight), out_dtype=torch.float32)
    assert torch.equal(y, (merged + layer._shared_expert_forward(norm, sizes)).to(torch.bfloat16))
    xv = mx.values(*mx.quantize(norm.double().cpu().numpy(), "floor"))
    wv = mx.values(*mx.quantize(layer.split_linear.weight.detach().double().cpu().numpy(), "floor"))
    ref, err = mx.product(xv, wv)
    assert np.all(np.abs(split.double().cpu().numpy() - ref) <= err + 2.0 ** -8 * (np.abs(ref) + err))
    # a changed weight is packed again, and the default path is the one it was
    with torch.no_grad():
        layer.merge_linear.weight.mul_(2.0)
    z = layer(x, groups)
    assert torch.equal(z, (2 * merged + layer._shared_expert_forward(norm, sizes)).to(torch.bfloat16))
    plain = make("bf16")
    out = plain(x, groups)
    shared = plain._shared_expert_forward(plain.pre_norm(x, cu_groups=cu), sizes)
    moe = plain.moe_mlp(torch.nn.functional.linear(plain.pre_norm(x, cu_groups=cu), plain.split_linear.weight))
    assert torch.equal(out, torch.addmm(shared, moe, plain.merge_linear.weight.t()))
    with pytest.raises(ValueError):
        make("int8")
