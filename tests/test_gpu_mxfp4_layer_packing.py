"""GPU: the MoE layer's packed MXFP4 weights on several streams, in captures and after updates."""
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


def _values(m):
    from flash_mh_moe.mxfp4 import mxfp4_dequantize
    return mxfp4_dequantize(m)


def _want(layer, name):
    from flash_mh_moe.mxfp4 import mxfp4_quantize
    return _values(mxfp4_quantize(getattr(layer, name).weight))


def _dirty(nbytes):
    """Blocks of the allocator that are handed out next hold ones, not zeros."""
    for stream in (torch.cuda.current_stream(), *_streams()):
        with torch.cuda.stream(stream):
            keep = [torch.full((nbytes,), 0x7f, dtype=torch.uint8, device="cuda") for _ in range(4)]
            del keep
    torch.cuda.synchronize()


_pool: list = []


def _streams():
    if not _pool:
        _pool.extend([torch.cuda.Stream(), torch.cuda.Stream()])
    return _pool


@torch.no_grad()
def test_first_use_on_one_stream_then_another():
    layer = _layer()
    a, b = _streams()
    want = _want(layer, "split_linear")
    _dirty(512 * 256)
    torch.cuda.synchronize()
    with torch.cuda.stream(a):
        torch.cuda._sleep(200_000_000)                     # a tenth of a second: the packing waits behind it
        layer._linear_mxfp4("split_linear")
    with torch.cuda.stream(b):
        got = _values(layer._linear_mxfp4("split_linear"))
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@torch.no_grad()
def test_first_use_inside_a_capture_then_eager():
    layer = _layer()
    x = torch.randn(40, 512, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").bfloat16()
    ref = _layer()
    want = ref(x)
    layer.moe_mlp.packed_weights(), layer.moe_mlp.router_planes(), layer.shared_packed()
    layer._shared_routing([40], x.device)
    _dirty(512 * 256)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lin = _values(layer._linear_mxfp4("split_linear"))
    assert torch.equal(layer(x), want)                     # before any replay
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(lin, _want(layer, "split_linear"))
    assert torch.equal(layer(x), want)


@torch.no_grad()
def test_weights_updated_under_a_captured_graph():
    """A graph that was captured with packed weights keeps them: an update packs into other memory, and nothing
    else is handed the old one while the graph can be replayed."""
    layer = _layer()
    first = _want(layer, "merge_linear")
    m = layer._linear_mxfp4("merge_linear")
    addresses = {m.data.data_ptr(), m.sf.data_ptr()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lin = _values(layer._linear_mxfp4("merge_linear"))
    del m
    layer.merge_linear.weight.mul_(2.0)
    second = _values(layer._linear_mxfp4("merge_linear"))
    other = [torch.full((512 * 256,), 0x33, dtype=torch.uint8, device="cuda") for _ in range(4)]
    assert not addresses & {t.data_ptr() for t in other}
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(lin, first) and torch.equal(second, 2 * first)


@torch.no_grad()
def test_update_while_another_stream_reads():
    """An update frees the old packed weights; a stream that still reads them keeps its memory."""
    layer = _layer()
    a, _ = _streams()
    first = _want(layer, "split_linear")
    layer._linear_mxfp4("split_linear")
    torch.cuda.synchronize()
    with torch.cuda.stream(a):
        torch.cuda._sleep(200_000_000)
        got = _values(layer._linear_mxfp4("split_linear"))
    layer.split_linear.weight.mul_(2.0)
    layer._linear_mxfp4("split_linear")
    other = [torch.full((512 * 256,), 0x33, dtype=torch.uint8, device="cuda") for _ in range(4)]
    torch.cuda.synchronize()
    assert torch.equal(got, first) and len(other) == 4


@torch.no_grad()
def test_copies_pack_for_themselves():
    import copy
    layer = _layer()
    m = layer._linear_mxfp4("split_linear")
    other = copy.deepcopy(layer)
    other.split_linear.weight.mul_(2.0)
    assert torch.equal(_values(other._linear_mxfp4("split_linear")), 2 * _values(m))
    assert layer._linear_mxfp4("split_linear") is m
