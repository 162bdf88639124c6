"""CPU: route_experts refuses sizes out of its range before it allocates or narrows them, and biases whose layout is
not the logits'.  (Meta tensors stand for the logits: nothing is read.)"""
import pytest
import torch


class _Logits:
    """A meta tensor that says it is on the GPU, so that the checks behind the device's are reached."""

    def __init__(self, *shape):
        self.t = torch.zeros((), device="meta").expand(*shape)

    def __getattr__(self, name):
        return True if name == "is_cuda" else getattr(self.t, name)


@pytest.fixture(autouse=True)
def no_launch(monkeypatch):
    from flash_mh_moe import _lib, route

    def launched(*args, **kwargs):
        raise AssertionError("the call was let through")
    monkeypatch.setattr(_lib, "launch", launched)
    monkeypatch.setattr(route, "_route_experts", launched)


@pytest.mark.parametrize("shape,kw", [
    ((1, 4, (1 << 32) + 8), dict(top_k=2)), ((1, 4, 1025), dict(top_k=2)), ((1, (1 << 32) + 4, 8), dict(top_k=2)),
    (((1 << 32) + 1, 1, 8), dict(top_k=2)), ((1 << 16, 1 << 15, 8), dict(top_k=2)), ((0, 4, 8), dict(top_k=2)),
    ((1, 4, 0), dict(top_k=1)), ((1, 4, 8), dict(top_k=0)), ((1, 4, 8), dict(top_k=-1)), ((1, 4, 8), dict(top_k=9)),
    ((1, 4, 64), dict(top_k=33)), ((1, 4, 64), dict(top_k=(1 << 32) + 2)), ((1, 4, 8), dict(top_k=2, num_groups=(1 << 32) + 1)),
    ((1, 4, 8), dict(top_k=2, num_groups=0)), ((1, 4, 8), dict(top_k=2, num_groups=3)),
    ((1, 4, 8), dict(top_k=2, num_groups=4, topk_groups=(1 << 32) + 1)), ((1, 4, 8), dict(top_k=2, num_groups=4, topk_groups=0)),
    ((1, 4, 8), dict(top_k=3, num_groups=4, topk_groups=1)), ((1, 4, 130), dict(top_k=2, num_groups=65, topk_groups=65))])
def test_sizes(shape, kw):
    from flash_mh_moe.route import route_experts
    with pytest.raises(ValueError):
        route_experts(_Logits(*shape), **kw)


@pytest.mark.parametrize("shape", [(8, 3), (4, 6), (2, 12), (8,), ()])
def test_bias_layout(shape):
    from flash_mh_moe.route import route_experts
    with pytest.raises(ValueError, match="expert_bias"):
        route_experts(_Logits(3, 4, 8), 2, expert_bias=torch.zeros(shape, device="meta"))


@pytest.mark.parametrize("kw", [dict(), dict(expert_bias=torch.zeros(3, 8, device="meta")), dict(num_groups=4, topk_groups=2),
                                dict(expert_bias=torch.zeros(24, device="meta"), num_groups=8, topk_groups=8),
                                dict(expert_bias=torch.zeros(3, 1, 8, device="meta")), dict(expert_bias=torch.zeros(24, 1, device="meta"))])
def test_what_is_let_through(kw):
    from flash_mh_moe.route import route_experts
    with pytest.raises(AssertionError, match="let through"):
        with torch.no_grad():
            route_experts(_Logits(3, 4, 8), 2, **kw)
