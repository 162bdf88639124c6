"""GPU: the device status word when the first call of a device is inside a graph capture or behind other work."""
import pytest
import torch

from flash_mh_moe import _lib

pytestmark = pytest.mark.gpu

ERR_ARGS = _lib.MHMOE_ERR_ARGS


def _weights(N, K):
    from flash_mh_moe.mxfp4 import MXFP4Matrix
    g = torch.Generator(device="cuda").manual_seed(N + K)
    data = torch.randint(0, 256, (N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.randint(118, 126, (N, K // 32), generator=g, device="cuda", dtype=torch.uint8)
    return MXFP4Matrix.from_blocks(data, scales)


def test_first_call_of_a_device_inside_a_capture():
    """A word made while a graph is captured is zero before any replay and no replay clears it."""
    from flash_mh_moe.mxfp4 import mxfp4_linear
    w = _weights(256, 512)
    x = torch.randn(50, 512, generator=torch.Generator(device="cuda").manual_seed(0), device="cuda").bfloat16()
    dev = x.device
    want = mxfp4_linear(x, w)
    torch.cuda.synchronize()
    before = _lib._status.pop(dev.index)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = mxfp4_linear(x, w)
        _lib.check_device_status(dev)
        _lib.device_status(dev).fill_(ERR_ARGS)
        graph.replay()
        with pytest.raises(ValueError):
            _lib.check_device_status(dev)
        graph.replay()
        _lib.check_device_status(dev)
        assert torch.equal(y, want)
    finally:
        torch.cuda.synchronize()
        _lib._status[dev.index] = before


def test_first_call_behind_a_busy_stream():
    """The word is 0 for every stream once it exists, whatever its memory held and however busy the first stream is."""
    dev = torch.device("cuda", torch.cuda.current_device())
    before = _lib.device_status(dev)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    try:
        with torch.cuda.stream(a):
            junk = [torch.full((128,), ERR_ARGS, dtype=torch.int32, device=dev) for _ in range(64)]
            torch.cuda.synchronize()
            del junk
            torch.cuda._sleep(200_000_000)
            _lib._status.pop(dev.index)
            word = _lib.device_status(dev)
        with torch.cuda.stream(b):
            seen = word.clone()
        torch.cuda.synchronize()
        assert int(seen) == 0
    finally:
        torch.cuda.synchronize()
        _lib._status[dev.index] = before
