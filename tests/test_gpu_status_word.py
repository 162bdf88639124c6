"""GPU: the device status word.  A recorded argument error is recoverable (the kernels clip or read
zeros), so it ends no wait of the call that recorded it nor of a later one; a wait that gave up is
recorded over it.  The products do not look at what earlier calls recorded at all."""
import pytest
import torch

from flash_mh_moe import _lib

pytestmark = pytest.mark.gpu

LIMIT_NS = 2_000_000   # 2 ms a wait
ERR_ARGS, ERR_TIMEOUT = _lib.MHMOE_ERR_ARGS, _lib.MHMOE_ERR_TIMEOUT


def _wait(mode, recorded):
    """(nanoseconds waited, status after) of the self test's wait for what never comes."""
    status = torch.full((1,), recorded, dtype=torch.int32, device="cuda")
    elapsed = torch.zeros(1, dtype=torch.int64, device="cuda")
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    _lib.check(_lib.lib().mhmoe_wait_selftest(flag.data_ptr(), 1, mode, LIMIT_NS, status.data_ptr(), elapsed.data_ptr(),
                                              _lib.stream_ptr(status.device)), "wait_selftest")
    return int(elapsed.item()), int(status.item())


@pytest.mark.parametrize("mode", [1, 2])
def test_argument_error_ends_no_wait(mode):
    ns, status = _wait(mode, ERR_ARGS)
    assert ns >= LIMIT_NS and status == ERR_TIMEOUT
    ns, status = _wait(mode, ERR_TIMEOUT)          # another role gave up: this one leaves too
    assert ns < LIMIT_NS and status == ERR_TIMEOUT


def _weights(n, N, K):
    from flash_mh_moe.mxfp4 import MXFP4Matrix
    g = torch.Generator(device="cuda").manual_seed(N + K)
    data = torch.randint(0, 256, (n, N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.randint(118, 126, (n, N, K // 32), generator=g, device="cuda", dtype=torch.uint8)
    return MXFP4Matrix.from_blocks(data, scales) if n > 1 else MXFP4Matrix.from_blocks(data[0], scales[0])


# one kernel form each: rows quantised inside, a cluster on the columns, flat tiles, wide tiles
@pytest.mark.parametrize("M,N,K", [(3, 256, 16384), (100, 384, 16384), (300, 512, 8192), (1300, 4096, 2048)])
@pytest.mark.parametrize("recorded", [ERR_ARGS, ERR_TIMEOUT])
def test_linear_with_an_error_recorded(M, N, K, recorded):
    from flash_mh_moe.mxfp4 import mxfp4_linear
    w = _weights(1, N, K)
    x = torch.randn(M, K, generator=torch.Generator(device="cuda").manual_seed(0), device="cuda").bfloat16()
    dev = x.device
    _lib.check_device_status(dev)
    want = mxfp4_linear(x, w)
    _lib.device_status(dev).fill_(recorded)
    got = [mxfp4_linear(x, w) for _ in range(4)]
    with pytest.raises((ValueError, _lib.MHMoEError)):
        _lib.check_device_status(dev)
    assert all(torch.equal(y, want) for y in got)
    _lib.check_device_status(dev)


# flat and wide tiles, rows quantised each or copied from tokens quantised once
@pytest.mark.parametrize("T,E,k,N,K", [(40, 64, 4, 512, 4096), (700, 8, 2, 1024, 2048), (3000, 8, 7, 512, 1024)])
def test_expert_rows_beside_a_bad_id(T, E, k, N, K):
    from flash_mh_moe import flash_mh_moe_global_sort
    from flash_mh_moe.mxfp4 import mxfp4_expert_linear
    w = _weights(E, N, K)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(T, K, generator=g, device="cuda").bfloat16()
    idx = torch.rand(T, E, generator=g, device="cuda").topk(k, 1).indices
    ids, rw, offs = flash_mh_moe_global_sort(torch.rand(1, T, k, generator=g, device="cuda"), idx[None], E)
    dev = x.device
    _lib.check_device_status(dev)
    want = mxfp4_expert_linear(x, w, offs, ids, rw, activation="swiglu7")
    bad = ids.clone()
    at = torch.tensor([0, T * k // 3, T * k - 1], device="cuda")
    bad[at] = torch.tensor([T, -1, 1 << 30], dtype=torch.int32, device="cuda")
    got = [mxfp4_expert_linear(x, w, offs, bad, rw, activation="swiglu7") for _ in range(3)]
    later = mxfp4_expert_linear(x, w, offs, ids, rw, activation="swiglu7")      # a good call, the error still recorded
    with pytest.raises(ValueError):
        _lib.check_device_status(dev)
    rest = torch.ones(T * k, dtype=torch.bool, device="cuda")
    rest[at] = False
    for y in got:
        assert torch.equal(y[rest], want[rest]) and (y[at] == 0).all()
    assert torch.equal(later, want)
