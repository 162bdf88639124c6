"""GPU: mxfp4_expert_linear's list of token tiles: more than 256 experts (its second round of 256), the most that
are accepted, and offsets that count rows many times over."""
import numpy as np
import pytest
import torch

from oracle import mxfp4_ref as mx

pytestmark = pytest.mark.gpu


def _w(n, N, K, seed):
    from flash_mh_moe.mxfp4 import MXFP4Matrix
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 16, (n, N, K)).astype(np.uint8)
    scales = rng.integers(118, 126, (n, N, (K + 31) // 32)).astype(np.uint8)
    m = MXFP4Matrix.from_blocks(torch.from_numpy(mx.pack(codes)).cuda(), torch.from_numpy(scales).cuda(), K)
    return m, mx.values(codes, scales)


def _offsets(n, R, seed, used=1.0):
    """Sorted offsets of n experts: most of the rows in a few, many experts without any."""
    rng = np.random.default_rng(seed)
    share = rng.exponential(size=n) ** 3 * (rng.random(n) < 0.6)
    o = np.concatenate([[0], np.round(np.cumsum(share) / share.sum() * R * used)]).astype(np.int64)
    return np.minimum(o, R)


# (experts, rows, tokens, weight rows, columns): flat tiles of 16 and 32 rows, wide tiles, copied rows
@pytest.mark.parametrize("n,R,T,N,K", [(257, 600, 600, 64, 96), (300, 4000, 700, 128, 160), (700, 20000, 20000, 66, 64),
                                       (513, 30000, 5000, 260, 128), (12288, 3000, 400, 2, 32), (12288, 200000, 900, 2, 64)])
@pytest.mark.parametrize("offsets", [torch.int64, torch.int32])
def test_many_experts(n, R, T, N, K, offsets):
    from flash_mh_moe import _lib
    from flash_mh_moe.mxfp4 import mxfp4_expert_linear
    w, wv = _w(n, N, K, n)
    rng = np.random.default_rng(R)
    x = torch.from_numpy(rng.standard_normal((T, K)).astype(np.float32)).half()
    ids = rng.integers(0, T, R).astype(np.int32)
    rw = rng.random(R).astype(np.float32)
    o = _offsets(n, R, n + R, 0.97)
    used = int(o[-1])
    y = mxfp4_expert_linear(x.cuda(), w, torch.from_numpy(o).to(offsets).cuda(), torch.from_numpy(ids).cuda(),
                            torch.from_numpy(rw).cuda(), scale_rounding="ceil")
    _lib.check_device_status(y.device)
    assert (y[used:] == 0).all()
    xv = mx.values(*mx.quantize(x.double().numpy(), "ceil"))
    rows = np.unique(np.concatenate([rng.integers(0, used, 1500), o[:-1][o[:-1] < used], np.maximum(o[1:] - 1, 0)]))
    rows = rows[rows < used]
    if len(rows) > 4000:
        rows = rows[:: len(rows) // 4000 + 1]
    e = np.searchsorted(o, rows, "right") - 1
    a, b = xv[ids[rows]], wv[e]
    ref = np.einsum("rk,rnk->rn", a, b) * rw[rows, None]
    # oracle/mxfp4_ref.py's bound of the fp32 sums, a rounding for the weight, half a step of fp16
    err = (K / 16 + 8) * 2.0 ** -23 * np.einsum("rk,rnk->rn", np.abs(a), np.abs(b)) * rw[rows, None] + 2.0 ** -23 * np.abs(ref)
    info = torch.finfo(torch.float16)
    got = y.double().cpu().numpy()[rows]
    bad = ~(np.abs(got - ref) <= err + info.eps / 2 * (np.abs(ref) + err) + info.tiny * info.eps)
    assert not bad.any(), np.argwhere(bad)[:4]


def test_offsets_that_count_rows_many_times():
    """0, R, 0, R, ...: every other one of 12288 experts claims all 45 million rows, 2.2e9 tiles.  The list holds what
    the scratch has room for, the error is recorded, and the next call is right."""
    from flash_mh_moe import _lib
    from flash_mh_moe.mxfp4 import mxfp4_expert_linear
    n, R, K = 12288, 45_000_000, 32
    w, wv = _w(n, 1, K, 0)
    x = torch.randn(8, K, generator=torch.Generator().manual_seed(0)).bfloat16()
    offs = torch.tensor([0, R] * (n // 2) + [0], device="cuda")
    ids = torch.zeros(R, dtype=torch.int32, device="cuda")
    _lib.check_device_status(ids.device)
    y = mxfp4_expert_linear(x.cuda(), w, offs, ids)
    assert y.shape == (R, 1)
    with pytest.raises(ValueError):
        _lib.check_device_status(ids.device)
    del y, ids
    torch.cuda.empty_cache()
    good = torch.arange(n + 1, device="cuda").clamp(max=8)
    got = mxfp4_expert_linear(x.cuda(), w, good, out_dtype=torch.float32).double().cpu().numpy()
    _lib.check_device_status(good.device)
    xv = mx.values(*mx.quantize(x.double().numpy(), "floor"))
    for r in range(8):
        ref, err = mx.product(xv[r:r + 1], wv[r])
        assert np.all(np.abs(got[r:r + 1] - ref) <= err + 2.0 ** -24 * (np.abs(ref) + err))
