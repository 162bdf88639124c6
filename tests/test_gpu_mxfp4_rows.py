"""GPU: rows of the MXFP4 products do not touch one another, in every form of the kernels: a row's bits stay
the same with other rows beside it, or with NaN and large ones.  And forms that take their activations in MXFP4."""
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
    d, s = torch.from_numpy(mx.pack(codes)).cuda(), torch.from_numpy(scales).cuda()
    return MXFP4Matrix.from_blocks(d if n > 1 else d[0], s if n > 1 else s[0], K), mx.values(codes, scales)


def _x(M, K, seed, dtype=torch.bfloat16):
    return torch.randn(M, K, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


# two row counts of one form each: rows quantised inside, flat tiles of 32, 64 and 128, two flat tiles, wide tiles
@pytest.mark.parametrize("few,many,N,K", [(2, 9, 384, 1024), (1, 16, 517, 900), (17, 32, 384, 1024), (40, 60, 384, 1024),
                                          (65, 128, 260, 700), (200, 250, 384, 1024), (1300, 1400, 4096, 300)])
@pytest.mark.parametrize("act", [None, "swiglu7"])
def test_a_row_keeps_its_bits(few, many, N, K, act):
    from flash_mh_moe.mxfp4 import mxfp4_linear
    N += N % 2 if act else 0
    w, _ = _w(1, N, K, 5)
    x = _x(many, K, 6)
    y = mxfp4_linear(x, w, activation=act, out_dtype=torch.float32)
    assert torch.equal(mxfp4_linear(x[:few], w, activation=act, out_dtype=torch.float32), y[:few])
    z = x.clone()
    z[1::3] = float("nan")
    z[2::3] *= 2.0 ** 60
    keep = torch.arange(0, many, 3, device="cuda")
    got = mxfp4_linear(z, w, activation=act, out_dtype=torch.float32)
    assert torch.equal(got[keep], y[keep]) and torch.isnan(got[1::3]).all()


@pytest.mark.parametrize("n,rows,N,K", [(9, 5, 130, 300), (4, 60, 384, 512), (3, 300, 256, 256), (40, 500, 640, 96)])
def test_an_expert_row_keeps_its_bits(n, rows, N, K):
    """Experts of `rows` rows and fewer; the neighbours of the rows looked at become NaN and large, and their
    experts' weights stay."""
    from flash_mh_moe.mxfp4 import mxfp4_expert_linear
    w, _ = _w(n, N, K, 1)
    cnt = [max(1, rows - 7 * (e % 5)) if e % 4 != 3 else 0 for e in range(n)]
    offs = torch.tensor(np.concatenate([[0], np.cumsum(cnt)]), device="cuda")
    R = int(offs[-1]) + 3
    x = _x(R, K, 2)
    y = mxfp4_expert_linear(x, w, offs, activation="swiglu7")
    z = x.clone()
    z[1::3] = float("nan")
    z[2::3] *= 2.0 ** 60
    got = mxfp4_expert_linear(z, w, offs, activation="swiglu7")
    assert torch.equal(got[0::3], y[0::3]) and (got[R - 3:] == 0).all()
    assert torch.isnan(got[1:R - 3:3]).all()


@pytest.mark.parametrize("M", [1, 16, 17, 33, 64, 100, 128, 129])
@pytest.mark.parametrize("out", [torch.float16, torch.bfloat16, torch.float32])
def test_quantized_activations(M, out):
    from flash_mh_moe.mxfp4 import mxfp4_linear, mxfp4_quantize
    N, K = 322, 420
    w, wv = _w(1, N, K, 3)
    x = _x(M, K, M, torch.float16)
    q = mxfp4_quantize(x, "ceil")
    bias = torch.randn(N, generator=torch.Generator().manual_seed(4))
    y = mxfp4_linear(q, w, bias.cuda(), "swiglu7", out_dtype=out)
    assert y.dtype == out and torch.equal(y, mxfp4_linear(x, w, bias.cuda(), "swiglu7", out_dtype=out, scale_rounding="ceil"))
    xv = mx.values(*mx.quantize(x.double().cpu().numpy(), "ceil"))
    ref, err = mx.product(xv, wv[0], bias.double().numpy(), "swiglu7")
    info = torch.finfo(out)
    got = y.double().cpu().numpy()
    assert np.all(np.abs(got - ref) <= err + info.eps / 2 * (np.abs(ref) + err) + info.tiny * info.eps)
