"""CPU: the MXFP4 and expert-routing entry points refuse bad calls before any launch, the scale
layout's conversions are inverse to one another, and the oracles agree with known values."""
import numpy as np
import pytest
import torch

from oracle import mxfp4_ref as mx
from oracle import route_experts_ref as rr

P = 0x10000
ERR_ARGS, ERR_ARCH = 1, 2


def test_codec_known_values():
    x = np.array([[0.0, -0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -6.0, 7.9] + [0.0] * 21])
    codes, s = mx.quantize(x, "floor")
    assert s.tolist() == [[127]]
    assert mx.values(codes, s)[0, :11].tolist() == [0, 0, 0, 1, 1, 2, 2, 4, 4, -6, 6]
    codes, s = mx.quantize(x, "ceil")
    assert s.tolist() == [[128]] and mx.values(codes, s)[0, 10] == 8
    assert mx.quantize(np.full((1, 5), np.inf), "floor")[1].tolist() == [[255]]
    assert mx.quantize(np.zeros((1, 40)), "floor")[1].tolist() == [[0, 0]]


@pytest.mark.parametrize("shape", [(1, 1), (5, 33), (128, 128), (130, 517), (3, 129, 260)])
def test_blocks_round_trip(shape):
    from flash_mh_moe.mxfp4 import MXFP4Matrix
    rng = np.random.default_rng(0)
    codes = rng.integers(0, 16, shape).astype(np.uint8)
    scales = rng.integers(0, 256, (*shape[:-1], (shape[-1] + 31) // 32)).astype(np.uint8)
    data = torch.from_numpy(mx.pack(codes))
    m = MXFP4Matrix.from_blocks(data, torch.from_numpy(scales), shape[-1])
    assert m.shape == shape
    d, s = m.to_blocks()
    assert torch.equal(d, data) and torch.equal(s, torch.from_numpy(scales))
    # the documented position of every scale
    sf = m.sf.view(m.num_matrices, -1)
    ka = (shape[-1] + 127) // 128
    sc = scales.reshape(m.num_matrices, shape[-2], -1)
    for row in (0, shape[-2] - 1):
        for c in (0, sc.shape[-1] - 1):
            off = ((row // 128) * ka + c // 4) * 512 + (row % 32) * 16 + (row % 128 // 32) * 4 + c % 4
            assert sf[-1, off] == sc[-1, row, c]


def test_from_blocks_refuses():
    from flash_mh_moe.mxfp4 import MXFP4Matrix
    d, s = torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8)
    MXFP4Matrix.from_blocks(d, s)
    for bad in [(d.float(), s, None), (d, s.int(), None), (d, s[:3], None), (d, s, 64), (d, s, 30), (d[0], s[0], None)]:
        with pytest.raises(ValueError):
            MXFP4Matrix.from_blocks(*bad)


def test_matrix_refuses_sizes_it_does_not_hold():
    from flash_mh_moe.mxfp4 import MXFP4Matrix
    d, s = torch.zeros(1, 5, 64, dtype=torch.uint8), torch.zeros(1, 512, dtype=torch.uint8)
    m = MXFP4Matrix(d, s, 5, 100, 1, False)
    assert m.to("cpu").shape == (5, 100)
    for bad in [(d[:0], s[:0], 5, 0, 1, False), (d[:0], s[:0], 0, 1 << 30, 1, False), (d, s, 6, 100, 1, False), (d, s, 5, 129, 1, False), (d, s[:, :100], 5, 100, 1, False),
                (d.float(), s, 5, 100, 1, False), (d, s, 5, 100, 2, True), (d.transpose(1, 2), s, 5, 100, 1, False),
                (torch.zeros(2, 5, 64, dtype=torch.uint8), torch.zeros(2, 512, dtype=torch.uint8), 5, 100, 2, False)]:
        with pytest.raises(ValueError):
            MXFP4Matrix(*bad)


def test_python_refusals_without_a_device():
    from flash_mh_moe import mxfp4
    from flash_mh_moe.route import route_experts
    w = mxfp4.MXFP4Matrix.from_blocks(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8))
    x = torch.zeros(2, 32)
    for call in [lambda: mxfp4.mxfp4_quantize(x),                                   # CPU tensors
                 lambda: mxfp4.mxfp4_quantize(x, "nearest"),
                 lambda: mxfp4.mxfp4_quantize(x.int()),
                 lambda: mxfp4.mxfp4_dequantize(w),
                 lambda: mxfp4.mxfp4_linear(x, w),
                 lambda: mxfp4.mxfp4_linear(x.double(), w),
                 lambda: mxfp4.mxfp4_expert_linear(x, w, torch.zeros(2, dtype=torch.int64)),
                 lambda: mxfp4.mxfp4_expert_linear(x[0], w, torch.zeros(2, dtype=torch.int64)),
                 lambda: route_experts(torch.zeros(1, 2, 8), 2),
                 lambda: route_experts(torch.zeros(2, 8), 2),
                 lambda: route_experts(torch.zeros(1, 2, 8, dtype=torch.int32), 2),
                 lambda: route_experts(torch.zeros(1, 2, 8), 2, score_func="tanh")]:
        with pytest.raises(ValueError):
            call()


@pytest.fixture(scope="module")
def L():
    if torch.cuda.is_available():
        pytest.skip("device present: the valid-argument calls would run")
    from flash_mh_moe import _lib
    return _lib.lib()


def _route(L, logits=P, dtype=0, H=1, S=4, E=16, K=2, score=0, groups=1, keep=1, w=P):
    return L.mhmoe_route_experts(logits, dtype, 64, 16, None, None, 0, H, S, E, K, score, groups, keep, 1, 1e-12, 1.0,
                                 w, P, None, None)


@pytest.mark.parametrize("bad", [dict(logits=None), dict(dtype=3), dict(H=0), dict(S=-1), dict(E=1025), dict(K=0),
                                 dict(K=33, E=64), dict(K=17), dict(score=2), dict(groups=3), dict(groups=0),
                                 dict(groups=4, keep=5), dict(groups=4, keep=0), dict(groups=8, keep=1, K=3),
                                 dict(E=130, groups=65), dict(w=None), dict(H=1 << 16, S=1 << 15)])
def test_route_experts_refuses(L, bad):
    assert _route(L, **bad) == ERR_ARGS


def test_route_experts_accepts(L):
    assert _route(L) == ERR_ARCH
    assert _route(L, groups=4, keep=1, K=4) == ERR_ARCH
    assert L.mhmoe_route_experts_bwd(None, 0, 0, 0, 1, 4, 16, 2, 1, 1, 1e-12, 1.0, P, 8, 2, P, P, P, None) == ERR_ARCH
    # softmax gradients read the logits
    assert L.mhmoe_route_experts_bwd(None, 0, 0, 0, 1, 4, 16, 2, 0, 1, 1e-12, 1.0, P, 8, 2, P, P, P, None) == ERR_ARGS


def _linear(L, x=P, xd=0, xq=None, M=4, cols=64, rounding=0, w=P, N=32, act=0, ws=P, y=P, yd=1, ys=32):
    return L.mhmoe_mxfp4_linear(x, xd, cols, xq, xq, M, cols, rounding, w, P, N, None, act, ws, y, yd, ys, None, 0, None)


@pytest.mark.parametrize("bad", [dict(x=None), dict(xd=4), dict(M=-1), dict(cols=0), dict(rounding=2), dict(w=None),
                                 dict(w=P + 8), dict(N=0), dict(act=2), dict(act=1, N=31), dict(M=200, ws=None), dict(M=200, ws=P + 4),
                                 dict(y=None), dict(yd=-1), dict(ys=31), dict(cols=(1 << 20) + 1)])
def test_linear_refuses(L, bad):
    assert _linear(L, **bad) == ERR_ARGS


def test_linear_accepts(L):
    assert _linear(L) == ERR_ARCH
    assert _linear(L, x=None, xq=P, ws=None) == ERR_ARCH
    assert _linear(L, act=1, ys=16) == ERR_ARCH
    # a few rows need no workspace
    assert L.mhmoe_mxfp4_workspace_bytes(4, 4, 1, 32, 64, 0) == 0
    assert _linear(L, ws=None) == ERR_ARCH
    assert L.mhmoe_mxfp4_workspace_bytes(200, 200, 1, 32, 64, 0) > 0


def _experts(L, x=P, x_rows=8, cols=64, n=4, N=32, offs=P, gids=None, R=8, ws=P, ys=32):
    return L.mhmoe_mxfp4_expert_linear(x, 1, cols, x_rows, cols, 0, P, P, n, N, offs, gids, R, None, None, 0, ws, P, 1,
                                       ys, 1, None, 0, None)


@pytest.mark.parametrize("bad", [dict(offs=None), dict(n=0), dict(n=12289), dict(R=9), dict(x=None), dict(ws=None),
                                 dict(R=1 << 30, gids=P), dict(ys=8)])
def test_expert_linear_refuses(L, bad):
    assert _experts(L, **bad) == ERR_ARGS


def test_expert_linear_accepts(L):
    assert _experts(L) == ERR_ARCH
    assert _experts(L, R=100, gids=P) == ERR_ARCH


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("norm", [True, False])
def test_gradient_formula_against_differences(score, norm):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((2, 3, 12))
    x[0, 1, 4] = -np.inf
    idx = rr.select(x, 4, score, bias=0.1 * rng.standard_normal((2, 12)), groups=3, keep=2)
    g = rng.standard_normal((2, 3, 4))
    dx, _ = rr.gradient(x, idx, g, score, norm, scale=2.5)
    for h, s, e in np.ndindex(x.shape):
        if np.isneginf(x[h, s, e]):
            assert dx[h, s, e] == 0
            continue
        up, dn = x.copy(), x.copy()
        up[h, s, e] += 1e-5
        dn[h, s, e] -= 1e-5
        num = ((rr.weights(up, idx, score, norm, scale=2.5) - rr.weights(dn, idx, score, norm, scale=2.5)) * g).sum() / 2e-5
        assert abs(num - dx[h, s, e]) < 1e-8      # differences: 1e-10 of curvature, 1e-11 of cancellation
