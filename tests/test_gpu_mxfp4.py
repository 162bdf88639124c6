"""GPU: MXFP4 quantisation and products against the 64-bit restatement (oracle/mxfp4_ref.py holds
the bound of the products' error; the quantisation has to be equal)."""
import numpy as np
import pytest
import torch

from oracle import mxfp4_ref as mx

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _x(shape, dtype, seed, spread=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g)
    if spread:
        x = x * torch.exp2(torch.randint(-6, 6, (*shape[:-1], 1), generator=g).float())
    return x.to(DT[dtype])


def _w(n, N, K, seed):
    """Weights with scales that vary from block to block: (MXFP4Matrix, values [n, N, K])."""
    from flash_mh_moe.mxfp4 import MXFP4Matrix
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 16, (n, N, K)).astype(np.uint8)
    scales = rng.integers(118, 126, (n, N, (K + 31) // 32)).astype(np.uint8)
    m = MXFP4Matrix.from_blocks(torch.from_numpy(mx.pack(codes)).cuda(), torch.from_numpy(scales).cuda(), K)
    return m, mx.values(codes, scales)


def _close(y, ref, err):
    info = torch.finfo(y.dtype)
    got = y.double().cpu().numpy()
    tol = err + info.eps / 2 * (np.abs(ref) + err) + info.tiny * info.eps
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), (int(bad.sum()), float(np.abs(got - ref)[bad].max()), np.argwhere(bad)[:4].tolist())


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rounding", ["floor", "ceil"])
@pytest.mark.parametrize("shape", [(1, 1), (1, 32), (3, 31), (7, 129), (128, 256), (130, 1000), (2, 65, 517), (3, 1, 64)])
def test_quantize_matches(shape, dtype, rounding):
    from flash_mh_moe.mxfp4 import mxfp4_dequantize, mxfp4_quantize
    x = _x(shape, dtype, sum(shape))
    m = mxfp4_quantize(x.cuda(), rounding)
    codes, scales = mx.quantize(x.double().numpy(), rounding)
    d, s = m.to_blocks()
    assert m.shape == shape
    assert np.array_equal(s.cpu().numpy(), scales) and np.array_equal(d.cpu().numpy(), mx.pack(codes))
    v = mx.values(codes, scales)
    for out in DT.values():
        got = mxfp4_dequantize(m, out).cpu()
        assert got.dtype == out and torch.equal(got, torch.from_numpy(v).to(out))


def test_quantize_special_values():
    from flash_mh_moe.mxfp4 import mxfp4_dequantize, mxfp4_quantize
    rows = [np.linspace(-8, 8, 65)[:64], np.zeros(64), np.full(64, -0.0), np.full(64, 2.0 ** -140),
            np.full(64, -3.4e38), np.array([2.0 ** -126] + [2.0 ** -129] * 63), np.arange(64) * 0.25,
            np.array([6.0 * 2.0 ** -127, 7.0 * 2.0 ** -127] * 32)]
    x = torch.tensor(np.stack(rows), dtype=torch.float32)
    for rounding in ("floor", "ceil"):
        codes, scales = mx.quantize(x.double().numpy(), rounding)
        d, s = mxfp4_quantize(x.cuda(), rounding).to_blocks()
        assert np.array_equal(s.cpu().numpy(), scales) and np.array_equal(d.cpu().numpy(), mx.pack(codes))
    for bad in (float("nan"), float("inf"), float("-inf")):
        y = torch.ones(2, 64)
        y[0, 40] = bad
        v = mxfp4_dequantize(mxfp4_quantize(y.cuda())).cpu()
        assert torch.isnan(v[0, 32:]).all() and (v[0, :32] == 1).all() and (v[1] == 1).all()


def test_quantize_strides_and_empty():
    from flash_mh_moe.mxfp4 import mxfp4_dequantize, mxfp4_quantize
    base = _x((6, 200, 75), "bf16", 3).cuda()
    for v in (base[:, :, 1:66], base[:, ::3], base[::2], base.transpose(1, 2), base[2, 5:], base[:1].expand(4, 200, 75)):
        a, b = mxfp4_quantize(v), mxfp4_quantize(v.contiguous().clone())
        assert torch.equal(a.data, b.data) and torch.equal(a.sf, b.sf)
    e = mxfp4_quantize(torch.zeros(0, 64, device="cuda"))
    assert e.shape == (0, 64) and mxfp4_dequantize(e).shape == (0, 64)


LINEAR = [(1, 1, 1), (1, 256, 64), (2, 130, 100), (5, 33, 32), (16, 128, 256), (17, 96, 1000), (33, 260, 129),
          (64, 512, 512), (77, 517, 1000), (128, 256, 1280), (129, 300, 384), (200, 1025, 96), (257, 640, 2048),
          (1, 1024, 4096), (8, 200, 4096), (300, 70, 33), (513, 513, 513)]


@pytest.mark.parametrize("M,N,K", LINEAR)
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_linear_matches(M, N, K, dtype):
    from flash_mh_moe.mxfp4 import mxfp4_linear, mxfp4_quantize
    x = _x((M, K), dtype, M + N, spread=False)
    w, wv = _w(1, N, K, K)
    w.batched = False
    g = torch.Generator().manual_seed(1)
    bias = torch.randn(N, generator=g)
    xv = mx.values(*mx.quantize(x.double().numpy(), "floor"))
    _close(mxfp4_linear(x.cuda(), w), *mx.product(xv, wv[0]))
    y = mxfp4_linear(x.cuda(), w, bias.cuda(), out_dtype=torch.float32)
    _close(y, *mx.product(xv, wv[0], bias.double().numpy()))
    # activations that are MXFP4 already
    assert torch.equal(mxfp4_linear(mxfp4_quantize(x.cuda()), w, bias.cuda(), out_dtype=torch.float32), y)
    if N % 2 == 0:
        _close(mxfp4_linear(x.cuda(), w, bias.cuda(), "swiglu7"), *mx.product(xv, wv[0], bias.double().numpy(), "swiglu7"))
    xv = mx.values(*mx.quantize(x.double().numpy(), "ceil"))
    _close(mxfp4_linear(x.cuda(), w, scale_rounding="ceil"), *mx.product(xv, wv[0]))


# (rows, weight rows, columns) whose tiles of 128 x 256 are enough for every SM: outputs whose rows start on
# 32 bytes, on 16, and on neither
WIDE = [(1300, 4096, 160), (1290, 4104, 130), (1281, 4097, 33), (2500, 2560, 544)]


@pytest.mark.parametrize("M,N,K", WIDE)
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_linear_of_many_tiles(M, N, K, dtype):
    from flash_mh_moe.mxfp4 import mxfp4_linear, mxfp4_quantize
    x = _x((M, K), dtype, M, spread=False)
    x[5, :] = float("nan")
    w, wv = _w(1, N, K, K)
    w.batched = False
    bias = torch.randn(N, generator=torch.Generator().manual_seed(1))
    keep = [r for r in range(0, M, 7) if r != 5] + [M - 1, 127, 128]
    xv = mx.values(*mx.quantize(x[keep].double().numpy(), "floor"))
    for kw in (dict(), dict(bias=bias.cuda(), out_dtype=torch.float32), dict(bias=bias.cuda(), activation="swiglu7")):
        if "activation" in kw and N % 2:
            continue
        y = mxfp4_linear(x.cuda(), w, **kw)
        assert torch.isnan(y[5]).all()
        _close(y[keep], *mx.product(xv, wv[0], bias.double().numpy() if kw else None, kw.get("activation")))
        assert torch.equal(torch.nan_to_num(mxfp4_linear(mxfp4_quantize(x.cuda()), w, out_dtype=y.dtype, **{
            k: v for k, v in kw.items() if k != "out_dtype"})), torch.nan_to_num(y))


def test_linear_shapes_strides_and_nan():
    from flash_mh_moe.mxfp4 import mxfp4_linear
    w, wv = _w(1, 96, 160, 0)
    w.batched = False
    x = _x((4, 6, 200), "bf16", 2).cuda()
    v = x[..., 7:167]
    y = mxfp4_linear(v, w)
    assert y.shape == (4, 6, 96) and torch.equal(y, mxfp4_linear(v.contiguous(), w))
    assert torch.equal(mxfp4_linear(v[2, 3], w), y[2, 3])
    assert mxfp4_linear(x[:0, :, :160], w).shape == (0, 6, 96)
    z = v.contiguous().reshape(24, 160).clone()
    z[3, 100], z[9, 0] = float("nan"), float("inf")
    yz = mxfp4_linear(z, w)
    keep = [r for r in range(24) if r not in (3, 9)]
    assert torch.isnan(yz[[3, 9]]).all() and torch.equal(yz[keep], y.reshape(24, 96)[keep])


def test_linear_is_the_same_in_every_batch():
    """A row's result does not depend on the rows beside it within one kernel variant, and runs repeat."""
    from flash_mh_moe.mxfp4 import mxfp4_linear
    w, wv = _w(1, 384, 1024, 5)
    w.batched = False
    x = _x((300, 1024), "bf16", 6, spread=False).cuda()
    a = mxfp4_linear(x, w, out_dtype=torch.float32)
    for _ in range(3):
        assert torch.equal(mxfp4_linear(x, w, out_dtype=torch.float32), a)
    for M in (1, 2, 9, 40, 100, 200):
        ref, err = mx.product(mx.values(*mx.quantize(x[:M].double().cpu().numpy(), "floor")), wv[0])
        _close(mxfp4_linear(x[:M], w, out_dtype=torch.float32), ref, err)


def _routed(T, E, k, seed, skew=0.0, drop=0.0):
    """(gather ids, row weights, offsets) of top-k routing, through the package's sort."""
    from flash_mh_moe import flash_mh_moe_global_sort
    g = torch.Generator().manual_seed(seed)
    pop = -skew * torch.log(torch.arange(1, E + 1).float())
    idx = torch.topk(pop + torch.randn(T, E, generator=g), k, 1).indices
    if drop:
        idx = torch.where(torch.rand(T, 1, generator=g) < drop, -1, idx)
    w = torch.rand(T, k, generator=g)
    return flash_mh_moe_global_sort(w[None].cuda(), idx[None].cuda(), E)


def _expert_ref(xv, wv, gids, offs, rw, bias, act):
    ys, es = [], []
    for e in range(wv.shape[0]):
        a, b = offs[e], offs[e + 1]
        y, err = mx.product(xv[gids[a:b]], wv[e], None if bias is None else bias[e], act, None if rw is None else rw[a:b])
        ys.append(y)
        es.append(err)
    return np.concatenate(ys), np.concatenate(es)


@pytest.mark.parametrize("T,E,k,N,K,skew,drop", [
    (1, 1, 1, 64, 64, 0, 0), (1, 8, 2, 128, 96, 0, 0), (3, 5, 1, 33, 129, 0, 0), (40, 16, 4, 256, 256, 0, 0),
    (100, 8, 3, 130, 300, 2.0, 0), (64, 60, 6, 320, 128, 2.4, 0.3), (300, 4, 2, 512, 640, 1.0, 0),
    (500, 3, 2, 200, 256, 0, 0.2), (17, 128, 8, 96, 512, 0, 0), (9, 7, 7, 1026, 1000, 0, 0), (700, 2, 1, 260, 96, 0, 0)])
@pytest.mark.parametrize("act", [None, "swiglu7"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_expert_linear_matches(T, E, k, N, K, skew, drop, act, dtype):
    from flash_mh_moe.mxfp4 import mxfp4_expert_linear
    N += N % 2
    x = _x((T, K), dtype, T, spread=False)
    w, wv = _w(E, N, K, N)
    gids, rw, offs = _routed(T, E, k, 3, skew, drop)
    used = int(offs[-1])
    bias = 0.5 * torch.randn(E, N, generator=torch.Generator().manual_seed(2))
    g, o = gids.cpu().numpy(), offs.tolist()
    xv = mx.values(*mx.quantize(x.double().numpy(), "floor"))
    rwn = rw.cpu().double().numpy()
    y = mxfp4_expert_linear(x.cuda(), w, offs, gids, rw, bias.cuda(), act)
    ref, err = _expert_ref(xv, wv, g, o, rwn, bias.double().numpy(), act)
    assert y.shape == (T * k, N // 2 if act else N) and y.dtype == x.dtype
    _close(y[:used], ref, err)
    assert (y[used:] == 0).all()                       # rows behind the last expert's
    # rows in place: no gather, no weights, an output of the caller's
    xs = x.cuda()[gids[:used].long()]
    out = torch.full((used + 5, y.shape[1] + 3), 7.0, dtype=torch.float32, device="cuda")
    pad = torch.cat([xs, torch.full((5, K), float("nan"), dtype=x.dtype, device="cuda")])
    r = mxfp4_expert_linear(pad, w, offs, activation=act, out_dtype=torch.float32, out=out[:, 1:-2])
    ref, err = _expert_ref(xv, wv, g, o, None, None, act)
    assert r.data_ptr() == out[:, 1:].data_ptr()
    _close(r[:used], ref, err)
    assert (out[used:] == 7).all() and (out[:, 0] == 7).all() and (out[:, -2:] == 7).all()


@pytest.mark.parametrize("T,E,k,N,K,skew,drop", [
    (400, 60, 6, 1030, 96, 0, 0), (700, 100, 4, 512, 160, 2.4, 0.1), (2100, 16, 8, 2560, 64, 1.0, 0.05),
    (3000, 8, 7, 128, 130, 0, 0)])
@pytest.mark.parametrize("act", [None, "swiglu7"])
def test_expert_linear_of_many_rows(T, E, k, N, K, skew, drop, act):
    """Wide tiles, and (from 16384 rows on) tokens quantised once and copied."""
    from flash_mh_moe.mxfp4 import mxfp4_expert_linear
    x = _x((T, K), "bf16", T, spread=False)
    w, wv = _w(E, N, K, N)
    gids, rw, offs = _routed(T, E, k, 3, skew, drop)
    used, o = int(offs[-1]), offs.tolist()
    bias = 0.5 * torch.randn(E, N, generator=torch.Generator().manual_seed(2))
    y = mxfp4_expert_linear(x.cuda(), w, offs, gids, rw, bias.cuda(), act)
    assert (y[used:] == 0).all()
    xv = mx.values(*mx.quantize(x.double().numpy(), "floor"))
    g, rwn = gids.cpu().numpy(), rw.cpu().double().numpy()
    for e in range(E):                                 # every expert's first and last rows and a few between
        rows = sorted(set(range(o[e], o[e + 1], 37)) | set(range(max(o[e], o[e + 1] - 2), o[e + 1])))
        if rows:
            ref, err = mx.product(xv[g[rows]], wv[e], bias[e].double().numpy(), act, rwn[rows])
            _close(y[rows], ref, err)
    # ids outside x read as zeros and are reported, copied rows too
    from flash_mh_moe import _lib
    _lib.check_device_status(y.device)
    ids = gids.clone()
    ids[used // 2] = T
    z = mxfp4_expert_linear(x.cuda(), w, offs, ids, rw, None, act)
    with pytest.raises(ValueError):
        _lib.check_device_status(y.device)
    assert (z[used // 2] == 0).all()


def test_expert_linear_no_rows_and_bad_inputs():
    from flash_mh_moe import _lib
    from flash_mh_moe.mxfp4 import mxfp4_expert_linear
    w, wv = _w(3, 64, 64, 0)
    x = _x((10, 64), "bf16", 1, spread=False).cuda()
    zero = torch.zeros(4, dtype=torch.int64, device="cuda")
    assert mxfp4_expert_linear(x[:0], w, zero).shape == (0, 64)
    assert (mxfp4_expert_linear(x, w, zero) == 0).all()                       # every expert empty
    assert mxfp4_expert_linear(x, w, zero, gather_ids=torch.zeros(0, dtype=torch.int32, device="cuda")).shape == (0, 64)
    dev = x.device
    _lib.check_device_status(dev)
    # a gather id outside x reads as zeros, offsets outside the rows are clipped; both are reported
    offs = torch.tensor([0, 4, 4, 10], device="cuda")
    ids = torch.tensor([0, 99, 2, -1, 4, 5, 6, 7, 8, 9], dtype=torch.int32, device="cuda")
    good = mxfp4_expert_linear(x, w, offs)
    y = mxfp4_expert_linear(x, w, offs, gather_ids=ids)
    with pytest.raises(ValueError):
        _lib.check_device_status(dev)
    keep = [0, 2, 4, 5, 6, 7, 8, 9]
    assert torch.equal(y[keep], good[keep]) and (y[[1, 3]] == 0).all()
    y = mxfp4_expert_linear(x, w, torch.tensor([-5, 4, 4, 1000], device="cuda"))
    with pytest.raises(ValueError):
        _lib.check_device_status(dev)
    assert torch.equal(y, good)
    for call in [lambda: mxfp4_expert_linear(x, w, offs[:3]), lambda: mxfp4_expert_linear(x[:, :32], w, offs),
                 lambda: mxfp4_expert_linear(x, w, offs.cpu()), lambda: mxfp4_expert_linear(x, w, offs, row_weights=x[:3, 0]),
                 lambda: mxfp4_expert_linear(x, w, offs, bias=torch.zeros(64, device="cuda")),
                 lambda: mxfp4_expert_linear(x, w, offs, out=torch.zeros(10, 64, device="cuda")[:, ::2]),
                 lambda: mxfp4_expert_linear(x, w, offs, out=torch.zeros(9, 64, dtype=torch.bfloat16, device="cuda")),
                 lambda: mxfp4_expert_linear(x.clone().requires_grad_(True), w, offs),
                 lambda: mxfp4_expert_linear(x, w, offs, bias=torch.zeros(3, 64, device="cuda", requires_grad=True)),
                 lambda: mxfp4_expert_linear(x, w, offs, row_weights=torch.ones(10, device="cuda", requires_grad=True)),
                 lambda: mxfp4_expert_linear(x, w, offs, gather_ids=ids.long()),
                 lambda: mxfp4_expert_linear(x, w, offs.float()),
                 lambda: mxfp4_expert_linear(x, w, offs, activation="gelu")]:
        with pytest.raises(ValueError):
            call()


def test_route_sort_products_combine():
    """The operators together, as an expert layer runs them: route, sort, gate/up with SwiGLU7, down
    with the routing weights, and the sum of each token's rows."""
    from flash_mh_moe.mxfp4 import mxfp4_expert_linear
    from flash_mh_moe.route import flash_mh_moe_global_sort_with_inverse, route_experts
    T, E, k, d, f = 150, 16, 4, 256, 192
    g = torch.Generator().manual_seed(0)
    x = torch.randn(T, d, generator=g).bfloat16().cuda()
    logits = torch.randn(1, T, E, generator=g).cuda()
    mask = torch.rand(T, generator=g).cuda() < 0.8
    gu, guv = _w(E, 2 * f, d, 1)
    dn, dnv = _w(E, d, f, 2)
    weights, idx = route_experts(logits, k, "sigmoid", num_groups=4, topk_groups=2, token_mask=mask)
    gids, ps, offs, inv = flash_mh_moe_global_sort_with_inverse(weights, idx, E)
    h = mxfp4_expert_linear(x, gu, offs, gids, activation="swiglu7")
    p = mxfp4_expert_linear(h, dn, offs, row_weights=ps, out_dtype=torch.float32)
    inv = inv.view(T, k).long()
    y = torch.where((inv >= 0)[..., None], p[inv.clamp(min=0)], 0.0).sum(1)
    # reference: the same rows token by token in 64 bits, the hidden as the first product returned it
    xv = mx.values(*mx.quantize(x.double().cpu().numpy(), "floor"))
    used = int(offs[-1])
    o, gi = offs.tolist(), gids.cpu().numpy()
    href, herr = _expert_ref(xv, guv, gi, o, None, None, "swiglu7")
    _close(h[:used], href, herr)
    hv = mx.values(*mx.quantize(h[:used].double().cpu().numpy(), "floor"))
    ref, err = _expert_ref(hv, dnv, np.arange(used), o, ps[:used].double().cpu().numpy(), None, None)
    yr, er = np.zeros((T, d)), np.zeros((T, d))
    np.add.at(yr, gi[:used], ref)
    np.add.at(er, gi[:used], err + 2.0 ** -22 * np.abs(ref))
    assert used == int(mask.sum()) * k
    assert np.all(np.abs(y.double().cpu().numpy() - yr) <= er + 2.0 ** -22 * np.abs(yr))


def test_streams_graphs_and_two_calls():
    from flash_mh_moe.mxfp4 import mxfp4_dequantize, mxfp4_expert_linear, mxfp4_linear, mxfp4_quantize
    w, _ = _w(4, 256, 512, 0)
    w1, _ = _w(1, 256, 512, 0)
    w1.batched = False
    x = _x((100, 512), "bf16", 1, spread=False).cuda()
    offs = torch.tensor([0, 10, 10, 60, 100], device="cuda")

    def all_ops(v):
        return (mxfp4_linear(v, w1), mxfp4_linear(v[:3], w1), mxfp4_expert_linear(v, w, offs),
                mxfp4_dequantize(mxfp4_quantize(v)))

    ref = [t.clone() for t in all_ops(x)]
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = {}
    for s in (s1, s2):
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for s in (s1, s2):
            with torch.cuda.stream(s):
                outs[s] = all_ops(x)
    torch.cuda.synchronize()
    for s in (s1, s2):
        assert all(torch.equal(a, b) for a, b in zip(ref, outs[s]))
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    xs = x.clone()
    with torch.cuda.graph(g1):
        o1 = all_ops(xs)
    with torch.cuda.graph(g2):
        o2 = all_ops(xs)
    xs.copy_(x.flip(0))
    want = [t.clone() for t in all_ops(xs)]
    with torch.cuda.stream(s1):
        g1.replay()
    with torch.cuda.stream(s2):
        g2.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, o1)) and all(torch.equal(a, b) for a, b in zip(want, o2))
