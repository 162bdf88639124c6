"""GPU: route_experts and its backward pass against the 64-bit restatement.

Tolerances.  A softmax score in fp32: the exponent's argument x - m is off by half a unit of
2^-23 of |x - m| <= 32 in these inputs (2^-19 relative in the score at most), the exponential by two
units, the sum of up to 1024 terms, added 32 at a time and then over a tree, by (32 + 5) halves of
2^-23, the quotients by one each: below 2^-17.  The weight adds the sum over K <= 32 terms and a
quotient: 2^-16 of the weight holds everything.  A gradient is at most three such factors and a sum
over K: 2^-14 of its terms' magnitudes, plus half a step of the output's type.
"""
import numpy as np
import pytest
import torch

from oracle import route_experts_ref as rr

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _case(H, S, E, dtype, seed, bias=True, masked=0.0):
    rng = np.random.default_rng(seed)
    x = torch.from_numpy(rng.standard_normal((H, S, E)).astype(np.float32) * 1.5)
    if masked:
        x[torch.from_numpy(rng.random((H, S, E)) < masked)] = float("-inf")
    x = x.to(DT[dtype])
    b = torch.from_numpy((0.1 * rng.standard_normal((H, E))).astype(np.float32)) if bias else None
    return x, b


def _check(x, b, K, score, groups=1, keep=1, norm=True, scale=1.0, mask=None, xg=None, seed=5):
    from flash_mh_moe.route import route_experts
    xg = (x.cuda() if xg is None else xg).detach().requires_grad_(True)
    w, idx = route_experts(xg, K, score, None if b is None else b.cuda(), groups, keep, norm, route_scale=scale,
                           token_mask=None if mask is None else mask.cuda())
    xn = x.double().numpy()
    mn = None if mask is None else np.broadcast_to(mask.numpy(), x.shape[:2])
    ref = rr.select(xn, K, score, None if b is None else b.numpy(), groups, keep, mn)
    assert np.array_equal(idx.cpu().numpy(), ref)
    wr = rr.weights(xn, ref, score, norm, scale=scale)
    assert w.dtype == torch.float32 and idx.dtype == torch.int64
    got = w.detach().cpu().double().numpy()
    # a softmax row with a logit of +inf is NaN by its formula: NaN there, and no NaN elsewhere
    assert np.array_equal(np.isnan(got), np.isnan(wr))
    assert np.all((np.abs(got - wr) <= 2.0 ** -16 * np.abs(wr) + 1e-37) | np.isnan(wr))
    g = torch.from_numpy(np.random.default_rng(seed).standard_normal(ref.shape).astype(np.float32))
    (dx,) = torch.autograd.grad(w, xg, g.cuda())
    dr, mag = rr.gradient(xn, ref, g.double().numpy(), score, norm, scale=scale)
    info = torch.finfo(x.dtype)
    tol = 2.0 ** -14 * mag + info.eps / 2 * np.abs(dr) + info.tiny * info.eps
    assert dx.dtype == x.dtype and dx.shape == x.shape
    assert np.all((np.abs(dx.cpu().double().numpy() - dr) <= tol) | np.isnan(dr))
    return w, idx, dx


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("norm", [True, False])
def test_types_scores_and_norm(dtype, score, norm):
    x, b = _case(2, 37, 64, dtype, 1)
    _check(x, b, 6, score, norm=norm, scale=2.5)
    _check(x, None, 6, score, norm=norm)


@pytest.mark.parametrize("H,S,E,K,groups,keep", [
    (1, 1, 1, 1, 1, 1), (1, 1, 2, 1, 2, 1), (1, 3, 31, 5, 1, 1), (1, 5, 33, 32, 1, 1), (2, 9, 160, 6, 8, 3),
    (1, 4, 256, 8, 8, 4), (3, 7, 96, 32, 3, 1), (1, 2, 1024, 32, 64, 2), (1, 3, 1000, 7, 5, 2), (2, 5, 1023, 31, 1, 1),
    (1, 6, 60, 6, 60, 6), (12, 11, 128, 16, 4, 4), (1, 5, 320, 9, 5, 5), (1, 5, 512, 4, 2, 1), (1, 4, 7, 7, 7, 7)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_sizes_and_groups(H, S, E, K, groups, keep, score):
    x, b = _case(H, S, E, "fp32", H * E + K)
    _check(x, b, K, score, groups, keep)
    _check(x, None, K, score, groups, keep, norm=False)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,keep", [(1, 1), (4, 2)])
def test_masked_experts_and_tokens(score, groups, keep):
    x, b = _case(2, 40, 24, "fp32", 7, masked=0.6)
    x[0, 3] = float("-inf")                       # a row with no expert left
    x[1, 4, :23] = float("-inf")                  # one left
    x[0, 6] = torch.finfo(torch.float32).min      # the lowest number is a number
    b[0, 5] = float("-inf")                       # an expert taken out by its bias
    mask = torch.rand(2, 40, generator=torch.Generator().manual_seed(0)) < 0.7
    x[1, ~mask[1]] = float("nan")                 # contents of masked tokens do not matter
    xc = x.clone()
    xc[1, ~mask[1]] = 0.0
    from flash_mh_moe.route import route_experts
    w, idx, dx = _check(xc, b, 8, score, groups, keep, mask=mask, xg=x.cuda())
    assert (idx.cpu()[~mask] == -1).all() and (w.detach().cpu()[~mask] == 0).all() and (dx.cpu()[~mask] == 0).all()
    assert (idx[0, 3] == -1).all() and not (idx[0] == 5).any()
    # one mask for every head
    _check(xc, b, 8, score, groups, keep, mask=mask[0])


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [True, False])
def test_ties_and_near_ties(score, with_bias):
    """Equal candidates go to the lower id; candidates whose fp32 scores round alike do not."""
    rng = np.random.default_rng(11)
    x = torch.from_numpy(rng.integers(-2, 3, (1, 64, 48)).astype(np.float32))       # many equal logits
    x[0, 32:] += torch.from_numpy(rng.integers(0, 4, (32, 48)).astype(np.float32)) * 2.0 ** -21   # a few units apart
    x[0, 60:] += 40.0                                                                # saturated sigmoids
    b = torch.from_numpy(rng.integers(0, 2, (1, 48)).astype(np.float32) * 0.25) if with_bias else None
    _check(x, b, 8, score)
    _check(x, b, 8, score, groups=6, keep=2)
    # sums that tie up to fp32 rounding but not in 64 bits
    b2 = torch.from_numpy((rng.integers(0, 3, (1, 48)) * 2.0 ** -27).astype(np.float32))
    _check(torch.zeros(1, 4, 48), b2, 8, score)


@pytest.mark.parametrize("H,S,E,K,groups,keep,dtype", [
    (2, 5001, 24, 5, 1, 1, "fp32"), (3, 3333, 40, 8, 4, 2, "bf16"), (1, 9999, 12, 4, 1, 1, "fp16"),
    (1, 5003, 36, 16, 1, 1, "fp32"), (7, 1500, 33, 7, 3, 2, "fp32"), (12, 801, 130, 3, 1, 1, "fp32")])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_many_rows(H, S, E, K, groups, keep, dtype, score):
    """Enough rows for two and four of them a warp: heads that end inside a warp's rows, equal and
    nearly equal candidates, masked experts and tokens among them."""
    x, b = _case(H, S, E, dtype, H + E, masked=0.02)
    x[:, 1::5] = torch.round(x[:, 1::5])                    # equal logits
    x[:, 2::7] = x[:, 2::7].float().abs().clamp(min=1).to(x.dtype).log2().round() * 2.0 ** -12
    x[0, 17] = float("-inf")
    mask = torch.rand(H, S, generator=torch.Generator().manual_seed(1)) < 0.9
    _check(x, b, K, score, groups, keep, mask=mask, scale=1.5)
    _check(x, None, K, score, groups, keep, norm=False)


def test_nan_ranks_last():
    from flash_mh_moe.route import route_experts
    x = torch.randn(1, 3, 16, generator=torch.Generator().manual_seed(0))
    x[0, 1, 3] = float("nan")
    x[0, 2, :12] = float("nan")
    b = 0.01 * torch.randn(1, 16, generator=torch.Generator().manual_seed(1))
    for bias in (b, None):
        w, idx = route_experts(x.cuda(), 6, "sigmoid", None if bias is None else bias.cuda(), route_norm=False)
        ref = rr.select(x.double().numpy(), 6, "sigmoid", None if bias is None else bias.numpy())
        assert np.array_equal(idx.cpu().numpy(), ref)
        assert torch.isnan(w[0, 2, 4:]).all() and not torch.isnan(w[0, :2]).any()
        w, idx = route_experts(x.cuda(), 6, "softmax", None if bias is None else bias.cuda())
        assert torch.isnan(w[0, 1:]).all() and not torch.isnan(w[0, 0]).any()
        assert ((idx >= 0) & (idx < 16)).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_strides_and_broadcast(dtype):
    x, b = _case(3, 20, 40, dtype, 2)
    base = x.cuda()
    wide = torch.zeros(20, 3, 47, dtype=x.dtype, device="cuda")
    view = wide.permute(1, 0, 2)[:, :, 3:43]
    view.copy_(base)
    _check(x, b, 5, "softmax", norm=False, xg=view)                     # odd offset and strides
    _check(x, b, 5, "sigmoid", xg=base.transpose(0, 1).contiguous().transpose(0, 1))
    _check(x, b, 5, "softmax", xg=base.transpose(1, 2).contiguous().transpose(1, 2))   # strided experts
    # a broadcast input: the gradient is summed over its copies
    from flash_mh_moe.route import route_experts
    one = base[:1, :1].clone().requires_grad_(True)
    w, idx = route_experts(one.expand(3, 20, 40), 5, "softmax", b.cuda(), route_norm=False)
    g = torch.randn_like(w)
    (dx,) = torch.autograd.grad(w, one, g)
    full = base[:1, :1].expand(3, 20, 40).contiguous().requires_grad_(True)
    wf, idf = route_experts(full, 5, "softmax", b.cuda(), route_norm=False)
    (df,) = torch.autograd.grad(wf, full, g)
    assert torch.equal(idx, idf) and torch.equal(w, wf) and torch.equal(dx, df.sum((0, 1), keepdim=True))
    # an expanded gradient
    (d1,) = torch.autograd.grad(route_experts(full, 5, route_norm=False)[0].sum(), full)
    (d2,) = torch.autograd.grad(route_experts(full, 5, route_norm=False)[0], full, torch.ones_like(w))
    assert torch.equal(d1, d2)


def test_gradient_against_differences():
    from flash_mh_moe.route import route_experts
    x = torch.randn(1, 1, 16, generator=torch.Generator().manual_seed(4)).cuda()
    g = torch.randn(1, 1, 4, generator=torch.Generator().manual_seed(5)).cuda()
    for score in ("softmax", "sigmoid"):
        for norm in (True, False):
            f = lambda v: (route_experts(v, 4, score, route_norm=norm)[0].double() * g).sum()
            xr = x.clone().requires_grad_(True)
            (dx,) = torch.autograd.grad(f(xr), xr)
            h = 2.0 ** -8
            for e in range(16):
                up, dn = x.clone(), x.clone()
                up[..., e] += h
                dn[..., e] -= h
                # fp32 weights: 4 * 2^-17 * max|g| / 2h of rounding, h^2 of curvature
                assert abs((f(up) - f(dn)) / (2 * h) - dx[0, 0, e]) < 4 * 2.0 ** -17 * g.abs().max() / (2 * h) + h * h


def test_empty_and_refusals():
    from flash_mh_moe.route import route_experts
    x = torch.zeros(2, 0, 8, device="cuda", requires_grad=True)
    w, idx = route_experts(x, 3)
    assert w.shape == idx.shape == (2, 0, 3)
    assert torch.autograd.grad(w.sum(), x)[0].shape == x.shape
    y = torch.zeros(2, 4, 8, device="cuda")
    for kw in [dict(top_k=0), dict(top_k=9), dict(top_k=2, num_groups=3), dict(top_k=3, num_groups=4, topk_groups=1),
               dict(top_k=2, num_groups=2, topk_groups=3), dict(top_k=2, expert_bias=torch.zeros(8, device="cuda")),
               dict(top_k=2, expert_bias=torch.zeros(16)), dict(top_k=2, token_mask=torch.ones(3, dtype=torch.bool, device="cuda")),
               dict(top_k=2, token_mask=torch.ones(4, device="cuda"))]:
        with pytest.raises(ValueError):
            route_experts(y, **kw)
    with pytest.raises(ValueError):
        route_experts(torch.zeros(1, 1, 1025, device="cuda"), 2)
    # second derivatives are refused, not wrong
    z = torch.randn(1, 2, 8, device="cuda", requires_grad=True)
    (d,) = torch.autograd.grad(route_experts(z, 2)[0].sum(), z, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()


def test_side_stream_and_graph():
    from flash_mh_moe.route import route_experts
    x, b = _case(2, 50, 64, "bf16", 9)
    xg, bg = x.cuda().requires_grad_(True), b.cuda()
    g = torch.randn(2, 50, 6, device="cuda")

    def step():
        w, idx = route_experts(xg, 6, "sigmoid", bg, 4, 2)
        (dx,) = torch.autograd.grad(w, xg, g)
        return w.detach(), idx, dx

    ref = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            out = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(ref, out))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    x2, _ = _case(2, 50, 64, "bf16", 10)
    with torch.no_grad():
        xg.copy_(x2)
    graph.replay()
    got = [t.clone() for t in static]
    assert all(torch.equal(a, c) for a, c in zip(got, step()))


def test_same_selection_as_the_serving_router():
    """Without groups the choice equals compute_topk_probs_and_indices's on tie-free inputs."""
    from flash_mh_moe import compute_topk_probs_and_indices
    from flash_mh_moe.route import route_experts
    x = torch.randn(2, 100, 128, generator=torch.Generator().manual_seed(1)).cuda()
    for score in ("softmax", "sigmoid"):
        w, i = route_experts(x, 8, score)
        p, j = compute_topk_probs_and_indices(x, 8, score)
        assert torch.equal(i, j) and torch.allclose(w, p, rtol=2.0 ** -15, atol=0)
