"""GPU: route_experts' norm_eps.  Sums of the chosen scores on both sides of it, norm_eps = 0, and slots
without an expert, against the 64-bit formulas.

Tolerances: those of tests/test_gpu_route_experts.py (2^-16 of a weight, 2^-14 of a gradient's terms and half a
step of its type); their derivation holds for any norm_eps, a constant of fp32 (its own rounding,
2^-24, is one more half step)."""
import numpy as np
import pytest
import torch

from oracle import route_experts_ref as rr

pytestmark = pytest.mark.gpu


def _check(x, K, score, eps, mask=None, bias=None, scale=1.0, gmul=1.0, **groups):
    from flash_mh_moe.route import route_experts
    xg = x.cuda().requires_grad_(True)
    w, idx = route_experts(xg, K, score, None if bias is None else bias.cuda(), norm_eps=eps, route_scale=scale,
                           token_mask=None if mask is None else mask.cuda(), num_groups=groups.get("groups", 1),
                           topk_groups=groups.get("keep", 1))
    xn = x.double().numpy()
    mn = None if mask is None else np.broadcast_to(mask.numpy(), x.shape[:2])
    ref = rr.select(xn, K, score, None if bias is None else bias.numpy(), groups.get("groups", 1), groups.get("keep", 1), mn)
    assert np.array_equal(idx.cpu().numpy(), ref)
    has = ref >= 0
    eps32 = float(np.float32(eps))
    with np.errstate(all="ignore"):
        wr = np.where(has, rr.weights(xn, ref, score, True, eps32, scale), 0.0)
    got = w.detach().cpu().double().numpy()
    assert (got[~has] == 0).all()
    assert np.all(np.abs(got - wr) <= 2.0 ** -16 * np.abs(wr) + 1e-37), np.argwhere(~(np.abs(got - wr) <= 2.0 ** -16 * np.abs(wr)))[:4]
    g = gmul * torch.from_numpy(np.random.default_rng(7).standard_normal(ref.shape).astype(np.float32))
    (dx,) = torch.autograd.grad(w, xg, g.cuda())
    with np.errstate(all="ignore"):
        dr, mag = rr.gradient(xn, ref, g.double().numpy(), score, True, eps32, scale)
    dr, mag = np.nan_to_num(dr, nan=0.0), np.nan_to_num(mag, nan=0.0)
    info = torch.finfo(x.dtype)
    tol = 2.0 ** -14 * mag + info.eps / 2 * np.abs(dr) + info.tiny * info.eps
    err = np.abs(dx.cpu().double().numpy() - dr)
    assert np.all(err <= tol), (np.argwhere(~(err <= tol))[:4], dr[~(err <= tol)][:4])
    # sums that a rounding could put on the other side of eps are not among the inputs
    p = np.where(has, np.take_along_axis(rr.scores(xn, score), np.maximum(ref, 0), -1), 0.0).sum(-1)
    assert not (np.abs(p / max(eps32, 1e-300) - 1) < 2.0 ** -12).any()
    return p, eps32


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("eps", [0.0, 1e-12])
@pytest.mark.parametrize("H,S,E,K,groups", [(1, 40, 24, 8, dict()), (2, 40, 24, 5, dict(groups=4, keep=2)), (2, 6000, 16, 4, dict()),
                                            (1, 6000, 20, 12, dict())])
def test_slots_without_an_expert_weigh_nothing(score, eps, H, S, E, K, groups):
    rng = np.random.default_rng(S + K)
    x = torch.from_numpy(rng.standard_normal((H, S, E)).astype(np.float32))
    x[torch.from_numpy(rng.random(x.shape) < 0.5)] = float("-inf")
    x[:, ::9] = float("-inf")                              # rows without an expert
    mask = torch.from_numpy(rng.random((H, S)) < 0.7)
    _check(x, K, score, eps, mask, scale=2.5, **groups)
    _check(x, K, score, eps, mask, bias=torch.from_numpy(0.1 * rng.standard_normal((H, E)).astype(np.float32)), **groups)


def test_slots_without_an_expert_in_a_row_of_nan():
    from flash_mh_moe.route import route_experts
    x = torch.full((1, 2, 8), float("-inf"))
    x[0, 0, 2], x[0, 0, 5] = float("nan"), 1.0
    x[0, 1, 3], x[0, 1, 4] = float("inf"), 0.0
    for norm in (True, False):
        w, idx = route_experts(x.cuda(), 4, "softmax", route_norm=norm)
        assert idx[0].tolist() == [[5, 2, -1, -1], [3, 4, -1, -1]]
        assert torch.isnan(w[0, :, :1]).all() and (w[0, :, 2:] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("score,eps,shift", [("softmax", 0.4, 0.0), ("sigmoid", 1e-12, 30.0), ("sigmoid", 0.9, 0.0)])
@pytest.mark.parametrize("H,S,E,K", [(1, 50, 48, 4), (3, 3001, 40, 6), (2, 5000, 64, 3)])
def test_sums_on_both_sides_of_eps(dtype, score, eps, shift, H, S, E, K):
    """Rows above and below norm_eps within one warp: below it the gradient has no spread term and, for
    softmax, an entry for every expert."""
    rng = np.random.default_rng(E)
    x = rng.standard_normal((H, S, E)) * 0.5
    if score == "softmax":
        x[:, ::2] *= 8.0                                   # peaked rows: the chosen hold most of the mass
    else:
        x[:, ::2] -= 4.0 + shift                           # small sums
        x[:, 1::2] += 2.0 if shift == 0 else -20.0
    x[:, ::5, 3:] = -np.inf                                # rows with empty slots
    x = torch.from_numpy(x.astype(np.float32)).to(dtype)
    p, e = _check(x, K, score, eps, torch.from_numpy(rng.random(S) < 0.9))
    assert (p > e).any() and ((p < e) & (p > 0)).any()


def test_tiny_sums_without_eps():
    """norm_eps = 0 with sigmoid scores of 2^-120 and gradients of 2^16: g / n alone is above the largest number."""
    rng = np.random.default_rng(0)
    x = torch.from_numpy((-83.0 + 3.0 * rng.random((2, 70, 24))).astype(np.float32))
    _check(x, 5, "sigmoid", 0.0, gmul=65536.0)
    # scores below the smallest normal number of fp32 count as 0, and so do weights and gradients over a sum of 0
    from flash_mh_moe.route import route_experts
    z = torch.full((1, 3, 8), -120.0, device="cuda", requires_grad=True)
    w, idx = route_experts(z, 3, "sigmoid", norm_eps=0.0)
    (dz,) = torch.autograd.grad(w.sum(), z)
    assert idx[0, 0].tolist() == [0, 1, 2] and (w == 0).all() and (dz == 0).all()
