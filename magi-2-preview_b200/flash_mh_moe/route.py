"""Routing and sorting — same call signatures as the reference's ``inference/flash_mh_moe/route.py``.

Both functions run on the B200 through libmhmoe; neither has a CPU path.

* ``compute_topk_probs_and_indices``  (reference ``route.py:157-199``)
* ``flash_mh_moe_global_sort``        (reference ``route.py:209-253``)
* ``router_logits``                   the fp32 einsum of ``CoreMultiHeadMoE._route``
  (``inference/model/magi2_preview.py:2588-2591``)
"""
from __future__ import annotations

from typing import Literal, TypeAlias

import torch

from . import _lib

TopKScoreFunc: TypeAlias = Literal["softmax", "sigmoid"]

score_func_name2id_map = {"softmax": 0, "sigmoid": 1}


def compute_topk_probs_and_indices(
    router_logits: torch.Tensor,
    top_k: int,
    score_func: TopKScoreFunc = "softmax",
    expert_bias: torch.Tensor | None = None,
    num_virtual_group: int = 1,
    topk_virtual_group: int = 0,
    route_norm: bool = True,
    norm_eps: float = 1e-12,
    route_scale: float = 1.0,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Top-k probabilities and indices from router logits [H, S, E].

    Returns (topk_probs fp32 [H, S, K], topk_indices int64 [H, S, K]); indices are
    sorted by descending (bias-adjusted) score, ties to the lower expert id.  With
    ``num_virtual_group > 1`` the reference returns the selected set unsorted; this
    returns the same set sorted.  ``route_scale`` (default 1.0, i.e. the reference
    contract) folds in ``CoreMultiHeadMoE._route``'s ``topk_probs * route_scale``.
    """
    if score_func not in score_func_name2id_map:
        raise ValueError(f"Unknown score_func: {score_func}")
    _lib.require_cuda(router_logits)
    H, S, E = router_logits.shape
    K = int(top_k)
    if num_virtual_group > 1:
        assert 0 < topk_virtual_group <= num_virtual_group, (
            f"topk_virtual_group ({topk_virtual_group}) must be in (0, num_virtual_group ({num_virtual_group})]")
        assert E % num_virtual_group == 0, (
            f"num_experts ({E}) must be divisible by num_virtual_group ({num_virtual_group})")
    logits = router_logits.float().contiguous()
    bias = None
    if expert_bias is not None:
        bias = expert_bias.reshape(H, E).float().contiguous()
    dev = logits.device
    probs = torch.empty(H, S, K, dtype=torch.float32, device=dev)
    idx = torch.empty(H, S, K, dtype=torch.int64, device=dev)
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().mhmoe_topk(
            logits.data_ptr(), _lib.ptr(bias), H, S, E, K, score_func_name2id_map[score_func],
            int(num_virtual_group), int(topk_virtual_group), int(bool(route_norm)), float(norm_eps),
            float(route_scale), probs.data_ptr(), idx.data_ptr(), _lib.stream_ptr(dev)),
            "compute_topk_probs_and_indices")
    return probs, idx


def _global_sort(topk_probs, topk_indices, num_experts, want_row_of_flat):
    _lib.require_cuda(topk_probs, topk_indices)
    H, S, K = topk_indices.shape
    E = int(num_experts)
    dev = topk_indices.device
    idx = topk_indices.to(torch.int64).contiguous()
    probs = topk_probs.float().contiguous()
    R = H * S * K
    gather_ids = torch.empty(R, dtype=torch.int32, device=dev)
    probs_sorted = torch.empty(R, dtype=torch.float32, device=dev)
    offsets = torch.empty(H * E + 1, dtype=torch.int64, device=dev)
    row_of_flat = torch.empty(R, dtype=torch.int32, device=dev) if want_row_of_flat else None
    L = _lib.lib()
    ws = torch.empty(L.mhmoe_global_sort_workspace_bytes(H, S, K, E), dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        _lib.check(L.mhmoe_global_sort(probs.data_ptr(), idx.data_ptr(), H, S, K, E, ws.data_ptr(),
                                       gather_ids.data_ptr(), probs_sorted.data_ptr(), offsets.data_ptr(),
                                       _lib.ptr(row_of_flat), _lib.device_status(dev).data_ptr(),
                                       _lib.stream_ptr(dev)), "flash_mh_moe_global_sort")
    return gather_ids, probs_sorted, offsets, row_of_flat


def flash_mh_moe_global_sort(
    topk_probs: torch.Tensor,
    topk_indices: torch.Tensor,
    num_experts: int,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Map per-head expert ids to global [0, H*E) and sort stably into CSR form.

    Returns gather_ids int32 [T], probs_sorted fp32 [T], expert_offsets int64 [H*E+1],
    bit-identical to the reference's ``argsort(stable=True)`` construction.
    """
    g, p, o, _ = _global_sort(topk_probs, topk_indices, num_experts, False)
    return g, p, o


def flash_mh_moe_global_sort_with_inverse(topk_probs, topk_indices, num_experts):
    """``flash_mh_moe_global_sort`` plus ``row_of_flat`` int32 [H*S*K]: the sorted
    position of each flat (h, s, k) entry (the combine uses it as token -> rows map)."""
    return _global_sort(topk_probs, topk_indices, num_experts, True)


def router_logits(x_heads: torch.Tensor, gate: torch.Tensor, num_experts: int) -> torch.Tensor:
    """fp32 router logits [H, S, E] for x_heads [S, H, dh] (bf16) and gate [H*E, dh]."""
    _lib.require_cuda(x_heads, gate)
    S, H, dh = x_heads.shape
    x = x_heads if x_heads.dtype == torch.bfloat16 else x_heads.to(torch.bfloat16)
    if x.stride(2) != 1:
        x = x.contiguous()
    g = gate.float().contiguous()
    dev = x.device
    out = torch.empty(H, S, num_experts, dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().mhmoe_router_logits(x.data_ptr(), x.stride(0), x.stride(1), g.data_ptr(), S, H, dh,
                                                   int(num_experts), out.data_ptr(), _lib.stream_ptr(dev)),
                   "router_logits")
    return out


# ───────────────────────── fused tensor-core router ─────────────────────────

def router_prepare(gate: torch.Tensor) -> tuple[torch.Tensor, int]:
    """Split the fp32 router weight [H*E, dh] into the fewest exact bf16 planes (1..3)
    the fused router needs (load-time work; reads back three flags)."""
    _lib.require_cuda(gate)
    g = gate.detach().float().contiguous()
    n, dh = g.shape
    dev = g.device
    L = _lib.lib()
    flags = torch.zeros(3, dtype=torch.int32, device=dev)
    full = torch.empty(n, 3 * dh, dtype=torch.bfloat16, device=dev)
    with torch.cuda.device(dev):
        _lib.check(L.mhmoe_router_prepare(g.data_ptr(), n, dh, 3, full.data_ptr(), flags.data_ptr(),
                                           _lib.stream_ptr(dev)), "router_prepare")
        f = flags.tolist()
        nsplit = 3 if f[2] else (2 if f[1] else 1)
        if nsplit == 3:
            return full, 3
        planes = torch.empty(n, nsplit * dh, dtype=torch.bfloat16, device=dev)
        _lib.check(L.mhmoe_router_prepare(g.data_ptr(), n, dh, nsplit, planes.data_ptr(), None,
                                           _lib.stream_ptr(dev)), "router_prepare")
    return planes, nsplit


def fused_router_supported(E: int, K: int, dh: int) -> bool:
    return E <= 256 and K <= 16 and dh % 64 == 0


def route_fused(x_heads: torch.Tensor, planes: torch.Tensor, nsplit: int, num_experts: int, top_k: int,
                score_func: str = "softmax", expert_bias: torch.Tensor | None = None, route_norm: bool = True,
                norm_eps: float = 1e-12, route_scale: float = 1.0, return_logits: bool = False,
                logit_bias: torch.Tensor | None = None):
    """Router logits + top-k in one tcgen05 kernel (``CoreMultiHeadMoE._route``).

    x_heads [S, H, dh] bf16 (heads contiguous).  Returns (probs fp32 [H,S,K], idx int64
    [H,S,K]) and, with ``return_logits``, the fp32 logits [H,S,E] as a third item.
    ``logit_bias`` [H*E] (optional) is added to the logits before scoring.
    """
    if score_func not in score_func_name2id_map:
        raise ValueError(f"Unknown score_func: {score_func}")
    _lib.require_cuda(x_heads, planes)
    S, H, dh = x_heads.shape
    E, K = int(num_experts), int(top_k)
    x = x_heads if x_heads.dtype == torch.bfloat16 else x_heads.to(torch.bfloat16)
    if x.stride(2) != 1 or x.stride(1) != dh or x.stride(0) % 8 or x.data_ptr() % 16:
        x = x.contiguous()
    dev = x.device
    probs = torch.empty(H, S, K, dtype=torch.float32, device=dev)
    idx = torch.empty(H, S, K, dtype=torch.int64, device=dev)
    logits = torch.empty(H, S, E, dtype=torch.float32, device=dev) if return_logits else None
    bias = None if expert_bias is None else expert_bias.reshape(-1).float().contiguous()
    lbias = None if logit_bias is None else logit_bias.reshape(-1).float().contiguous()
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().mhmoe_route(
            x.data_ptr(), x.stride(0), x.stride(1), planes.data_ptr(), int(nsplit), S, H, dh, E, K,
            score_func_name2id_map[score_func], _lib.ptr(lbias), _lib.ptr(bias), int(bool(route_norm)),
            float(norm_eps),
            float(route_scale), probs.data_ptr(), idx.data_ptr(), _lib.ptr(logits),
            _lib.device_status(dev).data_ptr(), _lib.stream_ptr(dev)), "route")
    return (probs, idx, logits) if return_logits else (probs, idx)


# ───────────────────────── routing with expert groups, masks and gradients ─────────────────────────

def _route_experts(logits, bias, mask, top_k, cfg, need_saved):
    """(weights, indices, saved) of validated inputs; cfg = (score id, groups, kept groups, norm, eps, scale)."""
    H, S, E = logits.shape
    sh, ss, _ = logits.stride()
    dev = logits.device
    weights = torch.empty((H, S, top_k), dtype=torch.float32, device=dev)
    idx = torch.empty((H, S, top_k), dtype=torch.int64, device=dev)
    saved = torch.empty((H, S, top_k), dtype=torch.float32, device=dev) if need_saved else None
    _lib.launch("mhmoe_route_experts", dev, logits.data_ptr(), _lib.DTYPES[logits.dtype], sh, ss,
                None if bias is None else bias.data_ptr(), None if mask is None else mask.data_ptr(),
                S if mask is not None and mask.dim() == 2 else 0, H, S, E, top_k, *cfg, weights.data_ptr(),
                idx.data_ptr(), saved.data_ptr() if need_saved else None)
    return weights, idx, saved


def _route_experts_grad(ctx, grad_w, _grad_idx):
    if grad_w is None:
        return (None,) * 5
    logits, idx, saved = ctx.saved_tensors
    dtype, E, (score_func, _, _, route_norm, norm_eps, route_scale) = ctx.meta
    H, S, K = idx.shape
    g = grad_w if grad_w.dtype == torch.float32 else grad_w.float()
    gh, gs, gk = g.stride()
    if gk != 1 and K > 1:
        g = g.contiguous()
        gh, gs, _ = g.stride()
    dev = idx.device
    out = torch.empty((H, S, E), dtype=dtype, device=dev)
    ptr, sh, ss = (None, 0, 0) if logits is None else (logits.data_ptr(), logits.stride(0), logits.stride(1))
    _lib.launch("mhmoe_route_experts_bwd", dev, ptr, _lib.DTYPES[dtype], sh, ss, H, S, E, K, score_func, route_norm,
                norm_eps, route_scale, g.data_ptr(), gh, gs, idx.data_ptr(), saved.data_ptr(), out.data_ptr())
    return out, None, None, None, None


class _RouteExperts(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, mask, top_k, cfg):
        weights, idx, saved = _route_experts(logits, bias, mask, top_k, cfg, True)
        ctx.mark_non_differentiable(idx)
        ctx.set_materialize_grads(False)      # no zeros for the indices' gradient
        # sigmoid gradients need the chosen experts' logits only, which `saved` holds
        ctx.save_for_backward(logits if cfg[0] == 0 else None, idx, saved)
        ctx.meta = (logits.dtype, logits.shape[2], cfg)
        return weights, idx

    @staticmethod
    def backward(ctx, grad_w, grad_idx):
        # second derivatives are refused; the guard is only set up where one could be asked for
        if torch.is_grad_enabled():
            return _route_experts_grad_once(ctx, grad_w, grad_idx)
        return _route_experts_grad(ctx, grad_w, grad_idx)


_route_experts_grad_once = torch.autograd.function.once_differentiable(_route_experts_grad)


def route_experts(
    logits: torch.Tensor,
    top_k: int,
    score_func: TopKScoreFunc = "softmax",
    expert_bias: torch.Tensor | None = None,
    num_groups: int = 1,
    topk_groups: int = 1,
    route_norm: bool = True,
    norm_eps: float = 1e-12,
    route_scale: float = 1.0,
    token_mask: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Trainable top-k gating of logits [H, S, E] (fp32, bf16 or fp16, any outer strides).

    Returns (weights fp32 [H, S, K], indices int64 [H, S, K]).  With s the softmax or sigmoid
    scores:

    * candidates are ranked by ``s + expert_bias`` ([H, E] or [H*E], fp32), or by the logits
      without a bias, as 64-bit values (no dependence on how 32-bit scores round); ties go to
      the lower id, NaN ranks below every number;
    * ``num_groups`` > 1 splits the E experts into equal consecutive groups and keeps the
      ``topk_groups`` groups whose two best candidates have the largest sum; unlike
      ``compute_topk_probs_and_indices``'s virtual groups, the other groups' experts are
      never chosen;
    * an expert whose logit or bias is -inf is never chosen; where fewer than ``top_k`` experts
      are left, the remaining slots hold index -1 and weight 0 (the global sort skips them);
    * ``token_mask`` (bool [S] or [H, S]): tokens that are False get -1 and 0 throughout, and
      their logits (NaN included) are not looked at;
    * weights are ``route_scale * s / max(sum of the chosen s, norm_eps)``, or
      ``route_scale * s`` without ``route_norm``.  With ``norm_eps = 0`` sigmoid scores below the
      smallest normal fp32 number count as 0, and over a sum of 0 weights and gradients are 0.

    The weights are differentiable in the logits (first order, backward mode; logits with a
    forward-mode tangent are refused); the bias only steers the
    selection and gets no gradient.  Forward and backward can be captured into a CUDA graph; as with
    any torch operator, no earlier autograd graph of the same leaf may be alive when a
    ``backward()`` that accumulates into it is captured (``torch.autograd.grad`` has no such
    limit).  H * S < 2^31, E <= 1024, K <= 32, at most 64 groups, and ``top_k`` may not exceed the experts of
    ``topk_groups`` groups (``ValueError``).
    """
    score = score_func_name2id_map.get(score_func)
    if score is None:
        raise ValueError(f"Unknown score_func: {score_func}")
    if logits.dim() != 3 or logits.dtype not in _lib.DTYPES:
        raise ValueError(f"logits must be [H, S, E] in fp32, bf16 or fp16, got {tuple(logits.shape)} {logits.dtype}")
    _lib.require_no_tangent("route_experts", logits)
    _lib.require_cuda(logits)
    H, S, E = logits.shape
    K, groups, keep = int(top_k), int(num_groups), int(topk_groups)
    if not (0 < H and H * S < 1 << 31 and 0 < E <= 1024 and 0 < groups <= 64 and E % groups == 0 and 0 < keep <= groups
            and 0 < K <= 32 and K <= keep * (E // groups)):
        raise ValueError(f"route_experts cannot choose {K} of {E} experts in {keep} of {groups} groups for logits "
                         f"{tuple(logits.shape)}")
    bias = mask = None
    if expert_bias is not None:
        if expert_bias.device != logits.device or (
                tuple(expert_bias.shape) != (H, E) and [d for d in expert_bias.shape if d != 1] not in (
                    [d for d in (H * E,) if d != 1], [d for d in (H, E) if d != 1])):
            raise ValueError(f"expert_bias must be [{H}, {E}] or [{H * E}] on {logits.device}, got "
                             f"{tuple(expert_bias.shape)} on {expert_bias.device}")
        bias = expert_bias if expert_bias.dtype == torch.float32 else expert_bias.detach().float()
        if not bias.is_contiguous():
            bias = bias.contiguous()
    if token_mask is not None:
        if (token_mask.dtype != torch.bool or tuple(token_mask.shape) not in ((S,), (H, S))
                or token_mask.device != logits.device):
            raise ValueError(f"token_mask must be bool [S] or [H, S] on {logits.device}, got "
                             f"{tuple(token_mask.shape)} {token_mask.dtype} on {token_mask.device}")
        mask = token_mask if token_mask.is_contiguous() else token_mask.contiguous()
    x = logits if E == 1 or logits.stride(2) == 1 else logits.contiguous()
    cfg = (score, groups, keep, int(bool(route_norm)), float(norm_eps), float(route_scale))
    if torch.is_grad_enabled() and logits.requires_grad:
        return _RouteExperts.apply(x, bias, mask, K, cfg)
    return _route_experts(x, bias, mask, K, cfg, False)[:2]
