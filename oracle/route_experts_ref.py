"""numpy restatement of route_experts and its gradient in 64 bits — test infrastructure."""
from __future__ import annotations

import numpy as np


def scores(logits: np.ndarray, score_func: str) -> np.ndarray:
    x = np.asarray(logits, np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        if score_func == "sigmoid":
            return 1 / (1 + np.exp(-x))
        e = np.exp(x - x.max(-1, keepdims=True))
        return e / e.sum(-1, keepdims=True)


def _order(keys: np.ndarray) -> list[int]:
    """Positions by descending key, equal keys in order; NaN last; -inf left out."""
    at = [i for i in range(len(keys)) if keys[i] != -np.inf]
    return sorted(at, key=lambda i: (np.isnan(keys[i]), 0 if np.isnan(keys[i]) else -keys[i], i))


def select(logits, top_k, score_func, bias=None, groups=1, keep=1, token_mask=None) -> np.ndarray:
    """Chosen ids [H, S, K], -1 where none is left."""
    H, S, E = logits.shape
    x = np.asarray(logits, np.float64)
    s = scores(x, score_func)
    out = np.full((H, S, top_k), -1, np.int64)
    per = E // groups
    for h in range(H):
        for t in range(S):
            if token_mask is not None and not token_mask[h, t]:
                continue
            gone = np.isneginf(x[h, t])
            value = s[h, t]
            if bias is not None:
                value = value + bias[h].astype(np.float64)
                gone = gone | np.isneginf(bias[h])
            key = np.where(gone, -np.inf, value if bias is not None else x[h, t])
            if groups > 1:
                total = np.full(groups, -np.inf)
                for g in range(groups):
                    v = np.where(gone, -np.inf, value)[g * per:(g + 1) * per]
                    best = [v[i] for i in _order(v)[:2]]
                    if best:
                        total[g] = sum(best)
                kept = _order(total)[:keep]
                for g in range(groups):
                    if g not in kept:
                        key[g * per:(g + 1) * per] = -np.inf
            ids = _order(key)[:top_k]
            out[h, t, :len(ids)] = ids
    return out


def weights(logits, idx, score_func, norm=True, eps=1e-12, scale=1.0) -> np.ndarray:
    s = scores(logits, score_func)
    p = np.where(idx >= 0, np.take_along_axis(s, np.maximum(idx, 0), -1), 0.0)
    if norm:
        p = p / np.maximum(p.sum(-1, keepdims=True), eps)
    return scale * p


def gradient(logits, idx, grad, score_func, norm=True, eps=1e-12, scale=1.0):
    """(dlogits, bound of the terms' magnitude) for the weights' gradient ``grad``."""
    x = np.asarray(logits, np.float64)
    s = scores(x, score_func)
    has = idx >= 0
    at = np.maximum(idx, 0)
    p = np.where(has, np.take_along_axis(s, at, -1), 0.0)
    g = np.where(has, grad * scale, 0.0)
    n = p.sum(-1, keepdims=True)
    d = np.maximum(n, eps) if norm else np.ones_like(n)
    ds, mag = g / d, np.abs(g) / d
    if norm:
        ds = ds - np.where(n > eps, (g * p).sum(-1, keepdims=True) / d ** 2, 0.0)
        mag = mag + (np.abs(g) * p).sum(-1, keepdims=True) / d ** 2
    ds = np.where(has, ds, 0.0)
    f = p if score_func == "softmax" else p * (1 - p)
    if score_func == "sigmoid":
        with np.errstate(over="ignore"):
            f = p * np.where(has, np.take_along_axis(1 / (1 + np.exp(x)), at, -1), 0.0)
    dx, bound = np.zeros_like(x), np.zeros_like(x)
    if score_func == "softmax":
        dot = (ds * p).sum(-1, keepdims=True)
        if norm:
            dot = np.where(n > eps, 0.0, dot)
        any_ = has.any(-1, keepdims=True)
        dx -= np.where(any_, s * dot, 0.0)
        bound += np.where(any_, s * (np.abs(ds) * p).sum(-1, keepdims=True) * (dot != 0), 0.0)
    for k in range(idx.shape[-1]):
        part = np.where(has[..., k], ds[..., k] * f[..., k], 0.0)
        pm = np.where(has[..., k], mag[..., k] * f[..., k], 0.0)
        np.put_along_axis(dx, at[..., k:k + 1], np.take_along_axis(dx, at[..., k:k + 1], -1) + part[..., None], -1)
        np.put_along_axis(bound, at[..., k:k + 1], np.take_along_axis(bound, at[..., k:k + 1], -1) + pm[..., None], -1)
    return dx, bound
