"""Cases and plain forms of the expert routing and MXFP4 operators.

Four operators, as a user of the package calls them:

* ``route_experts``: top-k gating from router logits with expert groups, masked experts and
  masked tokens (``route``), and the same with its backward pass (``route_train``);
* ``mxfp4_quantize`` followed by ``mxfp4_dequantize`` (``quantize``): the 4-bit form is
  returned as the values it stands for;
* ``mxfp4_linear`` (``linear``): a dense product with MXFP4 weights, the activations quantised
  on the way;
* ``mxfp4_expert_linear`` (``experts``): the same product per expert over rows sorted by expert.

``run`` computes a case in elementary torch operations, or through the package where ``own`` is
true.  ``exact`` gives the operators' definitions in 64 bits.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
_EPS = 1e-12


def _package():
    """(flash_mh_moe.route, flash_mh_moe.mxfp4)."""
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "magi-2-preview_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from flash_mh_moe import mxfp4, route
    return route, mxfp4


# ───────────────────────────── cases ─────────────────────────────

def _route(name, op, H, S, E, K, dtype, score, groups=1, keep=1, bias=True, norm=True, scale=1.0, tokens_masked=0.0,
           experts_masked=0.0):
    return {"name": name, "op": op, "H": H, "S": S, "E": E, "K": K, "dtype": dtype, "score": score, "groups": groups,
            "keep": keep, "bias": bias, "norm": norm, "scale": scale, "tokens_masked": tokens_masked,
            "experts_masked": experts_masked}


def _quantize(name, n, rows, cols, dtype, out, rounding):
    return {"name": name, "op": "quantize", "n": n, "rows": rows, "cols": cols, "dtype": dtype, "out": out,
            "rounding": rounding}


def _linear(name, M, N, K, dtype, out, bias, act, rounding="floor"):
    return {"name": name, "op": "linear", "M": M, "N": N, "K": K, "dtype": dtype, "out": out, "bias": bias, "act": act,
            "rounding": rounding}


def _experts(name, T, E, top_k, N, K, dtype, out, skew, gather, act, weights, bias=False, rounding="floor"):
    return {"name": name, "op": "experts", "T": T, "E": E, "top_k": top_k, "N": N, "K": K, "dtype": dtype, "out": out,
            "skew": skew, "gather": gather, "act": act, "weights": weights, "bias": bias, "rounding": rounding}


def listed():
    return [
        # one token of one head in a decode step: 256 experts in 8 groups, 4 groups kept
        _route("route_token", "route", 1, 1, 256, 8, "bf16", "sigmoid", groups=8, keep=4, scale=2.5),
        # the production head split's routing of a full batch (12 heads, 16384 tokens)
        _route("route_heads", "route", 12, 16384, 256, 6, "fp32", "sigmoid", scale=4.9),
        # router training on a padded batch of the 128-expert layer
        _route("route_train_softmax", "route_train", 1, 16381, 128, 8, "fp32", "softmax", bias=False,
               tokens_masked=0.03),
        # router training with groups, half-width logits and a few experts taken out
        _route("route_train_groups", "route_train", 4, 4099, 160, 6, "bf16", "sigmoid", groups=8, keep=3, scale=2.5,
               experts_masked=0.05),
        # activations of a short odd batch
        _quantize("quantize_tokens", 1, 251, 1280, "bf16", "bf16", "floor"),
        # the gate/up matrices of 128 experts packed from training weights
        _quantize("quantize_weights", 128, 2048, 1024, "fp32", "bf16", "ceil"),
        # one token through a dense layer
        _linear("linear_token", 1, 4096, 2048, "bf16", "bf16", True, "none"),
        # a short odd batch through odd sizes
        _linear("linear_odd", 77, 517, 1000, "fp16", "fp16", False, "none", rounding="ceil"),
        # a long prefill through the first half of a feed-forward
        _linear("linear_prefill", 8192, 8192, 4096, "bf16", "bf16", False, "swiglu7"),
        # a decode batch of 32 tokens, top-8 of 128 experts: gate/up with SwiGLU
        _experts("experts_decode", 32, 128, 8, 2048, 1024, "bf16", "bf16", 0.0, True, "swiglu7", False),
        # a full batch through the 128-expert layer's gate/up
        _experts("experts_prefill", 16384, 128, 8, 2048, 1024, "bf16", "bf16", 0.0, True, "swiglu7", False),
        # skewed routing, empty experts among them: the down product, weighted
        _experts("experts_skewed", 1999, 256, 6, 1280, 1280, "bf16", "bf16", 2.4, False, "none", True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["route", "route_train", "quantize", "linear", "linear", "experts", "experts"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    out = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op in ("route", "route_train"):
        groups = rng.choice([1, 1, 2, 4, 5, 8])
        per = _log_int(rng, 4, 96)
        E = min(1024, groups * per)
        E -= E % groups
        keep = rng.randint(1, groups)
        K = rng.randint(1, min(16, keep * (E // groups)))
        H = rng.choice([1, 1, 2, 4, 12])
        S = _log_int(rng, 1, 16384 // H if E > 256 else 16384)
        case = _route("", op, H, S, E, K, dtype, rng.choice(["softmax", "sigmoid"]), groups, keep,
                      rng.random() < 0.6, rng.random() < 0.7, rng.choice([1.0, 2.5, 4.9]),
                      rng.choice([0.0, 0.0, 0.2]), rng.choice([0.0, 0.0, 0.1]))
    elif op == "quantize":
        n = rng.choice([1, 1, 1, 3, 8])
        cols = _log_int(rng, 1, 8192)
        rows = _log_int(rng, 1, min(16384, (1 << 28) // (n * cols)))
        case = _quantize("", n, rows, cols, dtype, rng.choice(["fp32", "bf16", "bf16"]), rng.choice(["floor", "ceil"]))
    elif op == "linear":
        M, N, K = _log_int(rng, 1, 8192), _log_int(rng, 16, 8192), _log_int(rng, 32, 4096)
        act = rng.choice(["none", "none", "swiglu7"])
        N += (N % 2) if act == "swiglu7" else 0
        case = _linear("", M, N, K, dtype, out, rng.random() < 0.5, act, rng.choice(["floor", "ceil"]))
    else:
        E = rng.choice([1, 8, 60, 128, 256])
        top_k = rng.randint(1, min(8, E))
        T = _log_int(rng, 1, 4096)
        N, K = _log_int(rng, 64, 2048), _log_int(rng, 64, 1280)
        act = rng.choice(["none", "swiglu7"])
        N += (N % 2) if act == "swiglu7" else 0
        case = _experts("", T, E, top_k, N, K, dtype, out, rng.choice([0.0, 1.2, 2.4]), rng.random() < 0.5, act,
                        rng.random() < 0.5, rng.random() < 0.3, rng.choice(["floor", "ceil"]))
    del case["name"]
    return case


def work(case):
    op = case["op"]
    if op in ("route", "route_train"):
        rows = case["H"] * case["S"]
        read = rows * case["E"] * _SIZE[case["dtype"]]
        out = rows * case["K"] * 12
        if op == "route":
            return {"bytes": read + out, "flops": 4 * rows * case["E"]}
        # backward: the weights' gradient in, the logits' gradient out
        return {"bytes": 2 * read + out + rows * case["K"] * 4, "flops": 8 * rows * case["E"]}
    if op == "quantize":
        elems = case["n"] * case["rows"] * case["cols"]
        return {"bytes": elems * (_SIZE[case["dtype"]] + _SIZE[case["out"]]), "flops": 3 * elems}
    N, K = case["N"], case["K"]
    cols = N // 2 if case["act"] == "swiglu7" else N
    if op == "linear":
        rows, x_rows, used = case["M"], case["M"], 1
    else:
        rows = case["T"] * case["top_k"]
        x_rows = case["T"] if case["gather"] else rows
        used = min(case["E"], rows)
    blocks = (K + 31) // 32
    weights = used * N * ((K + 1) // 2 + blocks)
    return {"bytes": weights + x_rows * K * _SIZE[case["dtype"]] + rows * cols * _SIZE[case["out"]],
            "flops": 2 * rows * N * K}


# ───────────────────────────── inputs ─────────────────────────────

def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _weights(g, n, N, K):
    """n matrices [N, K] of N(0, 0.02) weights in MXFP4: packed bytes and scale bytes, row-major."""
    data = torch.empty(n, N, (K + 1) // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(n, N, (K + 31) // 32, dtype=torch.uint8, device="cuda")
    for e in range(n):
        codes, s = _encode(_normal(g, N, K) * 0.02, "floor")
        if K % 2:
            codes = torch.nn.functional.pad(codes, (0, 1))
        data[e] = codes[:, 0::2] | (codes[:, 1::2] << 4)
        scales[e] = s
    return data, scales


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    state = {"case": case}
    if op in ("route", "route_train"):
        H, S, E, K = case["H"], case["S"], case["E"], case["K"]
        logits = _normal(g, H, S, E) + 0.5 * _normal(g, H, 1, E)
        if case["experts_masked"]:
            gone = torch.rand(H, S, E, generator=g, device="cuda") < case["experts_masked"]
            logits = logits.masked_fill(gone, float("-inf"))
        state["logits"] = logits.to(_DTYPES[case["dtype"]])
        state["bias"] = (0.02 if case["score"] == "sigmoid" else 0.5 / E) * _normal(g, H, E) if case["bias"] else None
        state["mask"] = None
        if case["tokens_masked"]:
            state["mask"] = torch.rand(S, generator=g, device="cuda") >= case["tokens_masked"]
        if op == "route_train":
            state["grad"] = _normal(g, H, S, K)
            state["logits"].requires_grad_(own)
        return state
    if op == "quantize":
        n, rows, cols = case["n"], case["rows"], case["cols"]
        x = _normal(g, n, rows, cols) * torch.exp(_normal(g, n, rows, 1))
        state["x"] = x.to(_DTYPES[case["dtype"]])
        return state
    N, K = case["N"], case["K"]
    n = case["E"] if op == "experts" else 1
    data, scales = _weights(g, n, N, K)
    if op == "linear":
        data, scales = data[0], scales[0]
        x_rows = case["M"]
        state["bias"] = 0.1 * _normal(g, N) if case["bias"] else None
    else:
        T, E, k = case["T"], case["E"], case["top_k"]
        popularity = -case["skew"] * torch.log(torch.arange(1, E + 1, device="cuda").float())
        chosen = torch.topk(popularity + _normal(g, T, E), k, dim=1).indices.reshape(-1)
        order = torch.sort(chosen, stable=True).indices
        offsets = torch.zeros(E + 1, dtype=torch.int64, device="cuda")
        offsets[1:] = torch.cumsum(torch.bincount(chosen, minlength=E), 0)
        state["offsets"] = offsets
        state["offsets_host"] = offsets.tolist()
        state["gather"] = (order // k).to(torch.int32) if case["gather"] else None
        state["row_weights"] = torch.rand(T * k, generator=g, device="cuda") if case["weights"] else None
        state["bias"] = 0.1 * _normal(g, E, N) if case["bias"] else None
        x_rows = T if case["gather"] else T * k
    state["x"] = _normal(g, x_rows, K).to(_DTYPES[case["dtype"]])
    if own:
        state["weight"] = _package()[1].MXFP4Matrix.from_blocks(data, scales, K)
    else:
        state["data"], state["scales"] = data, scales
    return state


# ───────────────────────────── plain forms ─────────────────────────────

def _pow2(e):
    """2^e in fp32 for whole e in [-127, 127], from its bits (a power function may be off by a rounding)."""
    bits = torch.where(e > -127, (e.int() + 127) << 23, torch.full_like(e, 1 << 22, dtype=torch.int32))
    return bits.view(torch.float32)


def _block_exponent(amax, rounding):
    """Power-of-two exponent of a block's scale from its largest magnitude (fp32)."""
    mant, exp = torch.frexp(amax)                       # amax = mant * 2^exp, mant in [0.5, 1)
    e = exp - 3                                         # floor(log2 amax) - 2
    if rounding == "ceil":
        e = e + (mant > 0.75).to(e.dtype)               # smallest e with amax <= 6 * 2^e
    e = torch.where(amax == 0, torch.full_like(e, -127), e)
    return e.clamp(-127, 127)


def _round_e2m1(a):
    """Magnitudes to the E2M1 grid {0, .5, 1, 1.5, 2, 3, 4, 6}, ties to even, saturating."""
    low = torch.round(a * 2) / 2
    mid = torch.round(a)
    high = torch.round(a / 2) * 2
    return torch.where(a < 2, low, torch.where(a < 4, mid, high)).clamp(max=6.0)


def _blocks(x):
    cols = x.shape[-1]
    x = torch.nn.functional.pad(x.float(), (0, -cols % 32))
    return x.unflatten(-1, (-1, 32))


def _quantized_values(x, rounding):
    """The fp32 values the MXFP4 form of x stands for."""
    b = _blocks(x)
    e = _block_exponent(b.abs().amax(-1, keepdim=True), rounding)
    q = _round_e2m1(b.abs() * _pow2(-e))
    v = torch.copysign(q, b) * _pow2(e)
    return v.flatten(-2)[..., : x.shape[-1]]


def _encode(x, rounding):
    """MXFP4 codes [rows, cols] (one per byte) and scale bytes [rows, ceil(cols / 32)]."""
    b = _blocks(x)
    e = _block_exponent(b.abs().amax(-1, keepdim=True), rounding)
    q = _round_e2m1(b.abs() * _pow2(-e))
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=x.device)
    code = torch.searchsorted(grid, q) | (torch.signbit(b).long() << 3)
    return code.to(torch.uint8).flatten(-2)[..., : x.shape[-1]], (e[..., 0] + 127).to(torch.uint8)


def _decode(data, scales, cols):
    """fp32 values of row-major packed bytes and scale bytes."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=data.device)
    grid = torch.cat([grid, -grid])
    v = torch.stack([grid[(data & 15).long()], grid[(data >> 4).long()]], -1).flatten(-2)[..., :cols]
    s = _pow2(scales.int() - 127)
    return v * s.repeat_interleave(32, -1)[..., :cols]


def _swiglu7(z):
    gate = z[..., 0::2].clamp(max=7.0)
    up = z[..., 1::2].clamp(-7.0, 7.0)
    return gate * (1.0 / (1.0 + torch.exp(-1.702 * gate))) * (up + 1.0)


def _run_route(state):
    case, logits, bias, mask = state["case"], state["logits"].detach(), state["bias"], state["mask"]
    H, S, E, K = case["H"], case["S"], case["E"], case["K"]
    x = logits.float()
    if case["score"] == "softmax":
        ex = torch.exp(x - x.amax(-1, keepdim=True))
        score = ex / ex.sum(-1, keepdim=True)
    else:
        score = 1.0 / (1.0 + torch.exp(-x))
    # the selection in 64 bits: candidates whose 32-bit scores round alike stay in order
    key = logits.double()
    masked = torch.isneginf(key)
    if bias is not None or case["groups"] > 1:
        if case["score"] == "softmax":
            ex64 = torch.exp(key - key.amax(-1, keepdim=True))
            value = ex64 / ex64.sum(-1, keepdim=True)
        else:
            value = 1.0 / (1.0 + torch.exp(-key))
        if bias is not None:
            value = value + bias.double()[:, None, :]
            key = value
        if case["groups"] > 1:
            grouped = value.masked_fill(masked, float("-inf")).unflatten(-1, (case["groups"], -1))
            top2 = torch.sort(grouped, -1, descending=True).values[..., :2]
            none = torch.isneginf(top2[..., :1])
            total = torch.where(torch.isneginf(top2), torch.zeros_like(top2), top2).sum(-1, keepdim=True)
            total = torch.where(none, torch.full_like(total, float("-inf")), total)[..., 0]
            best = torch.sort(total, dim=-1, descending=True, stable=True).indices[..., : case["keep"]]
            kept = torch.zeros_like(total, dtype=torch.bool).scatter_(-1, best, True)
            masked = masked | ~kept.repeat_interleave(E // case["groups"], -1)
    if mask is not None:
        masked = masked | ~mask[None, :, None]
    key = key.masked_fill(masked, float("-inf"))
    top, idx = torch.sort(key, dim=-1, descending=True, stable=True)
    top, idx = top[..., :K], idx[..., :K]
    empty = torch.isneginf(top)
    p = score.gather(-1, idx).masked_fill(empty, 0.0)
    total = p.sum(-1, keepdim=True)
    w = p / total.clamp(min=_EPS) if case["norm"] else p
    w = w * case["scale"]
    out_idx = idx.masked_fill(empty, -1)
    if case["op"] == "route":
        return w, out_idx
    grad = (state["grad"] * case["scale"]).masked_fill(empty, 0.0)
    if case["norm"]:
        d = total.clamp(min=_EPS)
        spread = torch.where(total > _EPS, (grad * p).sum(-1, keepdim=True) / (d * d), torch.zeros_like(d))
        ds = (grad / d - spread).masked_fill(empty, 0.0)
    else:
        ds = grad
    if case["score"] == "softmax":
        dx = -score * (ds * p).sum(-1, keepdim=True)
        dx = dx.scatter_add(-1, idx, ds * p)
    else:
        q = (1.0 / (1.0 + torch.exp(x))).gather(-1, idx)       # 1 - score
        dx = torch.zeros_like(x).scatter_add(-1, idx, (ds * p * q).masked_fill(empty, 0.0))
    dx = dx.masked_fill(torch.isneginf(logits), 0.0)
    if mask is not None:
        dx = dx.masked_fill(~mask[None, :, None], 0.0)
    return w, out_idx, dx.to(logits.dtype)


def _finish(acc, bias, act, row_weights, dtype):
    if bias is not None:
        acc = acc + bias
    if act == "swiglu7":
        acc = _swiglu7(acc)
    if row_weights is not None:
        acc = acc * row_weights[:, None]
    return acc.to(dtype)


def _run_linear(state):
    case = state["case"]
    xq = _quantized_values(state["x"], case["rounding"])
    w = _decode(state["data"], state["scales"], case["K"])
    return _finish(xq @ w.t(), state["bias"], case["act"], None, _DTYPES[case["out"]])


def _run_experts(state):
    case, offsets = state["case"], state["offsets_host"]
    xq = _quantized_values(state["x"], case["rounding"])
    cols = case["N"] // 2 if case["act"] == "swiglu7" else case["N"]
    y = torch.empty(offsets[-1], cols, dtype=_DTYPES[case["out"]], device="cuda")
    for e in range(case["E"]):
        a, b = offsets[e], offsets[e + 1]
        if a == b:
            continue
        rows = xq[a:b] if state["gather"] is None else xq[state["gather"][a:b].long()]
        w = _decode(state["data"][e], state["scales"][e], case["K"])
        y[a:b] = _finish(rows @ w.t(), None if state["bias"] is None else state["bias"][e], case["act"],
                         None if state["row_weights"] is None else state["row_weights"][a:b], y.dtype)
    return y


def _run_own(state):
    route, mxfp4 = _package()
    case = state["case"]
    op = case["op"]
    if op in ("route", "route_train"):
        w, idx = route.route_experts(state["logits"], case["K"], score_func=case["score"], expert_bias=state["bias"],
                                     num_groups=case["groups"], topk_groups=case["keep"], route_norm=case["norm"],
                                     norm_eps=_EPS, route_scale=case["scale"], token_mask=state["mask"])
        if op == "route":
            return w, idx
        (grad,) = torch.autograd.grad(w, state["logits"], state["grad"])
        return w.detach(), idx, grad
    out = _DTYPES[case["out"]]
    if op == "quantize":
        return mxfp4.mxfp4_dequantize(mxfp4.mxfp4_quantize(state["x"], scale_rounding=case["rounding"]), out)
    act = None if case["act"] == "none" else case["act"]
    if op == "linear":
        return mxfp4.mxfp4_linear(state["x"], state["weight"], bias=state["bias"], activation=act, out_dtype=out,
                                  scale_rounding=case["rounding"])
    return mxfp4.mxfp4_expert_linear(state["x"], state["weight"], state["offsets"], gather_ids=state["gather"],
                                     row_weights=state["row_weights"], bias=state["bias"], activation=act,
                                     out_dtype=out, scale_rounding=case["rounding"])


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op in ("route", "route_train"):
        return _run_route(state)
    if op == "quantize":
        return _quantized_values(state["x"], state["case"]["rounding"]).to(_DTYPES[state["case"]["out"]])
    return _run_linear(state) if op == "linear" else _run_experts(state)


# ───────────────────────────── definitions in 64 bits ─────────────────────────────

def _exact_values(x, rounding):
    """MXFP4 values of x in 64 bits: exponents from log2 corrected by comparison, codes by
    counting the midpoints a magnitude lies above (a tie goes to the even code)."""
    x = x.double()
    cols = x.shape[-1]
    x = torch.nn.functional.pad(x, (0, -cols % 32))
    b = x.reshape(*x.shape[:-1], -1, 32)
    amax = b.abs().max(-1, keepdim=True).values

    def two_to(k):
        return ((k.long() + 1023) << 52).view(torch.float64)

    k = torch.floor(torch.log2(amax.clamp(min=2.0 ** -160)))
    k = k - (two_to(k) > amax).double()
    k = k + (two_to(k + 1) <= amax).double()
    e = k - 2
    if rounding == "ceil":
        e = e + (amax > 6 * two_to(e)).double()
    scale = two_to(e.clamp(-127, 127))
    a = b.abs() / scale
    code = torch.zeros_like(a)
    grid = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    for i in range(7):
        middle = (grid[i] + grid[i + 1]) / 2
        code += ((a > middle) if i % 2 == 0 else (a >= middle)).double()
    value = torch.tensor(grid, dtype=torch.float64, device=x.device)[code.long()] * scale * torch.sign(b)
    return value.reshape(x.shape)[..., :cols]


def _exact_weight(data, scales, cols):
    low, high = (data & 15).double(), (data >> 4).double()
    c = torch.stack([low, high], -1).reshape(*data.shape[:-1], -1)[..., :cols]
    sign = 1 - 2 * (c >= 8).double()
    c = torch.remainder(c, 8)
    exp, man = torch.floor(c / 2), torch.remainder(c, 2)
    mag = torch.where(exp == 0, man / 2, (1 + man / 2) * torch.where(exp == 3, 4.0, exp))
    s = ((scales.long() + (1023 - 127)) << 52).view(torch.float64)
    return sign * mag * s[..., torch.arange(cols, device=data.device) // 32]


def _exact_finish(acc, bias, act, row_weights):
    if bias is not None:
        acc = acc + bias.double()
    if act == "swiglu7":
        g = torch.minimum(acc[:, 0::2], torch.full_like(acc[:, 0::2], 7.0))
        u = acc[:, 1::2].clamp(-7, 7)
        acc = g / (1 + torch.exp(-1.702 * g)) * (u + 1)
    if row_weights is not None:
        acc = acc * row_weights.double().unsqueeze(1)
    return acc


def _exact_route(state):
    case = state["case"]
    H, S, E, K = case["H"], case["S"], case["E"], case["K"]
    x = state["logits"].detach().double()
    alive = x > float("-inf")
    if state["mask"] is not None:
        alive = alive & state["mask"].view(1, S, 1)
    score = torch.softmax(x, -1) if case["score"] == "softmax" else torch.sigmoid(x)
    value = score if state["bias"] is None else score + state["bias"].double().view(H, 1, E)
    key = x if state["bias"] is None else value
    ids = torch.arange(E, device="cuda")
    low = torch.tensor(float("-inf"), dtype=torch.float64, device="cuda")

    def best(keys, free, numbers):
        """Largest key among the free entries, the lowest number among equals (or -1)."""
        m = torch.where(free, keys, low).max(-1, keepdim=True).values
        at = torch.where(free & (keys == m), numbers, keys.shape[-1]).min(-1).values
        return torch.where(at < keys.shape[-1], at, -1)

    G = case["groups"]
    if G > 1:
        v, f = value.view(H, S, G, E // G), alive.view(H, S, G, E // G)
        first = torch.where(f, v, low).max(-1).values
        one = best(v, f, torch.arange(E // G, device="cuda"))
        f2 = f & (torch.arange(E // G, device="cuda") != one.unsqueeze(-1))
        second = torch.where(f2, v, low).max(-1).values
        total = torch.where(second > low, first + second, first)
        open_groups = f.any(-1)
        kept = torch.zeros_like(open_groups)
        for _ in range(case["keep"]):
            at = best(total, open_groups & ~kept, torch.arange(G, device="cuda"))
            kept = kept | (torch.arange(G, device="cuda") == at.unsqueeze(-1))
        alive = (alive.view(H, S, G, E // G) & kept.unsqueeze(-1)).view(H, S, E)
    picks = []
    free = alive.clone()
    for _ in range(K):
        at = best(key, free, ids)
        free = free & (ids != at.unsqueeze(-1))
        picks.append(at)
    idx = torch.stack(picks, -1)
    has = idx >= 0
    p = torch.where(has, score.gather(-1, idx.clamp(min=0)), 0.0)
    n = p.sum(-1, keepdim=True)
    d = n.clamp(min=_EPS) if case["norm"] else torch.ones_like(n)
    w = case["scale"] * p / d
    if case["op"] == "route":
        return w, idx
    g = torch.where(has, state["grad"].double() * case["scale"], 0.0)
    ds = g / d
    if case["norm"]:
        ds = torch.where(has & (n > _EPS), ds - (g * p).sum(-1, keepdim=True) / d ** 2, ds)
    if case["score"] == "softmax":
        dot = (ds * p).sum(-1, keepdim=True)
        if case["norm"]:
            dot = torch.where(n > _EPS, torch.zeros_like(dot), dot)
        dx = -score * dot
        part = ds * p
    else:
        dx = torch.zeros_like(x)
        part = ds * p * torch.sigmoid(-x).gather(-1, idx.clamp(min=0))
    dx = dx.scatter_add(-1, idx.clamp(min=0), torch.where(has, part, 0.0))
    dx = torch.where(torch.isneginf(x), 0.0, dx)
    if state["mask"] is not None:
        dx = torch.where(state["mask"].view(1, S, 1), dx, 0.0)
    return w, idx, dx


def exact(case, seed):
    global own
    before, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = before
    op = case["op"]
    if op in ("route", "route_train"):
        return _exact_route(state)
    if op == "quantize":
        return torch.stack([_exact_values(m, case["rounding"]) for m in state["x"]])
    if op == "linear":
        w = _exact_weight(state["data"], state["scales"], case["K"])
        return _exact_finish(_exact_values(state["x"], case["rounding"]) @ w.t(), state["bias"], case["act"], None)
    xq = _exact_values(state["x"], case["rounding"])
    parts = []
    for e in range(case["E"]):
        a, b = state["offsets_host"][e], state["offsets_host"][e + 1]
        rows = xq[a:b] if state["gather"] is None else xq[state["gather"][a:b].long()]
        w = _exact_weight(state["data"][e], state["scales"][e], case["K"])
        parts.append(_exact_finish(rows @ w.t(), None if state["bias"] is None else state["bias"][e], case["act"],
                                   None if state["row_weights"] is None else state["row_weights"][a:b]))
    return torch.cat(parts)
