"""MXFP4 matrices and their products.

Format: E2M1 values (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) with one power-of-two E8M0
scale per 32 consecutive columns, and no second-level scale.  It stands beside the package's
NVFP4 (``flash_mh_moe.nvfp4``: E4M3 scales per 16 and an fp32 scale per matrix or row), for
weights that come in this format and for dense layers.  The reference has no counterpart.

* ``mxfp4_quantize`` / ``mxfp4_dequantize``: a float matrix to ``MXFP4Matrix`` and back.
* ``MXFP4Matrix.from_blocks`` / ``to_blocks``: packed bytes and scale bytes in row-major order,
  as checkpoints hold them.
* ``mxfp4_linear``: y = act(Q(x) W^T + bias), the activations quantised on the way.
* ``mxfp4_expert_linear``: the same per expert, over rows in the order of
  ``flash_mh_moe_global_sort``.

Products of two quantised values are exact, sums are fp32, and each output is rounded once.
All functions enqueue on the current stream of the tensors' device and do not synchronise;
they have no backward pass (nor a forward-mode derivative), and the products refuse inputs that need one.
"""
from __future__ import annotations

import functools
from dataclasses import dataclass

import torch

from . import _lib

_ROUNDING = {"floor": 0, "ceil": 1}
_ACTIVATION = {None: 0, "swiglu7": 1}


def _atoms(cols: int) -> int:
    """128-column scale atoms of a row."""
    return (cols + 127) // 128


@dataclass
class MXFP4Matrix:
    """A matrix [rows, cols], or ``num_matrices`` of them ([n, rows, cols]), in MXFP4.

    ``data``: uint8 [n, rows, cols_p / 2], low nibble = even column, cols_p = cols rounded up to
    128 (padding zero).  ``sf``: uint8 [n, ceil(rows / 128) * (cols_p / 128) * 512], scale bytes
    in 512-byte atoms of 128 rows x 128 columns: row m, block c of an atom at
    (m % 32) * 16 + (m // 32) * 4 + c.
    """
    data: torch.Tensor
    sf: torch.Tensor
    rows: int
    cols: int
    num_matrices: int
    batched: bool

    def __post_init__(self):
        # the kernels read these sizes: a matrix that does not hold them is refused here
        n, rows, ka = self.num_matrices, self.rows, _atoms(self.cols)
        for name, t, size in (("data", self.data, n * rows * ka * 64),
                              ("sf", self.sf, n * ((rows + 127) // 128) * ka * 512)):
            if t.dtype != torch.uint8 or t.numel() != size or not t.is_contiguous():
                raise ValueError(f"MXFP4Matrix.{name} must be {size} contiguous uint8 values for {n} x [{rows}, "
                                 f"{self.cols}], got {tuple(t.shape)} {t.dtype}")
        if (self.data.device != self.sf.device or n < 0 or rows < 0 or not 0 < self.cols < 1 << 30
                or (n != 1 and not self.batched)):
            raise ValueError(f"bad MXFP4Matrix: {n} x [{rows}, {self.cols}], batched {self.batched}, on "
                             f"{self.data.device} and {self.sf.device}")

    def to(self, device) -> "MXFP4Matrix":
        return MXFP4Matrix(self.data.to(device), self.sf.to(device), self.rows, self.cols, self.num_matrices,
                           self.batched)

    @property
    def shape(self) -> tuple[int, ...]:
        return (self.num_matrices, self.rows, self.cols) if self.batched else (self.rows, self.cols)

    @property
    def device(self) -> torch.device:
        return self.data.device

    @staticmethod
    def from_blocks(data: torch.Tensor, scales: torch.Tensor, cols: int | None = None) -> "MXFP4Matrix":
        """From packed bytes [(n,) rows, ceil(cols/2)] (low nibble = even column) and E8M0 bytes
        [(n,) rows, ceil(cols/32)], both row-major uint8.  ``cols`` defaults to two per byte."""
        if data.dtype != torch.uint8 or scales.dtype != torch.uint8 or data.dim() not in (2, 3):
            raise ValueError("from_blocks takes uint8 [(n,) rows, bytes] data and scales")
        cols = 2 * data.shape[-1] if cols is None else int(cols)
        if cols < 1 or data.shape[-1] != (cols + 1) // 2 or scales.shape != (*data.shape[:-1], (cols + 31) // 32):
            raise ValueError(f"data {tuple(data.shape)} and scales {tuple(scales.shape)} do not fit {cols} columns")
        if scales.device != data.device:
            raise ValueError(f"scales are on {scales.device}, data on {data.device}")
        batched = data.dim() == 3
        d, s = (data, scales) if batched else (data[None], scales[None])
        n, rows, nbytes = d.shape
        ka, rp = _atoms(cols), (rows + 127) // 128 * 128
        packed = d.new_zeros(n, rows, ka * 64)
        packed[..., :nbytes] = d
        if cols % 2:
            packed[..., nbytes - 1] &= 15
        padded = s.new_zeros(n, rp, ka * 4)
        padded[:, :rows, :s.shape[-1]] = s
        sf = padded.view(n, rp // 128, 4, 32, ka, 4).permute(0, 1, 4, 3, 2, 5).reshape(n, rp * ka * 4)
        return MXFP4Matrix(packed, sf.contiguous(), rows, cols, n, batched)

    def to_blocks(self) -> tuple[torch.Tensor, torch.Tensor]:
        """(data, scales) as ``from_blocks`` takes them."""
        n, ka, rp = self.num_matrices, _atoms(self.cols), (self.rows + 127) // 128 * 128
        d = self.data[..., : (self.cols + 1) // 2].contiguous()
        s = self.sf.view(n, rp // 128, ka, 32, 4, 4).permute(0, 1, 4, 3, 2, 5).reshape(n, rp, ka * 4)
        s = s[:, : self.rows, : (self.cols + 31) // 32].contiguous()
        return (d, s) if self.batched else (d[0], s[0])


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(x_rows: int, R: int, n: int, N: int, cols: int, grouped: int, device: int) -> int:
    with torch.cuda.device(device):
        return _lib.lib().mhmoe_mxfp4_workspace_bytes(x_rows, R, n, N, cols, grouped)


def _as(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    return t if t.dtype == dtype and t.is_contiguous() else t.detach().to(dtype).contiguous()


def _quantized_matrix(data, sf, rows, cols, n, batched) -> MXFP4Matrix:
    """An MXFP4Matrix of tensors made here, without the constructor's checks."""
    m = object.__new__(MXFP4Matrix)
    m.data, m.sf, m.rows, m.cols, m.num_matrices, m.batched = data, sf, rows, cols, n, batched
    return m


def _check_rounding(scale_rounding: str) -> int:
    if scale_rounding not in _ROUNDING:
        raise ValueError(f"scale_rounding must be 'floor' or 'ceil', got {scale_rounding!r}")
    return _ROUNDING[scale_rounding]


def _check_float(x: torch.Tensor, name: str) -> None:
    if x.dtype not in _lib.DTYPES:
        raise ValueError(f"{name} must be fp32, bf16 or fp16, got {x.dtype}")


def _check_matrix(w, name: str, device: torch.device | None = None) -> None:
    if not isinstance(w, MXFP4Matrix):
        raise ValueError(f"{name} must be an MXFP4Matrix, got {type(w).__name__}")
    _lib.require_cuda(w.data, w.sf)
    if device is not None and w.device != device:
        raise ValueError(f"{name} is on {w.device}, the activations on {device}")


def mxfp4_quantize(x: torch.Tensor, scale_rounding: str = "floor") -> MXFP4Matrix:
    """MXFP4 form of x [rows, cols] or [n, rows, cols] (fp32, bf16 or fp16; detached).

    Per row and 32 columns with largest magnitude a, the scale is 2^(floor(log2 a) - 2)
    (``floor``: magnitudes above 6 scales saturate) or the smallest power of two with
    a <= 6 scales (``ceil``: nothing saturates); values round to nearest, ties to even.  A block
    that holds NaN or an infinity becomes NaN."""
    rounding = _check_rounding(scale_rounding)
    _check_float(x, "x")
    shape = x.shape
    if len(shape) not in (2, 3) or shape[-1] < 1:
        raise ValueError(f"mxfp4_quantize takes [rows, cols] or [n, rows, cols], got {tuple(shape)}")
    _lib.require_cuda(x)
    rows, cols = shape[-2:]
    if cols > 1 and x.stride(-1) != 1:
        x = x.detach().contiguous()
    batched = len(shape) == 3
    n, sn = (shape[0], x.stride(0)) if batched else (1, 0)
    dev = x.device
    ka = _atoms(cols)
    data = torch.empty((n, rows, ka * 64), dtype=torch.uint8, device=dev)
    sf = torch.empty((n, (rows + 127) // 128 * ka * 512), dtype=torch.uint8, device=dev)
    _lib.launch("mhmoe_mxfp4_quantize", dev, x.data_ptr(), _lib.DTYPES[x.dtype], sn, x.stride(-2), n, rows, cols, rounding,
                data.data_ptr(), sf.data_ptr())
    return _quantized_matrix(data, sf, rows, cols, n, batched)


def mxfp4_dequantize(m: MXFP4Matrix, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values of ``m`` in fp32, bf16 or fp16 (one rounding; exact in fp32, and in bf16 where
    the value does not overflow)."""
    _check_matrix(m, "m")
    if dtype not in _lib.DTYPES:
        raise ValueError(f"dtype must be fp32, bf16 or fp16, got {dtype}")
    dev = m.device
    out = torch.empty(m.shape, dtype=dtype, device=dev)
    _lib.launch("mhmoe_mxfp4_dequantize", dev, m.data.data_ptr(), m.sf.data_ptr(), m.num_matrices, m.rows, m.cols,
                _lib.DTYPES[dtype], out.data_ptr())
    return out


def _product_args(x, bias, activation, n, N, out_dtype, what, row_weights=None, out=None):
    if activation not in _ACTIVATION:
        raise ValueError(f"activation must be None or 'swiglu7', got {activation!r}")
    if activation and N % 2:
        raise ValueError(f"swiglu7 pairs columns: {N} weight rows are odd")
    if out_dtype not in _lib.DTYPES:
        raise ValueError(f"out_dtype must be fp32, bf16 or fp16, got {out_dtype}")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, row_weights, bias, out)):
        raise ValueError(f"{what} has no backward pass: call it under no_grad or detach its inputs")
    if bias is not None:
        if bias.dim() == 0 or bias.numel() != n * N or bias.shape[-1] != N:
            raise ValueError(f"bias must hold {n} x {N} values, got {tuple(bias.shape)}")
        if bias.device != x.device:
            raise ValueError(f"bias is on {bias.device}, the activations on {x.device}")
        if bias.dtype != torch.float32 or not bias.is_contiguous():
            bias = bias.detach().float().contiguous()
    return bias, _ACTIVATION[activation], (N // 2 if activation else N)


def mxfp4_linear(x: torch.Tensor | MXFP4Matrix, weight: MXFP4Matrix, bias: torch.Tensor | None = None,
                 activation: str | None = None, out_dtype: torch.dtype | None = None,
                 scale_rounding: str = "floor") -> torch.Tensor:
    """act(Q(x) W^T + bias) for x [..., cols] and an MXFP4 weight [N, cols].

    x: fp32, bf16 or fp16, quantised per row as ``mxfp4_quantize`` does, or an ``MXFP4Matrix``
    [M, cols].  bias: [N].  ``activation='swiglu7'`` combines column pairs (even gate, odd linear)
    into N/2 outputs: min(g, 7) sigmoid(1.702 min(g, 7)) (clamp(u, -7, 7) + 1).  The result has
    ``out_dtype`` (default: x's type, bf16 for an MXFP4 x)."""
    rounding = _check_rounding(scale_rounding)
    _lib.require_no_tangent("mxfp4_linear", x, bias)
    quantized = isinstance(x, MXFP4Matrix)
    if quantized:
        _check_matrix(x, "x")
        if x.batched:
            raise ValueError("an MXFP4 x must be one matrix [M, cols]")
        lead, cols, ref = (x.rows,), x.cols, x.data
    else:
        _check_float(x, "x")
        if x.dim() < 1:
            raise ValueError("x must be [..., cols]")
        _lib.require_cuda(x)
        lead, cols, ref = tuple(x.shape[:-1]), x.shape[-1], x
    _check_matrix(weight, "weight", ref.device)
    if weight.batched or weight.cols != cols:
        raise ValueError(f"weight {weight.shape} does not fit activations with {cols} columns")
    N = weight.rows
    dtype = out_dtype or (torch.bfloat16 if quantized else x.dtype)
    bias, act, n_out = _product_args(ref, bias, activation, 1, N, dtype, "mxfp4_linear")
    dev = ref.device
    M = x.rows if quantized else (x.numel() // cols if cols else 0)
    y = torch.empty((*lead, n_out), dtype=dtype, device=dev)
    x2, xd, xs, ws, xq, xsf = None, 0, 0, None, None, None
    if quantized:
        xq, xsf = x.data.data_ptr(), x.sf.data_ptr()
    else:
        x2 = x if x.dim() == 2 else x.detach().reshape(M, cols)
        if cols > 1 and x2.stride(1) != 1:
            x2 = x2.detach().contiguous()
        xd, xs = _lib.DTYPES[x.dtype], x2.stride(0)
        nbytes = _workspace_bytes(M, M, 1, N, cols, 0, dev.index)
        if nbytes:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _lib.launch("mhmoe_mxfp4_linear", dev, _lib.ptr(x2), xd, xs, xq, xsf, M, cols, rounding, weight.data.data_ptr(),
                weight.sf.data_ptr(), N, _lib.ptr(bias), act, _lib.ptr(ws), y.data_ptr(), _lib.DTYPES[dtype], n_out,
                _lib.device_status(dev).data_ptr(), 0)
    return y


def mxfp4_expert_linear(x: torch.Tensor, weight: MXFP4Matrix, expert_offsets: torch.Tensor,
                        gather_ids: torch.Tensor | None = None, row_weights: torch.Tensor | None = None,
                        bias: torch.Tensor | None = None, activation: str | None = None,
                        out_dtype: torch.dtype | None = None, scale_rounding: str = "floor",
                        out: torch.Tensor | None = None) -> torch.Tensor:
    """Expert products over rows sorted by expert (``flash_mh_moe_global_sort``'s order):

        y[r] = row_weights[r] * act(Q(x[gather_ids[r]]) W_e^T + bias_e),
        expert_offsets[e] <= r < expert_offsets[e + 1]

    x [T, cols] (fp32, bf16 or fp16); weight [n, N, cols]; expert_offsets int64 (or int32) [n + 1]
    on the device; gather_ids int32 [R] (default: row r of x itself, R = T); row_weights [R]; bias
    [n, N]; activation, out_dtype and scale_rounding as in ``mxfp4_linear``.

    Returns y [R, N] (N/2 with SwiGLU7).  The rows from ``expert_offsets[n]`` on belong to no
    expert: they are 0, or left as they were in ``out`` ([R, N] of the output's type, any row
    stride), which is returned when given.  Offsets outside [0, R] are clipped and a gather id
    outside [0, T) reads as a row of zeros; both record an error that
    ``_lib.check_device_status`` raises."""
    rounding = _check_rounding(scale_rounding)
    _lib.require_no_tangent("mxfp4_expert_linear", x, row_weights, bias, out)
    _check_float(x, "x")
    if x.dim() != 2:
        raise ValueError(f"x must be [T, cols], got {tuple(x.shape)}")
    _lib.require_cuda(x, expert_offsets, gather_ids, row_weights)
    _check_matrix(weight, "weight", x.device)
    T, cols = x.shape
    n, N = weight.num_matrices, weight.rows
    if not weight.batched or weight.cols != cols:
        raise ValueError(f"weight {weight.shape} is not [n, N, {cols}]")
    if tuple(expert_offsets.shape) != (n + 1,):
        raise ValueError(f"expert_offsets must be [{n + 1}], got {tuple(expert_offsets.shape)}")
    if expert_offsets.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"expert_offsets must be int64 or int32, got {expert_offsets.dtype}")
    if gather_ids is not None and (gather_ids.dim() != 1 or gather_ids.dtype != torch.int32):
        raise ValueError(f"gather_ids must be an int32 vector, got {tuple(gather_ids.shape)} {gather_ids.dtype}")
    R = T if gather_ids is None else gather_ids.numel()
    if row_weights is not None and tuple(row_weights.shape) != (R,):
        raise ValueError(f"row_weights must be [{R}], got {tuple(row_weights.shape)}")
    dev = x.device
    for name, t in (("expert_offsets", expert_offsets), ("gather_ids", gather_ids), ("row_weights", row_weights)):
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, x on {dev}")
    dtype = out_dtype or (x.dtype if out is None else out.dtype)
    bias, act, n_out = _product_args(x, bias, activation, n, N, dtype, "mxfp4_expert_linear", row_weights, out)
    if out is not None and (tuple(out.shape) != (R, n_out) or out.dtype != dtype or out.device != dev
                            or (n_out > 1 and out.stride(1) != 1) or (R > 1 and out.stride(0) < n_out)):
        raise ValueError(f"out must be [{R}, {n_out}] {dtype} on {dev} with unit inner stride")
    if cols > 1 and x.stride(1) != 1:
        x = x.detach().contiguous()
    offs = _as(expert_offsets, torch.int64)
    gids = gather_ids if gather_ids is None or gather_ids.is_contiguous() else gather_ids.contiguous()
    rw = None if row_weights is None else _as(row_weights, torch.float32)
    y = torch.empty((R, n_out), dtype=dtype, device=dev) if out is None else out
    ws = torch.empty(max(1, _workspace_bytes(T, R, n, N, cols, 1, dev.index)), dtype=torch.uint8, device=dev)
    _lib.launch("mhmoe_mxfp4_expert_linear", dev, x.data_ptr(), _lib.DTYPES[x.dtype], x.stride(0), T, cols, rounding,
                weight.data.data_ptr(), weight.sf.data_ptr(), n, N, offs.data_ptr(), _lib.ptr(gids), R, _lib.ptr(rw),
                _lib.ptr(bias), act, ws.data_ptr(), y.data_ptr(), _lib.DTYPES[dtype], max(y.stride(0), n_out),
                int(out is None), _lib.device_status(dev).data_ptr(), 0)
    if out is not None:
        torch.autograd.graph.increment_version(out)        # written in place
    return y
