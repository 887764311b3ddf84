"""Microscaled (OCP MX) operators on an MI355X: rows in 4 or 8 bits with one power-of-two scale per 32 columns, the norm that
produces them and the product of such rows with 4-bit weights (include/clipenc.h, `clipenc_op_*_mx`).  Inference only.

    w = quantize(weight)                                              # once: e2m1, 4.25 bits a value
    h, q = norm_quantize(x, gamma, residual=r)                        # h = x + r;  q = rms norm of h, e4m3 in blocks
    y = linear(q, w, bias=b, act="gelu")                              # or linear(x, w): quantises x first

The arithmetic runs in libclipenc_hip.so; there is no CPU path.  Calls are asynchronous on the current stream of the tensors'
device, allocate only what they return (`linear` from values also a scratch) and may be captured into a graph.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib

FORMATS = {"e2m1": 0, "e4m3": 1, "e4m3_row": 2}
NORMS = {"rms": 0, "layer": 1}
ACTS = {None: -1, "quick_gelu": 0, "gelu": 1}
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


class MXTensor(NamedTuple):
    """A quantised [rows, cols] matrix.  `data`: uint8 [rows, kp / 2] (e2m1, the lower column in the low half of a byte) or [rows, kp]
    (e4m3), kp = cols rounded up to 128, the added columns zero; `scale`: uint8 [rows, kp / 32], biased exponents (0xff: NaN).
    fmt "e4m3_row": e4m3 data with `scale` float32 [rows]."""
    data: torch.Tensor
    scale: torch.Tensor
    fmt: str
    cols: int

    @property
    def shape(self) -> Tuple[int, int]:
        return self.data.shape[0], self.cols


def _padded(cols: int) -> int:
    return (cols + 127) // 128 * 128


def _row_bytes(cols: int, fmt: str) -> int:
    return _padded(cols) // 2 if fmt == "e2m1" else _padded(cols)


def _check_values(what: str, x: torch.Tensor, name: str = "x"):
    """(dtype code, row stride in elements) of a [rows, cols] matrix of values whose columns lie side by side."""
    if x.device.type != "cuda":
        raise _lib.ClipencError(f"{what} needs GPU tensors ('cuda[:i]' under PyTorch-ROCm), got {name} on {x.device}: this build has no CPU path")
    if x.dtype not in _DTYPES:
        raise ValueError(f"{what}: {name} must be bfloat16, float16 or float32, got {x.dtype}")
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"{what}: expected {name} of shape [rows, cols], got {tuple(x.shape)}")
    rows, cols = x.shape
    if cols > 1 and x.stride(1) != 1:
        raise ValueError(f"{what}: the columns of {name} must lie side by side (stride 1), got strides {x.stride()}")
    ld = x.stride(0) if rows > 1 else cols
    if ld < cols:
        raise ValueError(f"{what}: the rows of {name} overlap (strides {x.stride()})")
    return _DTYPES[x.dtype], ld


def _check_quantised(what: str, q: MXTensor, formats, name: str) -> None:
    if q.fmt not in formats:
        raise ValueError(f"{what}: {name} must be one of {sorted(formats)}, got {q.fmt!r}")
    rows, cols = q.data.shape[0], q.cols
    if cols < 1:
        raise ValueError(f"{what}: {name} has {cols} columns")
    want = (rows,) if q.fmt == "e4m3_row" else (rows, _padded(cols) // 32)
    kind = torch.float32 if q.fmt == "e4m3_row" else torch.uint8
    if q.data.dtype != torch.uint8 or tuple(q.data.shape) != (rows, _row_bytes(cols, q.fmt)) or q.scale.dtype != kind or tuple(q.scale.shape) != want:
        raise ValueError(f"{what}: {name} of {cols} columns in {q.fmt} needs uint8 data of {_row_bytes(cols, q.fmt)} bytes a row and {kind} scales "
                         f"{want}, got {q.data.dtype} {tuple(q.data.shape)} and {q.scale.dtype} {tuple(q.scale.shape)}")
    if not (q.data.is_contiguous() and q.scale.is_contiguous()):
        raise ValueError(f"{what}: {name} must be contiguous")
    if q.data.device.type != "cuda":
        raise _lib.ClipencError(f"{what} needs GPU tensors, got {name} on {q.data.device}: this build has no CPU path")


def _check_vector(what: str, v: Optional[torch.Tensor], n: int, name: str) -> Optional[int]:
    if v is None:
        return None
    if v.dtype != torch.float32 or tuple(v.shape) != (n,) or not v.is_contiguous():
        raise ValueError(f"{what}: {name} must be a contiguous float32 [{n}], got {v.dtype} {tuple(v.shape)}")
    return v.data_ptr()


def _one_device(what: str, device: torch.device, *tensors) -> None:
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"{what}: all tensors must be on {device}, got one on {t.device}")


def _new(rows: int, cols: int, fmt: str, device) -> MXTensor:
    data = torch.empty((rows, _row_bytes(cols, fmt)), dtype=torch.uint8, device=device)
    if fmt == "e4m3_row":
        return MXTensor(data, torch.empty((rows,), dtype=torch.float32, device=device), fmt, cols)
    return MXTensor(data, torch.empty((rows, _padded(cols) // 32), dtype=torch.uint8, device=device), fmt, cols)


@torch.no_grad()
def quantize(x: torch.Tensor, fmt: str = "e2m1") -> MXTensor:
    """The rows of x [rows, cols] (bf16 / fp16 / fp32, rows may be strided) in blocks of 32 columns: fmt "e2m1" or "e4m3"."""
    if fmt not in ("e2m1", "e4m3"):
        raise ValueError(f"quantize: fmt must be 'e2m1' or 'e4m3', got {fmt!r}")
    dt, ld = _check_values("quantize", x)
    rows, cols = x.shape
    lib = _lib.load()
    with torch.cuda.device(x.device):
        q = _new(rows, cols, fmt, x.device)
        _lib.check(lib.clipenc_op_quant_mx(x.data_ptr(), dt, rows, cols, ld, FORMATS[fmt], q.data.data_ptr(), q.scale.data_ptr(),
                                           _lib.current_stream_ptr(x.device)), "quantize")
    return q


@torch.no_grad()
def dequantize(q: MXTensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values [rows, cols] that q stands for."""
    if dtype not in _DTYPES:
        raise ValueError(f"dequantize: dtype must be bfloat16, float16 or float32, got {dtype}")
    _check_quantised("dequantize", q, FORMATS, "q")
    device = q.data.device
    _one_device("dequantize", device, q.scale)
    rows, cols = q.shape
    lib = _lib.load()
    with torch.cuda.device(device):
        out = torch.empty((rows, cols), dtype=dtype, device=device)
        _lib.check(lib.clipenc_op_dequant_mx(q.data.data_ptr(), q.scale.data_ptr(), FORMATS[q.fmt], rows, cols, out.data_ptr(), _DTYPES[dtype],
                                             _lib.current_stream_ptr(device)), "dequantize")
    return out


@torch.no_grad()
def norm_quantize(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
                  norm: str = "rms", eps: float = 1e-6, fmt: str = "e4m3") -> Tuple[torch.Tensor, MXTensor]:
    """(h, q): h = x + residual (x itself without one), q = its norm ("rms" or "layer") times `weight` plus `bias`, quantised to fmt:
    "e4m3" / "e2m1" in blocks, or "e4m3_row" with one scale a row.  x, residual: [rows, cols] of one type; weight, bias: float32."""
    what = "norm_quantize"
    if norm not in NORMS or fmt not in FORMATS:
        raise ValueError(f"{what}: norm must be one of {sorted(NORMS)} and fmt one of {sorted(FORMATS)}, got {norm!r}, {fmt!r}")
    dt, ld = _check_values(what, x)
    rows, cols = x.shape
    ld_r = 0
    if residual is not None:
        dt_r, ld_r = _check_values(what, residual, "residual")
        if residual.shape != x.shape or dt_r != dt:
            raise ValueError(f"{what}: residual must be {x.dtype} {tuple(x.shape)}, got {residual.dtype} {tuple(residual.shape)}")
    if weight is None:
        raise ValueError(f"{what}: weight is needed")
    g, b = _check_vector(what, weight, cols, "weight"), _check_vector(what, bias, cols, "bias")
    _one_device(what, x.device, weight, bias, residual)
    lib = _lib.load()
    with torch.cuda.device(x.device):
        h = x if residual is None else torch.empty((rows, cols), dtype=x.dtype, device=x.device)
        q = _new(rows, cols, fmt, x.device)
        _lib.check(lib.clipenc_op_norm_quant_mx(x.data_ptr(), dt, rows, cols, ld, None if residual is None else residual.data_ptr(), ld_r,
                                                NORMS[norm], g, b, eps, FORMATS[fmt], None if residual is None else h.data_ptr(),
                                                q.data.data_ptr(), q.scale.data_ptr(), _lib.current_stream_ptr(x.device)), what)
    return h, q


@torch.no_grad()
def linear(x, w: MXTensor, bias: Optional[torch.Tensor] = None, act: Optional[str] = None, residual: Optional[torch.Tensor] = None,
           out_dtype: Optional[torch.dtype] = None, x_fmt: str = "e4m3") -> torch.Tensor:
    """act(x . w^T + bias) + residual, [rows, out].  x: an MXTensor ("e4m3" or "e2m1") or values [rows, cols], which are quantised to
    x_fmt first; w: e2m1 [out, cols]; bias float32 [out]; act None, "quick_gelu" or "gelu" (erf), not together with a residual;
    residual [rows, out] of out_dtype (default: the values' type, bf16 for an MXTensor)."""
    what = "linear"
    if act not in ACTS:
        raise ValueError(f"{what}: act must be None, 'quick_gelu' or 'gelu', got {act!r}")
    if act is not None and residual is not None:
        raise ValueError(f"{what}: activation and residual are exclusive")
    _check_quantised(what, w, ("e2m1",), "w")
    coded = isinstance(x, MXTensor)
    if coded:
        _check_quantised(what, x, ("e2m1", "e4m3"), "x")
        device = x.data.device
    else:
        if x_fmt not in ("e2m1", "e4m3"):
            raise ValueError(f"{what}: x_fmt must be 'e2m1' or 'e4m3', got {x_fmt!r}")
        dt, ld = _check_values(what, x)
        device = x.device
    rows, cols = x.shape
    n = w.data.shape[0]
    if cols != w.cols:
        raise ValueError(f"{what}: x has {cols} columns and w {w.cols}")
    out_dtype = out_dtype or (torch.bfloat16 if coded else x.dtype)
    if out_dtype not in _DTYPES:
        raise ValueError(f"{what}: out_dtype must be bfloat16, float16 or float32, got {out_dtype}")
    b = _check_vector(what, bias, n, "bias")
    if residual is not None and (residual.dtype != out_dtype or tuple(residual.shape) != (rows, n) or not residual.is_contiguous()):
        raise ValueError(f"{what}: residual must be a contiguous {out_dtype} [{rows}, {n}], got {residual.dtype} {tuple(residual.shape)}")
    _one_device(what, device, w.data, w.scale, bias, residual, *((x.scale,) if coded else ()))
    r = None if residual is None else residual.data_ptr()
    lib = _lib.load()
    with torch.cuda.device(device):
        out = torch.empty((rows, n), dtype=out_dtype, device=device)
        stream = _lib.current_stream_ptr(device)
        if coded:
            _lib.check(lib.clipenc_op_gemm_mx(x.data.data_ptr(), x.scale.data_ptr(), FORMATS[x.fmt], w.data.data_ptr(), w.scale.data_ptr(), rows, n,
                                              cols, b, ACTS[act], r, out.data_ptr(), _DTYPES[out_dtype], stream), what)
        else:
            need = lib.clipenc_op_linear_mx_ws_bytes(rows, cols, FORMATS[x_fmt])
            ws = torch.empty((need,), dtype=torch.uint8, device=device) if need else None
            _lib.check(lib.clipenc_op_linear_mx(x.data_ptr(), dt, ld, FORMATS[x_fmt], w.data.data_ptr(), w.scale.data_ptr(), rows, n, cols, b,
                                                ACTS[act], r, out.data_ptr(), _DTYPES[out_dtype], None if ws is None else ws.data_ptr(), need,
                                                stream), what)
    return out
