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


# A call on a few rows costs the host more than the GPU, so the checks below read each attribute once and the stream and the
# allocations take torch's cheaper forms (a raw stream handle instead of a Stream object, 0.1 against 1.8 us; empty_strided).
def _stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


def _on_device(index: int):
    """A guard for work on another device than the current one, None where it is the current one."""
    return None if index == torch.cuda.current_device() else torch.cuda.device(index)


def _run(device: torch.device, what: str, fn, *args) -> None:
    """fn(*args, stream) on `device`."""
    guard = _on_device(device.index)
    if guard is None:
        rc = fn(*args, _stream(device))
    else:
        with guard:
            rc = fn(*args, _stream(device))
    if rc:
        _lib.check(rc, what)


def _check_values(what: str, x: torch.Tensor, name: str = "x"):
    """(dtype code, device, rows, cols, row stride in elements) of a matrix of values whose columns lie side by side."""
    device = x.device
    if device.type != "cuda":
        raise _lib.ClipencError(f"{what} needs GPU tensors ('cuda[:i]' under PyTorch-ROCm), got {name} on {device}: this build has no CPU path")
    dt = _DTYPES.get(x.dtype)
    if dt is None:
        raise ValueError(f"{what}: {name} must be bfloat16, float16 or float32, got {x.dtype}")
    shape = x.shape
    if len(shape) != 2 or shape[1] < 1:
        raise ValueError(f"{what}: expected {name} of shape [rows, cols], got {tuple(shape)}")
    rows, cols = shape
    ld, step = x.stride()
    if step != 1 and cols > 1:
        raise ValueError(f"{what}: the columns of {name} must lie side by side (stride 1), got strides {x.stride()}")
    if rows <= 1:
        ld = cols
    elif ld < cols:
        raise ValueError(f"{what}: the rows of {name} overlap (strides {x.stride()})")
    return dt, device, rows, cols, ld


def _check_quantised(what: str, q: MXTensor, formats, name: str):
    """(format code, device, rows, cols) of a quantised matrix."""
    data, scale, fmt, cols = q
    if fmt not in formats:
        raise ValueError(f"{what}: {name} must be one of {sorted(formats)}, got {fmt!r}")
    kp = (cols + 127) // 128 * 128
    shape, device = data.shape, data.device
    rows = shape[0] if len(shape) == 2 else -1
    row_bytes = kp // 2 if fmt == "e2m1" else kp
    want, kind = ((rows,), torch.float32) if fmt == "e4m3_row" else ((rows, kp // 32), torch.uint8)
    if cols < 1 or rows < 0 or shape[1] != row_bytes or data.dtype is not torch.uint8 or scale.dtype is not kind or scale.shape != want:
        raise ValueError(f"{what}: {name} of {cols} columns in {fmt} needs uint8 data of {row_bytes} bytes a row and {kind} scales {want}, "
                         f"got {data.dtype} {tuple(shape)} and {scale.dtype} {tuple(scale.shape)}")
    if not (data.is_contiguous() and scale.is_contiguous()):
        raise ValueError(f"{what}: {name} must be contiguous")
    if device.type != "cuda":
        raise _lib.ClipencError(f"{what} needs GPU tensors, got {name} on {device}: this build has no CPU path")
    if scale.device != device:
        raise ValueError(f"{what}: the data of {name} is on {device}, its scales on {scale.device}")
    return FORMATS[fmt], device, rows, cols


def _check_vector(what: str, v: Optional[torch.Tensor], n: int, device: torch.device, name: str) -> Optional[int]:
    if v is None:
        return None
    if v.dtype is not torch.float32 or v.shape != (n,) or not v.is_contiguous():
        raise ValueError(f"{what}: {name} must be a contiguous float32 [{n}], got {v.dtype} {tuple(v.shape)}")
    if v.device != device:
        raise ValueError(f"{what}: all tensors must be on {device}, got {name} on {v.device}")
    return v.data_ptr()


def _matrix(rows: int, cols: int, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    return torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=device)


def _new(rows: int, cols: int, fmt: str, device: torch.device) -> MXTensor:
    kp = (cols + 127) // 128 * 128
    data = _matrix(rows, kp // 2 if fmt == "e2m1" else kp, torch.uint8, device)
    if fmt == "e4m3_row":
        return MXTensor(data, torch.empty_strided((rows,), (1,), dtype=torch.float32, device=device), fmt, cols)
    return MXTensor(data, _matrix(rows, kp // 32, torch.uint8, device), fmt, cols)


def quantize(x: torch.Tensor, fmt: str = "e2m1") -> MXTensor:
    """The rows of x [rows, cols] (bf16 / fp16 / fp32, rows may be strided) in blocks of 32 columns: fmt "e2m1" or "e4m3"."""
    if fmt != "e2m1" and fmt != "e4m3":
        raise ValueError(f"quantize: fmt must be 'e2m1' or 'e4m3', got {fmt!r}")
    dt, device, rows, cols, ld = _check_values("quantize", x)
    q = _new(rows, cols, fmt, device)
    _run(device, "quantize", _lib.load().clipenc_op_quant_mx, x.data_ptr(), dt, rows, cols, ld, FORMATS[fmt], q.data.data_ptr(), q.scale.data_ptr())
    return q


def dequantize(q: MXTensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values [rows, cols] that q stands for."""
    out_dt = _DTYPES.get(dtype)
    if out_dt is None:
        raise ValueError(f"dequantize: dtype must be bfloat16, float16 or float32, got {dtype}")
    fmt, device, rows, cols = _check_quantised("dequantize", q, FORMATS, "q")
    out = _matrix(rows, cols, dtype, device)
    _run(device, "dequantize", _lib.load().clipenc_op_dequant_mx, q.data.data_ptr(), q.scale.data_ptr(), fmt, rows, cols, out.data_ptr(), out_dt)
    return out


def norm_quantize(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
                  norm: str = "rms", eps: float = 1e-6, fmt: str = "e4m3") -> Tuple[torch.Tensor, MXTensor]:
    """(h, q): h = x + residual (x itself without one), q = its norm ("rms" or "layer") times `weight` plus `bias`, quantised to fmt:
    "e4m3" / "e2m1" in blocks, or "e4m3_row" with one scale a row.  x, residual: [rows, cols] of one type; weight, bias: float32."""
    what = "norm_quantize"
    if norm not in NORMS or fmt not in FORMATS:
        raise ValueError(f"{what}: norm must be one of {sorted(NORMS)} and fmt one of {sorted(FORMATS)}, got {norm!r}, {fmt!r}")
    dt, device, rows, cols, ld = _check_values(what, x)
    r = hp = None
    ld_r, h = 0, x
    if residual is not None:
        if residual.shape != x.shape or residual.dtype is not x.dtype or residual.device != device:
            raise ValueError(f"{what}: residual must be {x.dtype} {tuple(x.shape)} on {device}, got {residual.dtype} {tuple(residual.shape)} on {residual.device}")
        ld_r = _check_values(what, residual, "residual")[4]
        h = _matrix(rows, cols, x.dtype, device)
        r, hp = residual.data_ptr(), h.data_ptr()
    if weight is None:
        raise ValueError(f"{what}: weight is needed")
    g, b = _check_vector(what, weight, cols, device, "weight"), _check_vector(what, bias, cols, device, "bias")
    q = _new(rows, cols, fmt, device)
    _run(device, what, _lib.load().clipenc_op_norm_quant_mx, x.data_ptr(), dt, rows, cols, ld, r, ld_r, NORMS[norm], g, b, eps, FORMATS[fmt], hp,
         q.data.data_ptr(), q.scale.data_ptr())
    return h, q


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
    _, device, n, w_cols = _check_quantised(what, w, ("e2m1",), "w")
    coded = isinstance(x, MXTensor)
    if coded:
        fmt, x_device, rows, cols = _check_quantised(what, x, ("e2m1", "e4m3"), "x")
    else:
        if x_fmt != "e2m1" and x_fmt != "e4m3":
            raise ValueError(f"{what}: x_fmt must be 'e2m1' or 'e4m3', got {x_fmt!r}")
        fmt = FORMATS[x_fmt]
        dt, x_device, rows, cols, ld = _check_values(what, x)
    if x_device != device:
        raise ValueError(f"{what}: x is on {x_device} and w on {device}")
    if cols != w_cols:
        raise ValueError(f"{what}: x has {cols} columns and w {w_cols}")
    if out_dtype is None:
        out_dtype = torch.bfloat16 if coded else x.dtype
    out_dt = _DTYPES.get(out_dtype)
    if out_dt is None:
        raise ValueError(f"{what}: out_dtype must be bfloat16, float16 or float32, got {out_dtype}")
    b, r = _check_vector(what, bias, n, device, "bias"), None
    if residual is not None:
        if residual.dtype is not out_dtype or residual.shape != (rows, n) or not residual.is_contiguous() or residual.device != device:
            raise ValueError(f"{what}: residual must be a contiguous {out_dtype} [{rows}, {n}] on {device}, got {residual.dtype} {tuple(residual.shape)} on {residual.device}")
        r = residual.data_ptr()
    lib = _lib.load()
    out = _matrix(rows, n, out_dtype, device)
    if coded:
        _run(device, what, lib.clipenc_op_gemm_mx, x.data.data_ptr(), x.scale.data_ptr(), fmt, w.data.data_ptr(), w.scale.data_ptr(), rows, n, cols, b,
             ACTS[act], r, out.data_ptr(), out_dt)
    else:
        need = lib.clipenc_op_linear_mx_ws_bytes(rows, cols, fmt)
        ws = torch.empty_strided((need,), (1,), dtype=torch.uint8, device=device) if need else None
        _run(device, what, lib.clipenc_op_linear_mx, x.data_ptr(), dt, ld, fmt, w.data.data_ptr(), w.scale.data_ptr(), rows, n, cols, b, ACTS[act], r,
             out.data_ptr(), out_dt, ws.data_ptr() if need else None, need)
    return out
