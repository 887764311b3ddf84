"""Microscaled (OCP MX) operators on an MI355X: rows in 4 or 8 bits with one power-of-two scale per 32 columns, the norm that
produces them and the product of such rows with 4-bit weights (include/clipenc.h, `clipenc_op_*_mx`).  Inference only.

    w = quantize(weight)                                              # once: e2m1, 4.25 bits a value
    h, q = norm_quantize(x, gamma, residual=r)                        # h = x + r;  q = rms norm of h, e4m3 in blocks
    y = linear(q, w, bias=b, act="gelu")                              # or linear(x, w): quantises x first

They have no backward pass: with gradients enabled, tensors that require one are refused.  The arithmetic runs in libclipenc_hip.so; there
is no CPU path.  Calls are asynchronous on the current stream of the tensors' device, allocate only what they return (`linear` from
values also a scratch) and may be captured into a graph.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib

FORMATS = {"e2m1": 0, "e4m3": 1, "e4m3_row": 2}
NORMS = {"rms": 0, "layer": 1}
ACTS = {None: -1, "quick_gelu": 0, "gelu": 1}
_BLOCKS = {"e2m1": 0, "e4m3": 1}      # formats of a product's rows
_WEIGHTS = {"e2m1": 0}                # and of its weights
_MAX_ROWS = 1 << 30                   # what the library takes; checked here too, since an int argument keeps the low 32 bits of a larger number
_MAX_COLS = 1 << 20
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


# A call on a few rows costs the host more than the GPU: the checks read each attribute once (is_cuda and get_device instead of a
# device object), and the stream and the allocations take torch's cheaper forms (a raw stream handle, 0.1 us, instead of a Stream
# object, 1.8; empty_strided, 1.3, instead of empty, 1.7).
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_empty = torch.empty_strided
_grad_enabled = torch.is_grad_enabled


def _call(index: int, what: str, fn, *args) -> None:
    """fn(*args, stream) with device `index` current, on its current stream."""
    if index == _current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _lib.check(rc, what)


def _check_no_grad(what: str, *tensors) -> None:
    """None of these operators has a backward pass: a gradient that the caller expects would be lost without a word."""
    if _grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{what} has no backward pass: call it under torch.no_grad(), or with tensors that require no gradient")


def _check_values(what: str, x: torch.Tensor, name: str = "x"):
    """(dtype code, device index, rows, cols, row stride in elements) of a matrix of values whose columns lie side by side."""
    dt, shape = _DTYPES.get(x.dtype), x.shape
    if not x.is_cuda:
        raise _lib.ClipencError(f"{what} needs GPU tensors ('cuda[:i]' under PyTorch-ROCm), got {name} on {x.device}: this build has no CPU path")
    if dt is None:
        raise ValueError(f"{what}: {name} must be bfloat16, float16 or float32, got {x.dtype}")
    if len(shape) != 2 or shape[1] < 1:
        raise ValueError(f"{what}: expected {name} of shape [rows, cols], got {tuple(shape)}")
    rows, cols = shape
    if cols > _MAX_COLS:
        raise ValueError(f"{what}: at most {_MAX_COLS} columns, got {name} of shape {tuple(shape)}")
    ld, step = x.stride()
    if step != 1 and cols > 1:
        raise ValueError(f"{what}: the columns of {name} must lie side by side (stride 1), got strides {x.stride()}")
    if rows <= 1:
        ld = cols
    elif ld < cols:
        raise ValueError(f"{what}: the rows of {name} overlap (strides {x.stride()})")
    return dt, x.get_device(), rows, cols, ld


def _check_quantised(what: str, q: MXTensor, formats, name: str):
    """(format code, device index, rows, cols) of a quantised matrix."""
    data, scale, fmt, cols = q
    code = formats.get(fmt)
    if code is None:
        raise ValueError(f"{what}: {name} must be one of {sorted(formats)}, got {fmt!r}")
    if not 1 <= cols <= _MAX_COLS:
        raise ValueError(f"{what}: {name} has {cols} columns (1 .. {_MAX_COLS})")
    kp = (cols + 127) // 128 * 128
    shape = data.shape
    rows = shape[0] if len(shape) == 2 else -1
    want, kind = ((rows, kp // 32), torch.uint8) if code != 2 else ((rows,), torch.float32)
    row_bytes = kp if code else kp // 2
    if rows < 0 or shape[1] != row_bytes or data.dtype is not torch.uint8 or scale.dtype is not kind or scale.shape != want:
        raise ValueError(f"{what}: {name} of {cols} columns in {fmt} needs uint8 data of {row_bytes} bytes a row and {kind} scales {want}, "
                         f"got {data.dtype} {tuple(shape)} and {scale.dtype} {tuple(scale.shape)}")
    if not (data.is_contiguous() and scale.is_contiguous()):
        raise ValueError(f"{what}: {name} must be contiguous")
    if not data.is_cuda:
        raise _lib.ClipencError(f"{what} needs GPU tensors, got {name} on {data.device}: this build has no CPU path")
    index = data.get_device()
    if scale.get_device() != index:
        raise ValueError(f"{what}: the data of {name} is on {data.device}, its scales on {scale.device}")
    return code, index, rows, cols


def _check_vector(what: str, v: Optional[torch.Tensor], n: int, index: int, name: str) -> Optional[int]:
    if v is None:
        return None
    if v.dtype is not torch.float32 or v.shape != (n,) or not v.is_contiguous():
        raise ValueError(f"{what}: {name} must be a contiguous float32 [{n}], got {v.dtype} {tuple(v.shape)}")
    if v.get_device() != index:
        raise ValueError(f"{what}: all tensors must be on cuda:{index}, got {name} on {v.device}")
    return v.data_ptr()


def _new(rows: int, cols: int, fmt: str, device: torch.device) -> MXTensor:
    kp = (cols + 127) // 128 * 128
    width = kp // 2 if fmt == "e2m1" else kp
    data = _empty((rows, width), (width, 1), dtype=torch.uint8, device=device)
    if fmt == "e4m3_row":
        return MXTensor(data, _empty((rows,), (1,), dtype=torch.float32, device=device), fmt, cols)
    kp //= 32
    return MXTensor(data, _empty((rows, kp), (kp, 1), dtype=torch.uint8, device=device), fmt, cols)


def quantize(x: torch.Tensor, fmt: str = "e2m1") -> MXTensor:
    """The rows of x [rows, cols] (bf16 / fp16 / fp32, rows may be strided) in blocks of 32 columns: fmt "e2m1" or "e4m3"."""
    code = _BLOCKS.get(fmt)
    if code is None:
        raise ValueError(f"quantize: fmt must be 'e2m1' or 'e4m3', got {fmt!r}")
    _check_no_grad("quantize", x)
    dt, index, rows, cols, ld = _check_values("quantize", x)
    q = _new(rows, cols, fmt, x.device)
    _call(index, "quantize", _lib.load().clipenc_op_quant_mx, x.data_ptr(), dt, rows, cols, ld, code, q[0].data_ptr(), q[1].data_ptr())
    return q


def dequantize(q: MXTensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values [rows, cols] that q stands for."""
    out_dt = _DTYPES.get(dtype)
    if out_dt is None:
        raise ValueError(f"dequantize: dtype must be bfloat16, float16 or float32, got {dtype}")
    _check_no_grad("dequantize", q[1])                              # (a row's scale may be any float32 tensor)
    code, index, rows, cols = _check_quantised("dequantize", q, FORMATS, "q")
    data = q[0]
    out = _empty((rows, cols), (cols, 1), dtype=dtype, device=data.device)
    _call(index, "dequantize", _lib.load().clipenc_op_dequant_mx, data.data_ptr(), q[1].data_ptr(), code, rows, cols, out.data_ptr(), out_dt)
    return out


def norm_quantize(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
                  norm: str = "rms", eps: float = 1e-6, fmt: str = "e4m3") -> Tuple[torch.Tensor, MXTensor]:
    """(h, q): h = x + residual (x itself without one), q = its norm ("rms" or "layer") times `weight` plus `bias`, quantised to fmt:
    "e4m3" / "e2m1" in blocks, or "e4m3_row" with one scale a row.  x, residual: [rows, cols] of one type; weight, bias: float32."""
    what = "norm_quantize"
    kind, code = NORMS.get(norm), FORMATS.get(fmt)
    if kind is None or code is None:
        raise ValueError(f"{what}: norm must be one of {sorted(NORMS)} and fmt one of {sorted(FORMATS)}, got {norm!r}, {fmt!r}")
    _check_no_grad(what, x, weight, bias, residual)
    dt, index, rows, cols, ld = _check_values(what, x)
    device = x.device
    r = hp = None
    ld_r, h = 0, x
    if residual is not None:
        dt_r, index_r, rows_r, cols_r, ld_r = _check_values(what, residual, "residual")
        if dt_r != dt or rows_r != rows or cols_r != cols or index_r != index:
            raise ValueError(f"{what}: residual must be {x.dtype} {tuple(x.shape)} on {device}, got {residual.dtype} {tuple(residual.shape)} on {residual.device}")
        h = _empty((rows, cols), (cols, 1), dtype=x.dtype, device=device)
        r, hp = residual.data_ptr(), h.data_ptr()
    if weight is None:
        raise ValueError(f"{what}: weight is needed")
    g = _check_vector(what, weight, cols, index, "weight")
    b = None if bias is None else _check_vector(what, bias, cols, index, "bias")
    q = _new(rows, cols, fmt, device)
    _call(index, what, _lib.load().clipenc_op_norm_quant_mx, x.data_ptr(), dt, rows, cols, ld, r, ld_r, kind, g, b, eps, code, hp, q[0].data_ptr(),
          q[1].data_ptr())
    return h, q


def linear(x, w: MXTensor, bias: Optional[torch.Tensor] = None, act: Optional[str] = None, residual: Optional[torch.Tensor] = None,
           out_dtype: Optional[torch.dtype] = None, x_fmt: str = "e4m3") -> torch.Tensor:
    """act(x . w^T + bias) + residual, [rows, out], summed in fp32 and rounded once.  x: an MXTensor ("e4m3" or "e2m1") or values
    [rows, cols], which are quantised to x_fmt first; w: e2m1 [out, cols]; bias float32 [out]; act None, "quick_gelu" or "gelu" (erf),
    not together with a residual; residual [rows, out] of out_dtype (default: the values' type, bf16 for an MXTensor)."""
    what = "linear"
    act_code = ACTS.get(act)
    if act_code is None:
        raise ValueError(f"{what}: act must be None, 'quick_gelu' or 'gelu', got {act!r}")
    if residual is not None and act is not None:
        raise ValueError(f"{what}: activation and residual are exclusive")
    coded = isinstance(x, MXTensor)
    _check_no_grad(what, None if coded else x, bias, residual)
    _, index, n, w_cols = _check_quantised(what, w, _WEIGHTS, "w")
    if coded:
        fmt, x_index, rows, cols = _check_quantised(what, x, _BLOCKS, "x")
    else:
        fmt = _BLOCKS.get(x_fmt)
        if fmt is None:
            raise ValueError(f"{what}: x_fmt must be 'e2m1' or 'e4m3', got {x_fmt!r}")
        dt, x_index, rows, cols, ld = _check_values(what, x)
    if rows > _MAX_ROWS or n > _MAX_ROWS:
        raise ValueError(f"{what}: at most {_MAX_ROWS} rows of x and of w, got {rows} and {n}")
    if x_index != index or cols != w_cols:
        raise ValueError(f"{what}: x has {cols} columns on cuda:{x_index} and w {w_cols} on cuda:{index}")
    if out_dtype is None:
        out_dtype = torch.bfloat16 if coded else x.dtype
    out_dt = _DTYPES.get(out_dtype)
    if out_dt is None:
        raise ValueError(f"{what}: out_dtype must be bfloat16, float16 or float32, got {out_dtype}")
    b = None if bias is None else _check_vector(what, bias, n, index, "bias")
    r = None
    if residual is not None:
        if residual.dtype is not out_dtype or residual.shape != (rows, n) or not residual.is_contiguous() or residual.get_device() != index:
            raise ValueError(f"{what}: residual must be a contiguous {out_dtype} [{rows}, {n}] on cuda:{index}, got {residual.dtype} {tuple(residual.shape)} on "
                             f"{residual.device}")
        r = residual.data_ptr()
    lib = _lib.load()
    w_data = w[0]
    device = w_data.device
    out = _empty((rows, n), (n, 1), dtype=out_dtype, device=device)
    if coded:
        _call(index, what, lib.clipenc_op_gemm_mx, x[0].data_ptr(), x[1].data_ptr(), fmt, w_data.data_ptr(), w[1].data_ptr(), rows, n, cols, b, act_code, r,
              out.data_ptr(), out_dt)
        return out
    ws = None
    need = lib.clipenc_op_linear_mx_ws_bytes(rows, n, cols, fmt)
    if need:
        scratch = _empty((need,), (1,), dtype=torch.uint8, device=device)
        ws = scratch.data_ptr()
    _call(index, what, lib.clipenc_op_linear_mx, x.data_ptr(), dt, ld, fmt, w_data.data_ptr(), w[1].data_ptr(), rows, n, cols, b, act_code, r, out.data_ptr(),
          out_dt, ws, need)
    return out
