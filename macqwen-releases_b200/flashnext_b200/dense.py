"""Norms, 8-bit rows and matrix products: the dense steps around the block.

* :func:`add_rms_norm` adds the residual and normalises rows, and writes them
  in their own type, in 8 bits with a scale a row, or both, in one pass;
* :func:`quantize_rows` / :func:`dequantize_rows` take rows to 8 bits (an
  attention's output, a weight when it is laid out) and back;
* :func:`linear` is ``act(x W^T + bias) + residual`` for bfloat16 rows and
  weights, or for 8-bit ones with a scale a row.

A decode step runs them around :class:`~flashnext_b200.moe_block.SparseMoEBlock`
and :class:`~flashnext_b200.paged_q8.PagedKVCacheQ8`, and ends in
:func:`~flashnext_b200.sampling.sample`.  Every call is ordered on torch's
current stream, needs no workspace and reads nothing on the host, so a step can
be captured in a CUDA graph.  Rows may be slices of wider ones.  Forward only.
"""
from __future__ import annotations

from typing import Any, NamedTuple

import torch

from . import _lib
from .paged_q8 import _elsewhere, _want

_FLOATS = {torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32}
_CODES = {torch.int8: _lib.Q8_INT8, torch.float8_e4m3fn: _lib.Q8_E4M3}
_LINEAR = {torch.bfloat16: _lib.LINEAR_BF16, torch.int8: _lib.LINEAR_INT8, torch.float8_e4m3fn: _lib.LINEAR_E4M3}
_FLT_MAX = 3.4028234663852886e38
ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2, "relu": 3}


class NormedRows(NamedTuple):
    """What :func:`add_rms_norm` was asked for; the rest is None."""

    y: Any         # [rows, dim] in x's type
    residual: Any  # [rows, dim] x + residual, in the residual's type
    codes: Any     # [rows, dim] int8 or float8_e4m3fn
    scales: Any    # [rows] float32


def _float(t, what):
    """FNMOE_DTYPE_* of a bfloat16 or float32 tensor."""
    d = _FLOATS.get(t.dtype)
    if d is None:
        raise TypeError(f"{what} must be a bfloat16 or float32 tensor, not {t.dtype}")
    return d


def _matrix(t, what, index):
    """Pointer, rows, columns and row stride of a matrix on CUDA device ``index`` whose rows are contiguous."""
    shape = t.shape
    if len(shape) == 2 and t.get_device() == index >= 0:
        rows, dim = shape
        if t.is_contiguous():
            return t.data_ptr(), rows, dim, dim
        s0, s1 = t.stride()
        if (s1 == 1 or dim < 2) and (s0 >= dim or rows < 2):
            return t.data_ptr(), rows, dim, s0 if rows > 1 else dim
    # say what is wrong
    if len(shape) != 2:
        raise ValueError(f"{what} must have two dimensions, not {tuple(shape)}")
    if not t.is_cuda:
        raise TypeError(f"{what} must be a CUDA tensor")
    if t.get_device() != index:
        _elsewhere(t, index, what)
    if s1 != 1 and dim > 1:
        raise ValueError(f"{what}'s rows must be contiguous")
    raise ValueError(f"{what}'s rows overlap")


def _same(t, rows, dim, what, index):
    p, r, d, stride = _matrix(t, what, index)
    if r != rows or d != dim:
        raise ValueError(f"{what} has shape {(r, d)}, not {(rows, dim)}")
    return p, stride


def _new(rows, dim, dtype, like):
    """A new contiguous matrix on ``like``'s device (the cheapest of torch's ways to make one)."""
    return torch.empty_strided((rows, dim), (dim, 1), dtype=dtype, device=like.device)


def _ready_stream(index):
    """The current stream of CUDA device ``index``, which must be the current one, with the library started up."""
    if torch._C._cuda_getDevice() != index or not _lib._available.get(index):
        _lib.ensure_device_of(index)  # refuses, or starts the library up
    return torch._C._cuda_getCurrentRawStream(index)


def add_rms_norm(x, weight, residual=None, eps: float = 1e-6, *, unit_offset: bool = False, codes=None,
                 keep: bool | None = None, residual_out=None) -> NormedRows:
    """``y = s / sqrt(mean(s^2) + eps) * weight`` with ``s = x + residual``, row by row.

    ``x`` [rows, dim] and ``residual`` (or None) are bfloat16 or float32 each,
    ``weight`` [dim] either (``unit_offset``: kept as w - 1).  With a residual,
    ``s`` comes back in its type, in a new tensor or in ``residual_out`` (which
    may be ``residual``); the norm sees the unrounded sum.  ``codes``
    (torch.int8 or torch.float8_e4m3fn) asks for y in 8 bits with one float32
    scale a row, max|y| over the code type's largest value; ``keep`` says
    whether y comes back as well, in x's type (by default when no codes are
    asked for).  A row that is not finite gets NaN as its scale.  ``dim`` is at
    most 16384.
    """
    index, dtype = x.get_device(), x.dtype
    xd = _FLOATS.get(dtype)
    if xd is None:
        xd = _float(x, "x")
    xp, rows, dim, xs = _matrix(x, "x", index)
    wd = _FLOATS.get(weight.dtype)
    if wd is None:
        wd = _float(weight, "weight")
    wp = _want(weight, weight.dtype, (dim,), "weight", index)
    if keep is None:
        keep = codes is None
    if codes is None and not keep:
        raise ValueError("neither y nor codes are asked for")
    if not 0.0 <= eps <= _FLT_MAX:
        raise ValueError("eps must be finite and not negative")
    y = q = scales = None
    rp = op = yp = qp = sp = rs = rd = ct = 0
    stream = _ready_stream(index)
    if residual is not None:
        rd = _float(residual, "residual")
        rp, rs = _same(residual, rows, dim, "residual", index)
        if residual_out is None:
            residual_out = _new(rows, dim, residual.dtype, x)
            op = residual_out.data_ptr()
        else:
            op = _want(residual_out, residual.dtype, (rows, dim), "residual_out", index)
    elif residual_out is not None:
        raise ValueError("residual_out needs residual")
    if keep:
        y = _new(rows, dim, dtype, x)
        yp = y.data_ptr()
    if codes is not None:
        ct, q, qp, scales, sp = _code_rows(rows, dim, codes, x)
    code = _lib.packed["fnmoe_add_rms_norm"](_lib.pack_norm(
        _lib.ABI_VERSION, _lib.NORM_UNIT_OFFSET if unit_offset else 0, rows, dim, xd, rd, wd, ct, eps, 0, xp, xs, rp, rs, wp,
        yp, op, qp, sp), stream)
    if code:
        _lib.check(code, "add_rms_norm")
    return NormedRows(y, residual_out, q, scales)


def _code_rows(rows, dim, codes, like):
    """New codes and scales: (code type, codes, their pointer, scales, their pointer)."""
    ct = _CODES.get(codes)
    if ct is None:
        raise TypeError("codes must be torch.int8 or torch.float8_e4m3fn")
    q = _new(rows, dim, codes, like)
    scales = torch.empty_strided((rows,), (1,), dtype=torch.float32, device=like.device)
    return ct, q, q.data_ptr(), scales, scales.data_ptr()


def quantize_rows(x, codes=torch.int8):
    """``(codes, scales)`` of the rows of ``x`` [rows, dim] (bfloat16 or float32):
    ``scales[r] = max(max|x[r]|, 2^-100) / top`` and ``codes`` the nearest codes
    of ``x / scales``, ``top`` 127 (torch.int8) or 448 (torch.float8_e4m3fn); a
    quotient as near the middle of two codes as 2^-21 of itself may take either.
    A row that is not finite gets NaN as its scale.  ``dim`` is at most 16384."""
    index = x.get_device()
    xd = _float(x, "x")
    xp, rows, dim, xs = _matrix(x, "x", index)
    stream = _ready_stream(index)
    ct, q, qp, scales, sp = _code_rows(rows, dim, codes, x)
    code = _lib.packed["fnmoe_add_rms_norm"](_lib.pack_norm(
        _lib.ABI_VERSION, _lib.NORM_ROWS_AS_THEY_ARE, rows, dim, xd, 0, 0, ct, 0.0, 0, xp, xs, 0, 0, 0, 0, 0, qp, sp), stream)
    if code:
        _lib.check(code, "quantize_rows")
    return q, scales


def dequantize_rows(codes, scales, out_dtype=None, out=None):
    """The values ``codes[r] * scales[r]``, rounded once to ``out_dtype`` (bfloat16, the default, or float32)."""
    ct = _CODES.get(codes.dtype)
    if ct is None:
        raise TypeError("codes must be an int8 or float8_e4m3fn tensor")
    shape, index = codes.shape, codes.get_device()
    if len(shape) != 2:
        raise ValueError(f"codes must have two dimensions, not {tuple(shape)}")
    cp, sp = _want(codes, codes.dtype, shape, "codes", index), _want(scales, torch.float32, (shape[0],), "scales", index)
    stream = _ready_stream(index)
    if out is None:
        out = _new(shape[0], shape[1], torch.bfloat16 if out_dtype is None else out_dtype, codes)
        op = out.data_ptr()
    elif out_dtype is not None and out.dtype is not out_dtype:
        raise TypeError(f"out is {out.dtype}, out_dtype {out_dtype}")
    else:
        op = _want(out, out.dtype, shape, "out", index)
    code = _lib.packed["fnmoe_dequantize_rows"](_lib.pack_row_codes(
        _lib.ABI_VERSION, shape[0], shape[1], ct, _float(out, "out"), 0, cp, sp, op), stream)
    if code:
        _lib.check(code, "dequantize_rows")
    return out


def linear(x, weight, bias=None, *, activation: str | None = None, residual=None, x_scale=None, weight_scale=None,
           out_dtype=None, out=None):
    """``act(x W^T + bias) + residual`` -> [rows, out_width].

    ``x`` [rows, in_width] and ``weight`` [out_width, in_width] are both
    bfloat16, or both int8 or float8_e4m3fn codes with a float32 scale a row
    (``x_scale`` [rows], ``weight_scale`` [out_width]; :func:`add_rms_norm` and
    :func:`quantize_rows` make them).  Their rows, and the rows' starts, lie on
    16-byte boundaries, so ``in_width`` is a multiple of 8 (16) unless rows are
    padded.  ``bias`` [out_width] and ``residual`` [rows, out_width] are
    bfloat16 or float32; ``activation`` is "silu", "gelu" (by erf), "relu" or
    None.  Sums are float32 (int8: exact), rounded once to ``out_dtype``
    (bfloat16, the default, or float32).  ``out`` may be ``residual`` where
    types and strides are the same.
    """
    index = x.get_device()
    kind = _LINEAR.get(x.dtype)
    if kind is None or weight.dtype is not x.dtype:
        raise TypeError("x and weight must both be bfloat16, int8 or float8_e4m3fn tensors")
    xp, rows, k, xs = _matrix(x, "x", index)
    wp, n, wk, ws = _matrix(weight, "weight", index)
    if wk != k:
        raise ValueError(f"weight has {wk} columns, x has {k}")
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {', '.join(map(str, ACTIVATIONS))}, not {activation!r}")
    xsp = wsp = bp = rp = bd = rd = rs = 0
    if kind:
        if x_scale is None or weight_scale is None:
            raise ValueError("8-bit x and weight need x_scale and weight_scale")
        xsp = _want(x_scale, torch.float32, (rows,), "x_scale", index)
        wsp = _want(weight_scale, torch.float32, (n,), "weight_scale", index)
    elif x_scale is not None or weight_scale is not None:
        raise ValueError("bfloat16 x and weight have no scales")
    if bias is not None:
        bd, bp = _float(bias, "bias"), _want(bias, bias.dtype, (n,), "bias", index)
    if residual is not None:
        rd = _float(residual, "residual")
        rp, rs = _same(residual, rows, n, "residual", index)
    stream = _ready_stream(index)
    if out is None:
        out = _new(rows, n, torch.bfloat16 if out_dtype is None else out_dtype, x)
        op = out.data_ptr()
    elif out_dtype is not None and out.dtype is not out_dtype:
        raise TypeError(f"out is {out.dtype}, out_dtype {out_dtype}")
    else:
        op = _want(out, out.dtype, (rows, n), "out", index)
    od = _FLOATS.get(out.dtype)
    if od is None:
        od = _float(out, "out")
    code = _lib.packed["fnmoe_linear"](_lib.pack_linear(
        _lib.ABI_VERSION, kind, rows, k, n, act, bd, rd, od, 0, xp, xs, wp, ws, xsp, wsp, bp, rp, rs, op), stream)
    if code:
        _lib.check(code, "linear")
    return out
