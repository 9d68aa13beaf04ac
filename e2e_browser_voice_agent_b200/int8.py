"""Matrix products in 8-bit integers over torch CUDA tensors, with a scale for each token and each output channel: the
h2c_i8_* operators of libh2cuda (include/h2cuda.h states their formulas).

  w8, w_scale = quantize(weight)                 # once: [n, k] values -> int8 [n, k padded to 16], float32 [n]
  y = matmul(x, w8, w_scale, bias=bias)          # x [m, k] -> y [m, n], the tokens quantized on the way

or, where several products share their input, matmul(xq, w8, w_scale, x_scale=xs, k=k) with xq, xs = quantize(x). norm makes such
codes of a normed residual stream:

  n = norm(x, weight, eps, residual=r)           # n.sum = x + r, n.codes and n.scale of its root-mean-square norm
  y = matmul(n.codes, w8, w_scale, x_scale=n.scale, k=k)

Every call enqueues kernels on the current stream of the tensors' device and returns; nothing is kept between calls.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .kv8 import _TYPES, _call, _want


class Norm(NamedTuple):
    """What norm returns."""
    codes: torch.Tensor          # int8 [rows, k padded to a multiple of 16]
    scale: torch.Tensor          # float32 [rows]
    sum: Optional[torch.Tensor]  # x + residual, None without a residual


def _matrix(name: str, t: torch.Tensor, index: int) -> int:
    if t.dim() == 2 and t.get_device() == index and t.stride(1) == 1 and t.numel() < 2**31:  # (the usual case)
        return t.data_ptr()
    if t.dim() != 2:
        raise ValueError(f"{name}: a matrix is wanted, not {tuple(t.shape)}")
    if t.get_device() != index:
        raise ValueError(f"{name}: on {t.device}, not cuda:{index}")
    if t.numel() >= 2**31 and max(t.shape) >= 2**31:
        raise ValueError(f"{name}: {tuple(t.shape)} does not fit in 32 bits")
    if t.stride(1) != 1 and t.shape[1] > 1:
        raise ValueError(f"{name}: rows must be dense")
    return t.data_ptr()


def quantize(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows of x ([rows, k], float32, float16 or bfloat16, any row stride) as int8 codes [rows, k padded to a multiple of
    16] and float32 scales [rows] (h2c_i8_quantize)."""
    index = x.get_device()
    px = _matrix("x", x, index)
    if x.dtype not in _TYPES:
        raise TypeError(f"x: float32, float16 or bfloat16 is wanted, not {x.dtype}")
    rows, k = x.shape
    q = torch.empty(rows, (k + 15) // 16 * 16, dtype=torch.int8, device=x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    _call(index, _lib.load().h2c_i8_quantize, _TYPES[x.dtype], px, x.stride(0), rows, k, q.data_ptr(), q.shape[1],
          scale.data_ptr())
    return q, scale


def matmul(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
           x_scale: Optional[torch.Tensor] = None, k: Optional[int] = None, out_dtype: Optional[torch.dtype] = None,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y = x w^T in 8-bit integers, scaled, plus bias (h2c_i8_matmul). x is [m, k] values, or with x_scale the codes of
    quantize, whose k must then be given; w int8 [n, at least k] with rows a multiple of 16 apart; w_scale and bias
    float32 [n]. The result has x's type (float32 for codes) unless out_dtype or out says otherwise. out may be x's values, in
    place; it shares no memory with another argument."""
    index = x.get_device()
    px, pw = _matrix("x", x, index), _matrix("w", w, index)
    if w.dtype is not torch.int8:
        raise TypeError(f"w: int8 is wanted, not {w.dtype}")
    m, n = x.shape[0], w.shape[0]
    if x_scale is None:
        x_type, ps = _TYPES.get(x.dtype), None
        if x_type is None:
            raise TypeError(f"x: float32, float16 or bfloat16 is wanted, not {x.dtype} (codes come with x_scale)")
        if k is not None and k != x.shape[1]:
            raise ValueError(f"k: x has {x.shape[1]} columns")
        k = x.shape[1]
    else:
        if x.dtype is not torch.int8:
            raise TypeError(f"x: int8 codes are wanted with x_scale, not {x.dtype}")
        if k is None or k > x.shape[1]:
            raise ValueError("k: the number of codes that count is wanted with x_scale, at most x's columns")
        x_type, ps = _lib.TYPE_I8, _want("x_scale", x_scale, torch.float32, index, (m,))
    if w.shape[1] < k:
        raise ValueError(f"w: at least {k} columns are wanted, not {w.shape[1]}")
    if out is None:
        kind = out_dtype or (torch.float32 if x_scale is not None else x.dtype)
        y_type = _TYPES.get(kind)
        if y_type is None:
            raise TypeError(f"out_dtype: float32, float16 or bfloat16 is wanted, not {kind}")
        out = torch.empty(m, n, dtype=kind, device=x.device)
        py, y_row = out.data_ptr(), n
    else:
        if out.shape != (m, n) or (out_dtype is not None and out.dtype is not out_dtype):
            raise ValueError(f"out: {(m, n)} is wanted, not {tuple(out.shape)} {out.dtype}")
        y_type = _TYPES.get(out.dtype)
        if y_type is None:
            raise TypeError(f"out: float32, float16 or bfloat16 is wanted, not {out.dtype}")
        py, y_row = _matrix("out", out, index), out.stride(0)
    L = _lib.load()
    need = L.h2c_i8_matmul_workspace(x_type, m, k)
    work = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    _call(index, L.h2c_i8_matmul, x_type, px, x.stride(0), ps, pw, w.stride(0),
          _want("w_scale", w_scale, torch.float32, index, (n,)), m, n, k, y_type, py, y_row,
          None if bias is None else _want("bias", bias, torch.float32, index, (n,)), None if work is None else work.data_ptr(), need)
    return out


def norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None,
         out: Optional[torch.Tensor] = None) -> Norm:
    """The codes of rows of x ([rows, k], float32, float16 or bfloat16, any row stride), or of x + residual, normed by their root mean
    square and multiplied by weight (float32 [k]) (h2c_i8_norm). residual has x's type or float32 and gives the sum its type; out takes
    the sum: residual itself, x itself, a tensor that shares no memory with the arguments, or None for a new one."""
    index = x.get_device()
    px = _matrix("x", x, index)
    if x.dtype not in _TYPES:
        raise TypeError(f"x: float32, float16 or bfloat16 is wanted, not {x.dtype}")
    rows, k = x.shape
    pr = po = None
    r_type = r_row = o_row = 0
    if residual is not None:
        pr, r_row = _matrix("residual", residual, index), residual.stride(0)
        if residual.shape != x.shape:
            raise ValueError(f"residual: {tuple(x.shape)} is wanted, not {tuple(residual.shape)}")
        if residual.dtype is not x.dtype and residual.dtype is not torch.float32:
            raise TypeError(f"residual: {x.dtype} or float32 is wanted, not {residual.dtype}")
        r_type = _TYPES[residual.dtype]
        if out is None:
            out = residual.new_empty(rows, k)
            po, o_row = out.data_ptr(), k
        else:
            if out.shape != x.shape:
                raise ValueError(f"out: {tuple(x.shape)} is wanted, not {tuple(out.shape)}")
            if out.dtype is not residual.dtype:
                raise TypeError(f"out: {residual.dtype} is wanted, not {out.dtype}")
            po, o_row = _matrix("out", out, index), out.stride(0)
    elif out is not None:
        raise ValueError("out: there is no residual, so no sum")
    k_pad = (k + 15) // 16 * 16
    q = x.new_empty(rows, k_pad, dtype=torch.int8)
    scale = weight.new_empty(rows, dtype=torch.float32)
    _call(index, _lib.load().h2c_i8_norm, _TYPES[x.dtype], px, x.stride(0), r_type, pr, r_row, po, o_row,
          _want("weight", weight, torch.float32, index, (k,)), eps, rows, k, q.data_ptr(), k_pad, scale.data_ptr())
    return Norm(q, scale, out)


def values(codes: torch.Tensor, scale: torch.Tensor, k: Optional[int] = None, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """What codes of quantize or norm stand for: [rows, k] values of dtype (h2c_i8_values). k: how many of a row's codes count, all
    unless given."""
    index = codes.get_device()
    pq = _matrix("codes", codes, index)
    if codes.dtype is not torch.int8:
        raise TypeError(f"codes: int8 is wanted, not {codes.dtype}")
    if dtype not in _TYPES:
        raise TypeError(f"dtype: float32, float16 or bfloat16 is wanted, not {dtype}")
    rows = codes.shape[0]
    k = codes.shape[1] if k is None else k
    if not 0 < k <= codes.shape[1]:
        raise ValueError(f"k: 1 to {codes.shape[1]} is wanted, not {k}")
    y = codes.new_empty(rows, k, dtype=dtype)
    _call(index, _lib.load().h2c_i8_values, pq, codes.stride(0), _want("scale", scale, torch.float32, index, (rows,)), rows, k,
          _TYPES[dtype], y.data_ptr())
    return y
