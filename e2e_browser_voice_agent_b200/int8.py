"""Matrix products in 8-bit integers over torch CUDA tensors, with a scale for each token and each output channel: the
h2c_i8_* operators of libh2cuda (include/h2cuda.h states their formulas).

  w8, w_scale = quantize(weight)                 # once: [n, k] values -> int8 [n, k padded to 16], float32 [n]
  y = matmul(x, w8, w_scale, bias=bias)          # x [m, k] -> y [m, n], the tokens quantized on the way

or, where several products share their input, matmul(xq, w8, w_scale, x_scale=xs, k=k) with xq, xs = quantize(x). Every call
enqueues kernels on the current stream of the tensors' device and returns; nothing is kept between calls.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .kv8 import _TYPES, _call, _want


def _matrix(name: str, t: torch.Tensor, index: int) -> int:
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
