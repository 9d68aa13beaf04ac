"""Rotary positions over torch CUDA tensors: the h2c_rope operator of libh2cuda (include/h2cuda.h states its formula).

  f = frequencies(128, base=1e6)                                   # once: float64 [64], radians per position
  q, k = rotate(q, p.position, f, k=k)                             # q and k [tokens, heads, head dim], any strides

rotate enqueues one kernel on the current stream of the tensors' device and returns; nothing is kept between calls.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib
from .kv8 import _TYPES, _call, _want

SCALINGS = ("none", "linear", "ntk", "yarn", "turns")


def frequencies(rotary_dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0, original: int = 0,
                fast: float = 32.0, slow: float = 1.0, device="cuda") -> torch.Tensor:
    """The frequencies base ** (-2 j / rotary_dim) of a head's rotary_dim / 2 pairs, in radians per position (float64), as they are or
    for contexts `factor` times as long as the model's:
      linear  all divided by factor
      ntk     the base raised by factor ** (rotary_dim / (rotary_dim - 2)): the slowest is divided by factor, the fastest stays
      yarn    pairs that turn more than `fast` times within `original` positions stay, those that turn less than `slow` times are
              divided by factor, and between them (from the pair at or before the one to the pair at or after the other) the share of both goes
              linearly with the pair's number, as models with YaRN (Peng et al. 2023) are trained and run; the attention
              temperature that belongs to it is yarn_magnitude(factor), an argument of rotate
      turns   the same, but that the share goes linearly with the turns
    A model whose frequencies are made otherwise brings its own tensor."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim: an even number is wanted, not {rotary_dim}")
    if not base > 1 or not factor >= 1:
        raise ValueError(f"base {base}, factor {factor}: a base above 1 and a factor of at least 1 are wanted")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling: one of {SCALINGS} is wanted, not {scaling!r}")
    half = rotary_dim // 2
    if scaling == "ntk":
        if rotary_dim == 2:
            raise ValueError("scaling ntk: the one pair of rotary_dim 2 has nothing to be stretched against")
        base *= factor ** (rotary_dim / (rotary_dim - 2))
    f = [base ** (-2 * j / rotary_dim) for j in range(half)]
    if scaling == "linear":
        f = [x / factor for x in f]
    if scaling in ("yarn", "turns"):
        if original < 1 or not fast > slow > 0:
            raise ValueError(f"scaling {scaling}: original ({original}) positions and fast ({fast}) above slow ({slow}) are wanted")
        at = lambda turns: rotary_dim * math.log(original / (2 * math.pi * turns)) / (2 * math.log(base))  # the pair that turns so often
        low, high = max(0, math.floor(at(fast))), min(rotary_dim - 1, math.ceil(at(slow)))
        for j in range(half):
            if scaling == "yarn":
                kept = 1 - (j - low) / max(high - low, 0.001)
            else:
                kept = (f[j] * original / (2 * math.pi) - slow) / (fast - slow)
            kept = min(1.0, max(0.0, kept))
            f[j] *= kept + (1 - kept) / factor
    return torch.tensor(f, dtype=torch.float64, device=device)


def yarn_magnitude(factor: float) -> float:
    """The magnitude of queries and keys that goes with scaling yarn."""
    return 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0


def _vectors(name: str, t: torch.Tensor, like: torch.Tensor, index: int):
    """(address, row stride, head stride) of [tokens, heads, head dim] values, the last axis dense, of like's type and device."""
    if t.dim() != 3:
        raise ValueError(f"{name}: [tokens, heads, head dim] is wanted, not {tuple(t.shape)}")
    if t.dtype is not like.dtype:
        raise TypeError(f"{name}: {like.dtype} is wanted, not {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{name}: on {t.device}, not cuda:{index}")
    row, head, dense = t.stride()
    if dense != 1:
        raise ValueError(f"{name}: the head dimension must be dense")
    return t.data_ptr(), row, head


def rotate(q: torch.Tensor, position: torch.Tensor, frequency: torch.Tensor, k: Optional[torch.Tensor] = None,
           interleaved: bool = False, magnitude: float = 1.0, out: Optional[torch.Tensor] = None,
           k_out: Optional[torch.Tensor] = None):
    """q ([tokens, heads, head dim], float32, float16 or bfloat16, any row and head stride) and, with it, k with their first 2 *
    len(frequency) values turned to their tokens' positions (h2c_rope). position: int32, one per token or more; tokens whose
    position is negative stay as they are. Pairs are (j, j + len(frequency)), or neighbours with `interleaved`. out and k_out:
    q and k themselves (in place), tensors that share no memory with the arguments, or None for new ones. Returns q's, or (q's,
    k's) with k."""
    index = q.get_device()
    kind = _TYPES.get(q.dtype)
    if kind is None:
        raise TypeError(f"q: float32, float16 or bfloat16 is wanted, not {q.dtype}")
    pq, q_row, q_head = _vectors("q", q, q, index)
    tokens, heads, head_dim = shape = q.shape
    k_heads, pk, k_row, k_head, pko, ko_row, ko_head = 0, None, 0, 0, None, 0, 0
    if k is not None:
        pk, k_row, k_head = _vectors("k", k, q, index)
        k_tokens, k_heads, k_dim = k.shape
        if k_tokens != tokens or k_dim != head_dim:
            raise ValueError(f"k: [{tokens}, heads, {head_dim}] is wanted, not {tuple(k.shape)}")
        if k_out is None:
            k_out = k.new_empty(tokens, k_heads, head_dim)
            pko, ko_row, ko_head = k_out.data_ptr(), k_heads * head_dim, head_dim
        else:
            if k_out.shape != k.shape:
                raise ValueError(f"k_out: {tuple(k.shape)} is wanted, not {tuple(k_out.shape)}")
            pko, ko_row, ko_head = _vectors("k_out", k_out, q, index)
    elif k_out is not None:
        raise ValueError("k_out: there is no k")
    if out is None:
        out = q.new_empty(tokens, heads, head_dim)
        po, o_row, o_head = out.data_ptr(), heads * head_dim, head_dim
    else:
        if out.shape != shape:
            raise ValueError(f"out: {tuple(shape)} is wanted, not {tuple(out.shape)}")
        po, o_row, o_head = _vectors("out", out, q, index)
    if position.dim() != 1 or position.shape[0] < tokens:
        raise ValueError(f"position: at least {tokens} entries are wanted, not {tuple(position.shape)}")
    pairs = frequency.shape[0] if frequency.dim() == 1 else 0
    if not 1 <= pairs <= head_dim // 2:
        raise ValueError(f"frequency: 1 to {head_dim // 2} entries are wanted, not {tuple(frequency.shape)}")
    if tokens >= 2**31 or heads >= 2**31 or k_heads >= 2**31 or head_dim >= 2**31:
        raise ValueError(f"q: {tuple(q.shape)} does not fit in 32 bits")
    _call(index, _lib.load().h2c_rope, kind, pq, q_row, q_head, po, o_row, o_head, heads, pk, k_row, k_head, pko, ko_row, ko_head,
          k_heads, tokens, head_dim, _want("position", position, torch.int32, index),
          _want("frequency", frequency, torch.float64, index), 2 * pairs, 1 if interleaved else 0, magnitude)
    return out if k is None else (out, k_out)
