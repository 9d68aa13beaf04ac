"""Penalties for repeated tokens, biases and masks of allowed tokens on logits, over torch CUDA tensors: the h2c_logits_adjust operator
of libh2cuda (include/h2cuda.h states its formula).

  adjust(logits, tokens=said, length=n, repetition=r, presence=p, frequency=f,   # what each session said, and how strongly it counts
         bias_id=ids, bias=b, allowed=bits, out=logits)                          # biases, a grammar's next tokens; in place

One kernel on the current stream of the tensors' device; nothing is kept between calls.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .kv8 import _TYPES, _call, _want

MAX_BIASES = _lib.LOGITS_MAX_BIASES


def _lines(name: str, t: torch.Tensor, dtype: torch.dtype, index: int, rows: int, columns: Optional[int] = None):
    """(address, row stride) of [rows, columns] values with dense rows."""
    if t.dtype is not dtype:
        raise TypeError(f"{name}: {dtype} is wanted, not {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{name}: on {t.device}, not cuda:{index}")
    if t.dim() != 2 or t.shape[0] != rows or (columns is not None and t.shape[1] != columns):
        raise ValueError(f"{name}: [{rows}, {'columns' if columns is None else columns}] is wanted, not {tuple(t.shape)}")
    if t.stride(1) != 1 and t.shape[1] > 1:
        raise ValueError(f"{name}: rows must be dense")
    return t.data_ptr(), t.stride(0)


def adjust(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, length: Optional[torch.Tensor] = None,
           repetition: Optional[torch.Tensor] = None, presence: Optional[torch.Tensor] = None,
           frequency: Optional[torch.Tensor] = None, bias_id: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
           allowed: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """logits ([rows, vocabulary], float32, float16 or bfloat16, any row stride) as the next token is chosen from (h2c_logits_adjust).
    tokens int32 [rows, columns] and length int32 [rows]: row r's tokens so far are tokens[r, :length[r]]; repetition (divides
    positive logits of tokens that are among them and multiplies the others), frequency (is taken off once per occurrence) and presence
    (once) float32 [rows]. bias_id int32 and bias float32 [rows, up to 1024]: what is added to some tokens, an id of -1 to none.
    allowed int32 [rows, vocabulary / 32 rounded up]: bit i % 32 of word i / 32 says whether token i may come; the others become
    -infinity. out: logits itself, another tensor of its shape and type, or None for a new one."""
    index = logits.get_device()
    kind = _TYPES.get(logits.dtype)
    if kind is None:
        raise TypeError(f"logits: float32, float16 or bfloat16 is wanted, not {logits.dtype}")
    if logits.dim() != 2 or logits.shape[1] < 1 or max(logits.shape) >= 2**31:
        raise ValueError(f"logits: [rows, vocabulary] is wanted, not {tuple(logits.shape)}")
    rows, vocab = logits.shape
    p_in, in_row = _lines("logits", logits, logits.dtype, index, rows)
    if out is None:
        out = logits.new_empty(rows, vocab)
        p_out, out_row = out.data_ptr(), vocab
    else:
        p_out, out_row = _lines("out", out, logits.dtype, index, rows, vocab)
    said, said_row, columns, p_len, strengths = None, 0, 0, None, [None, None, None]
    if (tokens is None) != (length is None):
        raise ValueError("tokens and length belong together")
    if (bias_id is None) != (bias is None):
        raise ValueError("bias_id and bias belong together")
    if tokens is not None:
        said, said_row = _lines("tokens", tokens, torch.int32, index, rows)
        columns = tokens.shape[1]
        if columns >= 2**31:
            raise ValueError(f"tokens: {tuple(tokens.shape)} does not fit in 32 bits")
        if not columns:  # (an empty tensor may have no address)
            said = p_len = None
        else:
            p_len = _want("length", length, torch.int32, index, (rows,))
        f32, one = torch.float32, (rows,)
        strengths = [None if repetition is None else _want("repetition", repetition, f32, index, one),
                     None if presence is None else _want("presence", presence, f32, index, one),
                     None if frequency is None else _want("frequency", frequency, f32, index, one)]
        if not columns:
            strengths = [None, None, None]
    elif not (repetition is presence is frequency is None):
        name = "repetition" if repetition is not None else "presence" if presence is not None else "frequency"
        raise ValueError(f"{name}: the tokens that it is for are wanted with it")
    p_id = p_bias = None
    n_bias = 0
    if bias_id is not None:
        if bias_id.dim() != 2 or bias_id.shape[1] > MAX_BIASES:
            raise ValueError(f"bias_id: [{rows}, up to {MAX_BIASES}] is wanted, not {tuple(bias_id.shape)}")
        n_bias = bias_id.shape[1]
        p_id, p_bias = _want("bias_id", bias_id, torch.int32, index, (rows, n_bias)), _want("bias", bias, torch.float32, index, (rows, n_bias))
    p_bits, bits_row = (None, 0) if allowed is None else _lines("allowed", allowed, torch.int32, index, rows, (vocab + 31) // 32)
    _call(index, _lib.load().h2c_logits_adjust, kind, p_in, in_row, p_out, out_row, rows, vocab, said, said_row, columns, p_len,
          *strengths, p_id, p_bias, n_bias, p_bits, bits_row)
    return out
