"""A paged 8-bit KV cache over torch CUDA tensors: the h2c_kv8_* operators of libh2cuda (include/h2cuda.h states their
formulas).

One step of a serving loop, for requests that hold `cached` tokens and will hold `total`:

  p = plan(cached, total, block_table, free_pages, free_state, page_size, max_tokens)   # pages and slots, on the GPU
  append(kv, kv_scale, k, v, p.slot)                                                    # the new tokens' K and V rows
  out = attention(q, kv, kv_scale, block_table, p.q_start, p.kv_len, max_q, max_kv)     # single tokens and prompts alike

kv is int8 [pages, 2, kv heads, page size, head dim] and kv_scale float32 [pages, 2, kv heads] (allocate makes both). Every
call enqueues kernels on the current stream of the tensors' device and returns; nothing is kept between calls. Arguments
that do not fit raise ValueError or TypeError here, or H2CError from the library.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib

_TYPES = {torch.float32: _lib.TYPE_F32, torch.float16: _lib.TYPE_F16, torch.bfloat16: _lib.TYPE_BF16}


class Plan(NamedTuple):
    """What plan returns; all on the device. status is [0, 0], [1, missing pages] or [2, 0] (see h2c_kv8_plan)."""
    kv_len: torch.Tensor      # int32 [requests]
    q_start: torch.Tensor     # int32 [requests + 1]
    slot: torch.Tensor        # int32 [max_tokens]
    position: torch.Tensor    # int32 [max_tokens]
    free_state: torch.Tensor  # int64 [2], the free_state of the next step
    status: torch.Tensor      # int32 [2]


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


class _On:
    """The device of `t` as the current one, for the time of a call (most often it is already)."""

    def __init__(self, t: torch.Tensor):
        if not t.is_cuda:
            raise ValueError("a CUDA tensor is wanted")
        self.device, self.before = t.device, torch.cuda.current_device()

    def __enter__(self):
        if self.device.index != self.before:
            torch.cuda.set_device(self.device)
        return _stream(self.device)

    def __exit__(self, *_):
        if self.device.index != self.before:
            torch.cuda.set_device(self.before)


def _want(name: str, t: torch.Tensor, dtype: torch.dtype, device: torch.device, shape: Optional[Tuple] = None) -> int:
    """The address of a contiguous tensor of this type and shape on this device."""
    if t.dtype is not dtype:
        raise TypeError(f"{name}: {dtype} is wanted, not {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name}: on {t.device}, not {device}")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"{name}: shape {shape} is wanted, not {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")
    return t.data_ptr()


def _cache(kv: torch.Tensor, kv_scale: torch.Tensor):
    if kv.dim() != 5 or kv.shape[1] != 2:
        raise ValueError(f"kv: [pages, 2, kv heads, page size, head dim] is wanted, not {tuple(kv.shape)}")
    n_pages, _, kv_heads, page, head_dim = kv.shape
    return (_want("kv", kv, torch.int8, kv.device),
            _want("kv_scale", kv_scale, torch.float32, kv.device, (n_pages, 2, kv_heads)), n_pages, page, kv_heads, head_dim)


def _rows(name: str, t: torch.Tensor, device: torch.device, heads: int, head_dim: int) -> Tuple[int, int, int, int]:
    """(address, element type, row stride, head stride) of [rows, heads, head_dim] values, the last axis dense."""
    if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != head_dim:
        raise ValueError(f"{name}: [rows, {heads}, {head_dim}] is wanted, not {tuple(t.shape)}")
    if t.dtype not in _TYPES:
        raise TypeError(f"{name}: float32, float16 or bfloat16 is wanted, not {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name}: on {t.device}, not {device}")
    s = t.stride()
    if s[2] != 1:
        raise ValueError(f"{name}: the head dimension must be dense")
    return t.data_ptr(), _TYPES[t.dtype], s[0], s[1]


def allocate(n_pages: int, page_size: int, kv_heads: int, head_dim: int, device="cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """A cache and its scales. A page's contents mean nothing before rows are appended to it."""
    return (torch.zeros(n_pages, 2, kv_heads, page_size, head_dim, dtype=torch.int8, device=device),
            torch.zeros(n_pages, 2, kv_heads, dtype=torch.float32, device=device))


def free_pool(n_pages: int, device="cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """(free_pages, free_state) of a pool whose pages are all free."""
    return (torch.arange(n_pages, dtype=torch.int32, device=device),
            torch.tensor([0, n_pages], dtype=torch.int64, device=device))


def plan(cached: torch.Tensor, total: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
         free_state: torch.Tensor, page_size: int, max_tokens: int, out: Optional[Plan] = None) -> Plan:
    """Take and give back pages so that request r goes from cached[r] to total[r] tokens, and map the new tokens to
    slots (h2c_kv8_plan). block_table (int32 [requests, columns]) and free_pages (int32 [pages], a ring) change in place.
    out: a Plan of an earlier call of the same sizes, whose tensors are written again."""
    dev = cached.device
    n = cached.shape[0] if cached.dim() == 1 else -1
    if n < 0:
        raise ValueError(f"cached: one length per request is wanted, not {tuple(cached.shape)}")
    if block_table.dim() != 2 or block_table.shape[0] != n:
        raise ValueError(f"block_table: [{n}, columns] is wanted, not {tuple(block_table.shape)}")
    if free_pages.dim() != 1:
        raise ValueError(f"free_pages: one number per page is wanted, not {tuple(free_pages.shape)}")
    if max_tokens < 0:
        raise ValueError(f"max_tokens: {max_tokens}")
    with _On(cached) as stream:
        i32, i64 = torch.int32, torch.int64
        if out is None:
            # one allocation; the 64-bit state first
            buf = torch.empty(4 + 2 + n + (n + 1) + 2 * max_tokens, dtype=i32, device=dev)
            state, status, kv_len, q_start, slot, position = buf.split([4, 2, n, n + 1, max_tokens, max_tokens])
            out = Plan(kv_len, q_start, slot, position, state.view(i64), status)
        p = (_want("cached", cached, i32, dev), _want("total", total, i32, dev, (n,)),
             _want("block_table", block_table, i32, dev))
        _lib.check(_lib.load().h2c_kv8_plan(
            n, page_size, *p, block_table.shape[1], _want("free_pages", free_pages, i32, dev), free_pages.shape[0],
            _want("free_state", free_state, i64, dev, (2,)), _want("out.free_state", out.free_state, i64, dev, (2,)),
            _want("out.kv_len", out.kv_len, i32, dev, (n,)), _want("out.q_start", out.q_start, i32, dev, (n + 1,)),
            _want("out.slot", out.slot, i32, dev, (max_tokens,)),
            _want("out.position", out.position, i32, dev, (max_tokens,)), max_tokens,
            _want("out.status", out.status, i32, dev, (2,)), stream))
    return out


def append(kv: torch.Tensor, kv_scale: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slot: torch.Tensor) -> None:
    """Quantize rows of K and V ([rows, kv heads, head dim], any row and head stride) into the cache at slot
    (h2c_kv8_append); slot may hold more entries than there are rows."""
    pkv, ps, n_pages, page, kvh, hd = _cache(kv, kv_scale)
    dev = kv.device
    pk, tk, k_row, k_head = _rows("k", k, dev, kvh, hd)
    pv, tv, v_row, v_head = _rows("v", v, dev, kvh, hd)
    rows = k.shape[0]
    if v.shape[0] != rows or tv != tk:
        raise ValueError("k and v must have as many rows and the same type")
    if slot.dim() != 1 or slot.shape[0] < rows:
        raise ValueError(f"slot: at least {rows} entries are wanted, not {tuple(slot.shape)}")
    with _On(kv) as stream:
        _lib.check(_lib.load().h2c_kv8_append(pkv, ps, n_pages, page, kvh, hd, tk, pk, k_row, k_head, pv, v_row, v_head,
                                              rows, _want("slot", slot, torch.int32, dev), stream))


def read(kv: torch.Tensor, kv_scale: torch.Tensor, slot: torch.Tensor,
         dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
    """The cached K and V at slot, [slots, kv heads, head dim] each (h2c_kv8_read)."""
    pkv, ps, n_pages, page, kvh, hd = _cache(kv, kv_scale)
    if dtype not in _TYPES:
        raise TypeError(f"dtype: float32, float16 or bfloat16 is wanted, not {dtype}")
    if slot.dim() != 1:
        raise ValueError(f"slot: one entry per row is wanted, not {tuple(slot.shape)}")
    rows = slot.shape[0]
    with _On(kv) as stream:
        k, v = torch.empty(2, rows, kvh, hd, dtype=dtype, device=kv.device).unbind(0)
        _lib.check(_lib.load().h2c_kv8_read(pkv, ps, n_pages, page, kvh, hd,
                                            _want("slot", slot, torch.int32, kv.device), rows, _TYPES[dtype],
                                            k.data_ptr(), v.data_ptr(), stream))
    return k, v


def attention(q: torch.Tensor, kv: torch.Tensor, kv_scale: torch.Tensor, block_table: torch.Tensor,
              q_start: torch.Tensor, kv_len: torch.Tensor, max_q: int, max_kv: int, scale: Optional[float] = None,
              window: int = 0, out: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Causal grouped-query attention of a ragged batch over the cache (h2c_kv8_attention). q is [rows, heads, head dim]
    with any row and head stride; scale defaults to head_dim ** -0.5; window > 0 limits each query to that many positions.
    max_q and max_kv bound the requests' query counts and lengths. Returns out ([rows, heads, head dim], q's type), or
    (out, lse) with lse float32 [rows, heads]; rows that belong to no request keep what out held."""
    pkv, ps, n_pages, page, kvh, hd = _cache(kv, kv_scale)
    dev = kv.device
    if q.dim() != 3:
        raise ValueError(f"q: [rows, heads, {hd}] is wanted, not {tuple(q.shape)}")
    rows, heads = q.shape[0], q.shape[1]
    pq, tq, q_row, q_head = _rows("q", q, dev, heads, hd)
    n = kv_len.shape[0]
    if block_table.dim() != 2 or block_table.shape[0] != n:
        raise ValueError(f"block_table: [{n}, columns] is wanted, not {tuple(block_table.shape)}")
    i32 = torch.int32
    with _On(kv) as stream:
        if out is None:
            out = torch.empty(rows, heads, hd, dtype=q.dtype, device=dev)
        po, to, o_row, o_head = _rows("out", out, dev, heads, hd)
        if to != tq or out.shape[0] != rows:
            raise ValueError("out must have q's rows and type")
        lse = torch.empty(rows, heads, dtype=torch.float32, device=dev) if return_lse else None
        a = _lib.Kv8AttentionArgs(pq, q_row, q_head, po, o_row, o_head, lse.data_ptr() if return_lse else None, pkv, ps,
                                  n_pages, page, kvh, hd, heads, tq, _want("block_table", block_table, i32, dev),
                                  block_table.shape[1], n, _want("q_start", q_start, i32, dev, (n + 1,)),
                                  _want("kv_len", kv_len, i32, dev, (n,)), rows, max_q, max_kv, window,
                                  hd ** -0.5 if scale is None else scale, None, 0)
        L = _lib.load()
        need = L.h2c_kv8_attention_workspace(a)
        if need:
            work = torch.empty(need, dtype=torch.uint8, device=dev)
            a.workspace, a.workspace_bytes = work.data_ptr(), need
        _lib.check(L.h2c_kv8_attention(a, stream))
    return (out, lse) if return_lse else out
