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


# The current device and its current stream, without the Stream object that torch.cuda.current_stream makes of it (which
# costs as much as a launch).
_device = torch._C._cuda_getDevice
_stream = torch._C._cuda_getCurrentRawStream


def _call(index: int, fn, *args) -> None:
    """fn(*args, stream) with device `index` current, on its current stream."""
    if index < 0:
        raise ValueError("CUDA tensors are wanted")
    before = _device()
    if index == before:
        rc = fn(*args, _stream(index))
    else:
        torch.cuda.set_device(index)
        try:
            rc = fn(*args, _stream(index))
        finally:
            torch.cuda.set_device(before)
    if rc:
        _lib.check(rc)


def _int32(names: str, *numbers: int) -> None:
    """Refuse numbers that a 32-bit argument of the library would cut off."""
    if max(numbers) >= 2**31 or min(numbers) < -2**31:
        raise ValueError(f"{names}: {numbers}: not all fit in 32 bits")


def _want(name: str, t: torch.Tensor, dtype: torch.dtype, index: int, shape: Optional[Tuple] = None) -> int:
    """The address of a contiguous tensor of this type and shape on device `index`."""
    if t.dtype is dtype and t.get_device() == index and t.is_contiguous() and (shape is None or t.shape == shape):
        return t.data_ptr()
    if t.dtype is not dtype:
        raise TypeError(f"{name}: {dtype} is wanted, not {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{name}: on {t.device}, not cuda:{index}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name}: shape {shape} is wanted, not {tuple(t.shape)}")
    raise ValueError(f"{name}: must be contiguous")


def _cache(kv: torch.Tensor, kv_scale: torch.Tensor):
    """(device, address, address of the scales, pages, page size, kv heads, head dimension)"""
    shape = kv.shape
    if len(shape) != 5 or shape[1] != 2:
        raise ValueError(f"kv: [pages, 2, kv heads, page size, head dim] is wanted, not {tuple(shape)}")
    n_pages, _, kv_heads, page, head_dim = shape
    if n_pages >= 2**31 or kv_heads >= 2**31 or page >= 2**31 or head_dim >= 2**31:
        raise ValueError(f"kv: {tuple(shape)} does not fit in 32 bits")
    index = kv.get_device()
    return (index, _want("kv", kv, torch.int8, index),
            _want("kv_scale", kv_scale, torch.float32, index, (n_pages, 2, kv_heads)), n_pages, page, kv_heads, head_dim)


def _rows(name: str, t: torch.Tensor, index: int, heads: int, head_dim: int) -> Tuple[int, int, int, int]:
    """(address, element type, row stride, head stride) of [rows, heads, head_dim] values, the last axis dense."""
    shape = t.shape
    if len(shape) != 3 or shape[0] >= 2**31 or shape[1] != heads or shape[2] != head_dim:
        raise ValueError(f"{name}: [rows, {heads}, {head_dim}] is wanted, not {tuple(shape)}")
    kind = _TYPES.get(t.dtype)
    if kind is None:
        raise TypeError(f"{name}: float32, float16 or bfloat16 is wanted, not {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{name}: on {t.device}, not cuda:{index}")
    row, head, dense = t.stride()
    if dense != 1:
        raise ValueError(f"{name}: the head dimension must be dense")
    return t.data_ptr(), kind, row, head


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
    out: a Plan of an earlier call of the same sizes, whose tensors are written again; none of them may be, or share memory
    with, an argument of this call (cached = p.kv_len wants another Plan than p)."""
    if cached.dim() != 1:
        raise ValueError(f"cached: one length per request is wanted, not {tuple(cached.shape)}")
    index, n = cached.get_device(), cached.shape[0]
    if block_table.dim() != 2 or block_table.shape[0] != n:
        raise ValueError(f"block_table: [{n}, columns] is wanted, not {tuple(block_table.shape)}")
    if free_pages.dim() != 1:
        raise ValueError(f"free_pages: one number per page is wanted, not {tuple(free_pages.shape)}")
    if max_tokens < 0:
        raise ValueError(f"max_tokens: {max_tokens}")
    _int32("page_size, max_tokens, columns, pages, requests", page_size, max_tokens, block_table.shape[1], free_pages.shape[0], n)
    i32, i64 = torch.int32, torch.int64
    args = (n, page_size, _want("cached", cached, i32, index), _want("total", total, i32, index, (n,)),
            _want("block_table", block_table, i32, index), block_table.shape[1],
            _want("free_pages", free_pages, i32, index), free_pages.shape[0], _want("free_state", free_state, i64, index, (2,)))
    if out is None:
        # one allocation; the 64-bit state first
        buf = torch.empty(4 + 2 + n + (n + 1) + 2 * max_tokens, dtype=i32, device=cached.device)
        state, status, kv_len, q_start, slot, position = buf.split((4, 2, n, n + 1, max_tokens, max_tokens))
        out = Plan(kv_len, q_start, slot, position, state.view(i64), status)
        at = buf.data_ptr()
        places = (at, at + 24, at + 24 + 4 * n, at + 28 + 8 * n, at + 28 + 8 * n + 4 * max_tokens, max_tokens, at + 16)
    else:
        places = (_want("out.free_state", out.free_state, i64, index, (2,)), _want("out.kv_len", out.kv_len, i32, index, (n,)),
                  _want("out.q_start", out.q_start, i32, index, (n + 1,)), _want("out.slot", out.slot, i32, index, (max_tokens,)),
                  _want("out.position", out.position, i32, index, (max_tokens,)), max_tokens,
                  _want("out.status", out.status, i32, index, (2,)))
    _call(index, _lib.load().h2c_kv8_plan, *args, *places)
    return out


def append(kv: torch.Tensor, kv_scale: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slot: torch.Tensor) -> None:
    """Quantize rows of K and V ([rows, kv heads, head dim], any row and head stride) into the cache at slot
    (h2c_kv8_append); slot may hold more entries than there are rows."""
    index, *cache = _cache(kv, kv_scale)
    pk, tk, k_row, k_head = _rows("k", k, index, cache[4], cache[5])
    pv, tv, v_row, v_head = _rows("v", v, index, cache[4], cache[5])
    rows = k.shape[0]
    if v.shape[0] != rows or tv != tk:
        raise ValueError("k and v must have as many rows and the same type")
    if slot.dim() != 1 or slot.shape[0] < rows:
        raise ValueError(f"slot: at least {rows} entries are wanted, not {tuple(slot.shape)}")
    _call(index, _lib.load().h2c_kv8_append, *cache, tk, pk, k_row, k_head, pv, v_row, v_head, rows,
          _want("slot", slot, torch.int32, index))


def read(kv: torch.Tensor, kv_scale: torch.Tensor, slot: torch.Tensor,
         dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
    """The cached K and V at slot, [slots, kv heads, head dim] each (h2c_kv8_read)."""
    index, *cache = _cache(kv, kv_scale)
    if dtype not in _TYPES:
        raise TypeError(f"dtype: float32, float16 or bfloat16 is wanted, not {dtype}")
    if slot.dim() != 1:
        raise ValueError(f"slot: one entry per row is wanted, not {tuple(slot.shape)}")
    rows = slot.shape[0]
    _int32("rows", rows, 0)
    k, v = (torch.empty(rows, cache[4], cache[5], dtype=dtype, device=kv.device) for _ in range(2))
    _call(index, _lib.load().h2c_kv8_read, *cache, _want("slot", slot, torch.int32, index), rows, _TYPES[dtype], k.data_ptr(),
          v.data_ptr())
    return k, v


def _attention_args(q, kv, kv_scale, block_table, q_start, kv_len, max_q, max_kv, scale, window, out, return_lse):
    """(device, arguments without a workspace, out, lse)"""
    index, pkv, ps, n_pages, page, kvh, hd = _cache(kv, kv_scale)
    if q.dim() != 3:
        raise ValueError(f"q: [rows, heads, {hd}] is wanted, not {tuple(q.shape)}")
    rows, heads, _ = q.shape
    pq, tq, q_row, q_head = _rows("q", q, index, heads, hd)
    n = kv_len.shape[0]
    if block_table.dim() != 2 or block_table.shape[0] != n:
        raise ValueError(f"block_table: [{n}, columns] is wanted, not {tuple(block_table.shape)}")
    _int32("heads, max_q, max_kv, window, columns", heads, max_q, max_kv, window, block_table.shape[1])
    i32 = torch.int32
    if out is None:
        out = q.new_empty(rows, heads, hd)
        po, o_row, o_head = out.data_ptr(), heads * hd, hd
    else:
        po, to, o_row, o_head = _rows("out", out, index, heads, hd)
        if to != tq or out.shape[0] != rows:
            raise ValueError("out must have q's rows and type")
    lse = q.new_empty(rows, heads, dtype=torch.float32) if return_lse else None
    a = _lib.Kv8AttentionArgs(pq, q_row, q_head, po, o_row, o_head, lse.data_ptr() if return_lse else None, pkv, ps, n_pages,
                              page, kvh, hd, heads, tq, _want("block_table", block_table, i32, index), block_table.shape[1], n,
                              _want("q_start", q_start, i32, index, (n + 1,)), _want("kv_len", kv_len, i32, index, (n,)), rows,
                              max_q, max_kv, window, hd ** -0.5 if scale is None else scale, None, 0)
    return index, a, out, lse


def attention(q: torch.Tensor, kv: torch.Tensor, kv_scale: torch.Tensor, block_table: torch.Tensor,
              q_start: torch.Tensor, kv_len: torch.Tensor, max_q: int, max_kv: int, scale: Optional[float] = None,
              window: int = 0, out: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Causal grouped-query attention of a ragged batch over the cache (h2c_kv8_attention). q is [rows, heads, head dim]
    with any row and head stride; scale defaults to head_dim ** -0.5; window > 0 limits each query to that many positions.
    max_q and max_kv bound the requests' query counts and lengths. Returns out ([rows, heads, head dim], q's type), or
    (out, lse) with lse float32 [rows, heads]; rows that belong to no request keep what out held. out may be q itself, or
    share no memory with the arguments."""
    index, a, out, lse = _attention_args(q, kv, kv_scale, block_table, q_start, kv_len, max_q, max_kv, scale, window, out, return_lse)
    L = _lib.load()
    need = L.h2c_kv8_attention_workspace(a)
    if need:
        work = kv.new_empty(need, dtype=torch.uint8)
        a.workspace, a.workspace_bytes = work.data_ptr(), need
    _call(index, L.h2c_kv8_attention, a)
    return (out, lse) if return_lse else out


def prefix_attention(q: torch.Tensor, kv: torch.Tensor, kv_scale: torch.Tensor, prefix_table: torch.Tensor, prefix_len: torch.Tensor,
                     group_start: torch.Tensor, block_table: torch.Tensor, q_start: torch.Tensor, kv_len: torch.Tensor, max_q: int,
                     max_kv: int, max_prefix: int, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                     return_lse: bool = False):
    """attention of requests that share prefixes, whose keys are read once for all of them (h2c_kv8_prefix_attention). Requests
    group_start[g] .. group_start[g + 1] - 1 (int32 [groups + 1]) also see the first prefix_len[g] (int32 [groups]) positions of the
    pages prefix_table[g] (int32 [groups, columns]), which come before their own; block_table, kv_len and max_kv are of their own
    positions alone. max_prefix bounds the prefixes' lengths. The rest is as in attention."""
    index, own, out, lse = _attention_args(q, kv, kv_scale, block_table, q_start, kv_len, max_q, max_kv, scale, 0, out, return_lse)
    i32, n = torch.int32, prefix_len.shape[0]
    if prefix_table.dim() != 2 or prefix_table.shape[0] != n:
        raise ValueError(f"prefix_table: [{n}, columns] is wanted, not {tuple(prefix_table.shape)}")
    _int32("groups, columns, max_prefix", n, prefix_table.shape[1], max_prefix)
    a = _lib.Kv8PrefixArgs(own, _want("prefix_table", prefix_table, i32, index), _want("prefix_len", prefix_len, i32, index, (n,)),
                           _want("group_start", group_start, i32, index, (n + 1,)), prefix_table.shape[1], n, max_prefix)
    L = _lib.load()
    need = L.h2c_kv8_prefix_attention_workspace(a)
    if need:
        work = kv.new_empty(need, dtype=torch.uint8)
        a.own.workspace, a.own.workspace_bytes = work.data_ptr(), need
    _call(index, L.h2c_kv8_prefix_attention, a)
    return (out, lse) if return_lse else out
