"""Attention of query rows that share a long prefix, whose keys and values are read once for all of them (``csrc/kernels/shared_prefix.cu``): decode steps of several continuations of
one prompt, or questions behind one document. ``ops.decode.gqa_decode_attention`` reads them once for every row, and is as fast up to some 16000 shared positions of 2 rows, 2500 of 8,
700 of 32, 250 of 64 and of 200 (16 heads over 4 of 128 columns, 40 own positions; 32 over 8: 2500, 1000, 200, 500 and none).

Rows' own positions are taken for few: from 400 rows by key heads on a row's go to one CTA, from 1184 on to one warp. A row of tens of thousands of own positions - one that no group names, or that lies far
within its group's prefix - is better off in a call of the other kernel: beside 150 rows of 8 key heads it takes 2.5 ms here, the whole call 0.8 ms there."""
from __future__ import annotations

from ctypes import c_float
from functools import lru_cache
from typing import Optional

import torch

from . import _lib

BF16, I32 = torch.bfloat16, torch.int32
MAX_GROUPS = 64
MAX_ROWS = 1 << 20


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(f"shared_prefix: {what}")


def scratch_bytes(rows: int, heads: int, kv_heads: int, head_dim: int, groups: int = 1) -> int:
    """Bytes that :func:`attention` takes as ``scratch`` for a call of so many rows (and for any of fewer in as many groups, the most of all of them)."""
    _need(0 <= rows <= MAX_ROWS and 0 <= groups <= MAX_GROUPS and kv_heads >= 1 and heads >= 1 and heads % kv_heads == 0 and heads // kv_heads <= 16 and head_dim in (64, 128),
          f"{rows} rows of {heads} heads over {kv_heads} of {head_dim} columns in {groups} groups are not supported")
    return _lib.load().ifab_shared_prefix_scratch_up_to(rows, heads, kv_heads, head_dim, groups)


def launches(rows: int, heads: int, kv_heads: int, head_dim: int, groups: int, page_tokens: int, max_pages: int) -> int:
    """Kernels that :func:`attention` launches for so many rows, where a slot has room for ``max_pages`` pages."""
    n = _lib.load().ifab_shared_prefix_launches(rows, heads, kv_heads, head_dim, groups, page_tokens, max_pages)
    _need(n > 0, f"{rows} rows of {heads} heads over {kv_heads} of {head_dim} columns in {groups} groups are not supported")
    return n


def attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, page_table: torch.Tensor, groups: torch.Tensor, *, heads: int,
              kv_heads: int, head_dim: int, scale: float, scratch: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, status_ptr: Optional[int] = None) -> torch.Tensor:
    """Softmax attention of bf16 rows ``q`` ``[T, >= heads * head_dim]`` (the q columns of a packed projection's rows) over the positions up to their own. ``out`` ``[T, heads * head_dim]`` bf16.

    ``positions`` / ``slots`` int32 ``[T]``: a row's position (negative: nobody's row, whose result is left as it was) and the slot of its sequence; ``page_table`` int32 ``[slots, pages of one]``;
    caches bf16 ``[pages, page_tokens, kv_heads, head_dim]`` that hold the keys and values of these rows already. ``groups`` int32 ``[n, 4]`` on the device, up to 64: first row, rows, shared
    positions, slot. The rows of a group see the positions below the shared ones through that slot's pages, which are read once for all, and the others through their own; a row whose own position
    lies within the prefix sees the prefix up to it. Groups come in the order of their rows; rows that none names see everything through their own slot; a group of no rows counts as none.

    Heads of 64 or 128 columns, up to 16 of them over a key head. Scores, maxima, sums and sums of values are f32, of which the tensor cores add up 4096 keys at a time (and cut off
    2^-14.4 at most); weights enter their products with 15 bits, the result is rounded once. Pages that
    are not there, slots, positions and groups out of range are skipped and set ``IFAB_STATUS_BAD_INDEX`` in the status word; a row that sees nothing gets zeros. ``scratch``: uint8 on 16 bytes,
    :func:`scratch_bytes`; calls that may run at the same time need one each. ``out`` may lie in the queries' place, row over row, and overlaps nothing else that the call reads."""
    # what is wrong with a call is said in _refuse: messages that are made for every call cost as much as its launches. Numbers are left to the library's own checks
    qs, ks, ps, gs, dev = q.shape, k_cache.shape, page_table.shape, groups.shape, q.get_device()
    if not (len(qs) == 2 and len(ks) == 4 and len(ps) == 2 and len(gs) == 2 and dev >= 0 and q.dtype is BF16 and k_cache.dtype is BF16 and v_cache.dtype is BF16 and positions.dtype is I32
            and slots.dtype is I32 and page_table.dtype is I32 and groups.dtype is I32 and ks[2] == kv_heads and ks[3] == head_dim and v_cache.shape == ks and qs[1] >= heads * head_dim
            and positions.shape == qs[:1] and slots.shape == qs[:1] and gs[1] == 4 and q.stride(1) == 1 and k_cache.is_contiguous() and v_cache.is_contiguous() and page_table.is_contiguous()
            and groups.is_contiguous() and positions.is_contiguous() and slots.is_contiguous() and k_cache.get_device() == dev and v_cache.get_device() == dev and positions.get_device() == dev
            and slots.get_device() == dev and page_table.get_device() == dev and groups.get_device() == dev):
        _refuse(q, k_cache, v_cache, positions, slots, page_table, groups, heads, kv_heads, head_dim, scale, scratch, out)
    T, n, cols = qs[0], gs[0], heads * head_dim
    if out is None:
        out = torch.empty((T, cols), dtype=BF16, device=q.device)
        ldo = cols
    else:
        ldo = out.stride(0) if T > 1 and len(out.shape) == 2 else cols
        if not (out.dtype is BF16 and out.shape == (T, cols) and out.get_device() == dev and out.stride(1) == 1 and ldo >= cols and _apart(out, q, cols, (k_cache, v_cache, positions, slots, page_table, groups))):
            _refuse(q, k_cache, v_cache, positions, slots, page_table, groups, heads, kv_heads, head_dim, scale, scratch, out)
    if T == 0:
        return out
    need = _scratch(T, heads, kv_heads, head_dim, n)
    if scratch is None:
        scratch = torch.empty(need, dtype=torch.uint8, device=q.device)
    elif not (scratch.dtype is torch.uint8 and scratch.get_device() == dev and scratch.is_contiguous() and scratch.numel() >= need and _apart(out, q, cols, (scratch,))):
        _refuse(q, k_cache, v_cache, positions, slots, page_table, groups, heads, kv_heads, head_dim, scale, scratch, out)
    args = (q.data_ptr(), q.stride(0) if T > 1 else cols, k_cache.data_ptr(), v_cache.data_ptr(), positions.data_ptr(), slots.data_ptr(), page_table.data_ptr(), ps[0], ps[1], ks[1], ks[0],
            groups.data_ptr(), n, scale, T, heads, kv_heads, head_dim, scratch.data_ptr(), need, out.data_ptr(), ldo, status_ptr)
    if dev == torch.cuda.current_device():
        rc = _lib.load().ifab_shared_prefix_attention(*args, _lib.current_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = _lib.load().ifab_shared_prefix_attention(*args, _lib.current_stream(dev))
    if rc == -1:
        _refuse(q, k_cache, v_cache, positions, slots, page_table, groups, heads, kv_heads, head_dim, scale, scratch, out)
    _lib.check(rc, "shared_prefix.attention")
    return out


def _apart(out: torch.Tensor, q: torch.Tensor, cols: int, others) -> bool:
    """Whether no row of the output lies over queries, but in the place of its own, and none between the ends of the others."""
    T, o, p = out.shape[0], out.data_ptr(), q.data_ptr()
    if T == 0:
        return True
    ldo, ldq = (t.stride(0) if T > 1 else cols for t in (out, q))
    end = o + 2 * ((T - 1) * ldo + cols)
    for t in others:
        at = t.data_ptr()
        if at < end and o < at + t.nbytes:
            return False
    if (o == p and ldo == ldq) or o >= p + 2 * ((T - 1) * ldq + cols) or p >= end:
        return True
    ahead = (p - o) // 2 % ldo           # columns side by side, in rows of one pitch
    return ldo == ldq and ahead >= cols and ahead + cols <= ldo


@lru_cache(maxsize=256)
def _scratch(rows: int, heads: int, kv_heads: int, head_dim: int, groups: int) -> int:
    return _lib.load().ifab_shared_prefix_scratch(rows, heads, kv_heads, head_dim, groups) if rows >= 1 and kv_heads >= 1 and heads >= 1 and groups >= 0 else 0


def _refuse(q, k_cache, v_cache, positions, slots, page_table, groups, heads, kv_heads, head_dim, scale, scratch, out) -> None:
    dev, T = q.get_device(), q.shape[0] if q.dim() else 0
    _need(q.dim() == 2 and q.dtype == BF16 and q.stride(1) == 1, "queries must be bf16 [T, heads * head_dim], columns contiguous")
    _need(dev >= 0, "the queries are on the host")
    _need(kv_heads >= 1 and heads >= 1 and heads % kv_heads == 0 and heads // kv_heads <= 16 and head_dim in (64, 128), f"{heads} heads over {kv_heads} of {head_dim} columns are not supported")
    _need(T <= MAX_ROWS, f"{T} rows are not supported")
    _need(q.shape[1] >= heads * head_dim, f"queries of {q.shape[1]} columns for {heads} heads of {head_dim}")
    pages, pt = k_cache.shape[:2] if k_cache.dim() == 4 else (0, 0)
    for t, what in ((k_cache, "keys"), (v_cache, "values")):
        _need(t.dtype == BF16 and t.get_device() == dev and t.shape == (pages, pt, kv_heads, head_dim) and t.is_contiguous() and pages > 0 and pt > 0,
              f"{what} must be contiguous bf16 [pages, page_tokens, {kv_heads}, {head_dim}] beside the queries")
    for t, what in ((positions, "positions"), (slots, "slots")):
        _need(t.dtype == I32 and t.shape == (T,) and t.get_device() == dev and t.is_contiguous(), f"{what} must be contiguous int32 [{T}] beside the queries")
    for t, what in ((page_table, "page_table"), (groups, "groups")):
        _need(t.dim() == 2 and t.dtype == I32 and t.get_device() == dev and t.is_contiguous(), f"{what} must be contiguous int32 beside the queries")
    _need(groups.shape[0] <= MAX_GROUPS and groups.shape[1] == 4, f"groups must be [up to {MAX_GROUPS}, 4]")
    num_slots, max_pages = page_table.shape
    _need(num_slots >= 1 and max_pages >= 1 and pages * pt < 1 << 31 and max_pages * pt < (1 << 31) - 256, f"{pages} pages of {pt} positions, {max_pages} of {num_slots} slots are not supported")
    _need(0 < c_float(scale).value <= 2.35e38, f"a scale of {scale}: above 0, to 2.35e38, as f32")
    _need(out is None or (out.dtype == BF16 and out.shape == (T, heads * head_dim) and out.get_device() == dev and out.stride(1) == 1 and (T < 2 or out.stride(0) >= heads * head_dim)),
          f"the output must be bf16 [{T}, {heads * head_dim}] beside the queries, its rows apart")
    _need(out is None or _apart(out, q, heads * head_dim, (k_cache, v_cache, positions, slots, page_table, groups)),
          "the output must overlap nothing that is read, but for the queries row over row")
    need = _scratch(T, heads, kv_heads, head_dim, groups.shape[0])
    _need(scratch is None or (scratch.dtype == torch.uint8 and scratch.get_device() == dev and scratch.is_contiguous() and scratch.numel() >= need),
          f"scratch must be {need} bytes (uint8) beside the queries")
    _need(scratch is None or out is None or _apart(out, q, heads * head_dim, (scratch,)), "the output must not overlap the scratch")
    near = all(t is None or t.data_ptr() % 16 == 0 for t in (q, k_cache, v_cache, groups, scratch, out)) and all(t is None or T < 2 or t.stride(0) % 8 == 0 for t in (q, out))
    _need(near, "rows, caches, groups and scratch must lie on 16 bytes")
    raise RuntimeError(f"shared_prefix.attention: {T} rows of {heads} heads are too many for one call")
