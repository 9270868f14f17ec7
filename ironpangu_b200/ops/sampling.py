"""A token for every row of logits, drawn from the whole vocabulary with random numbers that the caller gives (``csrc/kernels/draw.cu``), on one rank.

``ops.decode.sample_topk`` is the other sampler: at most 64 candidates a row, vocabularies split over ranks, penalties, and random numbers of its own."""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _lib
from ._lib import check

F32, BF16, I32 = torch.float32, torch.bfloat16, torch.int32
MAX_VOCAB = 1 << 18
MAX_ROWS = 1 << 20


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(f"sampling: {what}")


def sample(logits: torch.Tensor, uniforms: torch.Tensor, *, inv_temperature: Optional[torch.Tensor] = None, top_k: Optional[torch.Tensor] = None,
           top_p: Optional[torch.Tensor] = None, min_p: Optional[torch.Tensor] = None, probs: bool = False, out_ids: Optional[torch.Tensor] = None,
           out_probs: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """One token id (int32 ``[T]``) for each row of ``logits`` ``[T, V]`` (f32 or bf16, columns contiguous, up to 2^18 of them), with ``probs`` or ``out_probs`` also its
    probability among the tokens that were kept (f32 ``[T]``).

    A token weighs ``w = exp((logit - largest logit) * inv_temperature)``; tokens are ordered by falling logits, equal ones by rising ids. Kept are the first ``top_k``; of them those with
    ``w >= min_p``; of them those ahead of which less than ``top_p`` of their mass lies; always the first one. Drawn is the first kept token, by rising ids, at which the sum of the kept weights exceeds
    ``uniforms`` times that of all. The sums are integers of 2^-44: no order of additions changes a result, and weights below 2^-45 count as 0. A weight is off by 2^-28 of
    itself and 2^-45 at most.

    Per-row values, contiguous ``[T]``, none: no such cut. ``uniforms`` f32 within [0, 1); from 1 on the last kept token is drawn, below 0 the first. ``inv_temperature`` f32: 0 and less, infinity and NaN take the first token
    (probability 1). ``top_k`` int32: below 1, or V and more, keeps all. ``top_p`` f32: 1 and more, or NaN, keeps all. ``min_p`` f32: 0 and less, or NaN, keeps all. Logits of -inf and NaN are never drawn;
    a row of nothing else gets id -1 and probability 0. Beside a logit of +inf only such logits are drawn.
    ``out_ids`` and ``out_probs`` may lie where one of the rows' values does, and overlap nothing else that the call reads or writes."""
    # what is wrong with a call is said in _refuse: messages that are made for every call cost as much as its launch
    shape, dev, dt = logits.shape, logits.get_device(), logits.dtype
    f32 = dt is F32
    if not (len(shape) == 2 and (f32 or dt is BF16) and dev >= 0 and (logits.stride(1) == 1 or shape[1] == 1)):
        _refuse(logits, uniforms, inv_temperature, top_k, top_p, min_p, out_ids, out_probs)
    T, V = shape
    given = [uniforms.data_ptr()] if _is_row(uniforms, F32, T, dev) else _refuse(logits, uniforms, inv_temperature, top_k, top_p, min_p, out_ids, out_probs)
    for t, want in ((inv_temperature, F32), (top_k, I32), (top_p, F32), (min_p, F32)):
        if t is None:
            given.append(None)
        elif t.dtype is want and t.shape == (T,) and t.get_device() == dev and t.is_contiguous():
            given.append(t.data_ptr())
        else:
            _refuse(logits, uniforms, inv_temperature, top_k, top_p, min_p, out_ids, out_probs)
    fresh = out_ids is None and out_probs is None
    if out_ids is None:
        out_ids = torch.empty(T, dtype=I32, device=logits.device)
    elif not _is_row(out_ids, I32, T, dev):
        _refuse(logits, uniforms, inv_temperature, top_k, top_p, min_p, out_ids, out_probs)
    if out_probs is None:
        if probs:
            out_probs = torch.empty(T, dtype=F32, device=logits.device)
    elif not _is_row(out_probs, F32, T, dev):
        _refuse(logits, uniforms, inv_temperature, top_k, top_p, min_p, out_ids, out_probs)
    if T:
        if not fresh and not _apart(logits, given, out_ids, out_probs):
            _refuse(logits, uniforms, inv_temperature, top_k, top_p, min_p, out_ids, out_probs)
        u, it, k, p, m = given
        args = (logits.data_ptr(), logits.stride(0) if T > 1 else V, f32, T, V, it, k, p, m, u, out_ids.data_ptr(), None if out_probs is None else out_probs.data_ptr())
        if dev == torch.cuda.current_device():
            rc = _lib.load().ifab_draw(*args, _lib.current_stream(dev))
        else:
            with torch.cuda.device(dev):
                rc = _lib.load().ifab_draw(*args, _lib.current_stream(dev))
        if rc == -1:
            _refuse(logits, uniforms, inv_temperature, top_k, top_p, min_p, out_ids, out_probs)
        check(rc, "sampling.sample")
    return out_ids if out_probs is None else (out_ids, out_probs)


def _is_row(t: Optional[torch.Tensor], dtype: torch.dtype, T: int, dev: int) -> bool:
    return t is not None and t.dtype is dtype and t.shape == (T,) and t.get_device() == dev and t.is_contiguous()


def _apart(logits: torch.Tensor, given, out_ids: torch.Tensor, out_probs: Optional[torch.Tensor]) -> bool:
    """Whether the results overlap neither the logits nor one another, and of the rows' values (pointers) none but in its own place."""
    T, V = logits.shape
    n, size = 4 * T, logits.element_size()
    first, pitch = logits.data_ptr(), (logits.stride(0) if T > 1 else V) * size
    outs = [t.data_ptr() for t in (out_ids, out_probs) if t is not None]
    for o in outs:
        if any(p is not None and p != o and o < p + n and p < o + n for p in given):
            return False
        if o < first + (T - 1) * pitch + V * size and first < o + n:
            ahead = (o - first) % max(pitch, 1)      # it may lie between two rows
            if pitch < V * size or o < first or ahead < V * size or ahead + n > pitch:
                return False
    return len(outs) < 2 or abs(outs[0] - outs[1]) >= n


def _refuse(logits, uniforms, inv_temperature, top_k, top_p, min_p, out_ids, out_probs) -> None:
    shape, dev = logits.shape, logits.get_device()
    _need(len(shape) == 2 and logits.dtype in (F32, BF16), "logits must be f32 or bf16 [T, V]")
    _need(dev >= 0, "the logits are on the host")
    T, V = shape
    _need(1 <= V <= MAX_VOCAB and T <= MAX_ROWS, f"{T} rows of {V} logits are not supported")
    _need(logits.stride(1) == 1 or V == 1, "a row's logits must lie one behind the other")
    _need(T < 2 or logits.stride(0) >= V, "rows of logits must lie apart")
    _need(uniforms is not None, "uniforms are missing")
    for t, dtype, what in ((uniforms, F32, "uniforms"), (inv_temperature, F32, "inv_temperature"), (top_k, I32, "top_k"), (top_p, F32, "top_p"), (min_p, F32, "min_p"), (out_ids, I32, "out_ids"),
                           (out_probs, F32, "out_probs")):
        _need(t is None or _is_row(t, dtype, T, dev), f"{what} must be contiguous {str(dtype)[6:]} [{T}] beside the logits")
    given = [None if t is None else t.data_ptr() for t in (uniforms, inv_temperature, top_k, top_p, min_p)]
    _need((out_ids is None and out_probs is None) or T == 0 or _apart(logits, given, *((out_ids, out_probs) if out_ids is not None else (out_probs, None))),
          "results must not overlap the logits or one another, nor the rows' values but in their own place")
    raise AssertionError("sampling.sample: a call was refused without a reason")
