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


def _row(t: Optional[torch.Tensor], dtype: torch.dtype, T: int, dev: int, what: str) -> Optional[int]:
    if t is None:
        return None
    if not (t.dtype is dtype and t.shape == (T,) and t.get_device() == dev and (T < 2 or t.stride(0) == 1)):
        _need(False, f"{what} must be contiguous {str(dtype)[6:]} [{T}] beside the logits")
    return t.data_ptr()


def sample(logits: torch.Tensor, uniforms: torch.Tensor, *, inv_temperature: Optional[torch.Tensor] = None, top_k: Optional[torch.Tensor] = None,
           top_p: Optional[torch.Tensor] = None, min_p: Optional[torch.Tensor] = None, probs: bool = False, out_ids: Optional[torch.Tensor] = None,
           out_probs: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """One token id (int32 ``[T]``) for each row of ``logits`` ``[T, V]`` (f32 or bf16, columns contiguous, up to 2^18 of them), with ``probs`` or ``out_probs`` also its
    probability among the tokens that were kept (f32 ``[T]``).

    A token weighs ``w = exp((logit - largest logit) * inv_temperature)``; tokens are ordered by falling logits, equal ones by rising ids. Kept are the first ``top_k``; of them those with
    ``w >= min_p``; of them those ahead of which less than ``top_p`` of their mass lies; always the first one. Drawn is the first kept token, by rising ids, at which the sum of the kept weights exceeds
    ``uniforms`` times that of all. The sums are integers of 2^-44: no order of additions changes a result, and weights below 2^-45 count as 0.

    Per-row values, contiguous ``[T]``, none: no such cut. ``uniforms`` f32 within [0, 1); from 1 on the last kept token is drawn, below 0 the first. ``inv_temperature`` f32: 0 and less, infinity and NaN take the first token
    (probability 1). ``top_k`` int32: below 1, or V and more, keeps all. ``top_p`` f32: 1 and more, or NaN, keeps all. ``min_p`` f32: 0 and less, or NaN, keeps all. Logits of -inf and NaN are never drawn;
    a row of nothing else gets id -1 and probability 0. Beside a logit of +inf only such logits are drawn."""
    shape, dev = logits.shape, logits.get_device()
    f32 = logits.dtype is F32
    if not (len(shape) == 2 and (f32 or logits.dtype is BF16) and 1 <= shape[1] <= MAX_VOCAB and shape[0] <= MAX_ROWS and dev >= 0 and (logits.stride(1) == 1 or shape[1] == 1)):
        _need(len(shape) == 2 and logits.dtype in (F32, BF16) and shape[1] >= 1, "logits must be f32 or bf16 [T, V]")
        _need(dev >= 0, "the logits are on the host")
        _need(shape[1] <= MAX_VOCAB and shape[0] <= MAX_ROWS, f"{shape[0]} rows of {shape[1]} logits are not supported")
        _need(False, "a row's logits must lie one behind the other")
    T, V = shape
    ld = logits.stride(0) if T > 1 else V
    _need(ld >= V, "rows of logits must lie apart")
    up = _row(uniforms, F32, T, dev, "uniforms")
    _need(up is not None, "uniforms are missing")
    args = (_row(inv_temperature, F32, T, dev, "inv_temperature"), _row(top_k, I32, T, dev, "top_k"), _row(top_p, F32, T, dev, "top_p"), _row(min_p, F32, T, dev, "min_p"), up)
    if out_ids is None:
        out_ids = torch.empty(T, dtype=I32, device=logits.device)
    if out_probs is None and probs:
        out_probs = torch.empty(T, dtype=F32, device=logits.device)
    outs = _row(out_ids, I32, T, dev, "out_ids"), _row(out_probs, F32, T, dev, "out_probs")
    if T:
        if dev == torch.cuda.current_device():
            check(_lib.load().ifab_draw(logits.data_ptr(), ld, f32, T, V, *args, *outs, _lib.current_stream(dev)), "sampling.sample")
        else:
            _lib.call_on(dev, "ifab_draw", logits.data_ptr(), ld, f32, T, V, *args, *outs)
    return out_ids if out_probs is None else (out_ids, out_probs)
