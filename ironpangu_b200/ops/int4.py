"""Linears with weights of 4 bits and a scale - and, if wanted, a zero point - per group of columns:  ``w[n, k] = s[n, k // G] (q[n, k] - z[n, k // G])`` with ``q`` and
``z`` in 0 .. 15 (``z = 8`` without zero points) and ``G`` of 32, 64 or 128 columns (``csrc/kernels/int4_pack.cu``, ``int4_rows.cu``, ``int4_tc.cu``).

A matrix is packed once (:func:`quantise` a bf16 matrix, :func:`pack` what a checkpoint holds) and then multiplied by :func:`linear` as often as wanted. Like all weights it is
written by nothing while linears read it: a linear's loads of it may begin before the kernel ahead of it in the stream has ended."""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _lib
from ._lib import call_on, check

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
GROUPS = (32, 64, 128)
NORM_ROWS = 8            # rows up to which a linear takes the norm ahead of it
STREAM_ROWS = 16         # rows up to which the weights' stream is the work; more go through the tensor cores' tiles
SPIN_LIMIT = 4000000     # polls of a wait inside a kernel


class IfabInt4(C.Structure):
    """Mirror of ``struct IfabInt4`` in ``csrc/kernels/ifab_kernels.h``."""

    _fields_ = [("units", C.c_void_p), ("N", C.c_int32), ("K", C.c_int32), ("group", C.c_int32), ("zeros", C.c_int32), ("gated", C.c_int32), ("f16", C.c_int32)]


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(f"int4: {what}")


def _pitch(t: torch.Tensor) -> int:
    """Elements from a row to the next one; of a single row, whose stride says nothing, its columns."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


class Int4Weight:
    """A packed matrix of ``rows`` x ``k`` weights; ``gated``: gate rows, then as many up rows. ``units`` holds codes, scales and zero points together."""

    def __init__(self, rows: int, k: int, *, group: int = 128, zeros: bool = False, gated: bool = False, f16: bool = False, device="cuda"):
        if not (group in GROUPS and rows >= 1 and k >= 8 and k % 8 == 0 and not (gated and rows % 2) and max(rows, k) <= 1 << 24):      # (messages only where they are wanted)
            _need(group in GROUPS, f"groups of {group} columns are not supported")
            _need(rows >= 1 and k >= 8 and k % 8 == 0, f"a matrix of {rows} x {k} is not supported (columns in eights)")
            _need(max(rows, k) <= 1 << 24, f"a matrix of {rows} x {k} is too large")
            _need(False, f"{rows} rows are not gate and up rows")
        self.rows, self.k, self.group, self.zeros, self.gated, self.f16 = rows, k, group, bool(zeros), bool(gated), bool(f16)
        self.n = rows // 2 if gated else rows                 # columns of a result
        self.units = torch.empty(_lib.load().ifab_int4_bytes(self.n, k, group, self.zeros, self.gated), dtype=torch.uint8, device=device)
        self.device, self.index = self.units.device, self.units.get_device()
        self.desc = IfabInt4(self.units.data_ptr(), self.n, k, group, self.zeros, self.gated, self.f16)
        self.ref = C.byref(self.desc)

    @property
    def nbytes(self) -> int:
        return self.units.numel()

    def dequantise(self, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The weights' values ``[rows, k]``, rounded to bf16."""
        _need(self.index >= 0, "the weights are on the host")
        if out is None:
            out = torch.empty(self.rows, self.k, dtype=BF16, device=self.device)
        _need(out.shape == (self.rows, self.k) and out.dtype == BF16 and out.stride(1) == 1 and out.device == self.device, "the output must be bf16 [rows, k] beside the weights")
        _need(_pitch(out) % 8 == 0 and _pitch(out) >= self.k and out.data_ptr() % 16 == 0, "the output's rows must lie on 16 bytes, one behind the other")
        call_on(self.index, "ifab_int4_dequantise", self.ref, out.data_ptr(), _pitch(out))
        return out


def quantise(w: torch.Tensor, *, group: int = 128, zeros: bool = False, gated: bool = False) -> Int4Weight:
    """The bf16 matrix ``w`` ``[rows, k]`` in 4 bits. Per row and group: ``s = bf16(max|w| / 7)``; with zero points ``lo = min(w, 0)``, ``hi = max(w, 0)``,
    ``s = bf16((hi - lo) / 15)``, ``z = rint(-lo / s)``; ``q = rint(w / s) + z``, within 0 .. 15. Where ``s`` is 0 (a group of zeros, or of less than bf16's smallest) the weights are 0; a group with an infinity or NaN gets a
    scale of NaN."""
    _need(w.dim() == 2 and w.dtype == BF16 and w.stride(1) == 1 and w.is_cuda, "the matrix must be bf16 [rows, k] on the device, columns contiguous")
    _need(w.shape[0] >= 1 and _pitch(w) % 8 == 0 and _pitch(w) >= w.shape[1] and w.data_ptr() % 16 == 0, "the matrix's rows must lie on 16 bytes, one behind the other")
    out = Int4Weight(w.shape[0], w.shape[1], group=group, zeros=zeros, gated=gated, device=w.device)
    call_on(out.index, "ifab_int4_quantise", out.ref, w.data_ptr(), _pitch(w))
    return out


def pack(codes: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None, *, group: int = 128, gated: bool = False) -> Int4Weight:
    """A checkpoint's matrix: ``codes`` uint8 ``[rows, k]`` (a code in the low four bits of a byte), ``scales`` bf16 or f16 and ``zeros`` uint8 (or none: 8), both
    ``[rows, ceil(k / group)]``."""
    _need(codes.dim() == 2 and codes.dtype == torch.uint8 and codes.stride(1) == 1 and codes.is_cuda, "codes must be uint8 [rows, k] on the device, columns contiguous")
    rows, k = codes.shape
    _need(rows >= 1 and _pitch(codes) >= k, "codes must be rows one behind the other")
    _need(group in GROUPS, f"groups of {group} columns are not supported")
    _need(scales.dtype in (BF16, F16), "scales must be bf16 or f16")
    for t, what in ((scales, "scales"), (zeros, "zero points")):
        _need(t is None or (t.shape == (rows, -(-k // group)) and t.is_contiguous() and t.device == codes.device), f"{what} must be contiguous [rows, groups] beside the codes")
    _need(zeros is None or zeros.dtype == torch.uint8, "zero points must be uint8")
    out = Int4Weight(rows, k, group=group, zeros=zeros is not None, gated=gated, f16=scales.dtype == F16, device=codes.device)
    call_on(out.index, "ifab_int4_pack", out.ref, codes.data_ptr(), _pitch(codes), scales.data_ptr(), None if zeros is None else zeros.data_ptr())
    return out


def linear(x: torch.Tensor, w: Int4Weight, *, norm_w: Optional[torch.Tensor] = None, eps: float = 1e-5, residual: Optional[torch.Tensor] = None, out_f32: bool = False,
           out: Optional[torch.Tensor] = None, status_ptr: Optional[int] = None) -> torch.Tensor:
    """``y = x @ w.T (+ residual)``, or of a gated matrix ``silu(x @ gate.T) * (x @ up.T)``, for any number of bf16 rows ``x`` ``[T, k]``. ``norm_w`` (up to eight rows): the
    rows are RMS-normalised first, as :func:`ops.decode.rmsnorm` does it. ``residual`` (bf16, not of a gated matrix) may be ``out``, or lie apart from it. Sums are f32 and the
    result is rounded once, to bf16 or with ``out_f32`` not at all. ``out``, whose rows lie apart, must not overlap ``x``.

    Beyond sixteen rows a weight is rounded to the 11 bits of f16 ahead of its product (in units of its row's largest scale, so that weights 2^-25 of that and less lose more), which
    is the largest error of an f32 result there; up to sixteen rows it is not, and sums run over ``16 + q``, which costs two bits of f32. ``status_ptr``: a status word for
    waits that run out."""
    # the checks say what is wrong in _refuse: a message that is made for every call costs as much as the launch. Device numbers, which are compared in a fifth of the time that
    # devices are, and each attribute is asked for once
    shape, dev, xp, n, k = x.shape, w.index, x.data_ptr(), w.n, w.k
    if not (len(shape) == 2 and shape[1] == k and x.dtype is BF16 and x.get_device() == dev and x.stride(1) == 1):
        _refuse(x, w, norm_w, residual, out)
    T = shape[0]
    ldx = x.stride(0) if T > 1 else k
    if xp % 16 or ldx % 8:
        _refuse(x, w, norm_w, residual, out)
    fresh = out is None
    if fresh:
        f32 = out_f32
        out = torch.empty((T, n), dtype=F32 if f32 else BF16, device=w.device)
        yp, ldy = out.data_ptr(), n
    else:
        yp, ldy, f32 = out.data_ptr(), out.stride(0), out.dtype is F32
        if not (out.shape == (T, n) and (f32 or out.dtype is BF16) and out.get_device() == dev and (out.stride(1) == 1 or n == 1) and (ldy >= n or T < 2)):
            _refuse(x, w, norm_w, residual, out)
        # most outputs lie wholly ahead of or behind the rows
        if yp < xp + 2 * ((T - 1) * ldx + k) and xp < yp + (4 if f32 else 2) * ((T - 1) * ldy + n) and _meet(x, out):
            _refuse(x, w, norm_w, residual, out)
    if norm_w is not None and not (norm_w.shape == (k,) and norm_w.dtype is BF16 and norm_w.get_device() == dev and norm_w.stride(0) == 1 and norm_w.data_ptr() % 16 == 0 and T <= NORM_ROWS):
        _refuse(x, w, norm_w, residual, out)
    rp, ldr = None, 0
    if residual is not None:
        if not (not w.gated and residual.shape == (T, n) and residual.dtype is BF16 and residual.get_device() == dev and (residual.stride(1) == 1 or n == 1)):
            _refuse(x, w, norm_w, residual, out)
        rp, ldr = residual.data_ptr(), residual.stride(0)
        if not (fresh or residual is out or _same(residual, out)) and _meet(residual, out):
            _refuse(x, w, norm_w, residual, out)
    if T == 0:
        return out
    if dev < 0:
        _need(False, "the weights are on the host")
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return linear(x, w, norm_w=norm_w, eps=eps, residual=residual, out=out, status_ptr=status_ptr)
    lib = _lib.load()
    if T > STREAM_ROWS:
        scratch = torch.empty(lib.ifab_int4_gemm_scratch(T, k), dtype=torch.uint8, device=w.device)
        check(lib.ifab_int4_gemm(w.ref, xp, ldx, rp, ldr, yp, ldy, f32, T, scratch.data_ptr(), SPIN_LIMIT, status_ptr, _lib.current_stream(dev)), "int4.linear")
        return out
    check(lib.ifab_int4_rows(w.ref, xp, ldx, None if norm_w is None else norm_w.data_ptr(), eps, rp, ldr, yp, ldy, f32, T, SPIN_LIMIT, status_ptr, _lib.current_stream(dev)),
          "int4.linear")
    return out


def _same(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two matrices ``[T, n]`` are one in memory."""
    return a.data_ptr() == b.data_ptr() and a.dtype == b.dtype and (a.shape[0] < 2 or a.stride(0) == b.stride(0))


def _meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two matrices of as many rows share a byte."""
    T = a.shape[0]
    if T == 0:
        return False
    (ap, aw, al), (bp, bw, bl) = ((t.data_ptr(), t.shape[1] * t.element_size(), (t.stride(0) if T > 1 else 0) * t.element_size()) for t in (a, b))
    if ap >= bp + (T - 1) * bl + bw or bp >= ap + (T - 1) * al + aw:
        return False
    if al != bl or al == 0:
        return True
    ahead = (bp - ap) % al                           # columns side by side, in rows of one pitch
    return ahead < aw or ahead + bw > al


def _refuse(x: torch.Tensor, w: Int4Weight, norm_w, residual, out) -> None:
    T = x.shape[0] if x.dim() else 0
    _need(x.dim() == 2 and x.shape[1] == w.k and x.dtype == BF16 and x.stride(1) == 1 and x.device == w.device, f"the rows must be bf16 [T, {w.k}] beside the weights")
    _need(x.data_ptr() % 16 == 0 and (T <= 1 or x.stride(0) % 8 == 0), "rows must lie on 16 bytes")
    if norm_w is not None:
        _need(norm_w.shape == (w.k,) and norm_w.dtype == BF16 and norm_w.is_contiguous() and norm_w.device == w.device and norm_w.data_ptr() % 16 == 0,
              f"gains must be bf16 [{w.k}] on 16 bytes")
        _need(T <= NORM_ROWS, f"a norm ahead of {T} rows is a launch of its own (ops.decode.rmsnorm)")
    _need(out is None or (out.shape == (T, w.n) and out.dtype in (BF16, F32) and (out.stride(1) == 1 or w.n == 1) and out.device == w.device),
          f"the output must be bf16 or f32 [T, {w.n}] beside the weights")
    _need(out is None or T < 2 or out.stride(0) >= w.n, "the output's rows must lie apart")
    _need(out is None or not _meet(x, out), "the output must not overlap the rows")
    if residual is not None:
        _need(not w.gated, "a gated unit takes no residual")
        _need(residual.shape == (T, w.n) and residual.dtype == BF16 and residual.stride(1) == 1 and residual.device == w.device,
              f"the residual must be bf16 [T, {w.n}] beside the weights")
        _need(out is None or _same(residual, out) or not _meet(residual, out), "the residual must be the output or lie apart from it")
    raise AssertionError("int4.linear: a call was refused without a reason")
