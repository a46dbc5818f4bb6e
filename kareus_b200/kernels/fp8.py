"""Matrices in 8-bit floating point with a power-of-two scale for each block of 128, and their product.

The contract of both calls is at :func:`kareus_b200.kernels.fp8_quantize` and :func:`kareus_b200.kernels.fp8_gemm`; the kernels are
``csrc/fp8_quantize.cu`` and ``csrc/gemm_fp8_sm100.cu``, the PyTorch statements are in :mod:`.ref`."""
from __future__ import annotations

import torch

import kareus_b200.kernels as _entry

from . import ref
from .cuda import KernelError, _check, _count, _rows_readable, _stream, lib, require_current_device, status_word

_FORMAT_CODE = {"e4m3": 0, "e5m2": 1}
_MOST = (1 << 31) - 512          # rows and columns, whose numbers are ints in the kernels
_DTYPE = {fmt: ref.FP8_FORMATS[fmt][0] for fmt in _FORMAT_CODE}


class Fp8Matrix:
    """``data`` (``[rows, cols]``, one byte each) times the powers of two in ``scales`` (uint8, ``[row blocks, piece blocks, 32, 4,
    4]``: see :func:`.ref.fp8_pack_scales`).  Pieces run along the rows, which is the direction that a product contracts."""

    __slots__ = ("data", "scales", "fmt")

    def __init__(self, data: torch.Tensor, scales: torch.Tensor, fmt: str = "e4m3"):
        self.data, self.scales, self.fmt = data, scales, fmt

    def __repr__(self):
        return f"Fp8Matrix({tuple(self.data.shape)}, {self.fmt}, {self.data.device})"

    @property
    def shape(self):
        return self.data.shape

    def dequantize(self, dtype=torch.float32) -> torch.Tensor:
        """What the matrix stands for."""
        return ref.fp8_dequantize(self.data, self.scales, dtype)


def _check_matrix(m, what: str) -> None:
    if not isinstance(m, Fp8Matrix):
        raise KernelError(f"{what} has to be an Fp8Matrix, got {type(m).__name__}")
    if m.fmt not in _FORMAT_CODE or m.data.dtype != ref.FP8_FORMATS[m.fmt][0] or m.data.dim() != 2:
        raise KernelError(f"{what}: {m.data.dtype} of {m.data.dim()} dimensions is no matrix of format {m.fmt!r}")
    rows, cols = m.data.shape
    want = (-(-rows // 128), -(-(-(-cols // 128)) // 4), 32, 4, 4)
    if m.scales.dtype != torch.uint8 or tuple(m.scales.shape) != want or not m.scales.is_contiguous():
        raise KernelError(f"{what}: scales have to be contiguous uint8 {want}, got {m.scales.dtype} {tuple(m.scales.shape)}")
    if m.scales.device != m.data.device:
        raise KernelError(f"{what}: data on {m.data.device}, scales on {m.scales.device}")


def _empty(rows: int, cols: int, fmt: str, device) -> Fp8Matrix:
    """Rows start on 16 bytes."""
    data = torch.empty(rows, -(-cols // 16) * 16, dtype=ref.FP8_FORMATS[fmt][0], device=device)[:, :cols]
    return Fp8Matrix(data, torch.empty(-(-rows // 128), -(-(-(-cols // 128)) // 4), 32, 4, 4, dtype=torch.uint8, device=device), fmt)


def _statement(x, fmt: str, square: bool) -> Fp8Matrix:
    data, scales = ref.fp8_quantize(x, fmt, square)
    m = _empty(*x.shape, fmt, x.device)
    m.data.copy_(data)
    m.scales = scales
    return m


def quantize(x, rows: bool = True, cols: bool = False, square: bool = False, fmt: str = "e4m3"):
    if _entry._OPS is not None and fmt in _FORMAT_CODE:
        r = _entry._OPS.fp8_quantize(x, rows, cols, square, _FORMAT_CODE[fmt])
        if r is not None:
            return (None if r[0] is None else Fp8Matrix(r[0], r[1], fmt)), (None if r[2] is None else Fp8Matrix(r[2], r[3], fmt))
    if fmt not in _FORMAT_CODE:
        raise KernelError(f"unknown 8-bit format {fmt!r}; known: {sorted(_FORMAT_CODE)}")
    if x.dim() != 2 or not x.is_floating_point():
        raise KernelError(f"fp8_quantize takes a matrix of floating-point numbers, got {x.dtype} of shape {tuple(x.shape)}")
    if not (rows or cols):
        raise KernelError("fp8_quantize: neither rows nor columns are wanted")
    if max(x.shape) > _MOST:
        raise KernelError(f"fp8_quantize: {tuple(x.shape)} is too large")
    if not (x.is_cuda and x.dtype == torch.bfloat16):
        return _statement(x, fmt, square) if rows else None, _statement(x.t(), fmt, square) if cols else None
    require_current_device("fp8_quantize", x)
    status_word(x.device)                     # the native call takes over from the next one on
    M, N = x.shape
    r = _empty(M, N, fmt, x.device) if rows else None
    c = _empty(N, M, fmt, x.device) if cols else None
    if not x.numel():
        return r, c
    x = _rows_readable(x, "an 8-bit quantisation")
    _check(lib().kb_fp8_quantize(x.data_ptr(), M, N, x.stride(0) if M > 1 else N,
                                 r.data.data_ptr() if rows else 0, r.data.stride(0) if rows else 0, r.scales.data_ptr() if rows else 0,
                                 c.data.data_ptr() if cols else 0, c.data.stride(0) if cols else 0, c.scales.data_ptr() if cols else 0,
                                 1 if square else 0, _FORMAT_CODE[fmt], _stream()), f"fp8_quantize {M}x{N}")
    _count()
    return r, c


def _operand(m: Fp8Matrix, what: str):
    """The bytes with rows that TMA can read, and their stride."""
    d = m.data
    ld = d.stride(0) if d.shape[0] > 1 else -(-d.shape[1] // 16) * 16
    if d.stride(1) != 1 or ld % 16 or ld < d.shape[1] or d.data_ptr() % 16 or m.scales.data_ptr() % 16:
        raise KernelError(f"{what}: rows have to be contiguous and start on 16 bytes, got strides {tuple(d.stride())}")
    return d, ld


def gemm(a: Fp8Matrix, b: Fp8Matrix, out_dtype=None, accumulate=None, out=None):
    if (_entry._OPS is not None and out is None and out_dtype is None and type(a) is Fp8Matrix and type(b) is Fp8Matrix
            and _DTYPE.get(a.fmt) is a.data.dtype and _DTYPE.get(b.fmt) is b.data.dtype):
        r = _entry._OPS.fp8_gemm(a.data, a.scales, b.data, b.scales, accumulate)
        if r is not None:
            return r
    _check_matrix(a, "fp8_gemm a")
    _check_matrix(b, "fp8_gemm b")
    (M, K), (N, Kb) = a.shape, b.shape
    if K != Kb:
        raise ValueError(f"fp8_gemm shape mismatch: K={K} vs {Kb}")
    if max(M, N, K) > _MOST:
        raise KernelError(f"fp8_gemm: {M} x {N} x {K} is too large")
    if accumulate is not None and (out is not None or out_dtype is not None):
        raise KernelError("fp8_gemm: accumulate names the result, out and out_dtype cannot be given with it")
    if out is not None and out_dtype is not None and out.dtype != out_dtype:
        raise KernelError(f"fp8_gemm: out is {out.dtype}, out_dtype {out_dtype}")
    dest = accumulate if accumulate is not None else out
    if dest is not None and tuple(dest.shape) != (M, N):
        raise KernelError(f"fp8_gemm: the result is {(M, N)}, got a destination of {tuple(dest.shape)}")
    tensors = [a.data, b.data] + ([] if dest is None else [dest])
    if len({t.device for t in tensors}) != 1:
        raise KernelError(f"fp8_gemm: operands on several devices: {[str(t.device) for t in tensors]}")
    if not a.data.is_cuda:
        r = ref.fp8_gemm((a.data, a.scales), (b.data, b.scales), out_dtype or (torch.bfloat16 if out is None else out.dtype), accumulate)
        return r if out is None else out.copy_(r)
    require_current_device("fp8_gemm", a.data)
    if accumulate is not None and accumulate.dtype != torch.float32:
        raise KernelError(f"fp8_gemm accumulates in fp32, got {accumulate.dtype}")
    dt = dest.dtype if dest is not None else out_dtype or torch.bfloat16
    if dt not in (torch.bfloat16, torch.float32):
        raise KernelError(f"fp8_gemm results are bf16 or fp32, not {dt}")
    if dest is None:
        dest = torch.empty(M, N, dtype=dt, device=a.data.device)
    if not dest.numel():
        return dest
    ldc = dest.stride(0) if M > 1 else N
    if dest.stride(1) != 1 and N > 1 or ldc < N:
        raise KernelError(f"fp8_gemm: the destination's rows have to be contiguous, got strides {tuple(dest.stride())}")
    if not K:
        return dest if accumulate is not None else dest.zero_()
    (da, lda), (db, ldb) = _operand(a, "fp8_gemm a"), _operand(b, "fp8_gemm b")
    _check(lib().kb_gemm_fp8(da.data_ptr(), a.scales.data_ptr(), _FORMAT_CODE[a.fmt], lda, db.data_ptr(), b.scales.data_ptr(),
                             _FORMAT_CODE[b.fmt], ldb, dest.data_ptr(), ldc, M, N, K, 1 if dt == torch.float32 else 0,
                             1 if accumulate is not None else 0, status_word(da.device).data_ptr(), _stream()),
           f"fp8_gemm M={M} N={N} K={K}")
    _count()
    return dest
