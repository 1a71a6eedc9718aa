"""Root-mean-square norm of rows: with the residual's addition, with an 8-bit result for the block-scaled
products, and its gradient.

    h = x + residual          y = h * w / sqrt(mean(h ** 2) + eps)

Rows are the last dimension of a 2-D CUDA tensor (bf16, fp16 or fp32) whose rows may lie apart; the weight has
the type of the rows or is fp32.  Everything is computed in fp32 and rounded once.
"""
from __future__ import annotations

import torch

from .. import _native as N
from ..utils.tracing import traced
from .gemm import GemmError

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


class NormError(GemmError):
    pass


def _rows(t, name, like=None):
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dim() == 2 and t.dtype in _TYPES
            and (t.stride(1) == 1 or t.shape[1] == 1)):
        raise NormError(f"{name} must be a 2-D CUDA tensor of bf16, fp16 or fp32 with dense rows")
    if like is not None and (t.shape != like.shape or t.dtype != like.dtype or t.device != like.device):
        raise NormError(f"{name} must have x's shape, type and device")


def _weight(w, x):
    if not (isinstance(w, torch.Tensor) and w.is_cuda and w.is_contiguous() and w.dim() == 1
            and w.shape[0] == x.shape[1] and w.dtype in (x.dtype, torch.float32) and w.device == x.device):
        raise NormError("weight must be a contiguous CUDA vector of the row's length, of x's type or fp32")
    return int(w.dtype == torch.float32)


def _new(stream, like, shape, dtype):
    return like.new_empty(shape, dtype=dtype) if stream is None else N.new_empty_on(stream, like, shape, dtype)


def _forward(x, weight, residual, eps, mode, status_ptr, stream):
    if stream is None:
        r = N.fast().rms_norm(x, weight, residual, eps, mode, status_ptr)
        if r is not None:
            return r
    _rows(x, "x")
    w_f32 = _weight(weight, x)
    if residual is not None:
        _rows(residual, "residual", x)
    rows, d = x.shape
    if mode and d % 128:
        raise NormError("the 8-bit form wants rows of a multiple of 128 elements")
    h = _new(stream, x, (rows, d), x.dtype) if residual is not None else None
    y = _new(stream, x, (rows, d), torch.float8_e4m3fn if mode else x.dtype)
    s = _new(stream, x, (rows, d // 128), torch.float32) if mode else None
    sf = _new(stream, x, ((d // 128 + 3) // 4, rows), torch.int32) if mode == 2 else None
    with torch.cuda.device(x.device):
        rc = N.load().cb_rms_norm(
            x.data_ptr(), residual.data_ptr() if residual is not None else 0, weight.data_ptr(), y.data_ptr(),
            h.data_ptr() if h is not None else 0, s.data_ptr() if mode else 0, sf.data_ptr() if mode == 2 else 0,
            x.stride(0), residual.stride(0) if residual is not None else 0, rows, d, _TYPES[x.dtype], w_f32, mode,
            eps, status_ptr, N.raw_stream(stream))
    if rc != 0:
        raise NormError(f"rms_norm failed: {N.last_error()}")
    return y, s, sf, h


@traced("cb200.rms_norm")
def rms_norm(x, weight, residual=None, eps: float = 1e-6, status_ptr: int = 0, stream=None):
    """``y`` [rows, D] in x's type; with ``residual`` ``(y, h)``, ``h = x + residual`` rounded to x's type
    (``y`` is computed from the sum before that rounding)."""
    y, _, _, h = _forward(x, weight, residual, eps, 0, status_ptr, stream)
    return y if residual is None else (y, h)


@traced("cb200.rms_norm_quant")
def rms_norm_quant(x, weight, residual=None, eps: float = 1e-6, pow2: bool = False, status_ptr: int = 0,
                   stream=None):
    """The normalised rows as e4m3 with one scale per row and 128 columns, rounded once from fp32.

    ``(q, scales, h)`` in the form of :func:`ops.gemm.quantize_blockscaled`, for ``gemm_fp8_blockscaled``; with
    ``pow2`` ``(q, scales, sf, h)`` as :func:`ops.gemm.quantize_blockscaled_pow2` gives them, for ``gemm_fp8_mx``.
    ``h`` is None without a residual."""
    q, s, sf, h = _forward(x, weight, residual, eps, 2 if pow2 else 1, status_ptr, stream)
    return (q, s, sf, h) if pow2 else (q, s, h)


@traced("cb200.rms_norm_backward")
def rms_norm_backward(dy, h, weight, dh=None, eps: float = 1e-6, status_ptr: int = 0, stream=None):
    """``(dx, dw)`` from the gradient ``dy`` of the normalised rows: ``h`` is what was normalised (x, or the sum
    that :func:`rms_norm` returned with it), ``dh`` the gradient that reaches that sum on its other way.  ``dx``
    is the gradient of x and of the residual alike; ``dw`` is fp32, summed in a fixed order."""
    if stream is None:
        r = N.fast().rms_norm_backward(dy, h, weight, dh, eps, status_ptr)
        if r is not None:
            return r
    _rows(h, "h")
    _rows(dy, "dy", h)
    if dh is not None:
        _rows(dh, "dh", h)
    w_f32 = _weight(weight, h)
    rows, d = h.shape
    dx = _new(stream, h, (rows, d), h.dtype)
    dw = _new(stream, h, (d,), torch.float32)
    if rows == 0:
        with torch.cuda.stream(stream if stream is not None else torch.cuda.current_stream(h.device)):
            return dx, dw.zero_()
    lib = N.load()
    args = (dy.data_ptr(), h.data_ptr(), weight.data_ptr(), dh.data_ptr() if dh is not None else 0, dx.data_ptr())
    shape = (dy.stride(0), h.stride(0), dh.stride(0) if dh is not None else 0, rows, d, _TYPES[h.dtype], w_f32)
    with torch.cuda.device(h.device):
        n = lib.cb_rms_norm_backward_floats(*args, *shape)
        if n < 0:
            raise NormError(f"rms_norm_backward failed: {N.last_error()}")
        part = h.new_empty((n,), dtype=torch.float32) if stream is None else \
            N.new_empty_on(stream, h, (n,), torch.float32, handed_out=False)
        rc = lib.cb_rms_norm_backward(*args, dw.data_ptr(), part.data_ptr(), *shape, eps, status_ptr,
                                      N.raw_stream(stream))
    if rc != 0:
        raise NormError(f"rms_norm_backward failed: {N.last_error()}")
    return dx, dw
