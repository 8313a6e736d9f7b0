"""Products in 8-bit integers with a scale per position and per channel (``afb_int8_linear``, include/afb.h).

The reference's dense maps are float32 layers (chessfly/model.py:95-105).  For inference that can give up
some of that accuracy, ``quantize`` turns a matrix into int8 with one float32 scale per row and
``int8_linear`` computes

    y_ij = (sum_k q_ik w_jk) s_i t_j + b_j        q_ik = rint(x_ik / s_i),  s_i = max_k |x_ik| / 127

with exact int32 sums.  Weights are quantised once (``quantize(layer.weight)``), positions within the call.
A row of x that holds an infinity or a NaN gives a row of NaN; the other rows do not see it.

These are products of inference.  Rounding has no gradient: ``quantize`` returns none, and a backward that comes to a
product with an input that wants one fails.
"""

from __future__ import annotations

import torch

from . import _lib
from .gemm import _device_status

TYPES = {torch.float32: _lib.T_F32, torch.float16: _lib.T_F16, torch.bfloat16: _lib.T_BF16}


def _source(x: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """(tensor, leading dimension, transposed) of a (rows, k) matrix as the library reads it."""
    rows, k = x.shape
    if x.stride(1) == 1 and x.stride(0) >= max(k, 1):
        return x, x.stride(0), 0
    if x.stride(0) == 1 and x.stride(1) >= max(rows, 1):
        return x, x.stride(1), 1
    return x.contiguous(), max(k, 1), 0


def _check_source(x: torch.Tensor, norm) -> None:
    if x.dim() != 2:
        raise ValueError(f"x must be (rows, k), got {tuple(x.shape)}")
    if x.dtype not in TYPES:
        raise TypeError(f"x must be float32, float16 or bfloat16, not {x.dtype}")
    if not x.is_cuda:
        raise RuntimeError("x must be a CUDA tensor")
    if norm is not None:
        for name, t in (("mean", norm.mean), ("var", norm.var)):
            if t.shape != (x.shape[1],) or t.dtype != torch.float32 or t.device != x.device or not t.is_contiguous():
                raise ValueError(f"norm.{name} must be float32 ({x.shape[1]},) on x's device")


def _norm_args(norm):
    return (None, None, 0.0, 0.0) if norm is None else (norm.mean.data_ptr(), norm.var.data_ptr(), float(norm.eps), float(norm.clip))


def _rows16(q: torch.Tensor, device, name: str) -> torch.Tensor:
    """``q`` with rows that start on 16-byte boundaries (a copy if they do not)."""
    if q.dim() != 2 or q.dtype != torch.int8 or q.device != device:
        raise ValueError(f"{name} must be int8 (rows, k) on x's device")
    if q.stride(1) == 1 and q.stride(0) % 16 == 0 and q.stride(0) >= q.shape[1] and q.data_ptr() % 16 == 0:
        return q
    return empty_rows(*q.shape, device).copy_(q)


def _vector(t: torch.Tensor | None, n: int, device, name: str) -> torch.Tensor | None:
    if t is None:
        return None
    if t.shape != (n,) or t.dtype != torch.float32 or t.device != device:
        raise ValueError(f"{name} must be float32 ({n},) on x's device")
    return t if t.is_contiguous() else t.contiguous()


def empty_rows(rows: int, k: int, device) -> torch.Tensor:
    """An uninitialised (rows, k) int8 matrix: its rows start on 128-byte boundaries, so that each of the product's
    loads is one cache line (the library asks for 16; 2,048 x 838 -> 17937: 37.4 us against 45.5)."""
    return torch.empty(rows, max(-(-k // 128) * 128, 128), dtype=torch.int8, device=device)[:, :k]


def quantize(x: torch.Tensor, norm=None) -> tuple[torch.Tensor, torch.Tensor]:
    """x (rows, k) float32, float16 or bfloat16, contiguous or transposed -> (q int8 (rows, k), scale float32
    (rows,)) with x ~ q * scale[:, None].  ``norm``: a ``RunningNorm`` whose running statistics are applied to x
    first (its eval mode)."""
    _check_source(x, norm)
    rows, k = x.shape
    x, ld, trans = _source(x)
    q = empty_rows(rows, k, x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    with _lib.on_device(x.device):
        _lib.call("afb_quantize_rows", rows, k, TYPES[x.dtype], x.data_ptr(), ld, trans, *_norm_args(norm), q.data_ptr(),
                  q.stride(0), scale.data_ptr(), _lib.stream_of(x.device))
    return q, scale


def _result(rows: int, n: int, k: int, w, w_scale, bias, out_dtype, device):
    if out_dtype not in TYPES:
        raise TypeError(f"out_dtype must be float32, float16 or bfloat16, not {out_dtype}")
    if w.dim() != 2 or w.shape[1] != k:
        raise ValueError(f"inner dimensions differ: k = {k} and w {tuple(w.shape)}")
    w = _rows16(w, device, "w")
    # rows on 16 bytes let the kernel store through TMA; on 128, where that is little padding, its stores are whole lines
    size = 4 if out_dtype == torch.float32 else 2
    unit = (128 if n * size >= 1024 else 16) // size
    y = torch.empty_strided((rows, n), (-(-n // unit) * unit, 1), dtype=out_dtype, device=device)
    return w, _vector(w_scale, n, device, "w_scale"), _vector(bias, n, device, "bias"), y


class _NoGradient(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, *sources):
        return y.view_as(y)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("the 8-bit product has no gradient: detach its inputs, or run it under torch.no_grad()")


def _without_gradient(y: torch.Tensor, a: torch.Tensor, b: torch.Tensor, c: torch.Tensor | None) -> torch.Tensor:
    """``y``, computed from the others outside autograd: a backward that asks one of them for a gradient fails, where it
    would otherwise pass it by."""
    if torch.is_grad_enabled() and (a.requires_grad or b.requires_grad or (c is not None and c.requires_grad)):
        return _NoGradient.apply(y, a, b, c)
    return y


def _empty_sum(y: torch.Tensor, bias) -> torch.Tensor:
    """The product over k = 0."""
    y.zero_()
    return y if bias is None else y.add_(bias.detach().to(y.dtype))


def int8_matmul(q: torch.Tensor, scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: torch.Tensor | None = None,
                out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """(q w^T) * scale[:, None] * w_scale + bias, (rows, n) of ``out_dtype`` (rounded once), a view whose rows start
    on 16-byte boundaries.  q (rows, k) and
    w (n, k) int8 as ``quantize`` returns them (other layouts are copied), k <= 131071."""
    if q.dim() != 2:
        raise ValueError(f"q must be (rows, k), got {tuple(q.shape)}")
    if not q.is_cuda:
        raise RuntimeError("q must be a CUDA tensor")
    rows, k = q.shape
    n, dev = w.shape[0], q.device
    sources = scale, w_scale, bias
    q = _rows16(q, dev, "q")
    scale = _vector(scale, rows, dev, "scale")
    w, w_scale, bias, y = _result(rows, n, k, w, w_scale, bias, out_dtype, dev)
    if k == 0:
        return _without_gradient(_empty_sum(y, bias), *sources)
    with _lib.on_device(dev):
        _lib.call("afb_int8_matmul", rows, n, k, q.data_ptr(), q.stride(0), scale.data_ptr(), w.data_ptr(), w.stride(0),
                  w_scale.data_ptr(), bias.data_ptr() if bias is not None else None, y.data_ptr(), TYPES[out_dtype], y.stride(0),
                  _device_status(dev).data_ptr(), _lib.stream_of(dev))
    return _without_gradient(y, *sources)


def int8_linear(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: torch.Tensor | None = None, norm=None,
                out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """``quantize(x, norm)`` times the quantised weight: x (rows, k) float32, float16 or bfloat16, contiguous or a
    transposed view; w (n, k) int8 and w_scale (n,) from ``quantize``; bias (n,) float32.  (rows, n) of
    ``out_dtype``, a view whose rows start on 16-byte boundaries."""
    _check_source(x, norm)
    rows, k = x.shape
    n, dev = w.shape[0], x.device
    sources = x, w_scale, bias
    w, w_scale, bias, y = _result(rows, n, k, w, w_scale, bias, out_dtype, dev)
    if k == 0:
        return _without_gradient(_empty_sum(y, bias), *sources)
    x, ld, trans = _source(x)
    lib = _lib.load()
    size = lib.afb_int8_linear_workspace(rows, k)
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    with _lib.on_device(dev):
        _lib.check(lib.afb_int8_linear(rows, n, k, TYPES[x.dtype], x.data_ptr(), ld, trans, *_norm_args(norm), w.data_ptr(),
                                       w.stride(0), w_scale.data_ptr(), bias.data_ptr() if bias is not None else None,
                                       y.data_ptr(), TYPES[out_dtype], y.stride(0), ws.data_ptr() if size else None, size,
                                       _device_status(dev).data_ptr(), _lib.stream_of(dev)))
    return _without_gradient(y, *sources)
