"""Layer norm in front of a block-scaled product, on PyTorch-ROCm tensors.

  layer_norm              (x - mean) * rstd * weight + bias, differentiable
  layer_norm_forward      the same with what its backward pass needs, layer_norm_backward the gradients (both can be captured)
  layer_norm_quantize     the result MX-quantised in the same pass, ready for a product

No reference counterpart among the ported paths.  Checks, errors and streams are those of ``ops.py`` and ``ffn.py``: work is enqueued
on the current stream of the tensors' device, nothing synchronises, and there is no PyTorch or CPU compute fallback.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _lib as L
from .errors import TileTypeError, TileValueError
from .ffn import _ELEM8, _FLOATS, _call, _mode, _no_tangents, _ref, _rows, _same_device, _up32
from .ops import _DTYPE_FMT, _FMT_CODE, _dtype_name, _raise_code, _workspace


def _check(x, weight, bias, eps):
    for name, t in (("x", x), ("weight", weight), ("bias", bias)):
        if t is not None and t.dtype not in _FLOATS:
            raise TileTypeError(f"Unsupported dtype {_dtype_name(t.dtype)} for {name}, expected float32, bfloat16 or float16")
    if not (math.isfinite(eps) and eps >= 0):
        raise TileValueError(f"eps must be a number of at least zero, got {eps}")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise TileTypeError(f"Expect x (..., H) with at least one column, got {tuple(x.shape)}")
    H = x.shape[-1]
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and tuple(t.shape) != (H,):
            raise ValueError(f"{name} must be ({H},) for x {tuple(x.shape)}, got {tuple(t.shape)}")
    dev = _same_device(x, *(t for t in (weight, bias) if t is not None))
    return dev, H


def _vector(t):
    return None if t is None else t.detach().contiguous()


def _opt(t):
    return None if t is None else _ref(t)


def _forward(x, weight, bias, eps, stats):
    r = L.host().layer_norm(x, weight, bias, eps, 1 if stats else 0)
    if type(r) is int:
        _raise_code(r)
    if r is not None:
        return r if stats else (r, None, None)
    if not stats:
        _no_tangents("layer_norm", x, weight, bias)
    dev, H = _check(x, weight, bias, eps)
    x2, w, b = _rows(x.detach()), _vector(weight), _vector(bias)
    T = x2.shape[0]
    y = torch.empty((T, H), dtype=x.dtype, device=dev)
    mean, rstd = (torch.empty(T, dtype=torch.float32, device=dev) if stats else None for _ in range(2))
    _call(dev, L.lib().mx_layer_norm, _ref(x2), _opt(w), _opt(b), float(eps), _ref(y), _opt(mean), _opt(rstd))
    return y.reshape(x.shape), mean, rstd


def layer_norm_forward(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *, eps: float = 1e-5):
    """:func:`layer_norm` without autograd: returns ``(y, mean, rstd)``, mean and rstd float32, one for each row, as
    :func:`layer_norm_backward` takes them.  Both can be captured into a HIP graph."""
    return _forward(x, weight, bias, eps, True)


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor, weight: Optional[torch.Tensor] = None, *,
                        need_dx: bool = True, need_dweight: bool = True, need_dbias: bool = True):
    """Gradients ``(dx, dweight, dbias)`` of :func:`layer_norm_forward`; None where not asked for.  ``dy`` has the shape and dtype of
    ``x``; ``dx`` is in that dtype, ``dweight`` and ``dbias`` in that of ``weight`` (float32 without one).  Sums over the rows are in 32
    bits and in a fixed order: the same call gives the same bits."""
    r = L.host().layer_norm_backward(dy, x, mean, rstd, weight, need_dx, need_dweight, need_dbias)
    if type(r) is tuple:
        return r
    if r is not None:
        _raise_code(r)
    return _backward(dy, x, mean, rstd, weight, need_dx, need_dweight, need_dbias, torch.float32 if weight is None else weight.dtype)


def _backward(dy, x, mean, rstd, weight, need_dx, need_dweight, need_dbias, bias_dtype):
    _check(x, weight, None, 0.0)
    dev = _same_device(x, dy, mean, rstd)
    if dy.dtype != x.dtype:
        raise TileTypeError(f"dy must have the dtype of x ({_dtype_name(x.dtype)}), got {_dtype_name(dy.dtype)}")
    if dy.shape != x.shape:
        raise ValueError(f"dy must have the shape of x {tuple(x.shape)}, got {tuple(dy.shape)}")
    x2, dy2, w, m2, r2 = _rows(x.detach()), _rows(dy.detach()), _vector(weight), _vector(mean), _vector(rstd)
    T, H = x2.shape
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t.dtype != torch.float32 or tuple(t.shape) != (T,):
            raise ValueError(f"{name} must be ({T},) float32 as the forward pass leaves it, got {tuple(t.shape)} {_dtype_name(t.dtype)}")
    make = torch.empty if T else torch.zeros    # no rows: the sums over them are zeros
    dx = torch.empty((T, H), dtype=x.dtype, device=dev) if need_dx else None
    dw = make(H, dtype=torch.float32 if weight is None else weight.dtype, device=dev) if need_dweight else None
    db = make(H, dtype=bias_dtype, device=dev) if need_dbias else None
    if T and (need_dx or need_dweight or need_dbias):
        lib = L.lib()
        need = lib.mx_layer_norm_backward_workspace_bytes(T, H)
        ws = _workspace(dev, need)
        _call(dev, lib.mx_layer_norm_backward, _ref(dy2), _ref(x2), _ref(m2), _ref(r2), _opt(w), _opt(dx), _opt(dw), _opt(db),
              ws.data_ptr(), need)
    return (dx.reshape(x.shape) if need_dx else None), dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps=eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad
        return (*_backward(dy.to(x.dtype), x, mean, rstd, weight, need[0], need[1], need[2], ctx.bias_dtype), None)   # (sums are rounded once)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *, eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis, differentiable in x, weight and bias.

    x (..., H), weight and bias (H,) or None (ones, zeros) are float32, bfloat16 or float16, of the same dtype or not; the result has
    that of x, every gradient that of what it is the gradient of.  In 32 bits with one rounding at the end; the variance is that of
    the differences from the mean.  A row with a NaN or an infinity is NaN, and one whose sum passes 3.4e38; where the sum of the squared differences
    does (differences around 1e19), 1 / sqrt of it is zero.

    With gradients enabled the call refuses to be captured into a HIP graph (autograd accumulates a leaf's gradient on the stream that
    first used it, which a capture must not touch): capture :func:`layer_norm_forward` and :func:`layer_norm_backward`.  Inputs of
    forward-mode differentiation are refused."""
    if not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias))):
        return _forward(x, weight, bias, eps, False)[0]
    r = L.host().layer_norm(x, weight, bias, eps, 2)
    if type(r) is int:
        _raise_code(r)
    if r is not None:
        return r
    _no_tangents("layer_norm", x, weight, bias)
    if x.is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("layer_norm with gradients cannot be captured into a graph: capture layer_norm_forward and layer_norm_backward")
    return _LayerNorm.apply(x, weight, bias, eps)


def layer_norm_quantize(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, dtype=torch.float8_e4m3fn, *,
                        eps: float = 1e-5, scale_mode: str = "floor"):
    """:func:`layer_norm` whose result leaves MX-quantised, in one pass: ``(q, scale)`` as :func:`block_quantize` gives them of the
    unrounded result (last axis zero-padded to a multiple of 32), the left operand of a block-scaled product.

    ``dtype``: ``torch.float8_e4m3fn``, ``torch.float8_e5m2`` or ``"e2m1"`` (FP4, two per byte); ``scale_mode`` as in
    :func:`block_quantize`.  H is at least 32.  No autograd: for serving."""
    mode = _mode(scale_mode)
    r = L.host().layer_norm_quantize(x, weight, bias, dtype, eps, mode)
    if type(r) is tuple:
        return r
    if r is not None:
        _raise_code(r)
    fmt = dtype if isinstance(dtype, str) else _DTYPE_FMT.get(dtype)
    if fmt not in _FMT_CODE:
        raise TileTypeError(f"Unsupported quantisation dtype {dtype} for layer_norm_quantize, expected float8_e4m3fn, float8_e5m2 or \"e2m1\"")
    dev, H = _check(x, weight, bias, eps)
    if H < 32:
        raise ValueError(f"The requested block size 32 is larger than the inner most dimension of the input tensor {H}")
    x2, w, b = _rows(x.detach()), _vector(weight), _vector(bias)
    rows, Hp, fp4 = x2.shape[0], _up32(H), fmt == "e2m1"
    q = torch.empty((rows, Hp // 2 if fp4 else Hp), dtype=torch.uint8, device=dev)
    scale = torch.empty((rows, Hp // 32), dtype=torch.uint8, device=dev)
    _call(dev, L.lib().mx_layer_norm_quantize, _ref(x2), _opt(w), _opt(b), float(eps),
          ctypes.byref(L.desc(q, _FMT_CODE[fmt], 1 if fp4 else -1)), _ref(scale, L.MX_E8M0), mode)
    lead = x.shape[:-1]
    if not fp4:
        q = q.view(_ELEM8[fmt])
    return q.reshape(*lead, q.shape[-1]), scale.view(torch.float8_e8m0fnu).reshape(*lead, Hp // 32)
