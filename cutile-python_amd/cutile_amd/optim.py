"""AdamW over many tensors at once, states in 32 or in 8 bits, on PyTorch-ROCm tensors.

The step behind the gradients that :func:`gated_feed_forward`, :func:`layer_norm` and their like compute.  No reference counterpart (the
reference trains nothing).  Checks, errors and streams are those of ``ops.py``: work is enqueued on the current stream of the tensors'
device, nothing synchronises, and there is no PyTorch or CPU compute fallback.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Sequence

import torch

from . import _lib as L
from .errors import TileTypeError, TileValueError
from .ffn import _call, _same_device, _up32
from .ops import _dtype_name, _raise_code

_PARAMS = (torch.float32, torch.bfloat16)


class AdamWState(NamedTuple):
    """The state of one parameter.  32 bits: both moments float32, in the parameter's shape.  8 bits: ``exp_avg`` holds the first
    moment and ``exp_avg_sq`` the ROOT of the second, MXFP8: ``float8_e4m3fn`` elements (flat, padded to a multiple of 32) with one
    ``float8_e8m0fnu`` scale for 32 of them."""
    exp_avg: torch.Tensor
    exp_avg_sq: torch.Tensor
    exp_avg_scale: Optional[torch.Tensor] = None
    exp_avg_sq_scale: Optional[torch.Tensor] = None


def adamw_state(param: torch.Tensor, bits: int = 32) -> AdamWState:
    """The state of a parameter before its first step: zeros, 8 bytes an element (``bits`` 32) or 2.06 (8)."""
    if bits not in (8, 32):
        raise TileValueError(f"states have 8 or 32 bits, got {bits}")
    if param.dtype not in _PARAMS:
        raise TileTypeError(f"Unsupported parameter dtype {_dtype_name(param.dtype)}, expected float32 or bfloat16")
    if bits == 32:
        return AdamWState(*(torch.zeros(param.shape, dtype=torch.float32, device=param.device) for _ in range(2)))
    n = _up32(param.numel())
    zeros = [torch.zeros(k, dtype=torch.uint8, device=param.device) for k in (n, n, n // 32, n // 32)]
    return AdamWState(*(t.view(torch.float8_e4m3fn) for t in zeros[:2]), *(t.view(torch.float8_e8m0fnu) for t in zeros[2:]))


def _number(name, v, dtype, dev):
    """(host value, device address) of a number or of a tensor of one element."""
    if not isinstance(v, torch.Tensor):
        return (float(v) if dtype == torch.float32 else int(v)), None
    if v.dtype != dtype or v.numel() != 1 or v.device != dev:
        raise ValueError(f"{name} must be a number or one {_dtype_name(dtype)} element on {dev}, got {tuple(v.shape)} {_dtype_name(v.dtype)} on {v.device}")
    return 0, v.data_ptr()


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[Optional[torch.Tensor]], states: Sequence[AdamWState], *, step, lr=1e-3,
               betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01, grad_scale=1.0, seed: int = 0,
               copies: Optional[Sequence[Optional[torch.Tensor]]] = None) -> None:
    """One AdamW step of all parameters, in place, one launch for some fifty of them:

        g = grad * grad_scale;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
        param = param (1 - lr weight_decay) - lr / (1 - b1^step) m / (sqrt(v / (1 - b2^step)) + eps)

    in 32 bits.  Parameters and gradients are float32 or bfloat16, contiguous (a gradient that is not is copied first); a gradient of None
    leaves its parameter and state as they are.  ``copies``: bfloat16 tensors that receive the new parameters as well (what the products
    take of float32 masters).  ``step`` is the number of this step, from 1 on.  ``step`` (int64), ``lr`` and ``grad_scale`` (float32) may be
    tensors of one element on the device, read when the kernel runs: a captured graph then goes on counting.

    With 8-bit states (:func:`adamw_state`) elements are rounded up or down at random, since a step of ``b2`` = 0.999 is far
    smaller than the distance of two E4M3 numbers; the random bits are a hash of ``seed``, ``step``, the place in the list and
    the element, the same for the same arguments.  All states of a call have the same number of bits.  Parameters, states and copies must
    not overlap one another (a parameter listed twice is refused) nor what the kernel reads beside them: a gradient, or a ``step``, ``lr`` or
    ``grad_scale`` on the device; gradients may be the same.  A NaN or an infinity of a gradient reaches its parameter, and with 8-bit states the 31
    states that share its scale."""
    beta1, beta2 = betas
    r = L.host().adamw(params, grads, states, copies, step, lr, beta1, beta2, eps, weight_decay, grad_scale, seed)
    if r is True:
        return
    if r is not None:
        _raise_code(r)
    params, grads, states = list(params), list(grads), list(states)
    copies = [None] * len(params) if copies is None else list(copies)
    if not (len(params) == len(grads) == len(states) == len(copies)):
        raise ValueError(f"as many gradients, states and copies as parameters are needed: {len(params)} parameters, {len(grads)}, {len(states)}, {len(copies)}")
    if not params:
        return
    items, written = (L.MxAdamwTensor * len(params))(), []
    bits, dev, kept = None, None, []
    for i, (p, g, s, c) in enumerate(zip(params, grads, states, copies)):
        if p.dtype not in _PARAMS or (g is not None and g.dtype not in _PARAMS):
            bad = p if p.dtype not in _PARAMS else g
            raise TileTypeError(f"tensor {i}: unsupported dtype {_dtype_name(bad.dtype)}, expected float32 or bfloat16")
        dev = _same_device(p, *(t for t in (dev and params[0], g, *s, c) if t is not None))
        items[i].param_dtype, items[i].grad_dtype = L._TORCH_TO_MX[p.dtype], L.MX_F32
        if g is None:
            continue
        if g.layout != torch.strided or g.shape != p.shape:
            raise ValueError(f"tensor {i}: the gradient must be dense and of the parameter's shape {tuple(p.shape)}, got {tuple(g.shape)} {g.layout}")
        small = s[0].dtype != torch.float32
        if bits not in (None, 8 if small else 32):
            raise ValueError("the states of a call must all have 8 or all have 32 bits")
        bits, n = 8 if small else 32, p.numel()
        sizes = ((_up32(n), torch.float8_e4m3fn),) * 2 + ((_up32(n) // 32, torch.float8_e8m0fnu),) * 2 if small else ((n, torch.float32),) * 2
        for k, (count, dtype) in enumerate(sizes):
            if s[k] is None or s[k].numel() != count or s[k].dtype != dtype:
                raise ValueError(f"tensor {i}: state {k} must have {count} elements of {_dtype_name(dtype)}, as adamw_state makes it")
        if not small and (len(s) > 2 and (s[2] is not None or s[3] is not None)):
            raise ValueError(f"tensor {i}: states in 32 bits have no scales")
        if c is not None and (c.dtype != torch.bfloat16 or c.shape != p.shape):
            raise ValueError(f"tensor {i}: the copy must be bfloat16 of the parameter's shape {tuple(p.shape)}, got {tuple(c.shape)} {_dtype_name(c.dtype)}")
        mine = [p, *s[:len(sizes)], *([c] if c is not None else [])]
        if not all(t.is_contiguous() for t in mine):
            raise TileTypeError(f"tensor {i}: parameter, states and copy must be contiguous")
        kept.append(g.detach().contiguous())
        t = items[i]
        t.param, t.grad, t.n, t.grad_dtype = p.data_ptr(), kept[-1].data_ptr(), n, L._TORCH_TO_MX[g.dtype]
        t.exp_avg, t.exp_avg_sq = s[0].data_ptr(), s[1].data_ptr()
        if small:
            t.exp_avg_scale, t.exp_avg_sq_scale = s[2].data_ptr(), s[3].data_ptr()
        if c is not None:
            t.copy = c.data_ptr()
        written += mine
    o = L.MxAdamwOpts()
    o.struct_size, o.state_bits, o.seed = ctypes.sizeof(L.MxAdamwOpts), bits or 32, int(seed) & 0xFFFFFFFF
    o.step, o.step_at = _number("step", step, torch.int64, dev)
    o.lr, o.lr_at = _number("lr", lr, torch.float32, dev)
    o.grad_scale, o.scale_at = _number("grad_scale", grad_scale, torch.float32, dev)
    o.beta1, o.beta2, o.eps, o.weight_decay = float(beta1), float(beta2), float(eps), float(weight_decay)
    _call(dev, L.lib().mx_adamw_step, len(params), items, ctypes.byref(o))
    for t in written:
        if not t.is_inference():
            torch.autograd.graph.increment_version(t)
