"""A linear layer on block-scaled operands, on PyTorch-ROCm tensors: bias, activation and residual in the product's epilogue.

  block_scaled_linear               act(A @ W.T + bias) + residual of quantised operands, rounded or quantised again (serving)
  linear                            the same of float tensors, differentiable: every product of a training step block-scaled (MXFP8)
  linear_forward / linear_backward  the same without autograd (both can be captured)

The reference's sample stops at the product (samples/BlockScaledMatMul.py:229-297).  Checks, errors and streams are those of ``ops.py``
and ``ffn.py``: work is enqueued on the current stream of the tensors' device, nothing synchronises, and there is no PyTorch or CPU
compute fallback.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib as L
from .errors import TileTypeError, TileValueError
from .ffn import _FLOATS, _call, _codes, _mode, _no_tangents, _ref, _rows, _same_device
from .ops import _FMT_CODE, PackedScales, _as_u8, _dtype_name, _elem_format, _opts, _raise_code, _scale_code, _scale_desc, _workspace

_ACTS = {None: L.MX_ACT_NONE, "relu": L.MX_ACT_RELU, "gelu": L.MX_ACT_GELU, "gelu_tanh": L.MX_ACT_GELU_TANH, "silu": L.MX_ACT_SILU}


def _act(activation) -> int:
    if activation not in _ACTS:
        raise TileValueError(f"unknown activation {activation!r}; expected None, 'relu', 'gelu', 'gelu_tanh' or 'silu'")
    return _ACTS[activation]


def _opt(t):
    return None if t is None else _ref(t)


def _around(bias, residual, shape):
    """Checks bias (N,) and residual (..., N) of a result of this shape."""
    for name, t in (("bias", bias), ("residual", residual)):
        if t is not None and t.dtype not in _FLOATS:
            raise TileTypeError(f"Unsupported dtype {_dtype_name(t.dtype)} for {name}, expected float32, bfloat16 or float16")
    if bias is not None and tuple(bias.shape) != (shape[-1],):
        raise ValueError(f"bias must be ({shape[-1]},), got {tuple(bias.shape)}")
    if residual is not None and tuple(residual.shape) != tuple(shape):
        raise ValueError(f"residual must be {tuple(shape)}, got {tuple(residual.shape)}")


def block_scaled_linear(A: torch.Tensor, A_scale, W: torch.Tensor, W_scale, bias: Optional[torch.Tensor] = None,
                        residual: Optional[torch.Tensor] = None, *, activation: Optional[str] = None, out_dtype=torch.bfloat16,
                        a_format: Optional[str] = None, w_format: Optional[str] = None, kernel: str = "auto"):
    """``act((A * A_scale) @ (W * W_scale).T + bias) + residual`` in one launch where the product's kernel can finish it.

    A (M, K) and W (N, K) hold MX elements as in :func:`block_scaled_matmul` (FP4 packed along K, ``"e2m1"`` formats for uint8
    storage); A_scale (M, K/32) and W_scale (N, K/32) are E8M0 tensors or :class:`PackedScales` (operand "a" / "b").  ``bias`` (N,) and
    ``residual`` (M, N) are float32, bfloat16 or float16; ``activation`` is None, "relu", "gelu" (exact), "gelu_tanh" or "silu".

    Returns (M, N) in ``torch.bfloat16`` or ``torch.float32``, or with ``out_dtype`` ``torch.float8_e4m3fn`` ``(q, scale)``, quantised from
    the unrounded result by the floor rule (N a multiple of 32): the left operand of the next product.  Sums are the scaled matrix
    instructions' (1.5e-5 of the result's norm; ``kernel="generic"`` sums in 32 bits, far slower), what is behind them is in 32 bits.  A NaN
    is NaN; gelu and silu of -inf are zero."""
    act = _act(activation)
    if kernel in L.KERNELS:
        r = L.host().linear_gemm(A, A_scale, W, W_scale, bias, residual, a_format, w_format, out_dtype, act, L.KERNELS[kernel])
        if type(r) is int:
            _raise_code(r)
        if r is not None:
            return r
    a_fmt, w_fmt = _elem_format(A, a_format), _elem_format(W, w_format)
    if a_fmt is None or w_fmt is None:
        bad = A if a_fmt is None else W
        raise TileTypeError(f"Unsupported input dtype {_dtype_name(bad.dtype)} for mma_scaled, supported input dtypes are "
                            "float8_e4m3fn, float8_e5m2, float4_e2m1fn")
    if A.dim() != 2 or W.dim() != 2:
        raise TileTypeError(f"Expect A and W to be 2D, got {tuple(A.shape)} and {tuple(W.shape)}")
    codes = out_dtype == "e4m3" or out_dtype == torch.float8_e4m3fn
    if not codes and out_dtype not in (torch.bfloat16, torch.float32):
        raise TileTypeError(f"Unsupported output dtype {out_dtype}, expected bfloat16, float32 or float8_e4m3fn")
    for name, s in (("A_scale", A_scale), ("W_scale", W_scale)):
        if not isinstance(s, PackedScales) and _scale_code(s) != L.MX_E8M0:
            raise TileTypeError(f"Unsupported scale dtype {_dtype_name(s.dtype)} for {name}, supported scale dtypes are "
                                "float8_e8m0fnu")
    dA = L.desc(_as_u8(A), _FMT_CODE[a_fmt], 1 if a_fmt == "e2m1" else -1)
    dW = L.desc(_as_u8(W), _FMT_CODE[w_fmt], 1 if w_fmt == "e2m1" else -1)
    (M, K), (N, Kw) = dA.shape[:2], dW.shape[:2]
    if K != Kw:
        raise ValueError(f"Incompatible matrices: K dimension of A ({K}) must match K dimension of W ({Kw})")
    if codes and N % 32 != 0:
        raise ValueError(f"W must have a multiple of 32 rows for a quantised result, got {N}")
    _around(bias, residual, (M, N))
    dev = _same_device(A, W, *(s.data if isinstance(s, PackedScales) else s for s in (A_scale, W_scale)), *(t for t in (bias, residual) if t is not None))
    bias = None if bias is None else bias.detach().contiguous()
    residual = None if residual is None else _rows(residual.detach())
    dAs, la = _scale_desc(A_scale, M, K, 32, False)
    dWs, lw = _scale_desc(W_scale, N, K, 32, True)
    o = _opts(False, la, lw, kernel, 32)
    if codes:
        c = _codes(M, N, dev)
        outs = c.refs(L.MX_E4M3)
    else:
        c = torch.empty((M, N), dtype=out_dtype, device=dev)
        outs = (_ref(c), None)
    lib = L.lib()
    need = lib.mx_linear_gemm_workspace_bytes(M, N, K, ctypes.byref(o))
    ws = _workspace(dev, need)
    _call(dev, lib.mx_linear_gemm, ctypes.byref(dA), ctypes.byref(dAs), ctypes.byref(dW), ctypes.byref(dWs), _opt(bias), _opt(residual), act, *outs, None,
          ctypes.byref(o), ws.data_ptr() if ws is not None else None, need)
    return c.views(torch.float8_e4m3fn) if codes else c


class LinearState(NamedTuple):
    """What :func:`linear_forward` leaves for the backward pass."""
    saved: torch.Tensor   # uint8: input and weight along their columns in 8.25 bits an element, with an activation its argument in bf16
    T: int
    K: int
    N: int
    x_dtype: torch.dtype
    w_dtype: torch.dtype
    bias_dtype: Optional[torch.dtype]
    activation: Optional[str]
    scale_mode: str


def _check(x, w, bias, residual):
    for name, t in (("x", x), ("w", w)):
        if t.dtype not in (torch.float32, torch.bfloat16):
            raise TileTypeError(f"Unsupported dtype {_dtype_name(t.dtype)} for {name}, expected float32 or bfloat16")
    if x.dim() < 2 or w.dim() != 2:
        raise TileTypeError(f"Expect x (..., K) and w (N, K), got {tuple(x.shape)} and {tuple(w.shape)}")
    K, N = x.shape[-1], w.shape[0]
    if w.shape[1] != K:
        raise ValueError(f"w must be (N, {K}) for x {tuple(x.shape)}, got {tuple(w.shape)}")
    if K == 0 or N == 0 or K % 32 or N % 32:
        raise ValueError(f"K ({K}) and N ({N}) must be multiples of 32")
    _around(bias, residual, (*x.shape[:-1], N))
    return _same_device(x, w, *(t for t in (bias, residual) if t is not None)), K, N


def _forward(x, w, bias, residual, act: int, mode: int, train: bool):
    r = L.host().linear(x, w, bias, residual, act, mode, 1 if train else 0)
    if type(r) is int:
        _raise_code(r)
    if r is not None:
        return r if train else (r, None)
    if not train:
        _no_tangents("linear", x, w, bias, residual)
    dev, K, N = _check(x, w, bias, residual)
    x2, w2, b2 = _rows(x.detach()), _rows(w.detach()), None if bias is None else bias.detach().contiguous()
    r2 = None if residual is None else _rows(residual.detach())
    T = x2.shape[0]
    lib = L.lib()
    y = torch.empty((T, N), dtype=x.dtype, device=dev)
    kept = lib.mx_linear_saved_bytes(T, K, N, act) if train else 0
    saved = torch.empty(kept, dtype=torch.uint8, device=dev) if train else None
    need = lib.mx_linear_forward_workspace_bytes(T, K, N)
    ws = _workspace(dev, need)
    _call(dev, lib.mx_linear_forward, _ref(x2), _ref(w2), _opt(b2), _opt(r2), act, _ref(y), mode, saved.data_ptr() if kept else None, kept,
          ws.data_ptr() if ws is not None else None, need)
    return y.reshape(*x.shape[:-1], N), saved


def linear_forward(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None, *,
                   activation: Optional[str] = None, scale_mode: str = "floor"):
    """:func:`linear` without autograd: returns ``(y, state)``, and ``linear_backward(dy, state)`` the gradients of x, w and bias (that of
    the residual is ``dy``).  Both can be captured into a HIP graph."""
    y, saved = _forward(x, w, bias, residual, _act(activation), _mode(scale_mode), True)
    K = x.shape[-1]
    return y, LinearState(saved, x.numel() // K, K, w.shape[0], x.dtype, w.dtype, None if bias is None else bias.dtype, activation, scale_mode)


def linear_backward(dy: torch.Tensor, state: LinearState, *, need_dx: bool = True, need_dw: bool = True, need_dbias: bool = True):
    """Gradients ``(dx, dw, dbias)`` of :func:`linear_forward` for the gradient ``dy`` (..., N) of its result, in the dtypes of x, w and
    bias (``dx`` in the shape of ``dy`` but for its last axis); None where not asked for, and dbias where there was no bias.  Reads the
    state and leaves it as it is, so it can be called again with another ``dy``."""
    s = state
    act, need_dbias = _act(s.activation), need_dbias and s.bias_dtype is not None
    r = L.host().linear_backward(dy, s.saved, s.T, s.K, s.N, s.x_dtype, s.w_dtype, s.bias_dtype if need_dbias else torch.float32, need_dx, need_dw,
                                 need_dbias, act, _mode(s.scale_mode))
    if type(r) is tuple:
        return r if dy.dim() == 2 or not need_dx else (r[0].view(*dy.shape[:-1], s.K), r[1], r[2])
    if r is not None:
        _raise_code(r)
    if dy.dtype not in _FLOATS:
        raise TileTypeError(f"Unsupported gradient dtype {_dtype_name(dy.dtype)}, expected float32, bfloat16 or float16")
    if dy.dim() < 2 or dy.shape[-1] != s.N or dy.numel() != s.T * s.N:
        raise ValueError(f"dy must hold {s.T} rows of {s.N}, got {tuple(dy.shape)}")
    dev = _same_device(dy, s.saved)
    make = torch.empty if s.T else torch.zeros    # no tokens: the sums over them are zeros
    dx = torch.empty((s.T, s.K), dtype=s.x_dtype, device=dev) if need_dx else None
    dw = make((s.N, s.K), dtype=s.w_dtype, device=dev) if need_dw else None
    db = make(s.N, dtype=s.bias_dtype, device=dev) if need_dbias else None
    if s.T and (need_dx or need_dw or need_dbias):
        lib = L.lib()
        dy2 = _rows(dy.detach())
        if s.T > 1 and dy2.stride(0) > 1 << 25:    # rows farther apart than the library takes them
            dy2 = dy2.contiguous()
        need = lib.mx_linear_backward_workspace_bytes(s.T, s.K, s.N)
        ws = _workspace(dev, need)
        _call(dev, lib.mx_linear_backward, _ref(dy2), s.saved.data_ptr(), s.saved.numel(), s.K, act, _opt(dx), _opt(dw), _opt(db), _mode(s.scale_mode),
              ws.data_ptr(), need)
    return dx.reshape(*dy.shape[:-1], s.K) if need_dx else None, dw, db


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, residual, activation, scale_mode):
        y, state = linear_forward(x, w, bias, residual, activation=activation, scale_mode=scale_mode)
        ctx.save_for_backward(state.saved)
        ctx.state = state._replace(saved=None)
        ctx.residual_dtype = None if residual is None else residual.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        state = ctx.state._replace(saved=ctx.saved_tensors[0])
        need = ctx.needs_input_grad
        grads = linear_backward(dy, state, need_dx=need[0], need_dw=need[1], need_dbias=need[2])
        return (*grads, dy.to(ctx.residual_dtype) if need[3] else None, None, None)


def linear(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None, *,
           activation: Optional[str] = None, scale_mode: str = "floor") -> torch.Tensor:
    """``act(x @ w.T + bias) + residual``, every product of the forward and of the backward pass block-scaled in MXFP8 (E4M3),
    differentiable in x, w, bias and residual.

    x (..., K) and w (N, K) are float32 or bfloat16, K and N multiples of 32; ``bias`` (N,) and ``residual`` (..., N) float32, bfloat16 or
    float16; ``activation`` None, "relu", "gelu" (exact), "gelu_tanh" or "silu".  The result has the dtype of x, every gradient the dtype of
    what it is the gradient of.  Each operand is quantised along the axis that its product sums over.  The backward pass is kept input and
    weight in 8.25 bits an element and, with an activation, its argument in bfloat16; neither x nor w is kept, so they may be updated in
    place in between.  No operand may have 2^31 elements or more.

    With few tokens (up to 64, or tokens times N up to 2^19) the activation's argument is summed in 32 bits; with more, its sums are the
    scaled matrix instructions' (:func:`block_scaled_linear`).  Under the floor rule an infinity of the input or of the gradient counts as
    the largest number of its block, so gradients made of it may be finite; ``scale_mode="ceil"`` makes its block NaN.

    With gradients enabled the call refuses to be captured into a HIP graph (autograd accumulates a leaf's gradient on the stream that
    first used it, which a capture must not touch): capture :func:`linear_forward` and :func:`linear_backward`.  Inputs of forward-mode
    differentiation are refused."""
    act, mode = _act(activation), _mode(scale_mode)
    if not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, w, bias, residual))):
        return _forward(x, w, bias, residual, act, mode, False)[0]
    r = L.host().linear(x, w, bias, residual, act, mode, 2)
    if type(r) is int:
        _raise_code(r)
    if r is not None:
        return r
    _no_tangents("linear", x, w, bias, residual)
    if x.is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("linear with gradients cannot be captured into a graph: capture linear_forward and linear_backward")
    return _Linear.apply(x, w, bias, residual, activation, scale_mode)
