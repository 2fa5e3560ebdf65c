"""A gated feed-forward block that is trained in 8 bits, and its parts, on PyTorch-ROCm tensors.

  block_quantize_both             MX codes of a matrix along its rows and, transposed, along its columns
  gated_block_scaled_matmul       silu(A @ Wg.T) * (A @ Wu.T) with block-scaled operands, optionally with an 8-bit checkpoint
  silu_and_mul_backward_quantize  the activation's backward pass from that checkpoint
  gated_feed_forward              the whole block, differentiable: all six products of a training step block-scaled (MXFP8)

The reference has the forward pieces in bf16 (silu_and_mul_kernel, test/kernels/fused_moe.py:85-108, and the gate_up GEMM of
samples/MoE.py:197-288) and no backward pass.  Checks, errors and streams are those of ``ops.py``: work is enqueued on the
current stream of the tensors' device, nothing synchronises, and there is no PyTorch or CPU compute fallback.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib as L
from .errors import TileTypeError, TileValueError
from .ops import (_DTYPE_FMT, _FMT_CODE, PackedScales, _as_u8, _dtype_name, _elem_format, _opts, _raise_code, _scale_code,
                  _scale_desc, _workspace)

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_ELEM8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}


def _mode(scale_mode: str) -> int:
    if scale_mode not in ("ceil", "floor"):
        raise TileValueError(f"scale_mode must be 'ceil' or 'floor', got {scale_mode!r}")
    return 0 if scale_mode == "ceil" else 1


def _same_device(*tensors):
    dev = tensors[0].device
    if any(t.device != dev for t in tensors):
        raise ValueError("Input tensors must be on the same device.")
    if dev.type != "cuda":
        raise ValueError("Input tensors must be on a CUDA device.")
    return dev


def _no_tangents(what, *tensors):
    """Refuses inputs of forward-mode differentiation: a result without its tangent would be taken for a constant."""
    for t in tensors:
        if t is not None and torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{what} has no forward-mode derivative")


def _call(dev, fn, *args):
    """fn(*args, stream) with `dev` as the current device, on its current stream."""
    if torch.cuda.current_device() == dev.index:
        rc = fn(*args, L.stream_ptr(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, L.stream_ptr(dev))
    if rc != L.MX_OK:
        _raise_code(rc)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as [rows, last axis] with contiguous rows (a copy only where its strides allow no such view)."""
    t2 = t.reshape(-1, t.shape[-1])
    if (t2.stride(1) != 1 and t2.shape[1] > 1) or (t2.shape[0] > 1 and t2.stride(0) < 0):
        t2 = t2.contiguous()
    return t2


def _ref(t: torch.Tensor, dtype: Optional[int] = None):
    return ctypes.byref(L.desc(t, L._TORCH_TO_MX[t.dtype] if dtype is None else dtype))


class _Codes(NamedTuple):
    q: torch.Tensor       # uint8
    scale: torch.Tensor   # uint8

    def refs(self, code):
        return _ref(self.q, code), _ref(self.scale, L.MX_E8M0)

    def views(self, dtype):
        return self.q.view(dtype), self.scale.view(torch.float8_e8m0fnu)


def _codes(rows: int, cols: int, dev) -> _Codes:
    """Room for the elements and scales of a matrix that is quantised along its rows (``cols`` a multiple of 32)."""
    return _Codes(torch.empty((rows, cols), dtype=torch.uint8, device=dev),
                  torch.empty((rows, cols // 32), dtype=torch.uint8, device=dev))


def _up32(n: int) -> int:
    return -(-n // 32) * 32


def block_quantize_both(x: torch.Tensor, dtype=torch.float8_e4m3fn, *, scale_mode: str = "floor"):
    """MX-quantises ``x`` along its last axis and along its rows, in one pass over it.  Returns
    ``(x_q, scale, xt_q, scale_t)``.

    ``x`` (..., K) is taken as a matrix of ``rows`` x K.  ``x_q`` and ``scale`` are what :func:`block_quantize` returns (last
    axis zero-padded to a multiple of 32).  ``xt_q`` (K, R) and ``scale_t`` (K, R / 32) are the same of the transposed
    matrix, R = ``rows`` rounded up to a multiple of 32 with zeros: the operand of a product whose sum runs over the rows,
    such as a weight's gradient, or a weight in the gradient of its input.  Kept instead of ``x`` from a forward to a
    backward pass, ``xt_q`` is a checkpoint of 8.25 bits an element.  ``dtype``: ``torch.float8_e4m3fn`` or
    ``torch.float8_e5m2`` for both; ``scale_mode`` as in :func:`block_quantize`."""
    mode = _mode(scale_mode)
    r = L.host().quantize_both(x, dtype, mode)
    if type(r) is tuple:
        return r
    if r is not None:
        _raise_code(r)
    fmt = dtype if isinstance(dtype, str) else _DTYPE_FMT.get(dtype)
    if fmt not in _ELEM8:
        raise TileTypeError(f"Unsupported quantisation dtype {dtype} for block_quantize_both, expected float8_e4m3fn or "
                            "float8_e5m2")
    if x.dtype not in _FLOATS:
        raise TileTypeError(f"Unsupported input dtype {_dtype_name(x.dtype)} for block_quantize_both")
    dev = _same_device(x)
    if x.dim() == 0 or x.shape[-1] < 32:
        raise ValueError("The requested block size 32 is larger than the inner most dimension of the input tensor "
                         f"{x.shape[-1] if x.dim() else 0}")
    x2 = _rows(x.detach())
    rows, K = x2.shape
    r, t = _codes(rows, _up32(K), dev), _codes(K, _up32(rows), dev)
    code = _FMT_CODE[fmt]
    _call(dev, L.lib().mx_quantize_both, _ref(x2), *r.refs(code), *t.refs(code), mode)
    q, scale = r.views(_ELEM8[fmt])
    lead = x.shape[:-1]
    return q.reshape(*lead, _up32(K)), scale.reshape(*lead, _up32(K) // 32), *t.views(_ELEM8[fmt])


def gated_block_scaled_matmul(A: torch.Tensor, A_scale, W: torch.Tensor, W_scale, *, out_dtype=torch.bfloat16,
                              scale_mode: str = "floor", checkpoint: bool = False, a_format: Optional[str] = None,
                              w_format: Optional[str] = None, kernel: str = "auto"):
    """Both projections of a gated feed-forward block, the activation and the product: with
    ``[G | U] = (A * A_scale) @ (W * W_scale).T``, rounded to bf16 as between the projections of :func:`cutile_moe_scaled`,
    ``silu(G) * U``.

    A (M, K) and W (2F, K), gate rows first, hold MX elements as in :func:`block_scaled_matmul` (FP4 packed along K,
    ``"e2m1"`` formats for uint8 storage); A_scale (M, K/32) and W_scale (2F, K/32) are E8M0 tensors or :class:`PackedScales`
    (operand "a" / "b"); F is a multiple of 32.  From one row (weights streamed) to many; of the kernels "stream", "decode" (up
    to 32 rows) and "pingpong" finish the result in the launch of the product where they can, and "auto" takes what is fastest.
    With the ceiling rule or an E5M2 result the product goes through memory.

    Every kernel sums on the scaled matrix instructions, which align an instruction's products with some 18 bits below the largest:
    G and U are within 1.5e-5 of their norm before they are rounded, and a result that is rounded again lies on the other side of a border where
    they are that close to it (8-bit results 0.0004 to 0.004 of their norm from the definition).  NaN and infinities do not depend on the
    kernel: a block with a NaN has the scale and the zeros that :func:`block_quantize` gives it, silu(-inf) is zero.

    Returns (M, F) in ``torch.bfloat16``, or with ``out_dtype`` an 8-bit format ``(h_q, h_scale)``, ready for the down
    projection.  With ``checkpoint`` also ``(gate_up_q, gate_up_scale)``, [G | U] in MXFP8 E4M3, which is all that
    :func:`silu_and_mul_backward_quantize` needs of the forward pass."""
    mode = _mode(scale_mode)
    if kernel in L.KERNELS:
        r = L.host().gated(A, A_scale, W, W_scale, a_format, w_format, out_dtype, mode, checkpoint, L.KERNELS[kernel])
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
    out_fmt = None if out_dtype == torch.bfloat16 else out_dtype if isinstance(out_dtype, str) else _DTYPE_FMT.get(out_dtype)
    if out_dtype != torch.bfloat16 and out_fmt not in _ELEM8:
        raise TileTypeError(f"Unsupported output dtype {out_dtype}, expected bfloat16, float8_e4m3fn or float8_e5m2")
    for name, s in (("A_scale", A_scale), ("W_scale", W_scale)):
        if not isinstance(s, PackedScales) and _scale_code(s) != L.MX_E8M0:
            raise TileTypeError(f"Unsupported scale dtype {_dtype_name(s.dtype)} for {name}, supported scale dtypes are "
                                "float8_e8m0fnu")
    dev = _same_device(A, W, *(s.data if isinstance(s, PackedScales) else s for s in (A_scale, W_scale)))
    dA = L.desc(_as_u8(A), _FMT_CODE[a_fmt], 1 if a_fmt == "e2m1" else -1)
    dW = L.desc(_as_u8(W), _FMT_CODE[w_fmt], 1 if w_fmt == "e2m1" else -1)
    (M, K), (N, Kw) = dA.shape[:2], dW.shape[:2]
    if K != Kw:
        raise ValueError(f"Incompatible matrices: K dimension of A ({K}) must match K dimension of W ({Kw})")
    if N == 0 or N % 64 != 0:
        raise ValueError(f"W must have 2F rows (gate and up projection) with F a multiple of 32, got {N}")
    dAs, la = _scale_desc(A_scale, M, K, 32, False)
    dWs, lw = _scale_desc(W_scale, N, K, 32, True)
    o = _opts(False, la, lw, kernel, 32)
    F = N // 2
    if out_fmt is None:
        h = torch.empty((M, F), dtype=torch.bfloat16, device=dev)
        outs = (_ref(h), None)
    else:
        h = _codes(M, F, dev)
        outs = h.refs(_FMT_CODE[out_fmt])
    kept = _codes(M, N, dev) if checkpoint else None
    lib = L.lib()
    need = lib.mx_gated_gemm_workspace_bytes(M, F, K, ctypes.byref(o))
    ws = _workspace(dev, need)
    _call(dev, lib.mx_gated_gemm, ctypes.byref(dA), ctypes.byref(dAs), ctypes.byref(dW), ctypes.byref(dWs), *outs,
          *(kept.refs(L.MX_E4M3) if checkpoint else (None, None)), mode, ctypes.byref(o), ws.data_ptr() if ws is not None else None, need)
    r = h if out_fmt is None else h.views(_ELEM8[out_fmt])
    if not checkpoint:
        return r
    return (r, *kept.views(torch.float8_e4m3fn)) if out_fmt is None else (*r, *kept.views(torch.float8_e4m3fn))


def silu_and_mul_backward_quantize(dh: torch.Tensor, gate_up_q: torch.Tensor, gate_up_scale: torch.Tensor, *,
                                   scale_mode: str = "floor"):
    """Backward pass of ``silu(g) * u`` from the 8-bit checkpoint of ``[g | u]``, with everything that the products of a
    feed-forward block's backward pass take, quantised (MXFP8 E4M3), in one pass.

    ``dh`` (M, F) bfloat16, the gradient of the activation; ``gate_up_q`` (M, 2F) ``float8_e4m3fn`` and ``gate_up_scale``
    (M, 2F/32) ``float8_e8m0fnu`` as :func:`gated_block_scaled_matmul` leaves them; F a multiple of 32.
    Returns ``(d_q, d_scale, dt_q, dt_scale, at_q, at_scale)``: the gradient of [g | u] along its rows (M, 2F) for
    ``dx = d @ w1``, transposed along the tokens (2F, R) for ``dw1 = d.T @ x``, and the activation, recomputed, transposed
    along the tokens (F, R) for ``dw2 = dy.T @ a``; R is M rounded up to a multiple of 32, the tail zero.

    The arithmetic is in 32 bits: before it is quantised a result is within 2^-18 of its value (2^-17 for gates below -32), or of the terms of
    ``1 + g (1 - s)`` where they cancel.  A NaN is NaN itself and leaves its block's scale to the other elements."""
    mode = _mode(scale_mode)
    r = L.host().silu_backward(dh, gate_up_q, gate_up_scale, mode)
    if type(r) is tuple:
        return r
    if r is not None:
        _raise_code(r)
    if dh.dtype != torch.bfloat16:
        raise TileTypeError(f"Unsupported gradient dtype {_dtype_name(dh.dtype)}, expected bfloat16")
    if gate_up_q.dtype not in (torch.float8_e4m3fn, torch.uint8) or _scale_code(gate_up_scale) != L.MX_E8M0:
        raise TileTypeError("the checkpoint must be float8_e4m3fn with float8_e8m0fnu scales, got "
                            f"{_dtype_name(gate_up_q.dtype)} and {_dtype_name(gate_up_scale.dtype)}")
    if dh.dim() != 2 or gate_up_q.dim() != 2 or gate_up_scale.dim() != 2:
        raise TileTypeError("dh and the checkpoint must be 2D")
    dev = _same_device(dh, gate_up_q, gate_up_scale)
    M, F = dh.shape
    if F == 0 or F % 32 != 0:
        raise ValueError(f"dh must have a multiple of 32 columns, got {F}")
    if tuple(gate_up_q.shape) != (M, 2 * F) or tuple(gate_up_scale.shape) != (M, F // 16):
        raise ValueError(f"the checkpoint of a ({M}, {F}) gradient must be ({M}, {2 * F}) with scales ({M}, {F // 16}), got "
                         f"{tuple(gate_up_q.shape)} and {tuple(gate_up_scale.shape)}")
    gu = _rows(_as_u8(gate_up_q))
    if gu.data_ptr() % 8 or (M > 1 and gu.stride(0) % 8):   # the kernel reads 8 codes at a time
        gu = gu.clone(memory_format=torch.contiguous_format)
    dh, gus = _rows(dh.detach()), _rows(_as_u8(gate_up_scale))
    d, dt, at = _codes(M, 2 * F, dev), _codes(2 * F, _up32(M), dev), _codes(F, _up32(M), dev)
    _call(dev, L.lib().mx_silu_mul_backward_quantize, _ref(dh), _ref(gu, L.MX_E4M3), _ref(gus, L.MX_E8M0), *d.refs(L.MX_E4M3), *dt.refs(L.MX_E4M3), *at.refs(L.MX_E4M3), mode)
    return (*d.views(torch.float8_e4m3fn), *dt.views(torch.float8_e4m3fn), *at.views(torch.float8_e4m3fn))


# ==================================================================================================
# The whole block
# ==================================================================================================
class FeedForwardState(NamedTuple):
    """What :func:`gated_feed_forward_forward` leaves for the backward pass."""
    saved: torch.Tensor   # uint8: input, gate and up, and both weights, in 8.25 bits an element each
    T: int
    H: int
    F: int
    H_out: int
    x_dtype: torch.dtype
    w1_dtype: torch.dtype
    w2_dtype: torch.dtype
    scale_mode: str


def _check_block(x, w1, w2):
    for name, t in (("x", x), ("w1", w1), ("w2", w2)):
        if t.dtype not in (torch.float32, torch.bfloat16):
            raise TileTypeError(f"Unsupported dtype {_dtype_name(t.dtype)} for {name}, expected float32 or bfloat16")
    if x.dim() < 2 or w1.dim() != 2 or w2.dim() != 2:
        raise TileTypeError(f"Expect x (..., H), w1 (2F, H) and w2 (H_out, F), got {tuple(x.shape)}, {tuple(w1.shape)} and "
                            f"{tuple(w2.shape)}")
    H, F, H_out = x.shape[-1], w1.shape[0] // 2, w2.shape[0]
    if w1.shape[0] % 2 != 0 or w1.shape[1] != H or w2.shape[1] != F:
        raise ValueError(f"w1 must be (2F, H) and w2 (H_out, F) for x (..., H), got {tuple(w1.shape)}, {tuple(w2.shape)} and "
                         f"{tuple(x.shape)}")
    if H == 0 or F == 0 or H_out == 0 or H % 32 or F % 32 or H_out % 32:
        raise ValueError(f"H ({H}), F ({F}) and H_out ({H_out}) must be multiples of 32")
    return _same_device(x, w1, w2), H, F, H_out


def _forward(x, w1, w2, mode: int, train: bool):
    r = L.host().feed_forward(x, w1, w2, mode, 1 if train else 0)
    if type(r) is int:
        _raise_code(r)
    if r is not None:
        return r if train else (r, None)
    if not train:
        _no_tangents("gated_feed_forward", x, w1, w2)
    dev, H, F, H_out = _check_block(x, w1, w2)
    x2, w1, w2 = _rows(x.detach()), _rows(w1.detach()), _rows(w2.detach())
    T = x2.shape[0]
    lib = L.lib()
    y = torch.empty((T, H_out), dtype=x.dtype, device=dev)
    kept = lib.mx_ffn_saved_bytes(T, H, F, H_out) if train else 0
    saved = torch.empty(kept, dtype=torch.uint8, device=dev) if train else None
    need = lib.mx_ffn_forward_workspace_bytes(T, H, F, H_out)
    ws = _workspace(dev, need)
    _call(dev, lib.mx_ffn_forward, _ref(x2), _ref(w1), _ref(w2), _ref(y), mode, saved.data_ptr() if kept else None, kept,
          ws.data_ptr() if ws is not None else None, need)
    return y.reshape(*x.shape[:-1], H_out), saved


def gated_feed_forward_forward(x: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor, *, scale_mode: str = "floor"):
    """:func:`gated_feed_forward` without autograd: returns ``(y, state)``, and
    ``gated_feed_forward_backward(dy, state)`` the gradients.  Both can be captured into a HIP graph."""
    y, saved = _forward(x, w1, w2, _mode(scale_mode), True)
    return y, FeedForwardState(saved, x.numel() // x.shape[-1], x.shape[-1], w1.shape[0] // 2, w2.shape[0], x.dtype, w1.dtype,
                               w2.dtype, scale_mode)


def gated_feed_forward_backward(dy: torch.Tensor, state: FeedForwardState, *, need_dx: bool = True, need_dw1: bool = True,
                                need_dw2: bool = True):
    """Gradients ``(dx, dw1, dw2)`` of :func:`gated_feed_forward_forward` for the gradient ``dy`` (..., H_out) of its result,
    in the dtypes of x, w1 and w2 (``dx`` in the shape of ``dy`` but for its last axis); None where not asked for.  Reads the state and
    leaves it as it is, so it can be called again with another ``dy``."""
    s = state
    r = L.host().feed_forward_backward(dy, s.saved, s.T, s.H, s.F, s.H_out, s.x_dtype, s.w1_dtype, s.w2_dtype, need_dx, need_dw1,
                                       need_dw2, _mode(s.scale_mode))
    if type(r) is tuple:
        return r if dy.dim() == 2 or not need_dx else (r[0].view(*dy.shape[:-1], s.H), r[1], r[2])
    if r is not None:
        _raise_code(r)
    if dy.dtype not in _FLOATS:
        raise TileTypeError(f"Unsupported gradient dtype {_dtype_name(dy.dtype)}, expected float32, bfloat16 or float16")
    if dy.dim() < 2 or dy.shape[-1] != s.H_out or dy.numel() != s.T * s.H_out:
        raise ValueError(f"dy must hold {s.T} rows of {s.H_out}, got {tuple(dy.shape)}")
    dev = _same_device(dy, s.saved)
    make = torch.empty if s.T else torch.zeros    # no tokens: the sums over them are zeros
    dx = torch.empty((s.T, s.H), dtype=s.x_dtype, device=dev) if need_dx else None
    dw1 = make((2 * s.F, s.H), dtype=s.w1_dtype, device=dev) if need_dw1 else None
    dw2 = make((s.H_out, s.F), dtype=s.w2_dtype, device=dev) if need_dw2 else None
    if s.T and (need_dx or need_dw1 or need_dw2):
        lib = L.lib()
        dy2 = _rows(dy.detach())
        need = lib.mx_ffn_backward_workspace_bytes(s.T, s.H, s.F, s.H_out)
        ws = _workspace(dev, need)
        _call(dev, lib.mx_ffn_backward, _ref(dy2), s.saved.data_ptr(), s.saved.numel(), s.H, s.F,
              *(None if t is None else _ref(t) for t in (dx, dw1, dw2)), _mode(s.scale_mode), ws.data_ptr(), need)
    return dx.reshape(*dy.shape[:-1], s.H) if need_dx else None, dw1, dw2


class _GatedFeedForward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w1, w2, scale_mode):
        y, state = gated_feed_forward_forward(x, w1, w2, scale_mode=scale_mode)
        ctx.save_for_backward(state.saved)
        ctx.state = state._replace(saved=None)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        state = ctx.state._replace(saved=ctx.saved_tensors[0])
        need = ctx.needs_input_grad
        return (*gated_feed_forward_backward(dy, state, need_dx=need[0], need_dw1=need[1], need_dw2=need[2]), None)


def gated_feed_forward(x: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor, *, scale_mode: str = "floor") -> torch.Tensor:
    """``(silu(x @ wg.T) * (x @ wu.T)) @ w2.T`` with ``[wg ; wu] = w1``, every product of the forward and of the backward
    pass block-scaled in MXFP8 (E4M3), differentiable in x, w1 and w2.

    x (..., H), w1 (2F, H), gate rows first, and w2 (H_out, F) are float32 or bfloat16, H, F and H_out multiples of 32.
    The result has the dtype of x, every gradient the dtype of what it is the gradient of.  Each operand is quantised along the
    axis that its product sums over: input, weights and gradients along both of theirs.  The backward pass is kept
    8.25 bits an element: of the input, of gate and up (the activation is recomputed from them) and of both
    weights; neither x nor the weights are kept, so they may be updated in place in between.  No operand may have 2^31 elements
    or more.

    With few tokens (up to 64, or tokens times F up to 2^19) gate, up and the activation's gradient are summed in 32 bits, and results are the
    definition's to their rounding; with more, those sums are the scaled matrix instructions' (:func:`gated_block_scaled_matmul`) and results
    are 0.0017 to 0.0026 of their norm from the definition, of which rounding to bf16 is 0.0017.  Under the floor rule an infinity of the
    input or of the gradient counts as the largest number of its block, so gradients made of it may be finite; ``scale_mode="ceil"`` makes its
    block NaN.  A NaN is NaN under both.

    With gradients enabled the call refuses to be captured into a HIP graph (autograd accumulates a leaf's gradient on the
    stream that first used it, which a capture must not touch): capture :func:`gated_feed_forward_forward` and
    :func:`gated_feed_forward_backward`.  Inputs of forward-mode differentiation are refused."""
    mode = _mode(scale_mode)
    if not (torch.is_grad_enabled() and (x.requires_grad or w1.requires_grad or w2.requires_grad)):
        return _forward(x, w1, w2, mode, False)[0]
    r = L.host().feed_forward(x, w1, w2, mode, 2)
    if type(r) is int:
        _raise_code(r)
    if r is not None:
        return r
    _no_tangents("gated_feed_forward", x, w1, w2)
    if x.is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("gated_feed_forward with gradients cannot be captured into a graph: capture "
                           "gated_feed_forward_forward and gated_feed_forward_backward")
    return _GatedFeedForward.apply(x, w1, w2, scale_mode)
