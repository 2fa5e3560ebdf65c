"""Calls of the linear layer beside the usual ones."""
import ctypes

import numpy as np
import pytest
import torch

from cutile_amd import _lib as L
from mxutil import randn_operand
from oracle import mx_oracle as O

pytestmark = pytest.mark.gpu

bf16, f16, f32 = torch.bfloat16, torch.float16, torch.float32


# ---- operands ---------------------------------------------------------------------------------------------------------------------
def call(a, w, M, K, N, dev, out):
    """The C entry, FP4 operands as (storage, packed dimension, scales) on the general kernel: the product goes through memory."""
    o, lib = L.MxGemmOpts(struct_size=32, kernel=L.KERNELS["generic"], block_size=32), L.lib()
    need = lib.mx_linear_gemm_workspace_bytes(M, N, K, ctypes.byref(o))
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    c = torch.empty((M, N), dtype=out, device=dev)
    operands = [ctypes.byref(L.desc(t.view(torch.uint8), f, p)) for q, d, s in (a, w) for t, f, p in ((q, L.MX_E2M1, d), (s, L.MX_E8M0, -1))]
    rc = lib.mx_linear_gemm(*operands, None, None, L.MX_ACT_NONE, ctypes.byref(L.desc(c, L._TORCH_TO_MX[out])), None, None, ctypes.byref(o), ws.data_ptr(), need,
                            L.stream_ptr(dev))
    assert rc == L.MX_OK, L.last_error()
    return c


@pytest.mark.parametrize("M", [2, 256, 258, 600])
@pytest.mark.parametrize("columns", [False, True])
def test_fp4_packed_along_the_rows(dev, M, columns):
    """Two rows to a byte, the K axis contiguous or the rows: 16384 columns are finished 256 rows at a time, each part of which begins half as
    many bytes into such an operand."""
    K, N = 64, 16384
    a, w = randn_operand(M, K, O.E2M1, 1, dev), randn_operand(N, K, O.E2M1, 2, dev, std=K ** -0.5)
    along = torch.from_numpy(np.ascontiguousarray(a.codes[0::2] | a.codes[1::2] << 4)).to(dev)      # [M / 2, K]
    if columns:
        along = along.T.contiguous().T
    weights = (w.storage, 1, w.scale_t)
    want = call((a.storage, 1, a.scale_t), weights, M, K, N, dev, f32)
    assert torch.equal(call((along, 0, a.scale_t), weights, M, K, N, dev, f32), want)
    A, W = (O.dequantize(t.codes, t.scales, t.fmt).double() for t in (a, w))
    exact = A @ W.T
    # 64 products and the sum's roundings in 32 bits
    assert bool(((want.cpu().double() - exact).abs() <= 66 * 2.0 ** -24 * (A.abs() @ W.abs().T)).all())


# ---- gradients ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T", [2, 3])
@pytest.mark.parametrize("pitch", [1 << 25, (1 << 25) + 1, (1 << 25) + 64])
def test_gradient_whose_rows_lie_far_apart(ct, dev, pitch, T):
    K, N = 96, 64
    g = torch.Generator().manual_seed(T)
    x, w, b = ((torch.randn(s, generator=g)).to(bf16).to(dev) for s in ((T, K), (N, K), (N,)))
    room = torch.zeros((T - 1) * pitch + N, dtype=bf16, device=dev)
    far = room.as_strided((T, N), (pitch, 1))
    near = torch.randn((T, N), generator=g).to(bf16).to(dev)
    far.copy_(near)
    _, state = ct.linear_forward(x, w, b, activation="gelu")
    want = ct.linear_backward(near, state)
    for got in (ct.linear_backward(far, state), ct.linear_backward(far.unsqueeze(0), state)):
        assert all(torch.equal(p.reshape(q.shape), q) for p, q in zip(got, want))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    got = torch.autograd.grad(ct.linear(*leaves, activation="gelu"), leaves, far)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("T", [40, 600])
@pytest.mark.parametrize("xt,rt", [(bf16, f32), (bf16, f16), (f32, bf16), (bf16, bf16)], ids=str)
def test_graph_of_the_residuals_gradient(ct, dev, T, xt, rt):
    """The residual's gradient is dy, in the residual's type: its graph is that of dy.  The others have none and say so."""
    K, N = 64, 96
    g = torch.Generator().manual_seed(7)
    x, w, b = ((torch.randn(s, generator=g)).to(xt).to(dev).requires_grad_() for s in ((T, K), (N, K), (N,)))
    r = torch.randn((T, N), generator=g).to(rt).to(dev).requires_grad_()
    dy = torch.randn((T, N), generator=g).to(xt).to(dev).requires_grad_()
    weight = torch.randn((T, N), generator=g).to(rt).to(dev)
    dx, dw, db, dr = torch.autograd.grad(ct.linear(x, w, b, r, activation="silu"), (x, w, b, r), dy, create_graph=True)
    assert dr.dtype == rt and torch.equal(dr.detach(), dy.detach().to(rt))
    (back,) = torch.autograd.grad((dr * weight).sum(), dy)
    assert torch.equal(back, weight.to(xt))
    for t in (dx, dw, db):
        with pytest.raises(RuntimeError, match="cannot be differentiated"):
            t.sum().backward(retain_graph=True)
