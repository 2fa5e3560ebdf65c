"""Calls of the linear layer beside the usual ones."""
import ctypes

import numpy as np
import pytest
import torch

from cutile_amd import _lib as L
from mxutil import randn_operand
from oracle import mx_oracle as O
from test_gpu_linear import d64

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


# ---- the activations alone ----------------------------------------------------------------------------------------------------
def exponent(p, act):
    """|z| of the exponential exp(-|z|) that an activation has in it."""
    return {"silu": p.abs(), "gelu": p * p / 2, "gelu_tanh": (2 * (2 / torch.pi) ** 0.5 * (p + 0.044715 * p ** 3)).abs()}[act]


def act_exact(p, act):
    """The activation where tanh(z / 2) + 1 and the like have lost their bits: x s(z) through exp."""
    if act == "gelu":
        return p * 0.5 * torch.special.erfc(-p * 0.5 ** 0.5)
    z = p if act == "silu" else 2 * (2 / torch.pi) ** 0.5 * (p + 0.044715 * p ** 3)
    return p * torch.sigmoid(z)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("kernel,M", [("stream", 1), ("stream", 40), ("mfma128", 200), ("pingpong", 300), ("generic", 2), ("auto", 70)])
def test_activation_to_its_stated_precision(ct, dev, kernel, M, act):
    """A product of zero and an fp32 result leave act(bias): within 2e-6 + 2.5e-7 |z| of its value, gelu below -7 within 4e-5 more; numbers below
    2e-36 may be zero.  (z: roundings of x^2, of its product and sum, of the last product, 2^-24 each, and constants off by 5e-8, are
    2.3e-7 of it at most, and so much of the exponential.  The rest: 2^x and reciprocals 2^-23 each, some 2^-24, gelu's fit 2.6e-7 up to 7 and
    3.5e-5 up to 12.75, from where on numbers are below 2e-36.)"""
    K, N = 256, 4096
    for lo, hi in ((-100.0, 100.0), (-14.0, 4.0), (-2.0, 2.0), (-1e-3, 1e-3)):
        bias = torch.linspace(lo, hi, N, dtype=f32, device=dev)
        a, w = torch.zeros((M, K), dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn), torch.zeros((N, K), dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
        one = lambda rows: torch.full((rows, K // 32), 127, dtype=torch.uint8, device=dev).view(torch.float8_e8m0fnu)  # noqa: E731
        y = d64(ct.block_scaled_linear(a, one(M), w, one(N), bias, activation=act, out_dtype=f32, kernel=kernel))
        p = d64(bias)
        want = act_exact(p, act)
        err = (2e-6 + 2.5e-7 * exponent(p, act)) * want.abs()
        if act == "gelu":
            err = err + torch.where(p < -7, 4e-5, 0.0) * want.abs()
        bad = ~((y - want).abs() <= err + 2e-36)
        assert not bool(bad.any()), (p[bad[0]][:4].tolist(), y[0][bad[0]][:4].tolist(), want[bad[0]][:4].tolist())
