"""Refusals of the linear layer's entry points, without a GPU: every rule is checked before anything touches a device."""
import ctypes

import pytest
import torch

import cutile_amd as ct
from cutile_amd import _lib as L
from test_norm_adamw_validation import P, desc, ref

bf16, f16, f32 = torch.bfloat16, torch.float16, torch.float32
E4M3, E5M2, E8M0 = torch.float8_e4m3fn, torch.float8_e5m2, torch.float8_e8m0fnu


def z(*shape, dtype=f32):
    return torch.zeros(shape, dtype=torch.uint8).view(dtype) if dtype in (E4M3, E5M2, E8M0) else torch.zeros(shape, dtype=dtype)


# ---- the Python entry points -----------------------------------------------------------------------------------
@pytest.mark.parametrize("over,error,message", [
    (dict(), ValueError, "CUDA device"),
    (dict(activation="tanh"), ct.TileValueError, "unknown activation 'tanh'"),
    (dict(A=z(4, 64, dtype=bf16)), ct.TileTypeError, "Unsupported input dtype bfloat16"),
    (dict(W=z(96, 64, dtype=torch.uint8)), ct.TileTypeError, "Unsupported input dtype uint8"),
    (dict(A=z(2, 4, 64, dtype=E4M3)), ct.TileTypeError, "2D"),
    (dict(out_dtype=f16), ct.TileTypeError, "Unsupported output dtype"),
    (dict(out_dtype=E5M2), ct.TileTypeError, "Unsupported output dtype"),
    (dict(A_scale=z(4, 2)), ct.TileTypeError, "Unsupported scale dtype float32 for A_scale"),
    (dict(W_scale=z(96, 2, dtype=E4M3)), ct.TileTypeError, "for W_scale"),
    (dict(W=z(96, 32, dtype=E4M3)), ValueError, r"K dimension of A \(64\) must match K dimension of W \(32\)"),
    (dict(W=z(97, 64, dtype=E4M3), out_dtype=E4M3, bias=None, residual=None), ValueError, "multiple of 32 rows"),
    (dict(bias=z(95)), ValueError, r"bias must be \(96,\)"),
    (dict(bias=z(1, 96)), ValueError, "bias must be"),
    (dict(bias=z(96, dtype=torch.float64)), ct.TileTypeError, "Unsupported dtype float64 for bias"),
    (dict(residual=z(4, 95)), ValueError, r"residual must be \(4, 96\)"),
    (dict(residual=z(96)), ValueError, "residual must be"),
    (dict(residual=z(4, 96, dtype=E4M3)), ct.TileTypeError, "for residual"),
])
def test_block_scaled_linear_refusals(over, error, message):
    a = dict(A=z(4, 64, dtype=E4M3), A_scale=z(4, 2, dtype=E8M0), W=z(96, 64, dtype=E4M3), W_scale=z(96, 2, dtype=E8M0), bias=z(96), residual=z(4, 96))
    with pytest.raises(error, match=message):
        ct.block_scaled_linear(**{**a, **over})


@pytest.mark.parametrize("over,error,message", [
    (dict(), ValueError, "CUDA device"),
    (dict(x=z(4, 64, dtype=f16)), ct.TileTypeError, "Unsupported dtype float16 for x"),
    (dict(w=z(96, 64, dtype=E4M3)), ct.TileTypeError, "for w"),
    (dict(x=z(64)), ct.TileTypeError, r"Expect x \(\.\.\., K\)"),
    (dict(w=z(1, 96, 64)), ct.TileTypeError, "Expect x"),
    (dict(w=z(96, 32)), ValueError, r"w must be \(N, 64\)"),
    (dict(x=z(4, 48), w=z(96, 48)), ValueError, "multiples of 32"),
    (dict(w=z(80, 64), bias=None, residual=None), ValueError, "multiples of 32"),
    (dict(x=z(4, 0), w=z(96, 0)), ValueError, "multiples of 32"),
    (dict(bias=z(64)), ValueError, r"bias must be \(96,\)"),
    (dict(residual=z(5, 96)), ValueError, r"residual must be \(4, 96\)"),
    (dict(residual=z(4, 96, dtype=torch.int32)), ct.TileTypeError, "for residual"),
    (dict(activation="swish"), ct.TileValueError, "unknown activation"),
    (dict(scale_mode="nearest"), ct.TileValueError, "scale_mode"),
])
@pytest.mark.parametrize("f", ["linear", "linear_forward"])
def test_linear_refusals(f, over, error, message):
    with pytest.raises(error, match=message):
        getattr(ct, f)(**{**dict(x=z(4, 64), w=z(96, 64), bias=z(96), residual=z(4, 96)), **over})


@pytest.mark.parametrize("dy,error,message", [
    (z(4, 96), ValueError, "CUDA device"),
    (z(5, 96), ValueError, "4 rows of 96"),
    (z(4, 64), ValueError, "4 rows of 96"),
    (z(4, 96, dtype=torch.float64), ct.TileTypeError, "Unsupported gradient dtype"),
])
def test_linear_backward_refusals(dy, error, message):
    state = ct.LinearState(torch.zeros(1 << 16, dtype=torch.uint8), 4, 64, 96, f32, f32, f32, "gelu", "floor")
    with pytest.raises(error, match=message):
        ct.linear_backward(dy, state)


# ---- the C entries -----------------------------------------------------------------------------------------------
F, B, H16, E = L.MX_F32, L.MX_BF16, L.MX_F16, L.MX_E4M3
GEMM = dict(A=desc(E, (4, 64)), As=desc(L.MX_E8M0, (4, 2)), W=desc(E, (96, 64)), Ws=desc(L.MX_E8M0, (96, 2)), bias=desc(F, (96,)), res=desc(B, (4, 96)),
            act=L.MX_ACT_GELU, out=desc(B, (4, 96)), scale=None, pre=None, opts=None, ws=P, bytes=1 << 30)


@pytest.mark.parametrize("over,code,message", [
    (dict(A=None), L.MX_ERR_INVALID, "null descriptor"),
    (dict(A=desc(E, (1, 4, 64))), L.MX_ERR_SHAPE, "2 dimensions"),
    (dict(A=desc(E, (-4, 64))), L.MX_ERR_SHAPE, "negative extent"),
    (dict(A=desc(E, (4, 32))), L.MX_ERR_SHAPE, "must match K dimension of W"),
    (dict(A=desc(E, (4, 64), ptr=None)), L.MX_ERR_INVALID, "A: null data pointer"),
    (dict(A=desc(E, (4, 64), (-64, 1))), L.MX_ERR_LAYOUT, "negative strides"),
    (dict(A=desc(B, (4, 64))), L.MX_ERR_DTYPE, "must be MX_E4M3"),
    (dict(As=desc(L.MX_E8M0, (4, 3))), L.MX_ERR_SHAPE, "A_scale must be"),
    (dict(Ws=desc(L.MX_E8M0, (64, 2))), L.MX_ERR_SHAPE, "W_scale must be"),
    (dict(Ws=desc(L.MX_E8M0, (96, 2), ptr=None)), L.MX_ERR_INVALID, "W_scale: null data pointer"),
    (dict(bias=desc(F, (64,))), L.MX_ERR_SHAPE, "bias must be"),
    (dict(bias=desc(F, (96,), (2,))), L.MX_ERR_LAYOUT, "contiguous"),
    (dict(bias=desc(E, (96,))), L.MX_ERR_DTYPE, "bias must be"),
    (dict(res=desc(B, (4, 97))), L.MX_ERR_SHAPE, "residual must be"),
    (dict(res=desc(B, (4, 96), (1, 4))), L.MX_ERR_LAYOUT, "contiguous"),
    (dict(res=desc(E, (4, 96))), L.MX_ERR_DTYPE, "residual must be"),
    (dict(act=5), L.MX_ERR_INVALID, "unknown activation 5"),
    (dict(act=-1), L.MX_ERR_INVALID, "unknown activation"),
    (dict(out=None), L.MX_ERR_INVALID, "out: null"),
    (dict(out=desc(H16, (4, 96))), L.MX_ERR_DTYPE, "out must be"),
    (dict(out=desc(B, (4, 96), (95, 1))), L.MX_ERR_LAYOUT, "out: rows overlap"),
    (dict(scale=desc(L.MX_E8M0, (4, 3))), L.MX_ERR_INVALID, "only an MX_E4M3 output"),
    (dict(out=desc(E, (4, 96))), L.MX_ERR_INVALID, "out_scale"),
    (dict(out=desc(E, (4, 96)), scale=desc(L.MX_E8M0, (4, 2))), L.MX_ERR_SHAPE, "out_scale must be"),
    (dict(out=desc(E, (4, 96), (100, 1)), scale=desc(L.MX_E8M0, (4, 3))), L.MX_ERR_LAYOUT, "aligned to 8"),
    (dict(pre=desc(F, (4, 96))), L.MX_ERR_DTYPE, "pre must be MX_BF16"),
    (dict(pre=desc(B, (4, 64))), L.MX_ERR_SHAPE, "pre must be"),
    (dict(pre=desc(B, (4, 96), (8, 1))), L.MX_ERR_LAYOUT, "pre: rows overlap"),
    (dict(opts=L.MxGemmOpts(struct_size=32, block_size=16)), L.MX_ERR_INVALID, "block_size must be 32"),
    (dict(ws=None), L.MX_ERR_WORKSPACE, "workspace"),
    (dict(bytes=1 << 10), L.MX_ERR_WORKSPACE, "workspace"),
    (dict(ws=P + 8), L.MX_ERR_WORKSPACE, "aligned"),
])
def test_linear_gemm_codes(over, code, message):
    a = {**GEMM, **over}
    rc = L.lib().mx_linear_gemm(*(ref(a[n]) for n in ("A", "As", "W", "Ws", "bias", "res")), a["act"], ref(a["out"]), ref(a["scale"]), ref(a["pre"]), ref(a["opts"]),
                                a["ws"], a["bytes"], None)
    assert rc == code and message in L.last_error(), L.last_error()


def test_linear_gemm_without_rows_or_columns():
    a = dict(GEMM, A=desc(E, (0, 64)), As=desc(L.MX_E8M0, (0, 2)), res=None, out=desc(B, (0, 96)))
    call = lambda: L.lib().mx_linear_gemm(*(ref(a[n]) for n in ("A", "As", "W", "Ws", "bias", "res")), 0, ref(a["out"]), None, None, None, None, 0, None)  # noqa: E731
    assert call() == L.MX_OK
    a.update(A=GEMM["A"], As=GEMM["As"], W=desc(E, (0, 64)), Ws=desc(L.MX_E8M0, (0, 2)), bias=None, out=desc(B, (4, 0)))
    assert call() == L.MX_OK
    assert L.lib().mx_linear_gemm_workspace_bytes(0, 96, 64, None) == 0


FWD = dict(x=desc(F, (4, 64)), w=desc(B, (96, 64)), bias=desc(F, (96,)), res=None, act=L.MX_ACT_SILU, y=desc(B, (4, 96)), mode=1, saved=P, kept=1 << 20, ws=P, bytes=1 << 20)


@pytest.mark.parametrize("over,code,message", [
    (dict(x=None), L.MX_ERR_INVALID, "x: null"),
    (dict(x=desc(E, (4, 64))), L.MX_ERR_DTYPE, "x must be"),
    (dict(w=desc(B, (96, 32))), L.MX_ERR_SHAPE, "w must be"),
    (dict(x=desc(F, (4, 48)), w=desc(B, (96, 48))), L.MX_ERR_SHAPE, "multiples of 32"),
    (dict(y=desc(H16, (4, 96))), L.MX_ERR_DTYPE, "y must be"),
    (dict(y=desc(B, (4, 96), (32, 1))), L.MX_ERR_LAYOUT, "overlap"),
    (dict(bias=desc(F, (95,))), L.MX_ERR_SHAPE, "bias must be"),
    (dict(res=desc(B, (3, 96))), L.MX_ERR_SHAPE, "residual must be"),
    (dict(act=9), L.MX_ERR_INVALID, "unknown activation"),
    (dict(mode=2), L.MX_ERR_INVALID, "scale_mode"),
    (dict(ws=None), L.MX_ERR_WORKSPACE, "workspace"),
    (dict(bytes=64), L.MX_ERR_WORKSPACE, "workspace"),
    (dict(kept=64), L.MX_ERR_WORKSPACE, "saved"),
    (dict(saved=P + 16), L.MX_ERR_WORKSPACE, "saved"),
    (dict(x=desc(F, (1 << 21, 1024)), w=desc(B, (32, 1024)), bias=None, y=desc(B, (1 << 21, 32))), L.MX_ERR_SHAPE, "2 GiB"),
])
def test_linear_forward_codes(over, code, message):
    a = {**FWD, **over}
    rc = L.lib().mx_linear_forward(*(ref(a[n]) for n in ("x", "w", "bias", "res")), a["act"], ref(a["y"]), a["mode"], a["saved"], a["kept"], a["ws"], a["bytes"], None)
    assert rc == code and message in L.last_error(), L.last_error()


BACK = dict(dy=desc(F, (4, 96)), saved=P, kept=1 << 20, K=64, act=L.MX_ACT_SILU, dx=desc(B, (4, 64)), dw=desc(F, (96, 64)), db=desc(B, (96,)), mode=1, ws=P, bytes=1 << 20)


@pytest.mark.parametrize("over,code,message", [
    (dict(dy=None), L.MX_ERR_INVALID, "dy: null"),
    (dict(dy=desc(E, (4, 96))), L.MX_ERR_DTYPE, "dy must be"),
    (dict(dy=desc(F, (4, 96), ((1 << 25) + 1, 1))), L.MX_ERR_LAYOUT, "2^25 elements apart"),
    (dict(K=48), L.MX_ERR_SHAPE, "multiples of 32"),
    (dict(act=-2), L.MX_ERR_INVALID, "unknown activation"),
    (dict(dx=desc(B, (4, 96))), L.MX_ERR_SHAPE, "dx must be"),
    (dict(dw=desc(H16, (96, 64))), L.MX_ERR_DTYPE, "dw must be"),
    (dict(dw=desc(F, (96, 64), (8, 1))), L.MX_ERR_LAYOUT, "dw: rows overlap"),
    (dict(db=desc(F, (64,))), L.MX_ERR_SHAPE, "dbias must be"),
    (dict(mode=-1), L.MX_ERR_INVALID, "scale_mode"),
    (dict(dy=desc(F, (0, 96)), dx=None), L.MX_ERR_SHAPE, "no tokens"),
    (dict(kept=64), L.MX_ERR_WORKSPACE, "saved"),
    (dict(saved=None), L.MX_ERR_WORKSPACE, "saved"),
    (dict(bytes=64), L.MX_ERR_WORKSPACE, "workspace"),
    (dict(dx=None, dw=None, db=None), L.MX_OK, ""),
])
def test_linear_backward_codes(over, code, message):
    a = {**BACK, **over}
    rc = L.lib().mx_linear_backward(ref(a["dy"]), a["saved"], a["kept"], a["K"], a["act"], ref(a["dx"]), ref(a["dw"]), ref(a["db"]), a["mode"], a["ws"], a["bytes"], None)
    assert rc == code and (code == L.MX_OK or message in L.last_error()), L.last_error()
