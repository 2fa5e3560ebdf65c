"""Refusals of the feed-forward block's entry points, without a GPU: every rule is checked before anything touches a device."""
import ctypes

import pytest
import torch

import cutile_amd as ct
from cutile_amd import _lib as L

E4M3, E5M2, E8M0 = torch.float8_e4m3fn, torch.float8_e5m2, torch.float8_e8m0fnu
bf16, f32, f16 = torch.bfloat16, torch.float32, torch.float16


def elems(*shape, dtype=E4M3):
    return torch.zeros(shape, dtype=torch.uint8).view(dtype)


# ---- the Python entry points -----------------------------------------------------------------------------------
@pytest.mark.parametrize("x,kw,error,message", [
    (torch.zeros(4, 64), dict(dtype=bf16), ct.TileTypeError, "Unsupported quantisation dtype"),
    (torch.zeros(4, 64), dict(dtype="e2m1"), ct.TileTypeError, "Unsupported quantisation dtype"),
    (torch.zeros(4, 64, dtype=torch.int32), {}, ct.TileTypeError, "Unsupported input dtype int32"),
    (torch.zeros(4, 64, dtype=torch.float64), {}, ct.TileTypeError, "Unsupported input dtype float64"),
    (torch.zeros(4, 64), dict(scale_mode="round"), ct.TileValueError, "scale_mode"),
    (torch.zeros(4, 64), {}, ValueError, "CUDA device"),
])
def test_quantize_both_refusals(x, kw, error, message):
    with pytest.raises(error, match=message):
        ct.block_quantize_both(x, **kw)


def gated(**over):
    a = dict(A=elems(4, 64), A_scale=elems(4, 2, dtype=E8M0), W=elems(128, 64), W_scale=elems(128, 2, dtype=E8M0))
    return ct.gated_block_scaled_matmul(**{**a, **over})


@pytest.mark.parametrize("over,error,message", [
    (dict(), ValueError, "CUDA device"),
    (dict(A=torch.zeros(4, 64)), ct.TileTypeError, "Unsupported input dtype float32"),
    (dict(W=torch.zeros(128, 64, dtype=f16)), ct.TileTypeError, "Unsupported input dtype float16"),
    (dict(A=elems(1, 4, 64)), ct.TileTypeError, "2D"),
    (dict(out_dtype=f32), ct.TileTypeError, "Unsupported output dtype"),
    (dict(out_dtype="e2m1"), ct.TileTypeError, "Unsupported output dtype"),
    (dict(A_scale=torch.zeros(4, 2)), ct.TileTypeError, "A_scale"),
    (dict(W_scale=torch.zeros(128, 2)), ct.TileTypeError, "W_scale"),
    (dict(scale_mode="up"), ct.TileValueError, "scale_mode"),
    (dict(kernel="fast"), Exception, "CUDA device|unknown kernel"),
])
def test_gated_refusals(over, error, message):
    with pytest.raises(error, match=message):
        gated(**over)


@pytest.mark.parametrize("dh,q,s,kw,error,message", [
    (torch.zeros(4, 64), elems(4, 128), elems(4, 4, dtype=E8M0), {}, ct.TileTypeError, "Unsupported gradient dtype float32"),
    (torch.zeros(4, 64, dtype=bf16), elems(4, 128, dtype=E5M2), elems(4, 4, dtype=E8M0), {}, ct.TileTypeError, "checkpoint"),
    (torch.zeros(4, 64, dtype=bf16), elems(4, 128), torch.zeros(4, 4), {}, ct.TileTypeError, "checkpoint|scale dtype"),
    (torch.zeros(2, 4, 64, dtype=bf16), elems(4, 128), elems(4, 4, dtype=E8M0), {}, ct.TileTypeError, "2D"),
    (torch.zeros(4, 64, dtype=bf16), elems(4, 128), elems(4, 4, dtype=E8M0), {}, ValueError, "CUDA device"),
    (torch.zeros(4, 64, dtype=bf16), elems(4, 128), elems(4, 4, dtype=E8M0), dict(scale_mode=1), ct.TileValueError, "scale_mode"),
])
def test_silu_backward_refusals(dh, q, s, kw, error, message):
    with pytest.raises(error, match=message):
        ct.silu_and_mul_backward_quantize(dh, q, s, **kw)


@pytest.mark.parametrize("form", [ct.gated_feed_forward, ct.gated_feed_forward_forward])
@pytest.mark.parametrize("x,w1,w2,error,message", [
    (torch.zeros(4, 64, dtype=f16), torch.zeros(128, 64), torch.zeros(32, 64), ct.TileTypeError, "float16 for x"),
    (torch.zeros(4, 64), torch.zeros(128, 64, dtype=f16), torch.zeros(32, 64), ct.TileTypeError, "float16 for w1"),
    (torch.zeros(4, 64), torch.zeros(128, 64), torch.zeros(32, 64, dtype=torch.float64), ct.TileTypeError, "float64 for w2"),
    (torch.zeros(64), torch.zeros(128, 64), torch.zeros(32, 64), ct.TileTypeError, "Expect x"),
    (torch.zeros(4, 64), torch.zeros(2, 128, 64), torch.zeros(32, 64), ct.TileTypeError, "Expect x"),
    (torch.zeros(4, 64), torch.zeros(128, 32), torch.zeros(32, 64), ValueError, "w1 must be"),
    (torch.zeros(4, 64), torch.zeros(129, 64), torch.zeros(32, 64), ValueError, "w1 must be"),
    (torch.zeros(4, 64), torch.zeros(128, 64), torch.zeros(32, 96), ValueError, "w1 must be"),
    (torch.zeros(4, 48), torch.zeros(128, 48), torch.zeros(32, 64), ValueError, "multiples of 32"),
    (torch.zeros(4, 64), torch.zeros(80, 64), torch.zeros(32, 40), ValueError, "multiples of 32"),
    (torch.zeros(4, 64), torch.zeros(128, 64), torch.zeros(33, 64), ValueError, "multiples of 32"),
    (torch.zeros(4, 64), torch.zeros(0, 64), torch.zeros(32, 0), ValueError, "multiples of 32"),
    (torch.zeros(4, 64), torch.zeros(128, 64), torch.zeros(32, 64), ValueError, "CUDA device"),
])
def test_block_refusals(form, x, w1, w2, error, message):
    with pytest.raises(error, match=message):
        form(x, w1, w2)
    with pytest.raises(error, match=message):
        form(x, w1.requires_grad_(), w2)


def test_block_scale_mode():
    for form in (ct.gated_feed_forward, ct.gated_feed_forward_forward):
        with pytest.raises(ct.TileValueError, match="scale_mode"):
            form(torch.zeros(4, 64), torch.zeros(128, 64), torch.zeros(32, 64), scale_mode="nearest")


@pytest.mark.parametrize("dy,error,message", [
    (torch.zeros(4, 32, dtype=torch.float64), ct.TileTypeError, "Unsupported gradient dtype"),
    (torch.zeros(5, 32), ValueError, "dy must hold"),
    (torch.zeros(4, 64), ValueError, "dy must hold"),
    (torch.zeros(128), ValueError, "dy must hold"),
    (torch.zeros(4, 32), ValueError, "CUDA device"),
])
def test_block_backward_refusals(dy, error, message):
    state = ct.FeedForwardState(torch.zeros(16, dtype=torch.uint8), 4, 64, 64, 32, f32, f32, f32, "floor")
    with pytest.raises(error, match=message):
        ct.gated_feed_forward_backward(dy, state)


# ---- the C entries ----------------------------------------------------------------------------------------------
BUF = torch.zeros(1 << 20, dtype=torch.uint8)
P = (BUF.data_ptr() + 4095) // 4096 * 4096
O = L


def d(dtype, *shape, ld=None, ptr=P, nd=None):
    t = L.MxTensor()
    t.ptr, t.dtype, t.ndim, t.packed_dim = ptr, dtype, nd or len(shape), -1
    stride = [1] * len(shape)
    for i in range(len(shape) - 2, -1, -1):
        stride[i] = stride[i + 1] * shape[i + 1]
    if ld is not None:
        stride[-2] = ld
    for i, (n, s) in enumerate(zip(shape, stride)):
        t.shape[i], t.stride[i] = n, s
    return t


def refs(args):
    return [ctypes.byref(a) if isinstance(a, L.MxTensor) else a for a in args]


def check(fn, good, cases):
    """Every case: (name or names of the arguments that differ, their values, code, part of the message)."""
    for change, code, message in cases:
        args = dict(good)
        args.update(change)
        rc = fn(*refs(args.values()), None)
        assert rc == code and message in L.last_error(), (change.keys(), rc, L.last_error())


def test_c_quantize_both():
    good = dict(x=d(L.MX_F32, 40, 64), q=d(L.MX_E4M3, 40, 64), s=d(L.MX_E8M0, 40, 2), qt=d(L.MX_E4M3, 64, 64), st=d(L.MX_E8M0, 64, 2), mode=1)
    check(L.lib().mx_quantize_both, good, [
        (dict(x=None), L.MX_ERR_INVALID, "x: null descriptor"),
        (dict(x=d(L.MX_F32, 40, 64, ptr=None)), L.MX_ERR_INVALID, "x: null data pointer"),
        (dict(x=d(L.MX_E4M3, 40, 64)), L.MX_ERR_DTYPE, "x must be"),
        (dict(x=d(L.MX_F32, 1, 40, 64)), L.MX_ERR_SHAPE, "2 dimensions"),
        (dict(x=d(L.MX_F32, 40, 64, ld=-64)), L.MX_ERR_LAYOUT, "x: rows"),
        (dict(x=d(L.MX_F32, 40, 31)), L.MX_ERR_SHAPE, "larger than the inner most dimension"),
        (dict(x=d(L.MX_F32, 1 << 40, 64)), L.MX_ERR_SHAPE, "out of range"),
        (dict(q=None), L.MX_ERR_INVALID, "xq: null descriptor"),
        (dict(q=d(L.MX_E4M3, 40, 96)), L.MX_ERR_SHAPE, "xq must be [40, 64]"),
        (dict(q=d(L.MX_E4M3, 40, 64, ptr=P + 4)), L.MX_ERR_LAYOUT, "xq: rows"),
        (dict(q=d(L.MX_E4M3, 40, 64, ld=32)), L.MX_ERR_LAYOUT, "xq: rows"),
        (dict(q=d(L.MX_E4M3, 40, 64, ld=68)), L.MX_ERR_LAYOUT, "xq: rows"),
        (dict(q=d(L.MX_E5M2, 40, 64)), L.MX_ERR_DTYPE, "both be"),
        (dict(q=d(L.MX_BF16, 40, 64), qt=d(L.MX_BF16, 64, 64)), L.MX_ERR_DTYPE, "MX_E4M3"),
        (dict(s=d(L.MX_E8M0, 40, 3)), L.MX_ERR_SHAPE, "scale must be [40, 2]"),
        (dict(s=d(L.MX_E4M3, 40, 2)), L.MX_ERR_DTYPE, "scale must be MX_E8M0"),
        (dict(s=d(L.MX_E8M0, 40, 2, ld=1)), L.MX_ERR_LAYOUT, "scale: rows overlap"),
        (dict(qt=d(L.MX_E4M3, 64, 40)), L.MX_ERR_SHAPE, "xt must be [64, 64]"),
        (dict(qt=d(L.MX_E4M3, 64, 64, ptr=P + 8)), L.MX_ERR_LAYOUT, "xt: rows"),
        (dict(st=None), L.MX_ERR_INVALID, "scale_t: null descriptor"),
        (dict(st=d(L.MX_E8M0, 64, 1)), L.MX_ERR_SHAPE, "scale_t must be"),
        (dict(mode=2), L.MX_ERR_INVALID, "scale_mode"),
    ])


def test_c_gated_gemm():
    lib = L.lib()
    M, K, F = 40, 128, 64
    need = lib.mx_gated_gemm_workspace_bytes(M, F, K, None)
    assert need >= M * 2 * F * 2 and lib.mx_gated_gemm_workspace_bytes(0, F, K, None) == 0
    good = dict(A=d(L.MX_E4M3, M, K), As=d(L.MX_E8M0, M, K // 32), W=d(L.MX_E4M3, 2 * F, K), Ws=d(L.MX_E8M0, 2 * F, K // 32),
                out=d(L.MX_E4M3, M, F), out_s=d(L.MX_E8M0, M, F // 32), gu=d(L.MX_E4M3, M, 2 * F), gus=d(L.MX_E8M0, M, F // 16), mode=1,
                opts=None, ws=P, ws_bytes=need)
    check(lib.mx_gated_gemm, good, [
        (dict(A=None), L.MX_ERR_INVALID, "null descriptor"),
        (dict(Ws=None), L.MX_ERR_INVALID, "null descriptor"),
        (dict(A=d(L.MX_E4M3, 1, M, K)), L.MX_ERR_SHAPE, "2 dimensions"),
        (dict(A=d(L.MX_E4M3, M, K, ptr=None)), L.MX_ERR_INVALID, "A: null data pointer"),
        (dict(W=d(L.MX_E4M3, 2 * F, K, ptr=None)), L.MX_ERR_INVALID, "W: null data pointer"),
        (dict(As=d(L.MX_E8M0, M, K // 32, ptr=None)), L.MX_ERR_INVALID, "A_scale: null data pointer"),
        (dict(Ws=d(L.MX_E8M0, 2 * F, K // 32, ptr=None)), L.MX_ERR_INVALID, "W_scale: null data pointer"),
        (dict(A=d(L.MX_E4M3, M, K, ld=-K)), L.MX_ERR_LAYOUT, "A: negative strides"),
        (dict(Ws=d(L.MX_E8M0, 2 * F, K // 32, ld=-4)), L.MX_ERR_LAYOUT, "W_scale: negative strides"),
        (dict(As=d(L.MX_E8M0, M, 3)), L.MX_ERR_SHAPE, "A_scale must be [40, 4]"),
        (dict(As=d(L.MX_E8M0, 2, M, K // 32)), L.MX_ERR_SHAPE, "A_scale must be [40, 4]"),
        (dict(Ws=d(L.MX_E8M0, F, K // 32)), L.MX_ERR_SHAPE, "W_scale must be [128, 4]"),
        (dict(W=d(L.MX_E4M3, 2 * F, 96)), L.MX_ERR_SHAPE, "K dimension of A (128) must match K dimension of W (96)"),
        (dict(W=d(L.MX_E4M3, 2 * F + 1, K)), L.MX_ERR_SHAPE, "2F rows"),
        (dict(W=d(L.MX_E4M3, 2 * F + 2, K)), L.MX_ERR_SHAPE, "multiple of 32"),
        (dict(W=d(L.MX_E4M3, 0, K)), L.MX_ERR_SHAPE, "multiple of 32"),
        (dict(out=d(L.MX_E4M3, M, 2 * F)), L.MX_ERR_SHAPE, "out must be"),
        (dict(out=d(L.MX_F32, M, F)), L.MX_ERR_DTYPE, "out must be MX_BF16"),
        (dict(out=d(L.MX_BF16, M, F)), L.MX_ERR_INVALID, "has none"),
        (dict(out=d(L.MX_BF16, M, F, ptr=P + 8), out_s=None), L.MX_ERR_LAYOUT, "out: rows"),
        (dict(out=d(L.MX_BF16, M, F, ld=F - 8), out_s=None), L.MX_ERR_LAYOUT, "out: rows"),
        (dict(out_s=None), L.MX_ERR_INVALID, "out_scale"),
        (dict(gu=None), L.MX_ERR_INVALID, "go together"),
        (dict(gus=None), L.MX_ERR_INVALID, "go together"),
        (dict(gu=d(L.MX_E5M2, M, 2 * F)), L.MX_ERR_DTYPE, "gate_up must be MX_E4M3"),
        (dict(gu=d(L.MX_E4M3, M, F)), L.MX_ERR_SHAPE, "gate_up must be"),
        (dict(mode=-1), L.MX_ERR_INVALID, "scale_mode"),
        (dict(ws=None), L.MX_ERR_WORKSPACE, "required"),
        (dict(ws=P + 16), L.MX_ERR_WORKSPACE, "aligned"),
        (dict(ws_bytes=need - 1), L.MX_ERR_WORKSPACE, "required"),
        (dict(A=d(L.MX_F16, M, K)), L.MX_ERR_DTYPE, "A/B must be"),
    ])
    for kernel, change in ((L.MX_KERNEL_STREAM, dict(A=d(L.MX_E4M3, 4, 96), As=d(L.MX_E8M0, 4, 3), W=d(L.MX_E4M3, 2 * F, 96), Ws=d(L.MX_E8M0, 2 * F, 3))),
                           (L.MX_KERNEL_MFMA_PINGPONG, dict(A=d(L.MX_E4M3, 4, K, ptr=P + 8), As=d(L.MX_E8M0, 4, 4)))):
        o = L.MxGemmOpts(struct_size=32, kernel=kernel, block_size=32)
        args = {**good, **change, "out": d(L.MX_E4M3, 4, F), "out_s": d(L.MX_E8M0, 4, F // 32), "gu": None, "gus": None, "opts": ctypes.byref(o),
                "ws_bytes": 1 << 19}
        assert lib.mx_gated_gemm(*refs(args.values()), None) == L.MX_ERR_LAYOUT, L.last_error()


def test_c_silu_backward():
    M, F = 40, 64
    good = dict(dh=d(L.MX_BF16, M, F), gu=d(L.MX_E4M3, M, 2 * F), gus=d(L.MX_E8M0, M, 4), q=d(L.MX_E4M3, M, 2 * F), s=d(L.MX_E8M0, M, 4),
                qt=d(L.MX_E4M3, 2 * F, 64), st=d(L.MX_E8M0, 2 * F, 2), at=d(L.MX_E4M3, F, 64), ats=d(L.MX_E8M0, F, 2), mode=1)
    check(L.lib().mx_silu_mul_backward_quantize, good, [
        (dict(dh=None), L.MX_ERR_INVALID, "dh: null descriptor"),
        (dict(dh=d(L.MX_F32, M, F)), L.MX_ERR_DTYPE, "dh must be MX_BF16"),
        (dict(dh=d(L.MX_BF16, M, 48)), L.MX_ERR_SHAPE, "multiple of 32"),
        (dict(dh=d(L.MX_BF16, M, 0)), L.MX_ERR_SHAPE, "multiple of 32"),
        (dict(gu=d(L.MX_E5M2, M, 2 * F)), L.MX_ERR_DTYPE, "gate_up must be MX_E4M3"),
        (dict(gu=d(L.MX_E4M3, M, F)), L.MX_ERR_SHAPE, "gate_up must be"),
        (dict(gu=d(L.MX_E4M3, M, 2 * F, ptr=P + 4)), L.MX_ERR_LAYOUT, "gate_up: rows"),
        (dict(gus=d(L.MX_E4M3, M, 4)), L.MX_ERR_DTYPE, "gate_up_scale"),
        (dict(gus=d(L.MX_E8M0, M, 2)), L.MX_ERR_SHAPE, "gate_up_scale must be"),
        (dict(q=d(L.MX_E4M3, M, F)), L.MX_ERR_SHAPE, "d must be"),
        (dict(s=None), L.MX_ERR_INVALID, "d_scale: null"),
        (dict(qt=d(L.MX_E4M3, 2 * F, 40)), L.MX_ERR_SHAPE, "dt must be"),
        (dict(at=d(L.MX_E4M3, F, 64, ptr=P + 8)), L.MX_ERR_LAYOUT, "at: rows"),
        (dict(at=d(L.MX_E5M2, F, 64)), L.MX_ERR_DTYPE, "MX_E4M3"),
        (dict(ats=d(L.MX_E8M0, F, 2, ld=1)), L.MX_ERR_LAYOUT, "at_scale: rows overlap"),
        (dict(mode=3), L.MX_ERR_INVALID, "scale_mode"),
    ])


def test_c_block():
    lib = L.lib()
    T, H, F, Ho = 40, 64, 96, 32
    kept, fwd, bwd = (f(T, H, F, Ho) for f in (lib.mx_ffn_saved_bytes, lib.mx_ffn_forward_workspace_bytes, lib.mx_ffn_backward_workspace_bytes))
    assert kept >= T * H + T * 2 * F + 2 * F * H + Ho * F and fwd > 0 and bwd > 0
    for f in (lib.mx_ffn_saved_bytes, lib.mx_ffn_forward_workspace_bytes, lib.mx_ffn_backward_workspace_bytes):
        assert f(0, H, F, Ho) == 0
    good = dict(x=d(L.MX_BF16, T, H), w1=d(L.MX_BF16, 2 * F, H), w2=d(L.MX_F32, Ho, F), y=d(L.MX_BF16, T, Ho), mode=1, saved=P, saved_bytes=kept,
                ws=P, ws_bytes=fwd)
    check(lib.mx_ffn_forward, good, [
        (dict(x=None), L.MX_ERR_INVALID, "x: null descriptor"),
        (dict(x=d(L.MX_E4M3, T, H)), L.MX_ERR_DTYPE, "x must be"),
        (dict(x=d(L.MX_BF16, T, 48), w1=d(L.MX_BF16, 2 * F, 48)), L.MX_ERR_SHAPE, "multiples of 32"),
        (dict(w1=d(L.MX_BF16, 2 * F, 32)), L.MX_ERR_SHAPE, "w1 must be"),
        (dict(w2=d(L.MX_BF16, Ho, 64)), L.MX_ERR_SHAPE, ""),
        (dict(w2=None), L.MX_ERR_INVALID, "w2: null descriptor"),
        (dict(y=d(L.MX_BF16, T, 64)), L.MX_ERR_SHAPE, "y must be"),
        (dict(y=d(L.MX_E4M3, T, Ho)), L.MX_ERR_DTYPE, "y must be"),
        (dict(y=d(L.MX_BF16, T, Ho, ld=16)), L.MX_ERR_LAYOUT, "y: rows overlap"),
        (dict(mode=7), L.MX_ERR_INVALID, "scale_mode"),
        (dict(saved_bytes=kept - 1), L.MX_ERR_WORKSPACE, "saved"),
        (dict(saved=P + 32), L.MX_ERR_WORKSPACE, "saved must be 256-byte aligned"),
        (dict(ws=None), L.MX_ERR_WORKSPACE, "workspace"),
        (dict(ws_bytes=fwd - 1), L.MX_ERR_WORKSPACE, "workspace"),
        # 2 GiB and more of one operand (the buffers are not read: the size is refused before)
        (dict(x=d(L.MX_BF16, 1 << 26, H), y=d(L.MX_BF16, 1 << 26, Ho)), L.MX_ERR_SHAPE, "2 GiB"),
    ])
    good = dict(dy=d(L.MX_BF16, T, Ho), saved=P, saved_bytes=kept, H=H, F=F, dx=d(L.MX_BF16, T, H), dw1=d(L.MX_F32, 2 * F, H), dw2=d(L.MX_F32, Ho, F),
                mode=1, ws=P, ws_bytes=bwd)
    check(lib.mx_ffn_backward, good, [
        (dict(dy=None), L.MX_ERR_INVALID, "dy: null descriptor"),
        (dict(dy=d(L.MX_E4M3, T, Ho)), L.MX_ERR_DTYPE, "dy must be"),
        (dict(H=48), L.MX_ERR_SHAPE, "multiples of 32"),
        (dict(F=0), L.MX_ERR_SHAPE, "multiples of 32"),
        (dict(dx=d(L.MX_BF16, T, F)), L.MX_ERR_SHAPE, "dx must be"),
        (dict(dw1=d(L.MX_F16, 2 * F, H)), L.MX_ERR_DTYPE, "dw1 must be"),
        (dict(dw2=d(L.MX_F32, Ho, F, ld=64)), L.MX_ERR_LAYOUT, "dw2: rows overlap"),
        (dict(dy=d(L.MX_BF16, 0, Ho), dx=None), L.MX_ERR_SHAPE, "no tokens"),
        (dict(saved=None), L.MX_ERR_WORKSPACE, "saved"),
        (dict(saved_bytes=kept - 256), L.MX_ERR_WORKSPACE, "saved"),
        (dict(ws=P + 128), L.MX_ERR_WORKSPACE, "workspace"),
        (dict(ws_bytes=0), L.MX_ERR_WORKSPACE, "workspace"),
    ])
    # nothing asked for: nothing enqueued
    assert lib.mx_ffn_backward(*refs({**good, "dx": None, "dw1": None, "dw2": None}.values()), None) == L.MX_OK
    assert lib.mx_ffn_forward(*refs({"x": d(L.MX_BF16, 0, H), "w1": d(L.MX_BF16, 2 * F, H), "w2": d(L.MX_BF16, Ho, F), "y": d(L.MX_BF16, 0, Ho),
                                     "mode": 1, "saved": None, "n": 0, "ws": None, "k": 0}.values()), None) == L.MX_OK


def test_sizes_grow_with_their_arguments():
    """Workspaces of a padded or larger call hold those of a smaller one."""
    lib = L.lib()
    for f in (lib.mx_ffn_saved_bytes, lib.mx_ffn_forward_workspace_bytes, lib.mx_ffn_backward_workspace_bytes):
        sizes = [f(T, 512, 1024, 512) for T in (1, 31, 32, 33, 64, 65, 512, 4096)]
        assert all(s % 256 == 0 for s in sizes) and sizes[-1] > sizes[-2] > sizes[0]
