"""Refusals of layer norm's and AdamW's entry points, without a GPU: every rule is checked before anything touches a device."""
import ctypes

import pytest
import torch

import cutile_amd as ct
from cutile_amd import _lib as L

bf16, f16, f32 = torch.bfloat16, torch.float16, torch.float32
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


# ---- the Python entry points -----------------------------------------------------------------------------------
@pytest.mark.parametrize("over,error,message", [
    (dict(), ValueError, "CUDA device"),
    (dict(x=torch.zeros(4, 64, dtype=torch.float64)), ct.TileTypeError, "Unsupported dtype float64 for x"),
    (dict(weight=torch.zeros(64, dtype=torch.int32)), ct.TileTypeError, "Unsupported dtype int32 for weight"),
    (dict(bias=torch.zeros(64, dtype=E4M3)), ct.TileTypeError, "for bias"),
    (dict(weight=torch.zeros(63)), ValueError, r"weight must be \(64,\)"),
    (dict(bias=torch.zeros(1, 64)), ValueError, r"bias must be \(64,\)"),
    (dict(x=torch.zeros(())), ct.TileTypeError, "at least one column"),
    (dict(x=torch.zeros(4, 0), weight=None, bias=None), ct.TileTypeError, "at least one column"),
    (dict(eps=-1e-5), ct.TileValueError, "eps"),
    (dict(eps=float("nan")), ct.TileValueError, "eps"),
])
@pytest.mark.parametrize("f", ["layer_norm", "layer_norm_forward", "layer_norm_quantize"])
def test_layer_norm_refusals(f, over, error, message):
    with pytest.raises(error, match=message):
        getattr(ct, f)(**{**dict(x=torch.zeros(4, 64), weight=torch.zeros(64), bias=torch.zeros(64)), **over})


@pytest.mark.parametrize("over,error,message", [
    (dict(dtype=bf16), ct.TileTypeError, "Unsupported quantisation dtype"),
    (dict(dtype="e3m4"), ct.TileTypeError, "Unsupported quantisation dtype"),
    (dict(scale_mode="round"), ct.TileValueError, "scale_mode"),
])
def test_layer_norm_quantize_refusals(over, error, message):
    with pytest.raises(error, match=message):
        ct.layer_norm_quantize(torch.zeros(4, 64), **over)


@pytest.mark.parametrize("over,error,message", [
    (dict(), ValueError, "CUDA device"),
    (dict(x=torch.zeros(4, 64, dtype=torch.int8)), ct.TileTypeError, "Unsupported dtype int8 for x"),
    (dict(weight=torch.zeros(32)), ValueError, "weight must be"),
])
def test_layer_norm_backward_refusals(over, error, message):
    a = dict(dy=torch.zeros(4, 64), x=torch.zeros(4, 64), mean=torch.zeros(4), rstd=torch.zeros(4), weight=torch.zeros(64))
    with pytest.raises(error, match=message):
        ct.layer_norm_backward(**{**a, **over})


def state(n, bits=32, dtype=f32):
    return ct.adamw_state(torch.zeros(n, dtype=dtype), bits)


@pytest.mark.parametrize("over,error,message", [
    (dict(), ValueError, "CUDA device"),
    (dict(grads=[]), ValueError, "as many gradients"),
    (dict(copies=[None, None]), ValueError, "as many gradients"),
    (dict(params=[torch.zeros(8, dtype=f16)]), ct.TileTypeError, "unsupported dtype float16"),
    (dict(grads=[torch.zeros(8, dtype=f16)]), ct.TileTypeError, "unsupported dtype float16"),
])
def test_adamw_refusals(over, error, message):
    a = dict(params=[torch.zeros(8)], grads=[torch.zeros(8)], states=[state(8)], step=1)
    with pytest.raises(error, match=message):
        ct.adamw_step(**{**a, **over})


def test_adamw_state():
    p = torch.zeros(3, 11, dtype=bf16)
    s = ct.adamw_state(p)
    assert s.exp_avg.shape == s.exp_avg_sq.shape == p.shape and s.exp_avg.dtype == f32 and s.exp_avg_scale is None
    s = ct.adamw_state(p, 8)
    assert s.exp_avg.shape == (64,) and s.exp_avg_sq.dtype == E4M3 and s.exp_avg_scale.shape == (2,) and s.exp_avg_sq_scale.dtype == E8M0
    assert all(bool((t.view(torch.uint8) == 0).all()) for t in s)
    with pytest.raises(ct.TileValueError, match="8 or 32"):
        ct.adamw_state(p, 16)
    with pytest.raises(ct.TileTypeError, match="float16"):
        ct.adamw_state(p.half())


# ---- the C entries -----------------------------------------------------------------------------------------------
BUF = torch.zeros(1 << 16, dtype=torch.uint8)
P = (BUF.data_ptr() + 255) // 256 * 256


def desc(dtype, shape, stride=None, ptr=P, packed=-1):
    d = L.MxTensor()
    d.ptr, d.dtype, d.ndim, d.packed_dim = ptr, dtype, len(shape), packed
    stride = stride or [int(torch.tensor(shape[i + 1:]).prod()) if i + 1 < len(shape) else 1 for i in range(len(shape))]
    for i, (s, st) in enumerate(zip(shape, stride)):
        d.shape[i], d.stride[i] = s, st
    return d


def ref(d):
    return None if d is None else ctypes.byref(d)


F, B, H16 = L.MX_F32, L.MX_BF16, L.MX_F16
NORM = dict(x=desc(B, (4, 64)), weight=desc(F, (64,)), bias=desc(B, (64,)), eps=1e-5, y=desc(B, (4, 64)), mean=desc(F, (4,)), rstd=desc(F, (4,)))


@pytest.mark.parametrize("over,code,message", [
    (dict(x=None), L.MX_ERR_INVALID, "x: null"),
    (dict(x=desc(L.MX_E4M3, (4, 64))), L.MX_ERR_DTYPE, "x must be"),
    (dict(x=desc(B, (4, 64), (1, 4))), L.MX_ERR_LAYOUT, "contiguous"),
    (dict(x=desc(B, (4, 64), (-64, 1))), L.MX_ERR_LAYOUT, "contiguous"),
    (dict(x=desc(B, (4, 0)), weight=None, bias=None, y=desc(B, (4, 0))), L.MX_ERR_SHAPE, "at least one column"),
    (dict(x=desc(B, (4, 64), ptr=None)), L.MX_ERR_INVALID, "null data pointer"),
    (dict(weight=desc(F, (63,))), L.MX_ERR_SHAPE, "weight must be"),
    (dict(weight=desc(F, (64,), (2,))), L.MX_ERR_LAYOUT, "contiguous"),
    (dict(bias=desc(L.MX_I32, (64,))), L.MX_ERR_DTYPE, "bias must be"),
    (dict(bias=desc(F, (64,), ptr=None)), L.MX_ERR_INVALID, "null data pointer"),
    (dict(eps=-1.0), L.MX_ERR_INVALID, "eps"),
    (dict(eps=float("nan")), L.MX_ERR_INVALID, "eps"),
    (dict(y=None), L.MX_ERR_INVALID, "y: null"),
    (dict(y=desc(F, (4, 64))), L.MX_ERR_DTYPE, "type of x"),
    (dict(y=desc(B, (4, 65))), L.MX_ERR_SHAPE, "y must be"),
    (dict(y=desc(B, (4, 64), (63, 1))), L.MX_ERR_LAYOUT, "overlap"),
    (dict(mean=desc(F, (3,))), L.MX_ERR_SHAPE, "mean must be"),
    (dict(rstd=desc(B, (4,))), L.MX_ERR_DTYPE, "rstd must be MX_F32"),
])
def test_layer_norm_codes(over, code, message):
    a = {**NORM, **over}
    rc = L.lib().mx_layer_norm(ref(a["x"]), ref(a["weight"]), ref(a["bias"]), a["eps"], ref(a["y"]), ref(a["mean"]), ref(a["rstd"]), None)
    assert rc == code and message in L.last_error(), L.last_error()


QUANT = dict(x=desc(B, (4, 60)), q=desc(L.MX_E4M3, (4, 64)), s=desc(L.MX_E8M0, (4, 2)), mode=1)


@pytest.mark.parametrize("over,code,message", [
    (dict(x=desc(B, (4, 31)), q=desc(L.MX_E4M3, (4, 32)), s=desc(L.MX_E8M0, (4, 1))), L.MX_ERR_SHAPE, "larger than the inner most"),
    (dict(q=None), L.MX_ERR_INVALID, "xq: null"),
    (dict(q=desc(B, (4, 64))), L.MX_ERR_DTYPE, "element format"),
    (dict(q=desc(L.MX_E4M3, (4, 60))), L.MX_ERR_SHAPE, "xq must be"),
    (dict(q=desc(L.MX_E4M3, (4, 64), (68, 1))), L.MX_ERR_LAYOUT, "aligned to 8"),
    (dict(q=desc(L.MX_E4M3, (4, 64), ptr=P + 4)), L.MX_ERR_LAYOUT, "aligned to 8"),
    (dict(q=desc(L.MX_E2M1, (4, 64), (32, 1))), L.MX_ERR_LAYOUT, "packed along H"),
    (dict(q=desc(L.MX_E2M1, (4, 62), (32, 1), packed=1)), L.MX_ERR_SHAPE, "xq must be"),
    (dict(q=desc(L.MX_E2M1, (4, 64), (34, 1), packed=1)), L.MX_ERR_LAYOUT, "aligned to 4"),
    (dict(s=desc(L.MX_E8M0, (4, 3))), L.MX_ERR_SHAPE, "scale must be"),
    (dict(s=desc(L.MX_E4M3, (4, 2))), L.MX_ERR_DTYPE, "scale must be"),
    (dict(s=desc(L.MX_E8M0, (4, 2), (1, 1))), L.MX_ERR_LAYOUT, "overlap"),
    (dict(mode=2), L.MX_ERR_INVALID, "scale_mode"),
])
def test_layer_norm_quantize_codes(over, code, message):
    a = {**QUANT, **over}
    rc = L.lib().mx_layer_norm_quantize(ref(a["x"]), None, None, 1e-5, ref(a["q"]), ref(a["s"]), a["mode"], None)
    assert rc == code and message in L.last_error(), L.last_error()


BACK = dict(dy=desc(B, (4, 64)), x=desc(B, (4, 64)), mean=desc(F, (4,)), rstd=desc(F, (4,)), weight=desc(F, (64,)), dx=desc(B, (4, 64)),
            dw=desc(F, (64,)), db=desc(B, (64,)), ws=P, bytes=1 << 14)


@pytest.mark.parametrize("over,code,message", [
    (dict(dy=desc(F, (4, 64))), L.MX_ERR_DTYPE, "dy must have the type of x"),
    (dict(dy=desc(B, (3, 64))), L.MX_ERR_SHAPE, "dy must be"),
    (dict(mean=None), L.MX_ERR_INVALID, "mean and rstd"),
    (dict(rstd=desc(F, (5,))), L.MX_ERR_SHAPE, "rstd must be"),
    (dict(mean=desc(B, (4,))), L.MX_ERR_DTYPE, "mean must be MX_F32"),
    (dict(dx=desc(F, (4, 64))), L.MX_ERR_DTYPE, "dx must have the type of x"),
    (dict(dw=desc(F, (65,))), L.MX_ERR_SHAPE, "dweight must be"),
    (dict(db=desc(L.MX_E4M3, (64,))), L.MX_ERR_DTYPE, "dbias must be"),
    (dict(ws=None), L.MX_ERR_WORKSPACE, "workspace"),
    (dict(bytes=16), L.MX_ERR_WORKSPACE, "workspace"),
    (dict(ws=P + 64), L.MX_ERR_WORKSPACE, "aligned"),
    (dict(dy=desc(B, (0, 64)), x=desc(B, (0, 64)), mean=desc(F, (0,)), rstd=desc(F, (0,)), dx=desc(B, (0, 64))), L.MX_ERR_SHAPE, "no rows"),
])
def test_layer_norm_backward_codes(over, code, message):
    a = {**BACK, **over}
    rc = L.lib().mx_layer_norm_backward(*(ref(a[n]) for n in ("dy", "x", "mean", "rstd", "weight", "dx", "dw", "db")), a["ws"], a["bytes"], None)
    assert rc == code and message in L.last_error(), L.last_error()
    assert L.lib().mx_layer_norm_backward_workspace_bytes(0, 64) == 0


def adam(tensors, **over):
    o = L.MxAdamwOpts(struct_size=ctypes.sizeof(L.MxAdamwOpts), state_bits=32, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, grad_scale=1.0, step=1)
    for k, v in over.items():
        setattr(o, k, v)
    items = (L.MxAdamwTensor * max(1, len(tensors)))(*tensors)
    return L.lib().mx_adamw_step(len(tensors), items, ctypes.byref(o), None)


def one(at=0, n=64, p=F, g=F, small=False, **over):
    q = P + at
    t = L.MxAdamwTensor(param=q, grad=q + 1024, exp_avg=q + 2048, exp_avg_sq=q + 3008, n=n, param_dtype=p, grad_dtype=g)
    if small:
        t.exp_avg_scale, t.exp_avg_sq_scale = q + 3500, q + 3600
    for k, v in over.items():
        setattr(t, k, v)
    return t


@pytest.mark.parametrize("tensors,over,code,message", [
    ([one()], dict(struct_size=8), L.MX_ERR_INVALID, "another version"),
    ([one()], dict(state_bits=16), L.MX_ERR_INVALID, "8 or 32 bits"),
    ([one()], dict(lr=-1.0), L.MX_ERR_INVALID, "learning rate"),
    ([one()], dict(lr=float("nan")), L.MX_ERR_INVALID, "learning rate"),
    ([one()], dict(beta1=1.0), L.MX_ERR_INVALID, "betas"),
    ([one()], dict(beta2=-0.1), L.MX_ERR_INVALID, "betas"),
    ([one()], dict(eps=-1e-8), L.MX_ERR_INVALID, "eps"),
    ([one()], dict(weight_decay=float("inf")), L.MX_ERR_INVALID, "weight decay"),
    ([one()], dict(grad_scale=float("nan")), L.MX_ERR_INVALID, "scale"),
    ([one()], dict(step=0), L.MX_ERR_INVALID, "from 1"),
    ([one(n=-1)], {}, L.MX_ERR_SHAPE, "tensor 0"),
    ([one(p=H16)], {}, L.MX_ERR_DTYPE, "tensor 0"),
    ([one(), one(at=8192, g=H16)], {}, L.MX_ERR_DTYPE, "tensor 1"),
    ([one(param=None)], {}, L.MX_ERR_INVALID, "null"),
    ([one(exp_avg_sq=None)], {}, L.MX_ERR_INVALID, "null"),
    ([one()], dict(state_bits=8), L.MX_ERR_INVALID, "null"),
    ([one(param=P + 2)], {}, L.MX_ERR_LAYOUT, "misaligned"),
    ([one(small=True, exp_avg=P + 2052)], dict(state_bits=8), L.MX_ERR_LAYOUT, "misaligned"),
    ([one(copy=P + 5001)], {}, L.MX_ERR_LAYOUT, "misaligned"),
    ([one(), one()], {}, L.MX_ERR_INVALID, "overlap"),
    ([one(), one(at=8192, param=P + 252)], {}, L.MX_ERR_INVALID, "overlap"),
    ([one(copy=P + 2300)], {}, L.MX_ERR_INVALID, "overlap"),
    ([one(small=True, exp_avg_sq_scale=P + 3501)], dict(state_bits=8), L.MX_ERR_INVALID, "overlap"),
])
def test_adamw_codes(tensors, over, code, message):
    assert adam(tensors, **over) == code and message in L.last_error(), L.last_error()


def test_nothing_to_do_is_fine():
    assert adam([]) == L.MX_OK and adam([one(n=0), one(n=0, param=None)]) == L.MX_OK
    ct.adamw_step([], [], [], step=1)
    assert L.lib().mx_adamw_step(-1, None, None, None) == L.MX_ERR_INVALID
    assert ctypes.sizeof(L.MxAdamwTensor) == 72 and ctypes.sizeof(L.MxAdamwOpts) == 96
