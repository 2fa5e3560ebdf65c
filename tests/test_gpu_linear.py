"""The linear layer's epilogue and its trained form against 64-bit arithmetic: every kernel that finishes it, every format, activation and
type around it, sizes at the edges of tiles, blocks and vectors."""
import ctypes

import pytest
import torch

import ffnutil as R
from cutile_amd import _lib as L
from mxutil import randn_operand
from oracle import mx_oracle as O
from test_gpu_ffn_elements import check_codes, tiles
from test_gpu_ffn_elements import sum_error as aligned

pytestmark = pytest.mark.gpu

bf16, f16, f32 = torch.bfloat16, torch.float16, torch.float32
FMT = {"e4m3": O.E4M3, "e5m2": O.E5M2, "e2m1": O.E2M1}
ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]


def sum_error(A, W):
    """Products are aligned to the power of two of the largest: mantissas below 2 make products below 4, so that the last bit kept, 2^-18 of the
    power of two above, is up to 2^-17 of the largest product, and each of the K is off by less than that.  (32 products, E4M3: 1.56 x 2^-18
    a product seen.)"""
    return 2 * aligned(A, W)


def u8(t):
    return t.view(torch.uint8)


def d64(t):
    return t.detach().cpu().double()


def act64(p, name):
    """The activation and its derivative."""
    if name is None:
        return p, torch.ones_like(p)
    if name == "relu":
        return p.clamp(min=0), (p > 0).double()
    if name == "gelu":
        t = torch.special.ndtr(p)
        return p * t, t + p * torch.exp(-p * p / 2) / (2 * torch.pi) ** 0.5
    if name == "silu":
        t = torch.sigmoid(p)
        return p * t, t * (1 + p * (1 - t))
    c = (2 / torch.pi) ** 0.5
    t = torch.tanh(c * (p + 0.044715 * p ** 3))
    return 0.5 * p * (1 + t), 0.5 * (1 + t) + 0.5 * p * (1 - t * t) * c * (1 + 0.134145 * p * p)


def around(dev, M, N, bt, rt, seed):
    g = torch.Generator().manual_seed(seed)
    return (None if bt is None else (0.5 * torch.randn(N, generator=g)).to(bt).to(dev),
            None if rt is None else torch.randn((M, N), generator=g).to(rt).to(dev))


def definition(a, w, bias, res, act):
    """(result, bound of a kernel's before it is rounded): the product's, through a slope of 1.13 at most; 2e-6 of the activation (its
    polynomial, the hardware's 2^x and reciprocal, exp's rounded argument); some roundings of 2^-24."""
    A, W = (O.dequantize(t.codes, t.scales, t.fmt).double() for t in (a, w))
    p = A @ W.T
    if bias is not None:
        p = p + d64(bias)
    y, _ = act64(p, act)
    err = 1.13 * (sum_error(A, W) + 2.0 ** -23 * p.abs()) + 2e-6 * y.abs()
    if res is not None:
        y, err = y + d64(res), err + 2.0 ** -23 * d64(res).abs()
    return p, y, err + 2.0 ** -23 * y.abs()


def check(got, want, err, dtype):
    bad = ~((d64(got) - want).abs() <= err + {f32: 2.0 ** -24, bf16: R.HALF_BF16}[dtype] * (want.abs() + err))
    assert not bool(bad.any()), (float((d64(got) - want).abs().max()), int(bad.sum()), bad.nonzero()[:4].tolist())


CASES = [
    # kernel, formats, M, K, N, bias, residual, activation
    ("auto", "e4m3", "e4m3", 1, 2048, 8192, bf16, None, "gelu_tanh"),
    ("auto", "e4m3", "e2m1", 32, 4096, 512, bf16, bf16, "gelu"),
    ("auto", "e4m3", "e4m3", 3, 512, 96, f32, None, "silu"),
    ("auto", "e4m3", "e4m3", 7, 160, 37, f32, f32, "gelu"),
    ("auto", "e5m2", "e5m2", 40, 1024, 224, None, bf16, "relu"),
    ("auto", "e5m2", "e2m1", 9, 256, 65, f16, f16, None),
    ("auto", "e2m1", "e2m1", 130, 544, 320, bf16, None, "gelu_tanh"),
    ("auto", "e4m3", "e4m3", 100, 96, 1, None, None, "silu"),
    ("auto", "e4m3", "e4m3", 333, 32, 130, bf16, f32, "gelu"),
    ("auto", "e4m3", "e4m3", 700, 1024, 1536, bf16, bf16, None),
    ("auto", "e4m3", "e2m1", 1300, 512, 1120, f32, None, "relu"),
    ("auto", "e4m3", "e4m3", 1531, 2048, 1088, bf16, bf16, "gelu"),
    ("auto", "e4m3", "e4m3", 200, 12288, 256, bf16, bf16, "silu"),
    ("auto", "e4m3", "e2m1", 17, 8192, 24640, bf16, bf16, "gelu"),  # many weights
    ("stream", "e4m3", "e4m3", 1, 128, 32, bf16, bf16, "gelu"),
    ("stream", "e4m3", "e4m3", 17, 1152, 97, f32, bf16, "gelu_tanh"),
    ("stream", "e4m3", "e2m1", 64, 4224, 160, None, f32, "silu"),
    ("stream", "e5m2", "e5m2", 33, 640, 1000, bf16, None, "relu"),
    ("stream", "e4m3", "e4m3", 100, 2048, 2944, bf16, bf16, None),
    ("stream", "e4m3", "e4m3", 2, 2048, 4099, f16, f32, "gelu"),   # units of sixteen columns where the result is not quantised
    ("stream", "e4m3", "e2m1", 16, 1024, 4096, bf16, bf16, "silu"),
    ("decode", "e4m3", "e2m1", 20, 1024, 9248, bf16, bf16, "gelu"),
    ("decode", "e4m3", "e2m1", 31, 512, 224, f32, None, "silu"),
    ("decode", "e4m3", "e2m1", 7, 8192, 96, f16, f32, "gelu"),
    ("decode", "e4m3", "e2m1", 32, 4608, 16480, bf16, bf16, "gelu_tanh"),
    ("decode", "e4m3", "e2m1", 16, 1536, 16416, None, f16, "relu"),
    ("decode", "e4m3", "e2m1", 5, 512, 48, bf16, bf16, "gelu"),
    ("decode", "e4m3", "e2m1", 40, 512, 64, bf16, bf16, None),
    ("mfma128", "e4m3", "e4m3", 1, 32, 64, bf16, None, "gelu"),
    ("mfma128", "e4m3", "e4m3", 257, 544, 192, f32, bf16, "gelu_tanh"),
    ("mfma128", "e2m1", "e2m1", 300, 1536, 450, bf16, f16, "silu"),
    ("mfma128", "e5m2", "e5m2", 1000, 512, 2500, bf16, f32, "relu"),
    ("mfma128", "e4m3", "e2m1", 130, 4096, 136, bf16, None, None),
    ("mfma128", "e4m3", "e4m3", 70, 8192, 72, bf16, bf16, "gelu"),
    ("pingpong", "e4m3", "e4m3", 1, 32, 64, bf16, None, "gelu"),
    ("pingpong", "e4m3", "e4m3", 257, 544, 192, f32, bf16, "gelu_tanh"),
    ("pingpong", "e4m3", "e2m1", 300, 1536, 449, bf16, f16, "silu"),
    ("pingpong", "e5m2", "e5m2", 513, 1024, 300, f16, f32, "relu"),
    ("pingpong", "e2m1", "e2m1", 1025, 1024, 2944, bf16, bf16, "gelu"),
    ("pingpong", "e4m3", "e4m3", 1531, 512, 1088, None, bf16, None),
    ("pingpong", "e4m3", "e4m3", 2305, 512, 4161, bf16, None, "gelu"),
    ("pingpong", "e4m3", "e4m3", 2305, 1024, 4160, bf16, bf16, "silu"),
    # tiles split along K: all of them; those behind a whole round
    ("pingpong", "e4m3", "e4m3", 500, 4096, 520, bf16, bf16, "gelu"),
    ("pingpong", "e4m3", "e4m3", 257, 8192, 288, f32, None, "silu"),
    ("pingpong", "e4m3", "e2m1", 1, 4096, 264, None, bf16, None),
    ("pingpong", "e4m3", "e2m1", 600, 6144, 544, bf16, None, "gelu_tanh"),
    ("pingpong", "e4m3", "e4m3", 4200, 4096, 4128, bf16, bf16, "gelu"),
    ("auto", "e4m3", "e4m3", 1531, 8192, 1088, bf16, bf16, "relu"),
    ("pingpong", "e2m1", "e2m1", 500, 8192, 520, bf16, bf16, "gelu"),
    ("pingpong", "e2m1", "e2m1", 300, 1536, 448, f32, None, "gelu_tanh"),
    ("pingpong", "e2m1", "e2m1", 1531, 1056, 1088, None, bf16, None),
    ("auto", "e2m1", "e2m1", 2048, 2048, 4096, bf16, bf16, "silu"),
    ("pingpong", "e4m3", "e4m3", 700, 640, 1088, bf16, f32, "gelu"),
    ("pingpong", "e4m3", "e4m3", 257, 640, 192, f32, bf16, "gelu_tanh"),
    ("pingpong", "e4m3", "e4m3", 300, 256, 320, bf16, None, "silu"),
    ("pingpong", "e4m3", "e4m3", 700, 544, 1088, bf16, f32, "gelu"),   # (results of both types: fp32 with fp32 residuals)
    ("pingpong", "e4m3", "e2m1", 500, 4096, 520, None, f32, "silu"),
    ("pingpong", "e2m1", "e2m1", 300, 1056, 448, f32, f32, None),
    # at the ping-pong kernel's sizes what it does not finish
    ("auto", "e5m2", "e5m2", 2048, 1024, 4096, bf16, bf16, "gelu"),
    ("auto", "e4m3", "e4m3", 2048, 1024, 4097, bf16, f32, "silu"),
    ("auto", "e4m3", "e2m1", 2048, 1024, 4096, f16, f16, "relu"),
    ("mfma256", "e4m3", "e4m3", 300, 512, 320, bf16, bf16, "gelu"),
    # through memory, some rows at a time
    ("mfma256", "e2m1", "e2m1", 2305, 256, 2080, bf16, bf16, "gelu"),
    ("pingpong32", "e4m3", "e4m3", 1500, 544, 4160, bf16, None, "silu"),
    ("pingpong", "e5m2", "e5m2", 1100, 1024, 8200, None, bf16, "relu"),
    ("generic", "e4m3", "e4m3", 33, 96, 64, bf16, bf16, "gelu"),
    ("generic", "e2m1", "e4m3", 5, 64, 30, f32, f32, "silu"),
]


@pytest.mark.parametrize("kernel,af,wf,M,K,N,bt,rt,act", CASES)
def test_product_with_epilogue(ct, dev, kernel, af, wf, M, K, N, bt, rt, act):
    a, w = randn_operand(M, K, FMT[af], M + K, dev), randn_operand(N, K, FMT[wf], N, dev, std=K ** -0.5)
    bias, res = around(dev, M, N, bt, rt, M + N)
    p, want, err = definition(a, w, bias, res, act)
    kw = dict(activation=act, a_format=a.fmt_kw, w_format=w.fmt_kw, kernel=kernel)
    scales = [(a.scale_t, w.scale_t)]
    if kernel in ("mfma128", "pingpong", "mfma256", "pingpong32"):
        scales.append(tuple(ct.pack_scales(t.scale_t, operand=o, kernel=kernel) for t, o in ((a, "a"), (w, "b"))))
    elif kernel in ("auto", "stream") and K % 128 == 0:
        scales.append((a.scale_t, ct.pack_scales(w.scale_t, operand="b")))
    for a_s, w_s in scales:
        args = (a.storage, a_s, w.storage, w_s, bias, res)
        for dtype in (bf16, f32):
            y = ct.block_scaled_linear(*args, out_dtype=dtype, **kw)
            assert y.dtype == dtype and y.shape == (M, N)
            check(y, want, err, dtype)
        if N % 32 == 0:
            q, s = ct.block_scaled_linear(*args, out_dtype=torch.float8_e4m3fn, **kw)
            assert q.shape == (M, N) and s.shape == (M, N // 32) and bool(q.float().isfinite().all())
            check_codes(q, s, want, err)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("kernel,M,K,N", [("stream", 20, 256, 96), ("stream", 1, 512, 8192), ("mfma128", 200, 288, 160), ("pingpong", 300, 544, 288), ("pingpong", 300, 640, 288), ("auto", 300, 512, 96),
                                          ("generic", 9, 64, 32)])
def test_every_activation_everywhere(ct, dev, kernel, M, K, N, act):
    """Arguments from -40 to 40, by way of the bias; every row the same product."""
    a, w = randn_operand(1, K, O.E4M3, K, dev), randn_operand(N, K, O.E4M3, N, dev, std=K ** -0.5)
    A, As = a.storage.expand(M, K), a.scale_t.expand(M, K // 32)
    bias = torch.linspace(-40, 40, N).to(dev)
    a.codes, a.scales = a.codes.repeat(M, 0), a.scales.repeat(M, 0)
    p, want, err = definition(a, w, bias, None, act)
    for dtype in (bf16, f32):
        y = ct.block_scaled_linear(A, As, w.storage, w.scale_t, bias, activation=act, out_dtype=dtype, kernel=kernel)
        check(y, want, err, dtype)


@pytest.mark.parametrize("kernel,M,K,N", [("stream", 20, 256, 96), ("mfma128", 200, 288, 160), ("pingpong", 300, 544, 288), ("pingpong", 300, 640, 288), ("pingpong", 1100, 1024, 1056), ("auto", 70, 512, 96)])
def test_not_finite(ct, dev, kernel, M, K, N):
    a, w = randn_operand(M, K, O.E4M3, M, dev), randn_operand(N, K, O.E4M3, N, dev, std=K ** -0.5)
    args, inf = (a.storage, a.scale_t, w.storage, w.scale_t), float("inf")
    bias = torch.zeros(N, device=dev)
    bias[0], bias[1], bias[2] = -inf, inf, float("nan")
    for act in ACTS:
        plain = ct.block_scaled_linear(*args, torch.zeros(N, device=dev), activation=act, kernel=kernel, out_dtype=f32)
        y = ct.block_scaled_linear(*args, bias, activation=act, kernel=kernel, out_dtype=f32)
        assert bool((y[:, 1] == inf).all()) and bool(y[:, 2].isnan().all()) and torch.equal(y[:, 3:], plain[:, 3:])
        assert bool((y[:, 0] == (-inf if act is None else 0)).all())
        q, s = ct.block_scaled_linear(*args, bias, activation=act, kernel=kernel, out_dtype="e4m3")
        clean, cs = ct.block_scaled_linear(*args, torch.zeros(N, device=dev), activation=act, kernel=kernel, out_dtype="e4m3")
        # block_quantize of a block with a NaN: its scale, zeros beside it (the infinity is the largest number of it: 1.75 x 2^128 / 2^120 = 448)
        want, ws = ct.block_quantize(y[:, :32].contiguous(), 32, scale_mode="floor")
        assert torch.equal(u8(s)[:, :1], u8(ws)) and torch.equal(q[:, 3:32].float(), want[:, 3:].float()) and bool(q[:, 2].float().isnan().all())
        assert torch.equal(u8(q)[:, 32:], u8(clean)[:, 32:]) and torch.equal(u8(s)[:, 1:], u8(cs)[:, 1:])


def test_views_around_the_product(ct, dev):
    """Bias and residual off 16-byte borders, of wider matrices, broadcast rows; a residual of three dimensions is none."""
    for kernel, M, K, N in (("stream", 5, 256, 64), ("mfma128", 150, 128, 96), ("pingpong", 300, 256, 290)):
        a, w = randn_operand(M, K, O.E4M3, M, dev), randn_operand(N, K, O.E4M3, N, dev)
        bias, res = around(dev, M, N + 7, bf16, bf16, 1)
        b = bias[3:3 + N]
        args = (a.storage, a.scale_t, w.storage, w.scale_t)
        for r in (res[:, 5:5 + N], res[:, :N].T.contiguous().T, res[:1, 1:1 + N].expand(M, N), res.repeat(2, 1)[::2, :N]):
            want = ct.block_scaled_linear(*args, b.clone(), r.contiguous(), kernel=kernel)
            assert torch.equal(ct.block_scaled_linear(*args, b, r, kernel=kernel), want)
        with pytest.raises(ValueError, match="residual must be"):
            ct.block_scaled_linear(*args, b, res[None, :, :N], kernel=kernel)


PAD, MARK = 64, 0xA5


def padded(dev, rows, cols, dtype, offset=0):
    """(whole buffer filled with a mark, descriptor of its [rows, cols] part, which begins `offset` elements into it)."""
    size = {L.MX_F32: 4, L.MX_BF16: 2}.get(dtype, 1)
    buf = torch.full((rows + 2, (cols + PAD) * size), MARK, dtype=torch.uint8, device=dev)
    t = L.MxTensor()
    t.ptr, t.dtype, t.ndim, t.packed_dim = buf.data_ptr() + offset * size, dtype, 2, -1
    t.shape[0], t.shape[1], t.stride[0], t.stride[1] = rows, cols, cols + PAD, 1
    return buf, t


def inner(buf, rows, cols, size, offset=0):
    at = slice(offset * size, (offset + cols) * size)
    got = buf[:rows, at].contiguous()
    rest = buf.clone()
    rest[:rows, at] = MARK
    assert bool((rest == MARK).all()), "written outside of the output"
    return got


@pytest.mark.parametrize("kernel,M,K,N", [("stream", 3, 640, 96), ("stream", 50, 256, 67), ("mfma128", 77, 288, 160), ("mfma128", 130, 4096, 100), ("pingpong", 300, 512, 320),
                                          ("pingpong", 500, 512, 333), ("pingpong", 300, 4096, 320), ("stream", 2, 1024, 4096), ("generic", 5, 64, 32)])
@pytest.mark.parametrize("out,offset", [("bf16", 0), ("bf16", 1), ("f32", 0), ("f32", 3), ("e4m3", 0)])
def test_padded_outputs(ct, dev, kernel, M, K, N, out, offset):
    if out == "e4m3" and N % 32:
        N = N // 32 * 32
    a, w = randn_operand(M, K, O.E4M3, M, dev), randn_operand(N, K, O.E4M3, N, dev, std=K ** -0.5)
    bias, res = around(dev, M, N, bf16, bf16, 2)
    o = L.MxGemmOpts(struct_size=32, kernel=L.KERNELS[kernel], block_size=32)
    lib = L.lib()
    need = lib.mx_linear_gemm_workspace_bytes(M, N, K, ctypes.byref(o))
    ws = torch.empty(max(need, 256), dtype=torch.uint8, device=dev)
    fmt, size, dtype = {"bf16": (L.MX_BF16, 2, bf16), "f32": (L.MX_F32, 4, f32), "e4m3": (L.MX_E4M3, 1, torch.float8_e4m3fn)}[out]
    c, dc = padded(dev, M, N, fmt, offset)
    s, ds = padded(dev, M, N // 32, L.MX_E8M0)
    p, dp = padded(dev, M, N, L.MX_BF16, 1)
    ref = lambda d: None if d is None else ctypes.byref(d)  # noqa: E731
    args = [ref(L.desc(u8(a.storage), L.MX_E4M3)), ref(L.desc(u8(a.scale_t), L.MX_E8M0)), ref(L.desc(u8(w.storage), L.MX_E4M3)),
            ref(L.desc(u8(w.scale_t), L.MX_E8M0)), ref(L.desc(bias, L.MX_BF16)), ref(L.desc(res, L.MX_BF16)), L.MX_ACT_GELU, ref(dc),
            ref(ds) if out == "e4m3" else None, ref(dp), ref(o), ws.data_ptr(), need, L.stream_ptr(dev)]
    assert lib.mx_linear_gemm(*args) == L.MX_OK, L.last_error()
    want = ct.block_scaled_linear(a.storage, a.scale_t, w.storage, w.scale_t, bias, res, activation="gelu", kernel=kernel, out_dtype=dtype)
    pre = ct.block_scaled_linear(a.storage, a.scale_t, w.storage, w.scale_t, bias, kernel=kernel)
    got_c, got_p = inner(c, M, N, size, offset), inner(p, M, N, 2, 1)
    got_s = inner(s, M, N // 32, 1) if out == "e4m3" else inner(s, 0, 0, 1)
    if kernel == "pingpong" and K >= 4096:
        # The call above splits K, this one does not (`pre` is off 16 bytes): the same products added in another order, so the two differ by
        # up to twice the bound of a sum.  Both are held to the definition instead, whose bound covers any order.
        P, y, err = definition(a, w, bias, res, "gelu")
        for q, z in ((got_c, got_s), (u8(want[0]), u8(want[1]))) if out == "e4m3" else ((got_c, None), (u8(want), None)):
            check_codes(q.view(dtype), z.view(torch.float8_e8m0fnu), y, err) if out == "e4m3" else check(q.view(dtype), y, err, dtype)
        for q in (got_p.view(bf16), pre):
            check(q, P, err + 2.0 ** -22 * P.abs(), bf16)
        return
    if out == "e4m3":
        assert torch.equal(got_c, u8(want[0])) and torch.equal(got_s, u8(want[1]))
    else:
        assert torch.equal(got_c, u8(want))
    assert torch.equal(got_p, u8(pre))


def raw(ct, dev, kernel, a, w, bias, res, out, act=L.MX_ACT_GELU, pre=None):
    """The C entry with views as they are."""
    M, K, N = a.storage.shape[0], a.storage.shape[1], w.storage.shape[0]
    o, lib = L.MxGemmOpts(struct_size=32, kernel=L.KERNELS[kernel], block_size=32), L.lib()
    need = lib.mx_linear_gemm_workspace_bytes(M, N, K, ctypes.byref(o))
    ws = torch.empty(max(need, 256), dtype=torch.uint8, device=dev)
    ref = lambda t: None if t is None else ctypes.byref(L.desc(t, L._TORCH_TO_MX[t.dtype]))  # noqa: E731
    rc = lib.mx_linear_gemm(ctypes.byref(L.desc(u8(a.storage), L.MX_E4M3)), ctypes.byref(L.desc(u8(a.scale_t), L.MX_E8M0)),
                            ctypes.byref(L.desc(u8(w.storage), L.MX_E4M3)), ctypes.byref(L.desc(u8(w.scale_t), L.MX_E8M0)), ref(bias), ref(res), act, ref(out), None,
                            ref(pre), ctypes.byref(o), ws.data_ptr(), need, L.stream_ptr(dev))
    assert rc == L.MX_OK, L.last_error()


@pytest.mark.parametrize("kernel", ["stream", "mfma128", "pingpong", "generic"])
def test_one_row_of_any_pitch(ct, dev, kernel):
    K, N = 256, 96
    a, w = randn_operand(1, K, O.E4M3, 1, dev), randn_operand(N, K, O.E4M3, 2, dev)
    bias, res = around(dev, 1, N, bf16, bf16, 3)
    want = ct.block_scaled_linear(a.storage, a.scale_t, w.storage, w.scale_t, bias, res, activation="gelu", kernel=kernel)
    pre = ct.block_scaled_linear(a.storage, a.scale_t, w.storage, w.scale_t, bias, kernel=kernel)
    for pitch in (1, 8, 5 * N):
        wide = torch.full((8 * N,), 7.0, device=dev)
        raw(ct, dev, kernel, a, w, bias, res.float().as_strided((1, N), (pitch, 1)), wide.as_strided((1, N), (pitch, 1)))
        assert torch.equal(wide[:N].to(bf16), want[0]) and bool((wide[N:] == 7).all())
        out, p = (torch.full((8 * N,), 7.0, dtype=bf16, device=dev) for _ in range(2))
        raw(ct, dev, kernel, a, w, bias, res.as_strided((1, N), (pitch, 1)), out.as_strided((1, N), (pitch, 1)), pre=p.as_strided((1, N), (pitch, 1)))
        assert torch.equal(out[:N], want[0]) and bool((out[N:] == 7).all())
        assert torch.equal(p[:N], pre[0]) and bool((p[N:] == 7).all())


@pytest.mark.parametrize("dtype", [bf16, f32])
@pytest.mark.parametrize("kernel", ["mfma128", "pingpong"])
def test_rows_far_apart(ct, dev, kernel, dtype):
    """Nine rows 2^27 bytes apart: 32 of such pitches are 2^32, where a tile's rows behind the last must not come round to."""
    M, K, N, pitch = 9, 256, 128, (1 << 27) // (2 if dtype == bf16 else 4)
    a, w = randn_operand(M, K, O.E4M3, 1, dev), randn_operand(N, K, O.E4M3, 2, dev)
    bias, res = around(dev, M, N, bf16, dtype, 3)
    want = ct.block_scaled_linear(a.storage, a.scale_t, w.storage, w.scale_t, bias, res, activation="gelu", kernel=kernel, out_dtype=dtype)
    far = torch.empty((M - 1) * pitch + N, dtype=dtype, device=dev).as_strided((M, N), (pitch, 1))
    far.copy_(res)
    raw(ct, dev, kernel, a, w, bias, far, far)                 # (the residual is the output itself)
    assert torch.equal(far, want)


@pytest.mark.parametrize("kernel,M,K,N", [("stream", 20, 256, 96), ("mfma128", 300, 288, 160), ("pingpong", 600, 640, 288), ("pingpong", 300, 4096, 320), ("generic", 9, 64, 32),
                                          ("mfma256", 300, 256, 96)])
def test_residual_in_place(ct, dev, kernel, M, K, N):
    a, w = randn_operand(M, K, O.E4M3, 1, dev), randn_operand(N, K, O.E4M3, 2, dev)
    bias, res = around(dev, M, N, f32, bf16, 3)
    want = ct.block_scaled_linear(a.storage, a.scale_t, w.storage, w.scale_t, bias, res, activation="silu", kernel=kernel)
    raw(ct, dev, kernel, a, w, bias, res, res, L.MX_ACT_SILU)
    assert torch.equal(res, want)


def test_empty(ct, dev):
    w = randn_operand(64, 128, O.E4M3, 1, dev)
    a = randn_operand(4, 128, O.E4M3, 2, dev)
    assert ct.block_scaled_linear(a.storage[:0], a.scale_t[:0], w.storage, w.scale_t, torch.ones(64, device=dev)).shape == (0, 64)
    assert ct.block_scaled_linear(a.storage, a.scale_t, w.storage[:0], w.scale_t[:0]).shape == (4, 0)
    bias = torch.randn(64, generator=torch.Generator().manual_seed(3)).to(dev)
    y = ct.block_scaled_linear(a.storage[:, :0], a.scale_t[:, :0], w.storage[:, :0], w.scale_t[:, :0], bias, activation="relu", out_dtype=f32)
    assert torch.equal(y, bias.clamp(min=0).expand(4, 64))        # an empty sum is zero


# ---- trained --------------------------------------------------------------------------------------------------------------------
def make(dev, T, K, N, dtype, seed, rt=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    x, w, b, dy = r(T, K).to(dtype), (r(N, K) * K ** -0.5).to(dtype), (0.3 * r(N)).to(dtype), (r(T, N) * 1e-2).to(dtype)
    return [t.to(dev) for t in (x, w, b, dy)] + [None if rt is None else r(T, N).to(rt).to(dev)]


def layer64(x, w, b, res, dy, act, mode="floor"):
    """y, dx, dw, dbias of the layer's definition, and P."""
    x, w, dy = d64(x), d64(w), d64(dy)
    how = ("e4m3", mode)
    p = R.rows(x, *how) @ R.rows(w, *how).T + (0 if b is None else d64(b))
    d = dy * act64(R.bf16(p), act)[1]
    y = act64(p, act)[0] + (0 if res is None else d64(res))
    return (y, R.rows(d, *how) @ R.columns(w, *how).T, R.columns(d, *how) @ R.columns(x, *how).T, d.sum(0)), p, d


# d differs from its definition's where P lies at a border of bf16 (a share 2^-14 / 2^-8 of the elements, by 2^-7 of a slope) and where what
# comes of it lies at a border of E4M3: a share 2^-9 of the elements at most, a step of 2^-3.  In norm: 2^-3 x 2^-4.5; with few tokens, where P is
# summed in 32 bits, the shares are 2^-5 of that.
FLIPS, FEW_FLIPS = 2.0 ** -7.5, 2.0 ** -10


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("T,K,N", [(1, 32, 32), (1, 1024, 2048), (16, 160, 224), (33, 544, 1056), (64, 512, 96), (77, 1024, 4096), (200, 288, 3040), (700, 256, 1024),
                                   (1100, 544, 1056), (1531, 512, 1088)])
def test_trained_layer(ct, dev, T, K, N, act):
    x, w, b, dy, res = make(dev, T, K, N, f32, T + N, bf16 if N % 3 else None)
    want, p, d = layer64(x, w, b, res, dy, act)
    y, st = ct.linear_forward(x, w, b, res, activation=act)
    got = ct.linear_backward(dy, st)
    few = T <= 64 or T * N <= 1 << 19
    X, W = R.rows(d64(x)), R.rows(d64(w))
    # in 32 bits: an instruction's 32 products, instruction after instruction, eight ranges of K: K / 32 + 40 roundings of 2^-24 of the products' sum
    sums = (K / 32 + 40) * 2.0 ** -24 * (X.abs() @ W.abs().T) if few else sum_error(X, W)
    err = 1.13 * sums + 2.0 ** -20 * (want[0].abs() + p.abs() + d64(b).abs())
    check(y, want[0], err + 2e-6 * want[0].abs(), f32)
    for g, t in zip(got[:2], want[1:3]):
        assert R.rel(g, t) <= (FEW_FLIPS if few else FLIPS) + 2.0 ** -14
        tiles(g, t)
    # the bias's gradient: P as it was summed is rounded to a bf16 number between those of the bounds of its sum, which gives slopes between
    # theirs (and 2^-18 for the arithmetic); then a sum of T numbers in 32 bits
    db = d64(got[2])
    slope = lambda v: act64(R.bf16(v), act)[1]  # noqa: E731
    off = torch.maximum((slope(p + sums) - slope(p)).abs(), (slope(p - sums) - slope(p)).abs()) + 2.0 ** -18
    assert bool(((db - want[3]).abs() <= (d64(dy).abs() * off).sum(0) + T * 2.0 ** -24 * d.abs().sum(0)).all())
    # (relu's slope jumps: a share 1.5e-5 x 0.8 of the arguments is that close to zero, and a whole element of dy hangs on each: the bound above)
    assert act == "relu" or R.rel(db, want[3]) <= (2.0 ** -12 if few else 2.0 ** -9)
    again = ct.linear_backward(dy, st)
    assert all(torch.equal(a, c) for a, c in zip(got, again))
    only = ct.linear_backward(dy, st, need_dx=False, need_dbias=False)
    assert only[0] is None and only[2] is None and torch.equal(only[1], got[1])
    only = ct.linear_backward(dy, st, need_dw=False)
    assert only[1] is None and torch.equal(only[0], got[0]) and torch.equal(only[2], got[2])
    assert torch.equal(ct.linear(x, w, b, res, activation=act), y)


@pytest.mark.parametrize("T,K,N,act", [(40, 256, 320, "gelu"), (900, 256, 1024, "silu"), (300, 96, 2048, None)])
def test_ceiling_rule(ct, dev, T, K, N, act):
    x, w, b, dy, _ = make(dev, T, K, N, f32, 5)
    want, p, d = layer64(x, w, b, None, dy, act, "ceil")
    y, st = ct.linear_forward(x, w, b, activation=act, scale_mode="ceil")
    for g, t in zip((y, *ct.linear_backward(dy, st)), want):
        assert R.rel(g, t) <= FLIPS


@pytest.mark.parametrize("xt,wt,bt,rt", [(bf16, bf16, bf16, None), (bf16, f32, f32, f32), (f32, bf16, None, bf16), (bf16, bf16, f16, f16), (f32, f32, None, None)])
@pytest.mark.parametrize("act", [None, "gelu"])
def test_autograd(ct, dev, xt, wt, bt, rt, act):
    T, K, N = 60, 256, 384
    x, w, b, dy, res = make(dev, T, K, N, f32, 6, f32)
    x, w, b, res = x.to(xt), w.to(wt), None if bt is None else b.to(bt), None if rt is None else res.to(rt)
    dy = dy.to(xt)
    want, _, _ = layer64(x, w, b, res, dy, act)
    leaves = [t.requires_grad_() for t in (x, w, b, res) if t is not None]
    y = ct.linear(x.view(3, 20, K), w, b, None if res is None else res.view(3, 20, N), activation=act)
    assert y.shape == (3, 20, N) and y.dtype == xt
    y.backward(dy.view(3, 20, N))
    wants = [want[1], want[2]] + ([want[3]] if b is not None else []) + ([d64(dy)] if res is not None else [])
    for t, g in zip(leaves, wants):
        assert t.grad.dtype == t.dtype and t.grad.shape == t.shape
        half = {f32: 0, bf16: R.HALF_BF16, f16: 2.0 ** -11}[t.dtype]
        assert R.rel(t.grad, g) <= FEW_FLIPS + 2.0 ** -12 + half
    (g,) = torch.autograd.grad(ct.linear(x, w, b, activation=act).float().sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        g.float().sum().backward()


def test_gradients_against_differences(ct, dev):
    """Of the layer without its quantisation: what is quantised once on either side is off by 2^-5 in the root mean square at most, a gradient
    of two such operands by the root of two times that, and by as much again through P."""
    T, K, N = 50, 128, 96
    x, w, b, dy, _ = make(dev, T, K, N, f32, 7)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    ct.linear(*leaves, activation="gelu").backward(dy)
    at = [d64(t) for t in leaves]
    f = lambda x, w, b: (act64(x @ w.T + b, "gelu")[0] * d64(dy)).sum()  # noqa: E731
    for k, t in enumerate(leaves):
        g = torch.autograd.functional.jacobian(lambda v: f(*at[:k], v, *at[k + 1:]), at[k])
        assert R.rel(t.grad, g) <= 2 * 2 ** 0.5 * 2.0 ** -5
        i = int(g.abs().argmax())
        step = torch.zeros(g.numel(), dtype=torch.float64)
        step[i] = 1e-5
        diff = (f(*at[:k], at[k] + step.view(g.shape), *at[k + 1:]) - f(*at[:k], at[k] - step.view(g.shape), *at[k + 1:])) / 2e-5
        assert abs(float(diff - g.flatten()[i])) <= 1e-6 * float(g.abs().max())


@pytest.mark.parametrize("T", [33, 600])
def test_any_strides(ct, dev, T):
    """Transposed, broadcast and strided inputs and gradients give what their copies give."""
    K, N = 128, 1024
    x, w, b, dy, res = make(dev, T, K, N, f32, 16, f32)
    views = [x.T.contiguous().T, torch.stack([w, w], 2)[:, :, 0], torch.stack([b, b], 1)[:, 0], res.T.contiguous().T]
    plain = [t.clone().requires_grad_() for t in (x, w, b, res)]
    odd = [t.detach().requires_grad_() for t in views]
    assert not any(t.is_contiguous() for t in odd)
    y, z = ct.linear(*plain, activation="silu"), ct.linear(*odd, activation="silu")
    assert torch.equal(y, z)
    y.backward(dy)
    z.backward(dy.T.contiguous().T)
    assert all(torch.equal(p.grad, o.grad) for p, o in zip(plain, odd))
    one, x1 = torch.ones((), device=dev), x[:1].expand(T, K)
    g = [torch.autograd.grad(ct.linear(t, plain[1], plain[2], activation="gelu"), plain[1:3], d) for t, d in ((x1, one.expand(T, N)), (x1.clone(), torch.ones((T, N), device=dev)))]
    assert all(torch.equal(a, c) for a, c in zip(*g))
    _, st = ct.linear_forward(views[0], views[1], views[2], views[3], activation="relu")
    _, st2 = ct.linear_forward(x, w, b, res, activation="relu")
    assert all(torch.equal(a, c) for a, c in zip(ct.linear_backward(dy.T.contiguous().T, st), ct.linear_backward(dy, st2)))


def test_residual_alone_and_no_tokens(ct, dev):
    x, w, b, dy, res = make(dev, 8, 64, 32, bf16, 8, bf16)
    res.requires_grad_()
    ct.linear(x, w, b, res, activation="relu").backward(dy)
    assert torch.equal(res.grad, dy)
    x0 = x[:0].clone().requires_grad_()
    w.requires_grad_()
    b.requires_grad_()
    y = ct.linear(x0, w, b)
    y.sum().backward()
    assert y.shape == (0, 32) and bool((w.grad == 0).all()) and bool((b.grad == 0).all()) and x0.grad.shape == (0, 64)


def test_streams_and_graphs(ct, dev):
    for T, K, N in ((40, 256, 320), (700, 256, 1024)):
        x, w, b, dy, res = make(dev, T, K, N, bf16, 9, bf16)
        a_q, a_s = ct.block_quantize(x, 32, scale_mode="floor")
        w_q, w_s = ct.block_quantize(w, 32, scale_mode="floor")

        def everything():
            y, st = ct.linear_forward(x, w, b, res, activation="gelu")
            return (y, *ct.linear_backward(dy, st), ct.block_scaled_linear(a_q, a_s, w_q, w_s, b, res, activation="silu"),
                    *(u8(t) for t in ct.block_scaled_linear(a_q, a_s, w_q, w_s, b, activation="gelu_tanh", out_dtype="e4m3")))

        want = everything()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = everything()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, c) for a, c in zip(got, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = everything()
        for seed in (10, 11, 12):
            fresh = make(dev, T, K, N, bf16, seed, bf16)
            for t, f in zip((x, w, b, dy, res), fresh):
                t.copy_(f)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(held, everything()))
        leaf = x.clone().requires_grad_()
        refused = torch.cuda.CUDAGraph()
        with torch.cuda.graph(refused):
            with pytest.raises(RuntimeError, match="cannot be captured"):
                ct.linear(leaf, w, b)
            keep = x + 1                                       # (a graph of something)


def test_weights_may_change_before_the_backward_pass(ct, dev):
    x, w, b, dy, _ = make(dev, 70, 128, 96, bf16, 13)
    y, st = ct.linear_forward(x, w, b, activation="silu")
    want = ct.linear_backward(dy, st)
    y, st = ct.linear_forward(x, w, b, activation="silu")
    w.zero_()
    x.zero_()
    assert all(torch.equal(a, c) for a, c in zip(ct.linear_backward(dy, st), want))


def test_gradient_that_is_not_finite(ct, dev):
    for T in (40, 600):
        x, w, b, dy, _ = make(dev, T, 128, 1024, bf16, 14)
        dy[3, 40] = float("nan")
        _, st = ct.linear_forward(x, w, b, activation="gelu")
        dx, dw, db = ct.linear_backward(dy, st)
        assert bool(dx[3].isnan().all()) and not bool(dx[[0, 1, 2, 4]].isnan().any())
        assert bool(dw[40].isnan().all()) and not bool(dw[:32].isnan().any()) and bool(db[40].isnan()) and int(db.isnan().sum()) == 1


@pytest.mark.parametrize("mode", ["floor", "ceil"])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("T", [40, 600])
def test_what_is_not_finite_stays_in_its_place(ct, dev, T, bad, mode):
    """One element of dy: its row of dx, its row of dw and its column's sum are not finite (under the floor rule an infinity is the largest
    number of its block); blocks that do not hold it give what they gave."""
    x, w, b, dy, _ = make(dev, T, 96, 1024, f32, 15)
    _, st = ct.linear_forward(x, w, b, activation="relu", scale_mode=mode)
    clean = ct.linear_backward(dy, st)
    n = int((x @ w.T + b)[5].argmax())                         # a column whose slope is one there
    dy[5, n] = bad
    dx, dw, db = ct.linear_backward(dy, st)
    others = [t for t in range(T) if t != 5]
    assert torch.equal(dx[others], clean[0][others])
    blocks = [k for k in range(1024) if k != n]
    assert torch.equal(dw[blocks], clean[1][blocks]) and torch.equal(db[blocks], clean[2][blocks])
    assert not bool(db[n].isfinite())
    if mode == "ceil" or bad != bad:
        assert bool(dx[5].isnan().all()) and bool(dw[n].isnan().all())
    else:
        assert not torch.equal(dx[5], clean[0][5]) and not torch.equal(dw[n], clean[1][n])
