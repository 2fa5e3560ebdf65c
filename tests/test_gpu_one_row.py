"""One row: its pitch names nothing, so any is allowed, 0 and 1 as well, of every operand and result."""
import ctypes

import pytest
import torch

from cutile_amd import _lib as L
from mxutil import randn_operand
from oracle import mx_oracle as O

pytestmark = pytest.mark.gpu


def u8(t):
    return t.view(torch.uint8)


def described(t, dtype, pitch):
    d = L.desc(t, dtype)
    d.stride[0] = pitch
    return d


def results(dev, *shapes, pitch):
    """[(tensor of a mark, descriptor)], the pitch of those with one row `pitch`"""
    out = []
    for rows, cols, dtype in shapes:
        t = torch.full((rows, cols), 0xA5, dtype=torch.uint8, device=dev) if dtype != L.MX_BF16 else torch.full((rows, cols), -7.0, dtype=torch.bfloat16, device=dev)
        out.append((t, described(t, dtype, pitch if rows == 1 else cols)))
    return out


def refs(args):
    return [ctypes.byref(a) if isinstance(a, L.MxTensor) else a for a in args]


@pytest.mark.parametrize("pitch", [0, 1, 8, 16, 1 << 40])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K", [32, 96, 256, 300])
def test_quantize_both(ct, dev, K, src, pitch):
    x = torch.randn((1, K), generator=torch.Generator().manual_seed(K)).to(src).to(dev)
    Kp = (K + 31) // 32 * 32
    outs = results(dev, (1, Kp, L.MX_E4M3), (1, Kp // 32, L.MX_E8M0), (K, 32, L.MX_E4M3), (K, 1, L.MX_E8M0), pitch=pitch)
    for x_pitch in (K, pitch):
        args = [described(x, L._TORCH_TO_MX[src], x_pitch), *(d for _, d in outs), 1, L.stream_ptr(dev)]
        assert L.lib().mx_quantize_both(*refs(args)) == L.MX_OK, L.last_error()
        for (t, _), want in zip(outs, ct.block_quantize_both(x)):
            assert torch.equal(t, u8(want))


@pytest.mark.parametrize("pitch", [0, 8, 16])
@pytest.mark.parametrize("F", [32, 160, 256])
def test_silu_backward(ct, dev, F, pitch):
    g = torch.Generator().manual_seed(F)
    dh = torch.randn((1, F), generator=g).to(torch.bfloat16).to(dev)
    q, s = ct.block_quantize(torch.randn((1, 2 * F), generator=g).to(dev), 32, torch.float8_e4m3fn, scale_mode="floor")
    outs = results(dev, (1, 2 * F, L.MX_E4M3), (1, F // 16, L.MX_E8M0), (2 * F, 32, L.MX_E4M3), (2 * F, 1, L.MX_E8M0), (F, 32, L.MX_E4M3), (F, 1, L.MX_E8M0),
                   pitch=pitch)
    args = [described(dh, L.MX_BF16, pitch), described(u8(q), L.MX_E4M3, pitch), described(u8(s), L.MX_E8M0, pitch), *(d for _, d in outs), 1,
            L.stream_ptr(dev)]
    assert L.lib().mx_silu_mul_backward_quantize(*refs(args)) == L.MX_OK, L.last_error()
    for (t, _), want in zip(outs, ct.silu_and_mul_backward_quantize(dh, q, s)):
        assert torch.equal(t, u8(want))


@pytest.mark.parametrize("pitch", [0, 16])
@pytest.mark.parametrize("kernel,w_fmt", [("auto", O.E4M3), ("stream", O.E4M3), ("pingpong", O.E4M3), ("mfma128", O.E4M3), ("decode", O.E2M1)])
def test_gated_product(ct, dev, kernel, w_fmt, pitch):
    K, F = 512, 192
    a, w = randn_operand(1, K, O.E4M3, 1, dev), randn_operand(2 * F, K, w_fmt, 2, dev, std=K ** -0.5)
    o = L.MxGemmOpts(struct_size=32, kernel=L.KERNELS[kernel], block_size=32)
    need = L.lib().mx_gated_gemm_workspace_bytes(1, F, K, ctypes.byref(o))
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    outs = results(dev, (1, F, L.MX_E4M3), (1, F // 32, L.MX_E8M0), (1, 2 * F, L.MX_E4M3), (1, F // 16, L.MX_E8M0), pitch=pitch)
    fp4 = w_fmt == O.E2M1
    args = [described(u8(a.storage), L.MX_E4M3, pitch), described(u8(a.scale_t), L.MX_E8M0, pitch),
            L.desc(u8(w.storage), L.MX_E2M1 if fp4 else L.MX_E4M3, 1 if fp4 else -1), L.desc(u8(w.scale_t), L.MX_E8M0), *(d for _, d in outs), 1, ctypes.byref(o),
            ws.data_ptr(), need, L.stream_ptr(dev)]
    assert L.lib().mx_gated_gemm(*refs(args)) == L.MX_OK, L.last_error()
    want = ct.gated_block_scaled_matmul(a.storage, a.scale_t, w.storage, w.scale_t, w_format=w.fmt_kw, out_dtype="e4m3", checkpoint=True, kernel=kernel)
    for (t, _), v in zip(outs, want):
        assert torch.equal(t, u8(v))


def test_block(ct, dev):
    g = torch.Generator().manual_seed(9)
    x, dy = (torch.randn((1, n), generator=g).to(torch.bfloat16).to(dev) for n in (128, 96))
    w1, w2 = (torch.randn(s, generator=g).to(torch.bfloat16).to(dev) for s in ((128, 128), (96, 64)))
    y, st = ct.gated_feed_forward_forward(x, w1, w2)
    want = (y, *ct.gated_feed_forward_backward(dy, st))
    for pitch in (0, 1):
        y, st = ct.gated_feed_forward_forward(x.as_strided((1, 128), (pitch, 1)), w1, w2)
        got = (y, *ct.gated_feed_forward_backward(dy.as_strided((1, 96), (pitch, 1)), st))
        assert all(torch.equal(p, q) for p, q in zip(got, want))
