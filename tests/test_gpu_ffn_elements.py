"""The gated product element by element, and the block tile by tile: what a norm over a whole result would pass, such as one column group or
one MX block of an edge tile that is zero, or one scale that is a power of two off."""
import pytest
import torch

import ffnutil as R
from mxutil import randn_operand
from oracle import mx_oracle as O
from test_gpu_ffn import make

pytestmark = pytest.mark.gpu


def sum_error(A, W):
    """Bound of a scaled MFMA's sum of K products, element by element: an instruction aligns its products to the largest and keeps 18 bits of
    them, so that each of the K is off by at most 2^-18 of the row's largest times the column's; adding the instructions' sums up is 2^-23 of them
    a time, which the same bound covers where there are fewer instructions than products."""
    return A.shape[1] * 2.0 ** -18 * A.abs().amax(1, keepdim=True) * W.abs().amax(1)


def gated_bounds(A, W):
    """(gate and up in bf16, h, bound of a kernel's gate and up, bound of its h before h is rounded)."""
    s, err = A @ W.T, sum_error(A, W)
    gu = R.bf16(s)
    # rounded from a sum that is off by err: err, and half a step on either side
    e_gu = err + 2 * R.HALF_BF16 * (s.abs() + err)
    g, u = gu.chunk(2, -1)
    e_g, e_u = e_gu.chunk(2, -1)
    # |silu'| <= 1.1, |silu(g)| <= |g|; 2^-20: the hardware's 2^x and reciprocal
    e_h = 1.1 * e_g * (u.abs() + e_u) + (g * torch.sigmoid(g)).abs() * e_u
    h = R.silu_mul(gu)
    return gu, h, e_gu, e_h + 2.0 ** -20 * h.abs()


def check_codes(q, s, want, err, limit=448.0):
    """Codes of numbers that are `err` from `want`: that, and the rounding to E4M3, half a step 2^-4 of the value, or where the floor rule ends at
    448 for up to 512 of the scale, 2^-3 of the value; numbers below the smallest normal one are off by half of 2^-9 of the scale."""
    v = R.value(q, s)
    scale = torch.ldexp(torch.ones(s.shape, dtype=torch.float64), s.cpu().view(torch.uint8).int() - 127).repeat_interleave(32, -1)
    bad = (v - want).abs() > err + 0.125 * (want.abs() + err) + 2.0 ** -10 * scale
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist())
    # the scale is the block's: its largest code is in the top binade, or its neighbours' where the largest lies at the border
    top = (want.abs() + err).reshape(want.shape[0], -1, 32).amax(-1)
    low = (want.abs() - err).clamp(min=0).reshape(want.shape[0], -1, 32).amax(-1)
    e = s.cpu().view(torch.uint8).int() - 127 + 8
    exps = [torch.frexp(t.clamp(min=1e-300))[1] - 1 for t in (low, top)]
    ok = (e >= exps[0].clamp(min=-119)) & (e <= exps[1].clamp(min=-119))
    assert bool(ok.all()), (~ok).nonzero()[:4].tolist()


CASES = [
    ("stream", O.E4M3, 1, 128, 32), ("stream", O.E4M3, 17, 1152, 96), ("stream", O.E2M1, 32, 4224, 160), ("stream", O.E4M3, 32, 2048, 2944),
    ("decode", O.E2M1, 1, 512, 32), ("decode", O.E2M1, 31, 4608, 224), ("decode", O.E2M1, 20, 1024, 9248),
    ("pingpong", O.E4M3, 1, 32, 64), ("pingpong", O.E4M3, 257, 544, 192), ("pingpong", O.E2M1, 300, 1536, 448), ("pingpong", O.E4M3, 1025, 1024, 2944),
    ("pingpong", O.E4M3, 1531, 512, 1088), ("pingpong", O.E4M3, 2305, 256, 4160),
    ("auto", O.E4M3, 3, 512, 96), ("auto", O.E4M3, 40, 1024, 224), ("auto", O.E2M1, 100, 544, 320), ("auto", O.E4M3, 700, 1024, 1536), ("auto", O.E4M3, 1300, 512, 1120),
]


@pytest.mark.parametrize("kernel,w_fmt,M,K,F", CASES)
def test_gated_product_elements(ct, dev, kernel, w_fmt, M, K, F):
    a, w = randn_operand(M, K, O.E4M3, M + K, dev), randn_operand(2 * F, K, w_fmt, F, dev, std=K ** -0.5)
    gu, want, e_gu, e_h = gated_bounds(O.dequantize(a.codes, a.scales, a.fmt).double(), O.dequantize(w.codes, w.scales, w.fmt).double())
    packed = kernel in ("pingpong", "stream")
    for ws in (w.scale_t, ct.pack_scales(w.scale_t, operand="b")) if packed else (w.scale_t,):
        args, kw = (a.storage, a.scale_t, w.storage, ws), dict(w_format=w.fmt_kw, kernel=kernel)
        h = ct.gated_block_scaled_matmul(*args, **kw).cpu().double()
        bad = (h - want).abs() > e_h + R.HALF_BF16 * (want.abs() + e_h)
        assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist())
        q, s, cq, cs = ct.gated_block_scaled_matmul(*args, out_dtype="e4m3", checkpoint=True, **kw)
        check_codes(q, s, want, e_h)
        check_codes(cq, cs, gu, e_gu)


# An operand whose every element is a step of 2^-3 off, independently, changes a tile's norm by 2^-3; a lane's eight columns of 32 that are missing
# by one half, a row of 16 by one quarter, an MX block's scale by more.  (What the roundings make of single elements is far below: BLOCK of test_gpu_ffn.)
TILE = 2.0 ** -3


def tiles(got, want, rows=16, cols=32):
    got, want = got.cpu().double(), want.double()
    e = torch.zeros((-(-want.shape[0] // rows) * rows, -(-want.shape[1] // cols) * cols), dtype=torch.float64)
    n = e.clone()
    e[:want.shape[0], :want.shape[1]] = (got - want) ** 2
    n[:want.shape[0], :want.shape[1]] = want ** 2
    e, n = (t.reshape(t.shape[0] // rows, rows, -1, cols).sum((1, 3)).sqrt() for t in (e, n))
    bad = e > TILE * n
    assert not bool(bad.any()), (float((e / n.clamp(min=1e-300)).max()), bad.nonzero()[:4].tolist())


@pytest.mark.parametrize("mode", ["floor", "ceil"])
@pytest.mark.parametrize("T,H,F,Ho", [(1, 1024, 2048, 512), (16, 160, 224, 96), (33, 544, 1056, 288), (64, 512, 1504, 320), (200, 544, 1056, 288), (513, 288, 992, 96),
                                      (700, 256, 1024, 512), (1100, 544, 1056, 288), (1531, 512, 1088, 160)])
def test_block_tiles(ct, dev, T, H, F, Ho, mode):
    x, w1, w2, dy = make(T, H, F, Ho, T + F, dev, torch.float32)
    y, st = ct.gated_feed_forward_forward(x, w1, w2, scale_mode=mode)
    got = (y, *ct.gated_feed_forward_backward(dy, st))
    for g, w in zip(got, R.block(*(t.cpu().double() for t in (x, w1, w2, dy)), "e4m3", mode)):
        tiles(g, w)
