"""block_quantize_both and silu_and_mul_backward_quantize on the GPU, against the oracle's quantiser and 64-bit arithmetic."""
import numpy as np
import pytest
import torch

import ffnutil as R
from oracle import mx_oracle as O

pytestmark = pytest.mark.gpu
FMT = {"e4m3": O.E4M3, "e5m2": O.E5M2}
SRC = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def u8(t):
    return t.view(torch.uint8).cpu().numpy()


def check_both(ct, x, fmt, mode):
    """x on the device; both directions bit for bit.  Blocks with an infinity or a NaN under the floor rule are block_quantize's: the
    rule (OCP MX v1.0) leaves them to the implementation, and the oracle's choice is another than the device's."""
    got = ct.block_quantize_both(x, R.ELEM[fmt], scale_mode=mode)
    f = x.detach().float().cpu().reshape(-1, x.shape[-1])
    K = f.shape[1]
    r = torch.nn.functional.pad(f, (0, -K % 32))
    for got_q, got_s, m in ((got[0], got[1], r), (got[2], got[3], R.padded_t(f))):
        q, s = O.block_quantize(np.ascontiguousarray(m.numpy()), 32, FMT[fmt], mode)
        if mode == "floor":
            odd = ~np.isfinite(m.numpy()).reshape(m.shape[0], -1, 32).all(-1)
            dq, ds = (u8(t) for t in ct.block_quantize(m.to(x.device), 32, R.ELEM[fmt], scale_mode=mode)) if odd.any() else (q, s)
            q, s = np.where(odd.repeat(32, -1), dq, q), np.where(odd, ds, s)
        assert np.array_equal(u8(got_q).reshape(q.shape), q)
        assert np.array_equal(u8(got_s).reshape(s.shape), s)
    return got


@pytest.mark.parametrize("rows,K", [(1, 32), (1, 4096), (31, 64), (32, 96), (33, 128), (127, 160), (129, 130), (300, 1000),
                                    (8, 33), (513, 544), (160, 2080)])
@pytest.mark.parametrize("src,fmt,mode", [("bf16", "e4m3", "floor"), ("bf16", "e5m2", "ceil"), ("f32", "e4m3", "ceil"),
                                          ("f16", "e4m3", "floor"), ("f32", "e5m2", "floor")])
def test_both_directions_bit_exact(ct, dev, rows, K, src, fmt, mode):
    g = torch.Generator().manual_seed(rows * 7919 + K)
    x = torch.randn((rows, K), generator=g) * torch.exp2(torch.randint(-12, 12, (rows, 1), generator=g).float())
    check_both(ct, x.to(SRC[src]).to(dev), fmt, mode)


@pytest.mark.parametrize("mode", ["floor", "ceil"])
@pytest.mark.parametrize("src", ["bf16", "f32", "f16"])
def test_both_directions_special_values(ct, dev, src, mode):
    """Zero blocks, subnormal and extreme blocks, infinities and NaN: the blocks that the hardware conversions do not take."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn((200, 256), generator=g)
    x[0:32] = 0
    x[3, 7] = -0.0
    x[40:72, 0:64] *= 2.0 ** -120 if src != "f16" else 2.0 ** -14
    x[64:96, 64:96] *= 1e-40 if src != "f16" else 2.0 ** -22
    x[100, 200] = float("inf")
    x[140, 10] = float("-inf")
    x[141, 70] = float("nan")
    x[180:, 128:] *= 1e38 if src != "f16" else 4e4
    check_both(ct, x.to(SRC[src]).to(dev), "e4m3", mode)
    check_both(ct, x.to(SRC[src]).to(dev), "e5m2", mode)


def test_both_directions_of_views(ct, dev):
    g = torch.Generator().manual_seed(6)
    base = torch.randn((70, 300), generator=g).to(torch.bfloat16).to(dev)
    for x in (base[:, 1:257], base[3:, 8:200], base[::2, :96], base.t()[:256], base[:1].expand(40, 300), base[:60].view(3, 20, 300)):
        check_both(ct, x, "e4m3", "floor")
    q, s, qt, st = ct.block_quantize_both(torch.empty((0, 64), dtype=torch.bfloat16, device=dev))
    assert q.shape == (0, 64) and s.shape == (0, 2) and qt.shape == (64, 0) and st.shape == (64, 0)
    q, s, qt, st = check_both(ct, base[0], "e4m3", "floor")
    assert q.shape == (320,) and s.shape == (10,) and qt.shape == (300, 32) and st.shape == (300, 1)


def test_both_directions_past_32_bits(ct, dev):
    """Offsets beyond 2^31 elements and 2^32 bytes of a wide fp32 matrix: its last rows and columns."""
    rows, K = 260, 8_400_000 // 32 * 32
    x = torch.zeros((rows, K), device=dev)
    x[:, -96:] = torch.randn((rows, 96), generator=torch.Generator().manual_seed(2)).to(dev)
    assert x.numel() * 4 > 2 ** 32 and x.numel() > 2 ** 31
    q, s, qt, st = ct.block_quantize_both(x)
    tail = x[:, -96:].cpu()
    for got_q, got_s, m in ((q[:, -96:], s[:, -3:], tail), (qt[-96:], st[-96:], R.padded_t(tail))):
        eq, es = O.block_quantize(np.ascontiguousarray(m.numpy()), 32, O.E4M3, "floor")
        assert np.array_equal(u8(got_q.contiguous()), eq) and np.array_equal(u8(got_s.contiguous()), es)
    assert int(q[:, :-96].view(torch.uint8).max()) == 0 and int(qt[:-96].view(torch.uint8).max()) == 0


def checkpoint(ct, gu):
    return ct.block_quantize(gu, 32, torch.float8_e4m3fn, scale_mode="floor")


# d and a come from 32-bit arithmetic of a dozen operations and two hardware approximations, each good to 2^-22 or better:
# 2^-18 of the value, where the sum 1 + g (1 - s) cancels (g near -1.28) of its terms.
FORMULA = 2.0 ** -18


@pytest.mark.parametrize("mode", ["floor", "ceil"])
@pytest.mark.parametrize("M,F", [(1, 32), (1, 4096), (31, 64), (33, 96), (77, 160), (128, 128), (129, 1408), (300, 224)])
def test_silu_backward(ct, dev, M, F, mode):
    g = torch.Generator().manual_seed(M * 131 + F)
    gu = torch.randn((M, 2 * F), generator=g) * 3
    dh = (torch.randn((M, F), generator=g) * 1e-3).to(torch.bfloat16)
    gq, gs = checkpoint(ct, gu.to(dev))
    got = ct.silu_and_mul_backward_quantize(dh.to(dev), gq, gs, scale_mode=mode)
    d, a = R.silu_mul_backward(dh.double(), R.value(gq, gs))
    # a value of the formula that is off by FORMULA may round to the other neighbour, or its block may take the other scale,
    # where it lies that close to the border: such elements are left out of the comparison, which has to be few of them
    checked = total = 0
    for got_q, got_s, m in ((got[0], got[1], d), (got[2], got[3], R.padded_t(d)), (got[4], got[5], R.padded_t(a))):
        assert got_q.shape == m.shape and got_s.shape == (m.shape[0], m.shape[1] // 32)
        assert got_q.dtype == torch.float8_e4m3fn and got_s.dtype == torch.float8_e8m0fnu
        lo, hi = (R.quantize(m * (1 + f), "e4m3", mode) for f in (-FORMULA, FORMULA))
        # (cancelled sums: their absolute error may be larger than FORMULA of the value)
        sure = (R.value(*lo) == R.value(*hi)) & (m.abs() >= 0.02 * m.abs().reshape(m.shape[0], -1, 32).amax(-1).repeat_interleave(32, -1))
        same = R.value(got_q, got_s) == R.value(*lo)
        assert bool(same[sure].all())
        # ... and those are within a step of the block's largest value
        off = (R.value(got_q, got_s) - m).abs() / m.abs().reshape(m.shape[0], -1, 32).amax(-1).repeat_interleave(32, -1).clamp(min=1e-300)
        assert float(off.max()) <= 0.125 + 2.0 ** -6     # saturation of the floor rule: 448 for up to 512
        checked, total = checked + int((sure & (m != 0)).sum()), total + int((m != 0).sum())   # (the padding is zeros)
    assert checked > 0.5 * total or M < 32


def test_silu_backward_special_values(ct, dev):
    """Zero checkpoints (a dead unit, padding) and gates far out give finite gradients; NaN and infinity stay in their blocks."""
    M, F = 64, 128
    g = torch.Generator().manual_seed(3)
    gu = torch.randn((M, 2 * F), generator=g)
    gu[:, :32] = 0
    gu[:32, 32:64] = 200.0
    gu[:32, 64:96] = -200.0
    dh = torch.randn((M, F), generator=g).to(torch.bfloat16)
    dh[40, 100] = float("nan")
    gq, gs = checkpoint(ct, gu.to(dev))
    got = ct.silu_and_mul_backward_quantize(dh.to(dev), gq, gs)
    d, a = R.silu_mul_backward(dh.double(), R.value(gq, gs))
    for got_q, got_s, m in ((got[0], got[1], d), (got[2], got[3], R.padded_t(d)), (got[4], got[5], R.padded_t(a))):
        nan = m.isnan().reshape(m.shape[0], -1, 32).any(-1).repeat_interleave(32, -1)
        v = R.value(got_q, got_s)
        assert not bool(v[~nan].isnan().any())
        assert bool(v[m.isnan()].isnan().all())
        top = m.abs().nan_to_num(0).reshape(m.shape[0], -1, 32).amax(-1).repeat_interleave(32, -1)
        # a step at most of the block's largest value; what 32 bits do not hold is zero: sigmoid(-200) = 2^-289
        assert bool(((v - m).abs()[~nan] <= 0.141 * top[~nan] + 2.0 ** -126).all())


def test_silu_backward_nan_in_the_checkpoint(ct, dev):
    """NaN codes and NaN scales of the checkpoint, and nothing else, give NaN."""
    M, F = 64, 64
    g = torch.Generator().manual_seed(7)
    gq, gs = checkpoint(ct, torch.randn((M, 2 * F), generator=g).to(dev))
    gq.view(torch.uint8)[5, 7] = 0x7F
    gq.view(torch.uint8)[6, F + 9] = 0xFF
    gs.view(torch.uint8)[9, 1] = 0xFF
    dh = torch.randn((M, F), generator=g).to(torch.bfloat16)
    for mode in ("floor", "ceil"):
        got = ct.silu_and_mul_backward_quantize(dh.to(dev), gq, gs, scale_mode=mode)
        d, a = R.silu_mul_backward(dh.double(), torch.where(gq.cpu().float().isnan(), float("nan"), R.value(gq.cpu().float().nan_to_num(), gs))
                                   + torch.where(gs.cpu().view(torch.uint8) == 255, float("nan"), 0.0).repeat_interleave(32, -1))
        for got_q, m in ((got[0], d), (got[2], R.padded_t(d)), (got[4], R.padded_t(a))):
            assert torch.equal(got_q.float().isnan().cpu(), m.isnan())


def test_silu_backward_of_views(ct, dev):
    """Rows that are not aligned, or apart, give the bits of contiguous ones."""
    M, F = 50, 96
    g = torch.Generator().manual_seed(4)
    gq, gs = checkpoint(ct, torch.randn((M, 2 * F), generator=g).to(dev))
    dh = torch.randn((M, F), generator=g).to(torch.bfloat16).to(dev)
    want = ct.silu_and_mul_backward_quantize(dh, gq, gs)
    wide = torch.zeros((M, F + 11), dtype=torch.bfloat16, device=dev)
    wide[:, 3:3 + F] = dh
    gwide = torch.zeros((M, 2 * F + 21), dtype=torch.uint8, device=dev)
    gwide[:, 5:5 + 2 * F] = gq.view(torch.uint8)
    swide = torch.zeros((M, F // 16 + 3), dtype=torch.uint8, device=dev)
    swide[:, 1:1 + F // 16] = gs.view(torch.uint8)
    got = ct.silu_and_mul_backward_quantize(wide[:, 3:3 + F], gwide[:, 5:5 + 2 * F].view(torch.float8_e4m3fn),
                                            swide[:, 1:1 + F // 16].view(torch.float8_e8m0fnu))
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    empty = ct.silu_and_mul_backward_quantize(dh[:0], gq[:0], gs[:0])
    assert [tuple(t.shape) for t in empty] == [(0, 2 * F), (0, F // 16), (2 * F, 0), (2 * F, 0), (F, 0), (F, 0)]
