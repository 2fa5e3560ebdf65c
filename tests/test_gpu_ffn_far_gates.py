"""The SiLU backward pass for gates far out: sigmoid is one or zero in 32 bits, and the gradient of the gate is dh u or zero."""
import pytest
import torch

import ffnutil as R
from test_gpu_ffn_quantize import FORMULA

pytestmark = pytest.mark.gpu
# A sigmoid below 2^-126, the smallest normal number of 32 bits, is zero: gates below -87.3.  What is lost is at most 2^-126 |g u| with |g| <= 2^7 where it is
# not smaller than that by itself, and |u| <= 2^3 here.
TINY = 2.0 ** -116
LARGEST = 448.0 * 2.0 ** 119                          # of E4M3 codes with a scale that a float's block has


def steps(got_q, got_s, m, mode):
    """Codes and scales against the formula's numbers `m` [rows, a multiple of 32], as in test_silu_backward: equal where FORMULA of the value
    decides no rounding, and within a step of the block's largest value everywhere."""
    lo, hi = (R.quantize(m * (1 + f), "e4m3", mode) for f in (-FORMULA, FORMULA))
    top = m.abs().reshape(m.shape[0], -1, 32).amax(-1).repeat_interleave(32, -1)
    sure = (R.value(*lo) == R.value(*hi)) & (m.abs() >= 0.02 * top) & ((m.abs() >= TINY) | (m == 0))
    v = R.value(got_q, got_s)
    assert not bool(v.isnan().any())
    assert torch.equal(v[sure], R.value(*lo)[sure])
    # (saturation of the floor rule: 448 for up to 512.  The ceiling rule's scale is at least 1e-12 rounded up, 2^-39, whose smallest code is 2^-48:
    # half of that is what a block of smaller numbers is off by)
    assert bool(((v - m).abs() <= (0.125 + 2.0 ** -6) * top + (2.0 ** -49 if mode == "ceil" else TINY)).all())


@pytest.mark.parametrize("mode", ["floor", "ceil"])
@pytest.mark.parametrize("M,F", [(1, 32), (40, 64), (130, 160)])
@pytest.mark.parametrize("low,high", [(4, 14), (14, 24), (20, 30), (23, 26), (30, 60), (60, 100), (100, 127)])
def test_far_gates(ct, dev, M, F, low, high, mode):
    """Gates of 2^low to 2^high, of both signs; a row's block of 32 has one sign, a token's block of 32 both."""
    g = torch.Generator().manual_seed(low * 128 + M)
    gate = torch.exp2(low + (high - low) * torch.rand((M, F), generator=g, dtype=torch.float64)).clamp(max=LARGEST)
    gate = gate * (1 - 2 * torch.randint(0, 2, (M, F // 32), generator=g)).repeat_interleave(32, -1)
    gu = torch.cat((gate.float(), torch.randn((M, F), generator=g)), -1)
    # (dh small enough for dh g, a = g u to stay within 32 bits)
    dh = (torch.randn((M, F), generator=g) * (1e-3 if high < 100 else 2.0 ** -20)).to(torch.bfloat16)
    if high >= 100:
        gu[:, F:] *= 2.0 ** -20
    gq, gs = ct.block_quantize(gu.to(dev), 32, torch.float8_e4m3fn, scale_mode="floor")
    got = ct.silu_and_mul_backward_quantize(dh.to(dev), gq, gs, scale_mode=mode)
    d, a = R.silu_mul_backward(dh.double(), R.value(gq, gs))
    for q, s, m in ((got[0], got[1], d), (got[2], got[3], R.padded_t(d)), (got[4], got[5], R.padded_t(a))):
        steps(q, s, m, mode)


@pytest.mark.parametrize("byte", [246, 247, 250, 254])
@pytest.mark.parametrize("sign", [0x00, 0x80])
def test_gates_at_the_end_of_the_format(ct, dev, byte, sign):
    """The largest numbers that codes and scales hold, beyond 32-bit floats too: the gate's gradient is dh u, or zero, and no other result is NaN."""
    M, F = 33, 64
    g = torch.Generator().manual_seed(byte)
    gq, gs = ct.block_quantize(torch.randn((M, 2 * F), generator=g).to(dev), 32, torch.float8_e4m3fn, scale_mode="floor")
    gq.view(torch.uint8)[:, :F] = 0x7E | sign
    gs.view(torch.uint8)[:, :F // 32] = byte
    dh = torch.randn((M, F), generator=g).to(torch.bfloat16)
    dh[3, 5] = 0
    for mode in ("floor", "ceil"):
        got = ct.silu_and_mul_backward_quantize(dh.to(dev), gq, gs, scale_mode=mode)
        d, _ = R.silu_mul_backward(dh.double(), R.value(gq, gs))
        steps(got[0][:, :F], got[1][:, :F // 32], d[:, :F], mode)
        steps(got[2][:F], got[3][:F], R.padded_t(d[:, :F]), mode)
        for t in (got[0], got[2], got[4]):
            assert mode == "ceil" or not bool(t.float().isnan().any())
