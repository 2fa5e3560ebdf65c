"""NaN and infinities of gate and up: what the gated product makes of them does not depend on the kernel that is taken."""
import pytest
import torch

import ffnutil as R
from mxutil import randn_operand
from oracle import mx_oracle as O

pytestmark = pytest.mark.gpu
KERNELS = [("stream", O.E4M3, 20), ("stream", O.E2M1, 9), ("decode", O.E2M1, 20), ("pingpong", O.E4M3, 20), ("pingpong", O.E4M3, 300), ("pingpong", O.E2M1, 70)]


def u8(t):
    return t.view(torch.uint8)


def both(ct, a, w, **kw):
    """Results of the kernel named and of the product through memory: (h, h_q, h_scale, gate_up_q, gate_up_scale)."""
    def run(kernel):
        args = (a.storage, a.scale_t, w.storage, w.scale_t)
        h = ct.gated_block_scaled_matmul(*args, w_format=w.fmt_kw, kernel=kernel)
        return (h, *ct.gated_block_scaled_matmul(*args, w_format=w.fmt_kw, kernel=kernel, out_dtype="e4m3", checkpoint=True))
    return run(kw["kernel"]), run("mfma128")


def same_values(got, want, sure):
    """Codes as numbers and scale bytes, where `sure` [rows, columns of whole blocks]"""
    (gq, gs), (wq, ws) = got, want
    x, y = gq.float().cpu(), wq.float().cpu()
    assert torch.equal(x.isnan()[sure], y.isnan()[sure]) and torch.equal(x.nan_to_num(0)[sure], y.nan_to_num(0)[sure])
    blocks = sure.reshape(sure.shape[0], -1, 32).all(-1)
    assert torch.equal(u8(gs).cpu()[blocks], u8(ws).cpu()[blocks])


@pytest.mark.parametrize("kernel,w_fmt,M", KERNELS)
def test_a_block_with_nan(ct, dev, kernel, w_fmt, M):
    """NaN is the largest of its block under the floor rule: the scale is that of an infinity, and the finite numbers beside it are zeros."""
    K, F = 1024, 256
    a, w = randn_operand(M, K, O.E4M3, 1, dev), randn_operand(2 * F, K, w_fmt, 2, dev, std=K ** -0.5)
    for row, block in ((70, 3), (F + 131, 31), (F + 64, 0)):       # a gate row and two up rows: NaN scales
        u8(w.scale_t)[row, block] = 0xFF
    got, want = both(ct, a, w, kernel=kernel)
    nan = [70, 131, 64]
    assert bool(got[0][:, nan].isnan().all()) and bool(want[0][:, nan].isnan().all())
    assert int(got[0].isnan().sum()) == M * 3
    odd = torch.zeros((M, 2 * F), dtype=torch.bool)               # blocks that hold a NaN (others: sums' last bits may differ)
    for c in (70, F + 131, F + 64):
        odd[:, c // 32 * 32:c // 32 * 32 + 32] = True
    same_values(got[3:5], want[3:5], odd)
    oddh = odd[:, :F] | odd[:, F:]
    same_values(got[1:3], want[1:3], oddh)
    assert bool((u8(got[4]).cpu()[:, 70 // 32] == 247).all()) and bool((u8(got[2]).cpu()[:, 70 // 32] == 247).all())
    # a NaN in a row of A: every block of the row
    u8(a.scale_t)[M // 2, 5] = 0xFF
    got, want = both(ct, a, w, kernel=kernel)
    row = torch.zeros((M, 2 * F), dtype=torch.bool)
    row[M // 2] = True
    same_values(got[3:5], want[3:5], row)
    same_values(got[1:3], want[1:3], row[:, :F])


@pytest.mark.parametrize("kernel,w_fmt,M", KERNELS)
def test_gates_without_bound(ct, dev, kernel, w_fmt, M):
    """Sums beyond bf16's and beyond 32-bit numbers: silu(-inf) u is zero, silu(inf) u infinite, and what bf16 rounds up to infinity is that."""
    K, F = 512, 128
    a, w = randn_operand(M, K, O.E4M3, 1, dev), randn_operand(2 * F, K, w_fmt, 2, dev)
    # rows of A: 2^127 (1, 0, ..), so that a column is W's first element times that; codes of 1, and of W's elements, in E4M3 or E2M1
    u8(a.storage).zero_()
    u8(a.storage)[:, 0] = 0x38
    u8(a.scale_t)[:] = 254
    u8(a.scale_t)[::3] = 127
    wq, ws = u8(w.storage), u8(w.scale_t)
    wq.zero_()
    one, four = (0x38, 0x48) if w_fmt == O.E4M3 else (2, 6)
    sign = 0x80 if w_fmt == O.E4M3 else 8
    for c in range(F):
        wq[c, 0] = (one, one | sign, four, four | sign)[c % 4]     # gates: +-2^127, +-2^129
        wq[F + c, 0] = one | (sign if c & 4 else 0)                # up: +-2^(127 - 27 - c / 8)
        ws[F + c, 0] = 100 - c // 8
    ws[:F, 0] = 127
    got, want = both(ct, a, w, kernel=kernel)
    assert bool(want[0].isinf().any()) and not bool(want[0].isnan().any())
    assert torch.equal(got[0], want[0])
    every = torch.ones((M, 2 * F), dtype=torch.bool)
    same_values(got[3:5], want[3:5], every)
    same_values(got[1:3], want[1:3], every[:, :F])


@pytest.mark.parametrize("kernel,M", [("stream", 20), ("pingpong", 20), ("pingpong", 300)])
def test_gates_that_round_up_to_infinity(ct, dev, kernel, M):
    """Sums of 32 bits between bf16's largest number and 2^128: infinite in bf16 whichever kernel rounds them."""
    K, F = 512, 128
    a, w = randn_operand(M, K, O.E4M3, 1, dev), randn_operand(2 * F, K, O.E4M3, 2, dev)
    u8(a.storage).zero_()
    u8(a.scale_t)[:] = 127
    u8(a.storage)[:, :3] = torch.tensor([0x3F, 0x1F, 0x03], dtype=torch.uint8, device=dev)     # 1.875, 2^-3 15/16, 3 2^-9: 1.998 in all
    u8(a.scale_t)[:, 0] = 254
    u8(w.storage).zero_()
    u8(w.storage)[:, :3] = 0x38
    u8(w.storage)[1:F:2, :3] = 0xB8
    u8(w.scale_t)[:] = 127
    u8(w.scale_t)[F:, 0] = 27                                                                  # up: 2^-100 of it
    got, want = both(ct, a, w, kernel=kernel)
    assert bool(want[0][:, ::2].isinf().all()) and bool((want[0][:, 1::2] == 0).all())
    assert torch.equal(got[0], want[0])
    every = torch.ones((M, 2 * F), dtype=torch.bool)
    same_values(got[3:5], want[3:5], every)
    same_values(got[1:3], want[1:3], every[:, :F])
