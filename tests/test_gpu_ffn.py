"""The gated product and the whole feed-forward block on the GPU, against 64-bit arithmetic and the single operators."""
import pytest
import torch

import ffnutil as R
from mxutil import randn_operand
from oracle import mx_oracle as O

pytestmark = pytest.mark.gpu

# The scaled MFMA's products of E4M3 and E2M1 elements with power-of-two scales are summed in 32 bits with the instruction's own
# alignment: within 2^-14 of the result's norm for the lengths here.  A value that is rounded to bf16 (half a step 2^-8 at most, 2^-9.8 in
# the root mean square) or to E4M3 behind it lands on the other neighbour where it lies that close to the border.
MFMA = 2.0 ** -14
# norm of the difference that this makes in a result quantised to E4M3: a share MFMA / step of the elements is a step, up to 2^-3, off
E4M3_FLIPS = (MFMA * 2.0 ** -3) ** 0.5
BF16_FLIPS = (MFMA * 2.0 ** -7) ** 0.5


def u8(t):
    return t.view(torch.uint8)


@pytest.mark.parametrize("w_fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("M,K,F", [(1, 256, 64), (3, 512, 96), (17, 160, 32), (40, 1024, 224), (100, 544, 320), (257, 512, 1024),
                                   (700, 1024, 1536), (1300, 512, 1120), (1024, 768, 2048)])
def test_gated_product(ct, dev, M, K, F, w_fmt):
    a = randn_operand(M, K, O.E4M3, M + K, dev)
    w = randn_operand(2 * F, K, O.E2M1 if w_fmt == "e2m1" else O.E4M3, F, dev, std=K ** -0.5)
    A = O.dequantize(a.codes, a.scales, O.E4M3).double()
    W = O.dequantize(w.codes, w.scales, w.fmt).double()
    gu = R.bf16(A @ W.T)
    kw = dict(w_format=w.fmt_kw)
    for ws in (w.scale_t, ct.pack_scales(w.scale_t, operand="b")):
        h = ct.gated_block_scaled_matmul(a.storage, a.scale_t, w.storage, ws, **kw)
        assert h.dtype == torch.bfloat16 and h.shape == (M, F)
        # half a step of h's own rounding, and what flips of gate and up make of it
        assert R.rel(h, R.silu_mul(gu)) <= R.HALF_BF16 + 2 * BF16_FLIPS
        q, s, cq, cs = ct.gated_block_scaled_matmul(a.storage, a.scale_t, w.storage, ws, out_dtype=torch.float8_e4m3fn, checkpoint=True, **kw)
        assert R.rel(R.value(q, s), R.rows(R.silu_mul(gu))) <= 2 * E4M3_FLIPS
        assert R.rel(R.value(cq, cs), R.rows(gu)) <= 2 * E4M3_FLIPS
        h2, cq2, cs2 = ct.gated_block_scaled_matmul(a.storage, a.scale_t, w.storage, ws, checkpoint=True, **kw)
        assert torch.equal(h2, h) and torch.equal(u8(cq2), u8(cq)) and torch.equal(u8(cs2), u8(cs))
        q2, s2 = ct.gated_block_scaled_matmul(a.storage, a.scale_t, w.storage, ws, out_dtype="e4m3", **kw)
        assert torch.equal(u8(q2), u8(q)) and torch.equal(u8(s2), u8(s))


@pytest.mark.parametrize("a_fmt,w_fmt", [("e4m3", "e4m3"), ("e4m3", "e2m1"), ("e5m2", "e5m2"), ("e2m1", "e2m1")])
@pytest.mark.parametrize("M,K,F", [(1, 32, 64), (100, 544, 192), (257, 512, 128), (300, 1536, 448), (770, 1024, 2112), (1025, 2048, 2944)])
def test_gated_product_in_one_kernel(ct, dev, M, K, F, a_fmt, w_fmt):
    """Tiles that overhang rows and columns, one and several tiles a workgroup, K that is no whole number of stages."""
    fmt = {"e4m3": O.E4M3, "e5m2": O.E5M2, "e2m1": O.E2M1}
    a, w = randn_operand(M, K, fmt[a_fmt], M + K, dev), randn_operand(2 * F, K, fmt[w_fmt], F, dev, std=K ** -0.5)
    gu = R.bf16(O.dequantize(a.codes, a.scales, a.fmt).double() @ O.dequantize(w.codes, w.scales, w.fmt).double().T)
    kw = dict(a_format=a.fmt_kw, w_format=w.fmt_kw, kernel="pingpong")
    for a_s, w_s in ((a.scale_t, w.scale_t), (ct.pack_scales(a.scale_t, operand="a"), ct.pack_scales(w.scale_t, operand="b"))):
        h, cq, cs = ct.gated_block_scaled_matmul(a.storage, a_s, w.storage, w_s, checkpoint=True, **kw)
        q, s = ct.gated_block_scaled_matmul(a.storage, a_s, w.storage, w_s, out_dtype="e4m3", **kw)
        assert R.rel(h, R.silu_mul(gu)) <= R.HALF_BF16 + 2 * BF16_FLIPS
        assert R.rel(R.value(q, s), R.rows(R.silu_mul(gu))) <= 2 * E4M3_FLIPS
        assert R.rel(R.value(cq, cs), R.rows(gu)) <= 2 * E4M3_FLIPS
    # its codes are those of the single operators for its own bf16 numbers, but where silu's last bits decide
    wq, ws = ct.block_quantize(h, 32, torch.float8_e4m3fn, scale_mode="floor")
    # (h was rounded to bf16 before: up to 2^-8 off, of which a share of 2^-8 / step elements move by a step of up to 2^-3)
    assert R.rel(R.value(q, s), R.value(wq, ws)) <= (R.HALF_BF16 * 2.0 ** -3) ** 0.5


@pytest.mark.parametrize("a_fmt,w_fmt", [("e4m3", "e4m3"), ("e4m3", "e2m1"), ("e5m2", "e5m2"), ("e5m2", "e2m1")])
@pytest.mark.parametrize("M,K,F", [(1, 128, 32), (2, 640, 96), (7, 1152, 64), (16, 2048, 160), (17, 512, 32), (29, 1664, 224), (32, 4224, 96)])
def test_gated_product_streamed(ct, dev, M, K, F, a_fmt, w_fmt):
    """Few rows: one and two row tiles, one to four K ranges of unequal lengths, K within a range's last 512, F of odd multiples of 32, strided rows."""
    fmt = {"e4m3": O.E4M3, "e5m2": O.E5M2, "e2m1": O.E2M1}
    a, w = randn_operand(M, K, fmt[a_fmt], M + K, dev), randn_operand(2 * F, K, fmt[w_fmt], F, dev, std=K ** -0.5)
    gu = R.bf16(O.dequantize(a.codes, a.scales, a.fmt).double() @ O.dequantize(w.codes, w.scales, w.fmt).double().T)
    kw = dict(a_format=a.fmt_kw, w_format=w.fmt_kw, kernel="stream")
    wide = torch.full((M, K + 48), 0x7F, dtype=torch.uint8, device=dev)      # rows with NaN codes behind them
    wide[:, :K] = u8(a.storage)
    strided = wide.view(a.storage.dtype)[:, :K]
    first = None
    for a_q, w_s in ((a.storage, w.scale_t), (strided, ct.pack_scales(w.scale_t, operand="b"))):
        h, cq, cs = ct.gated_block_scaled_matmul(a_q, a.scale_t, w.storage, w_s, checkpoint=True, **kw)
        q, s = ct.gated_block_scaled_matmul(a_q, a.scale_t, w.storage, w_s, out_dtype="e4m3", **kw)
        assert R.rel(h, R.silu_mul(gu)) <= R.HALF_BF16 + 2 * BF16_FLIPS
        assert R.rel(R.value(q, s), R.rows(R.silu_mul(gu))) <= 2 * E4M3_FLIPS
        assert R.rel(R.value(cq, cs), R.rows(gu)) <= 2 * E4M3_FLIPS
        got = [u8(t).clone() for t in (h, cq, cs, q, s)]
        assert first is None or all(torch.equal(x, y) for x, y in zip(got, first))
        first = got


def test_gated_product_streamed_nan(ct, dev):
    """NaN elements and scales of a row stay in it; a NaN in W reaches its column, and its MX block, of every row."""
    M, K, F = 20, 1024, 256
    a, w = randn_operand(M, K, O.E4M3, 1, dev), randn_operand(2 * F, K, O.E4M3, 2, dev, std=K ** -0.5)
    want, wcq, wcs = ct.gated_block_scaled_matmul(a.storage, a.scale_t, w.storage, w.scale_t, checkpoint=True, kernel="stream")
    u8(a.storage)[4, 1000] = 0x7F
    u8(a.scale_t)[18, 3] = 0xFF
    u8(w.storage)[70, 5] = 0xFF                       # a gate row
    u8(w.scale_t)[F + 131, 31] = 0xFF                 # an up row
    h, cq, cs = ct.gated_block_scaled_matmul(a.storage, a.scale_t, w.storage, w.scale_t, checkpoint=True, kernel="stream")
    rows, cols = [i for i in range(M) if i not in (4, 18)], [j for j in range(F) if j not in (70, 131)]
    assert bool(h[[4, 18]].isnan().all()) and bool(h[:, [70, 131]].isnan().all()) and bool(cq[[4, 18]].float().isnan().all())
    assert torch.equal(h[rows][:, cols], want[rows][:, cols])
    keep = [j for j in range(2 * F) if j // 32 not in (70 // 32, (F + 131) // 32)]
    assert torch.equal(u8(cq)[rows][:, keep], u8(wcq)[rows][:, keep])
    assert bool(cq[:, [70, F + 131]].float().isnan().all())


@pytest.mark.parametrize("a_fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("M,K,F", [(1, 512, 32), (5, 1024, 96), (17, 4096, 224), (32, 8192, 512), (16, 4608, 64), (20, 5120, 9216)])
def test_gated_product_decode(ct, dev, M, K, F, a_fmt):
    """The decode kernel: one and both halves of its rows, both lengths of a K slice, fewer units of 32 columns than workgroups and more."""
    a, w = randn_operand(M, K, O.E4M3 if a_fmt == "e4m3" else O.E5M2, M + K, dev), randn_operand(2 * F, K, O.E2M1, F, dev, std=K ** -0.5)
    gu = R.bf16(O.dequantize(a.codes, a.scales, a.fmt).double() @ O.dequantize(w.codes, w.scales, w.fmt).double().T)
    kw = dict(a_format=a.fmt_kw, w_format="e2m1", kernel="decode")
    h, cq, cs = ct.gated_block_scaled_matmul(a.storage, a.scale_t, w.storage, w.scale_t, checkpoint=True, **kw)
    q, s, cq2, cs2 = ct.gated_block_scaled_matmul(a.storage, a.scale_t, w.storage, w.scale_t, out_dtype="e4m3", checkpoint=True, **kw)
    assert R.rel(h, R.silu_mul(gu)) <= R.HALF_BF16 + 2 * BF16_FLIPS
    assert R.rel(R.value(q, s), R.rows(R.silu_mul(gu))) <= 2 * E4M3_FLIPS
    assert R.rel(R.value(cq, cs), R.rows(gu)) <= 2 * E4M3_FLIPS
    assert torch.equal(u8(cq2), u8(cq)) and torch.equal(u8(cs2), u8(cs))


def test_gated_product_decode_nan(ct, dev):
    """NaN elements and scales reach their rows and columns, in a workgroup's first unit and in its second, and nothing else."""
    M, K, F = 20, 1024, 9216                           # 288 units for 256 workgroups
    a, w = randn_operand(M, K, O.E4M3, 1, dev), randn_operand(2 * F, K, O.E2M1, 2, dev, std=K ** -0.5)
    kw = dict(w_format="e2m1", kernel="decode", checkpoint=True)
    want, wcq, _ = ct.gated_block_scaled_matmul(a.storage, a.scale_t, w.storage, w.scale_t, **kw)
    u8(a.storage)[4, 1000] = 0x7F
    u8(a.scale_t)[18, 3] = 0xFF
    bad = [5, 70, 8200, 9215]
    for n, j in enumerate(bad):
        u8(w.scale_t)[j + F * (n % 2), 7 * n] = 0xFF   # gate rows and up rows
    h, cq, cs = ct.gated_block_scaled_matmul(a.storage, a.scale_t, w.storage, w.scale_t, **kw)
    rows, cols = [i for i in range(M) if i not in (4, 18)], [j for j in range(F) if j not in bad]
    assert bool(h[[4, 18]].isnan().all()) and bool(h[:, bad].isnan().all()) and bool(cq[[4, 18]].float().isnan().all())
    assert torch.equal(h[rows][:, cols], want[rows][:, cols]) and not bool(h[rows][:, cols].isnan().any())
    clean = [j for j in range(2 * F) if j % F // 32 not in [b // 32 for b in bad]]
    assert torch.equal(u8(cq)[rows][:, clean], u8(wcq)[rows][:, clean])


def test_gated_product_is_chosen_by_size(ct, dev):
    """Where the streaming kernel is taken by default, its bits; explicit kernels and the others agree to their bounds."""
    for M, K, F, w_fmt in ((1, 2048, 4096, O.E4M3), (32, 8192, 2048, O.E4M3), (32, 8192, 1024, O.E2M1), (33, 1024, 512, O.E4M3),
                          (24, 4096, 512, O.E2M1), (12, 4608, 16384, O.E2M1)):
        a, w = randn_operand(M, K, O.E4M3, 1, dev), randn_operand(2 * F, K, w_fmt, 2, dev, std=K ** -0.5)
        got = ct.gated_block_scaled_matmul(a.storage, a.scale_t, w.storage, w.scale_t, w_format=w.fmt_kw)
        for kernel in ("stream", "pingpong", "mfma128"):
            other = ct.gated_block_scaled_matmul(a.storage, a.scale_t, w.storage, w.scale_t, w_format=w.fmt_kw, kernel=kernel)
            # elements whose gate and up flip at no kernel are the same; a flip of each, and the result's own rounding behind them
            assert R.rel(got, other.cpu().double()) <= 4 * BF16_FLIPS


def test_gated_product_in_one_kernel_extremes(ct, dev):
    """Blocks of zeros, of subnormal and of very large numbers, NaN: rows and scales of the operands that lead to them."""
    M, K, F = 300, 512, 512
    a, w = randn_operand(M, K, O.E4M3, 1, dev), randn_operand(2 * F, K, O.E4M3, 2, dev, std=K ** -0.5)
    u8(a.storage)[5] = 0
    u8(a.scale_t)[6:9] = torch.tensor([[3], [20], [200]], dtype=torch.uint8, device=dev)
    u8(a.storage)[10, 3] = 0x7F
    u8(w.storage)[64:96] = 0
    gu = ct.block_scaled_matmul(a.storage, a.scale_t, w.storage.T, w.scale_t.T, out_dtype=torch.bfloat16, kernel="pingpong")
    h, cq, cs = ct.gated_block_scaled_matmul(a.storage, a.scale_t, w.storage, w.scale_t, checkpoint=True, kernel="pingpong")
    wq, ws = ct.block_quantize(gu, 32, torch.float8_e4m3fn, scale_mode="floor")
    keep = [i for i in range(M) if i != 10]
    assert torch.equal(u8(cq)[keep], u8(wq)[keep]) and torch.equal(u8(cs)[keep], u8(ws)[keep])
    assert bool(h[10].isnan().all()) and bool(cq[10].float().isnan().all()) and not bool(h[keep].isnan().any())
    assert float(h[5].abs().max()) == 0 and float(h[:, 64:96][keep].abs().max()) == 0


def test_gated_product_in_one_kernel_nan(ct, dev):
    """A NaN element and a NaN scale reach their row's every column, in the first and in later tiles of a workgroup's walk, and no other row."""
    M, K, F = 2400, 512, 4096                          # more tiles than workgroups
    a, w = randn_operand(M, K, O.E4M3, 1, dev), randn_operand(2 * F, K, O.E4M3, 2, dev, std=K ** -0.5)
    want = ct.gated_block_scaled_matmul(a.storage, a.scale_t, w.storage, w.scale_t, kernel="pingpong")
    rows = list(range(3, M, 97))
    for n, r in enumerate(rows):
        if n % 2:
            u8(a.scale_t)[r, n % 16] = 0xFF
        else:
            u8(a.storage)[r, 17 * n % K] = 0x7F
    got, cq, cs = ct.gated_block_scaled_matmul(a.storage, a.scale_t, w.storage, w.scale_t, checkpoint=True, kernel="pingpong")
    q, s = ct.gated_block_scaled_matmul(a.storage, a.scale_t, w.storage, w.scale_t, out_dtype="e4m3", kernel="pingpong")
    keep = [i for i in range(M) if i not in set(rows)]
    assert bool(got[rows].isnan().all()) and bool(cq[rows].float().isnan().all()) and bool(q[rows].float().isnan().all())
    assert torch.equal(got[keep], want[keep]) and not bool(cq[keep].float().isnan().any())


@pytest.mark.parametrize("M,K,F,mode", [(5, 256, 64, "ceil"), (300, 512, 512, "ceil"), (300, 512, 512, "floor")])
def test_gated_product_is_the_pair_of_operators(ct, dev, M, K, F, mode):
    """The same bits as the projections in bf16, then silu_and_mul_quantize, and block_quantize of the former."""
    a, w = randn_operand(M, K, O.E4M3, 1, dev), randn_operand(2 * F, K, O.E4M3, 2, dev, std=K ** -0.5)
    gu = ct.block_scaled_matmul(a.storage, a.scale_t, w.storage.T, w.scale_t.T, out_dtype=torch.bfloat16)
    for fmt in ("e4m3", "e5m2"):
        q, s, cq, cs = ct.gated_block_scaled_matmul(a.storage, a.scale_t, w.storage, w.scale_t, out_dtype=R.ELEM[fmt], checkpoint=True,
                                                    scale_mode=mode)
        wq, ws = ct.silu_and_mul_quantize(gu, R.ELEM[fmt], scale_mode=mode)
        wcq, wcs = ct.block_quantize(gu, 32, torch.float8_e4m3fn, scale_mode=mode)
        for x, y in ((q, wq), (s, ws), (cq, wcq), (cs, wcs)):
            assert torch.equal(u8(x), u8(y))


def test_gated_product_nan_stays_in_its_row(ct, dev):
    M, K, F = 300, 512, 512
    a, w = randn_operand(M, K, O.E4M3, 1, dev), randn_operand(2 * F, K, O.E4M3, 2, dev, std=K ** -0.5)
    want = ct.gated_block_scaled_matmul(a.storage, a.scale_t, w.storage, w.scale_t)
    u8(a.storage)[7, 3] = 0x7F
    u8(a.scale_t)[250, 2] = 0xFF
    got = ct.gated_block_scaled_matmul(a.storage, a.scale_t, w.storage, w.scale_t)
    keep = [i for i in range(M) if i not in (7, 250)]
    assert bool(got[7].isnan().all()) and bool(got[250].isnan().all()) and torch.equal(got[keep], want[keep])
    none = ct.gated_block_scaled_matmul(a.storage[:0], a.scale_t[:0], w.storage, w.scale_t, checkpoint=True)
    assert [tuple(t.shape) for t in none] == [(0, F), (0, 2 * F), (0, F // 16)]


def make(T, H, F, Ho, seed, dev, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((T, H), generator=g).to(dtype)
    w1 = (torch.randn((2 * F, H), generator=g) * H ** -0.5).to(dtype)
    w2 = (torch.randn((Ho, F), generator=g) * F ** -0.5).to(dtype)
    dy = (torch.randn((T, Ho), generator=g) * 1e-3).to(dtype)
    return [t.to(dev) for t in (x, w1, w2, dy)]


# Every product of the block takes operands with flips of E4M3 of their own, at most three on a path (gate and up, the activation
# or its gradient, dh through bf16): their norms add up in the worst case.
BLOCK = 3 * 2 * E4M3_FLIPS


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,H,F,Ho", [(1, 64, 96, 32), (5, 160, 64, 96), (33, 256, 512, 256), (64, 256, 384, 256), (65, 512, 320, 512),
                                      (200, 544, 1056, 288), (300, 512, 1024, 512), (1030, 256, 768, 512)])
def test_block_forward_and_backward(ct, dev, T, H, F, Ho, dtype):
    x, w1, w2, dy = make(T, H, F, Ho, T + H, dev, dtype)
    for t in (x, w1, w2):
        t.requires_grad_()
    y = ct.gated_feed_forward(x, w1, w2)
    got = (y, *torch.autograd.grad(y, (x, w1, w2), dy))
    want = R.block(*(t.detach().cpu().double() for t in (x, w1, w2, dy)))
    half = R.HALF_BF16 if dtype == torch.bfloat16 else 2.0 ** -24
    for g, w, like in zip(got, want, (y, x, w1, w2)):
        assert g.shape == w.shape and g.dtype == dtype and g.shape == like.shape
        assert R.rel(g, w) <= half + BLOCK
    with torch.no_grad():
        assert torch.equal(ct.gated_feed_forward(x, w1, w2), y)


def test_block_functional_form_and_parts(ct, dev):
    """The functional form gives autograd's bits, each gradient alone those of all together, and the state can be read again."""
    x, w1, w2, dy = make(130, 256, 320, 192, 3, dev)
    y, state = ct.gated_feed_forward_forward(x, w1, w2)
    want = ct.gated_feed_forward_backward(dy, state)
    for k in range(8):
        need = [bool(k >> b & 1) for b in range(3)]
        got = ct.gated_feed_forward_backward(dy, state, need_dx=need[0], need_dw1=need[1], need_dw2=need[2])
        for g, w, n in zip(got, want, need):
            assert torch.equal(g, w) if n else g is None
    leaves = [t.clone().requires_grad_() for t in (x, w1, w2)]
    out = ct.gated_feed_forward(*leaves)
    assert torch.equal(out, y)
    with torch.no_grad():
        leaves[1].zero_()                # an update in place between the passes: the quantised weights were kept
    for g, w in zip(torch.autograd.grad(out, leaves, dy), want):
        assert torch.equal(g, w)


def test_block_leading_axes_and_strides(ct, dev):
    x, w1, w2, dy = make(60, 128, 96, 160, 4, dev)
    want = ct.gated_feed_forward(x, w1, w2)
    xs = torch.zeros((60, 200), dtype=x.dtype, device=dev)
    xs[:, 5:133] = x
    assert torch.equal(ct.gated_feed_forward(xs[:, 5:133].unflatten(0, (3, 20)), w1.t().contiguous().t(), w2), want.view(3, 20, 160))
    x3 = x.view(3, 20, 128).clone().requires_grad_()
    y = ct.gated_feed_forward(x3, w1, w2)
    y.backward(dy.view(3, 20, 160))
    assert x3.grad.shape == x3.shape and w1.grad is None
    # the gradient of a sum: a dy whose rows are one row
    y = ct.gated_feed_forward(x3, w1, w2)
    s1, = torch.autograd.grad(y.sum(), x3)
    y = ct.gated_feed_forward(x3, w1, w2)
    s2, = torch.autograd.grad(y, x3, torch.ones_like(y))
    assert torch.equal(s1, s2)


def test_block_without_tokens(ct, dev):
    _, w1, w2, _ = make(1, 64, 96, 32, 5, dev)
    x = torch.empty((0, 64), dtype=torch.bfloat16, device=dev, requires_grad=True)
    w1.requires_grad_()
    w2.requires_grad_()
    y = ct.gated_feed_forward(x, w1, w2)
    assert y.shape == (0, 32)
    dx, d1, d2 = torch.autograd.grad(y, (x, w1, w2), torch.empty_like(y))
    assert dx.shape == (0, 64) and not bool(d1.any()) and not bool(d2.any())


def test_gradients_against_differences(ct, dev):
    """The formula that the other tests hold the kernels to is the derivative of the block (differences in 64 bits), and the
    8-bit gradients are that derivative but for the quantisation: six roundings to E4M3 on a path, each 2^-4.8 of the norm at most
    (the root mean square of a uniform error of up to half a step of 2^-3), which add up to 0.21 if all of one sign."""
    T, H, F, Ho = 96, 128, 192, 160
    x, w1, w2, dy = make(T, H, F, Ho, 6, dev)
    v64 = [t.cpu().double() for t in (x, w1, w2)]
    d64 = dy.cpu().double()
    gu = v64[0] @ v64[1].T
    d, a = R.silu_mul_backward(d64 @ v64[2], gu)
    formula = (d @ v64[1], d.T @ v64[0], d64.T @ a)
    g = torch.Generator().manual_seed(7)
    for k in range(3):
        v, eps = torch.randn(v64[k].shape, generator=g, dtype=torch.float64), 1e-5
        up, down = list(v64), list(v64)
        up[k], down[k] = up[k] + eps * v, down[k] - eps * v
        diff = float(((R.block_unquantized(*up) - R.block_unquantized(*down)) * d64).sum()) / (2 * eps)
        assert abs(diff - float((formula[k] * v).sum())) <= 1e-6 * float(formula[k].norm() * v.norm())
    y, state = ct.gated_feed_forward_forward(x, w1, w2)
    for got, want in zip(ct.gated_feed_forward_backward(dy, state), formula):
        assert R.rel(got, want) <= 6 * 2.0 ** -4.8


def test_block_in_a_training_loop(ct, dev):
    """Runs as a module's forward, with an optimiser; micro-batches accumulate into the leaves' gradients."""
    x, w1, w2, dy = make(48, 64, 96, 64, 8, dev, torch.float32)
    w1, w2 = torch.nn.Parameter(w1), torch.nn.Parameter(w2)
    opt = torch.optim.SGD([w1, w2], lr=0.1)
    for _ in range(3):
        opt.zero_grad()
        for part, d in ((x[:20], dy[:20]), (x[20:], dy[20:])):
            ct.gated_feed_forward(part, w1, w2).backward(d)
        assert bool(w1.grad.isfinite().all()) and bool(w2.grad.isfinite().all()) and float(w1.grad.norm()) > 0
        opt.step()


def test_block_streams_and_graph(ct, dev):
    x, w1, w2, dy = make(300, 256, 512, 256, 9, dev)
    want_y, state = ct.gated_feed_forward_forward(x, w1, w2)
    want = ct.gated_feed_forward_backward(dy, state)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, st = ct.gated_feed_forward_forward(x, w1, w2)
        got = ct.gated_feed_forward_backward(dy, st)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, want_y) and all(torch.equal(a, b) for a, b in zip(got, want))
    sx, sdy = x.clone(), dy.clone()
    graphs = []
    for _ in range(2):                                 # two graphs, replayed in turn, with eager calls between
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            gy, gst = ct.gated_feed_forward_forward(sx, w1, w2)
            gd = ct.gated_feed_forward_backward(sdy, gst)
            gq = ct.block_quantize_both(sx)
        graphs.append((g, gy, gd, gq))
    for k in range(4):
        nx, _, _, ndy = make(300, 256, 512, 256, 20 + k, dev)
        sx.copy_(nx)
        sdy.copy_(ndy)
        ey, est = ct.gated_feed_forward_forward(nx, w1, w2)
        for g, gy, gd, gq in graphs:
            g.replay()
            ed = ct.gated_feed_forward_backward(ndy, est)
            torch.cuda.synchronize()
            assert torch.equal(gy, ey) and all(torch.equal(a, b) for a, b in zip(gd, ed))
            assert all(torch.equal(u8(a), u8(b)) for a, b in zip(gq, ct.block_quantize_both(nx)))
    x.requires_grad_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        sx.add_(0)
        with pytest.raises(RuntimeError, match="cannot be captured"):
            ct.gated_feed_forward(x, w1, w2)
    g.replay()
    torch.cuda.synchronize()


def test_two_threads(ct, dev):
    import threading
    data = [make(100 + 50 * i, 256, 320, 256, 30 + i, dev) for i in range(2)]
    want = []
    for x, w1, w2, dy in data:
        y, st = ct.gated_feed_forward_forward(x, w1, w2)
        want.append((y, *ct.gated_feed_forward_backward(dy, st)))
    torch.cuda.synchronize()
    bad = []

    def work(i):
        x, w1, w2, dy = data[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                y, st = ct.gated_feed_forward_forward(x, w1, w2)
                got = (y, *ct.gated_feed_forward_backward(dy, st))
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    bad.append(i)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad
