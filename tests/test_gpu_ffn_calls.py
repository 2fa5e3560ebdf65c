"""How the feed-forward block's operators may be called: padded outputs through the C entries, offsets past 32 bits, other streams, graphs
replayed in turn, views and shared tensors, dtypes mixed, gradients asked for twice."""
import ctypes

import pytest
import torch

import ffnutil as R
from cutile_amd import _lib as L
from mxutil import randn_operand
from oracle import mx_oracle as O
from test_gpu_ffn import BF16_FLIPS, BLOCK, make, u8

pytestmark = pytest.mark.gpu

PAD, MARK = 64, 0xA5


def padded(dev, rows, cols, dtype):
    """(whole buffer filled with a mark, descriptor of its [rows, cols] part); dtype: an 8-bit MX type or MX_BF16."""
    size = 2 if dtype == L.MX_BF16 else 1
    buf = torch.full((rows + 2, (cols + PAD) * size), MARK, dtype=torch.uint8, device=dev)
    t = L.MxTensor()
    t.ptr, t.dtype, t.ndim, t.packed_dim = buf.data_ptr(), dtype, 2, -1
    t.shape[0], t.shape[1], t.stride[0], t.stride[1] = rows, cols, cols + PAD, 1
    return buf, t


def inner(buf, rows, cols, size=1):
    got = buf[:rows, :cols * size].contiguous()
    rest = buf.clone()
    rest[:rows, :cols * size] = MARK
    assert bool((rest == MARK).all()), "written outside of the output"
    return got


def refs(args):
    return [ctypes.byref(a) if isinstance(a, L.MxTensor) else a for a in args]


@pytest.mark.parametrize("M,K,F,kernel", [(3, 640, 96, "auto"), (20, 512, 64, "stream"), (77, 288, 160, "auto"), (300, 512, 320, "pingpong")])
@pytest.mark.parametrize("out", ["bf16", "e4m3"])
def test_gated_gemm_into_padded_rows(ct, dev, M, K, F, kernel, out):
    a, w = randn_operand(M, K, O.E4M3, M, dev), randn_operand(2 * F, K, O.E4M3, F, dev, std=K ** -0.5)
    o = L.MxGemmOpts(struct_size=32, kernel=L.KERNELS[kernel], block_size=32)
    lib = L.lib()
    need = lib.mx_gated_gemm_workspace_bytes(M, F, K, ctypes.byref(o))
    ws = torch.empty(max(need, 256), dtype=torch.uint8, device=dev)
    fmt = L.MX_BF16 if out == "bf16" else L.MX_E4M3
    h, dh = padded(dev, M, F, fmt)
    s, ds = padded(dev, M, F // 32, L.MX_E8M0)
    c, dc = padded(dev, M, 2 * F, L.MX_E4M3)
    cs, dcs = padded(dev, M, F // 16, L.MX_E8M0)
    args = [L.desc(u8(a.storage), L.MX_E4M3), L.desc(u8(a.scale_t), L.MX_E8M0), L.desc(u8(w.storage), L.MX_E4M3), L.desc(u8(w.scale_t), L.MX_E8M0),
            dh, None if out == "bf16" else ds, dc, dcs, 1, ctypes.byref(o), ws.data_ptr(), need, L.stream_ptr(dev)]
    assert lib.mx_gated_gemm(*refs(args)) == L.MX_OK, L.last_error()
    want = ct.gated_block_scaled_matmul(a.storage, a.scale_t, w.storage, w.scale_t, kernel=kernel, checkpoint=True,
                                        out_dtype=torch.bfloat16 if out == "bf16" else torch.float8_e4m3fn)
    if out == "bf16":
        assert torch.equal(inner(h, M, F, 2), u8(want[0]))
        inner(s, 0, 0)
    else:
        assert torch.equal(inner(h, M, F), u8(want[0])) and torch.equal(inner(s, M, F // 32), u8(want[1]))
    assert torch.equal(inner(c, M, 2 * F), u8(want[-2])) and torch.equal(inner(cs, M, F // 16), u8(want[-1]))


@pytest.mark.parametrize("M,F", [(1, 32), (40, 96), (300, 416)])
def test_quantizers_into_padded_rows(ct, dev, M, F):
    lib, Rp = L.lib(), (M + 31) // 32 * 32
    x = torch.randn((M, 2 * F), generator=torch.Generator().manual_seed(M)).to(torch.bfloat16).to(dev)
    outs = [(M, 2 * F, L.MX_E4M3), (M, F // 16, L.MX_E8M0), (2 * F, Rp, L.MX_E4M3), (2 * F, Rp // 32, L.MX_E8M0)]
    b = [padded(dev, *o) for o in outs]
    assert lib.mx_quantize_both(*refs([L.desc(x, L.MX_BF16), *(t for _, t in b), 1, L.stream_ptr(dev)])) == L.MX_OK, L.last_error()
    for (buf, _), (r, c, _), want in zip(b, outs, ct.block_quantize_both(x)):
        assert torch.equal(inner(buf, r, c), u8(want))
    dh = torch.randn((M, F), generator=torch.Generator().manual_seed(F)).to(torch.bfloat16).to(dev)
    q, s = ct.block_quantize(x, 32, torch.float8_e4m3fn, scale_mode="floor")
    outs += [(F, Rp, L.MX_E4M3), (F, Rp // 32, L.MX_E8M0)]
    b = [padded(dev, *o) for o in outs]
    args = [L.desc(dh, L.MX_BF16), L.desc(u8(q), L.MX_E4M3), L.desc(u8(s), L.MX_E8M0), *(t for _, t in b), 1, L.stream_ptr(dev)]
    assert lib.mx_silu_mul_backward_quantize(*refs(args)) == L.MX_OK, L.last_error()
    for (buf, _), (r, c, _), want in zip(b, outs, ct.silu_and_mul_backward_quantize(dh, q, s)):
        assert torch.equal(inner(buf, r, c), u8(want))


def test_past_32_bits(ct, dev):
    """Results of more than 2^31 elements: the first and the last rows are those of a call with these rows alone."""
    M, F, K = 40000, 28672, 32
    assert M * 2 * F > 2 ** 31
    a, w = randn_operand(M, K, O.E4M3, 1, dev), randn_operand(2 * F, K, O.E4M3, 2, dev, std=K ** -0.5)
    W = O.dequantize(w.codes, w.scales, w.fmt).double()
    last = M - 64
    for kernel in ("auto", "pingpong", "mfma128"):
        h, cq, cs = ct.gated_block_scaled_matmul(a.storage, a.scale_t, w.storage, w.scale_t, checkpoint=True, kernel=kernel)
        for r in (0, last):
            gu = R.bf16(O.dequantize(a.codes[r:r + 64], a.scales[r:r + 64], a.fmt).double() @ W.T)
            assert R.rel(h[r:r + 64], R.silu_mul(gu)) <= R.HALF_BF16 + 2 * BF16_FLIPS
            assert R.rel(R.value(cq[r:r + 64], cs[r:r + 64]), R.rows(gu)) <= 2 * (2.0 ** -14 * 2.0 ** -3) ** 0.5
    dh = h
    got = ct.silu_and_mul_backward_quantize(dh, cq, cs)
    for r in (0, last):
        want = ct.silu_and_mul_backward_quantize(dh[r:r + 64], cq[r:r + 64], cs[r:r + 64])
        for i, (g, w_) in enumerate(zip(got, want)):
            part = g[r:r + 64] if i < 2 else g[:, r:r + 64] if i % 2 == 0 else g[:, r // 32:r // 32 + 2]
            assert torch.equal(u8(part.contiguous()), u8(w_))


def test_operators_on_a_side_stream_and_in_graphs(ct, dev):
    """The single operators: enqueued on the current stream, and captured twice and replayed in turn beside eager calls."""
    a, w = randn_operand(9, 512, O.E4M3, 1, dev), randn_operand(256, 512, O.E4M3, 2, dev, std=512 ** -0.5)
    big = randn_operand(600, 512, O.E4M3, 3, dev)
    dh = torch.randn((600, 128), generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(dev)

    def calls(sa, sas, sb, sbs, sdh):
        few = ct.gated_block_scaled_matmul(sa, sas, w.storage, w.scale_t, out_dtype="e4m3")
        many = ct.gated_block_scaled_matmul(sb, sbs, w.storage, w.scale_t, checkpoint=True)
        return (*few, *many, *ct.silu_and_mul_backward_quantize(sdh, many[1], many[2]))

    args = [a.storage, a.scale_t, big.storage, big.scale_t, dh]
    want = calls(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = calls(*args)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(u8(x), u8(y)) for x, y in zip(got, want))
    held = [t.clone() for t in args]
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = calls(*held)
        graphs.append((g, out))
    for k in range(4):
        for t, n in ((held[0], randn_operand(9, 512, O.E4M3, 10 + k, dev).storage), (held[2], randn_operand(600, 512, O.E4M3, 20 + k, dev).storage)):
            u8(t).copy_(u8(n))
        want = calls(*held)
        for g, out in graphs:
            g.replay()
            eager = calls(*held)
            torch.cuda.synchronize()
            assert all(torch.equal(u8(x), u8(y)) and torch.equal(u8(x), u8(z)) for x, y, z in zip(out, want, eager))


def test_gradients_asked_for_twice(ct, dev):
    x, w1, w2, dy = make(70, 64, 96, 64, 3, dev, torch.float32)
    leaves = [t.requires_grad_() for t in (x, w1, w2)]
    y = ct.gated_feed_forward(*leaves)
    first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    again = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    only, = torch.autograd.grad(y, (w2,), dy, retain_graph=True)
    assert torch.equal(only, first[2])
    g, = torch.autograd.grad(y, (x,), dy, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        (g.square().sum() + x.sum()).backward()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, leaves, dy) and torch.autograd.grad(y, leaves, dy)     # the state was freed


def test_mixed_dtypes_and_views_of_the_gradient(ct, dev):
    x, w1, w2, dy = make(50, 96, 64, 128, 5, dev, torch.float32)
    x16 = x.to(torch.bfloat16)
    y, st = ct.gated_feed_forward_forward(x16, w1, w2)
    assert y.dtype == torch.bfloat16
    dy16 = dy.to(torch.bfloat16)
    want = ct.gated_feed_forward_backward(dy16, st)
    assert [t.dtype for t in want] == [torch.bfloat16, torch.float32, torch.float32]
    ref = R.block(*(t.cpu().double() for t in (x16, w1, w2, dy16)))
    # (the bounds of the block's own test: rounding of the result, flips of E4M3 on a path)
    for g, w in zip(want, ref[1:]):
        assert R.rel(g, w) <= R.HALF_BF16 + 8 * (2.0 ** -14 * 2.0 ** -3) ** 0.5
    wide = torch.full((50, 300), float("nan"), dtype=torch.bfloat16, device=dev)
    wide[:, 100:228] = dy16
    for view in (wide[:, 100:228], dy16.t().contiguous().t(), dy16.float()):
        assert all(torch.equal(a, b) for a, b in zip(ct.gated_feed_forward_backward(view, st), want))
    one = dy16[:1].expand(50, 128)
    assert all(torch.equal(a, b) for a, b in zip(ct.gated_feed_forward_backward(one, st), ct.gated_feed_forward_backward(one.contiguous(), st)))
    assert all(torch.equal(a, b) for a, b in zip(ct.gated_feed_forward_backward(dy16.half(), st),
                                                 ct.gated_feed_forward_backward(dy16.half().float(), st)))


def test_one_tensor_for_several_arguments(ct, dev):
    """A tensor that is input and weight at once: its gradient is the sum of both."""
    t = (torch.randn((128, 64), generator=torch.Generator().manual_seed(6)) * 0.1).to(torch.bfloat16).to(dev).requires_grad_()
    w2 = torch.randn((64, 64), generator=torch.Generator().manual_seed(7)).to(torch.bfloat16).to(dev)
    y = ct.gated_feed_forward(t, t, w2)
    g, = torch.autograd.grad(y, (t,), torch.ones_like(y))
    _, st = ct.gated_feed_forward_forward(t.detach(), t.detach(), w2)
    dx, dw1, _ = ct.gated_feed_forward_backward(torch.ones_like(y), st)
    assert torch.equal(g, dx + dw1)


# Few tokens: gate, up and dh are sums in 32 bits, off by 2^-22 of a norm at most; the shares of their elements that flip at a rounding to bf16 and on
# to E4M3 follow as in test_gpu_ffn.py, on three operands of a path, two flips each.  The last product is the scaled MFMA's (2^-14).
FEW = 3 * 2 * (2.0 ** -22 * 2.0 ** -3) ** 0.5 + 2.0 ** -14


@pytest.mark.parametrize("mode", ["floor", "ceil"])
@pytest.mark.parametrize("T,H,F,Ho", [(1, 1024, 2048, 1024), (1, 32, 32, 32), (2, 160, 96, 64), (16, 2080, 224, 96), (17, 1024, 512, 1024), (32, 96, 1056, 4128),
                                      (33, 1024, 512, 256), (64, 544, 1504, 320), (65, 512, 512, 512), (100, 1024, 544, 1024), (513, 288, 992, 96)])
def test_few_tokens_are_exact(ct, dev, T, H, F, Ho, mode):
    """Every result of a step with few tokens is its definition's, but for the few elements that lie that close to a border."""
    x, w1, w2, dy = make(T, H, F, Ho, T + F, dev, torch.float32)
    y, st = ct.gated_feed_forward_forward(x, w1, w2, scale_mode=mode)
    got = (y, *ct.gated_feed_forward_backward(dy, st))
    for g, w in zip(got, R.block(*(t.cpu().double() for t in (x, w1, w2, dy)), "e4m3", mode)):
        assert R.rel(g, w) <= FEW + 2.0 ** -24


def test_few_tokens_powers_of_two(ct, dev):
    """Scales far from one: the input up and the weight down by 2^60 give the same bits, a gradient of 2^-100 bits scaled by it."""
    x, w1, w2, dy = make(9, 288, 160, 96, 11, dev, torch.float32)
    y, st = ct.gated_feed_forward_forward(x, w1, w2)
    dx, dw1, dw2 = ct.gated_feed_forward_backward(dy, st)
    y2, st2 = ct.gated_feed_forward_forward(x * 2.0 ** 60, w1 * 2.0 ** -60, w2)
    dx2, dw12, dw22 = ct.gated_feed_forward_backward(dy * 2.0 ** -40, st2)
    assert torch.equal(y, y2) and torch.equal(dx2, dx * 2.0 ** -100) and torch.equal(dw12, dw1 * 2.0 ** 20) and torch.equal(dw22, dw2 * 2.0 ** -40)


def test_few_tokens_nan(ct, dev):
    """A NaN in a token reaches its row of y and dx; one in a weight what is multiplied by it."""
    x, w1, w2, dy = make(20, 128, 96, 64, 12, dev, torch.float32)
    y, st = ct.gated_feed_forward_forward(x, w1, w2)
    dx = ct.gated_feed_forward_backward(dy, st)[0]
    bad = x.clone()
    bad[7, 100] = float("nan")
    y2, st2 = ct.gated_feed_forward_forward(bad, w1, w2)
    dx2, dw1, _ = ct.gated_feed_forward_backward(dy, st2)
    keep = [i for i in range(20) if i != 7]
    assert bool(y2[7].isnan().all()) and bool(dx2[7].isnan().all()) and torch.equal(y2[keep], y[keep]) and torch.equal(dx2[keep], dx[keep])
    assert bool(dw1.isnan().any())
    worse = w1.clone()
    worse[3, 5] = float("nan")
    assert bool(ct.gated_feed_forward_forward(x, worse, w2)[0].isnan().all())


@pytest.mark.parametrize("T", [31, 32, 33, 63, 64, 65, 480, 512, 513])
def test_a_padded_batch(ct, dev, T):
    """Tokens of zeros behind a batch, and a gradient of zeros for them, change no result of the others and no weight's gradient."""
    x, w1, w2, dy = make(T, 96, 64, 64, T, dev)
    more = 96
    px, pdy = (torch.cat((t, torch.zeros((more, t.shape[1]), dtype=t.dtype, device=dev))) for t in (x, dy))
    y, st = ct.gated_feed_forward_forward(x, w1, w2)
    py, pst = ct.gated_feed_forward_forward(px, w1, w2)
    got, want = ct.gated_feed_forward_backward(pdy, pst), ct.gated_feed_forward_backward(dy, st)
    assert not bool(py[T:].any()) and not bool(got[0][T:].any())
    # (other kernels may be chosen: elements that lie at a rounding's border)
    for a, b in ((py[:T], y), (got[0][:T], want[0]), (got[1], want[1]), (got[2], want[2])):
        assert R.rel(a, b.cpu().double()) <= R.HALF_BF16 + 8 * (2.0 ** -14 * 2.0 ** -3) ** 0.5


@pytest.mark.parametrize("mode", ["floor", "ceil"])
@pytest.mark.parametrize("T,H,F,Ho", [(70, 256, 8224, 64), (600, 160, 992, 96), (1100, 544, 1056, 288), (1531, 256, 416, 128), (2100, 96, 320, 64),
                                      (520, 1024, 1088, 544), (129, 512, 4160, 256)])
def test_block_beyond_few_tokens(ct, dev, T, H, F, Ho, mode):
    """More than 2^19 elements of the activation: F of odd and even multiples of 32, tokens of no and of whole groups of 64 and 512."""
    assert T > 64 and T * F > 2 ** 19
    x, w1, w2, dy = make(T, H, F, Ho, T + F, dev, torch.float32)
    y, st = ct.gated_feed_forward_forward(x, w1, w2, scale_mode=mode)
    got = (y, *ct.gated_feed_forward_backward(dy, st))
    for g, w in zip(got, R.block(*(t.cpu().double() for t in (x, w1, w2, dy)), "e4m3", mode)):
        assert R.rel(g, w) <= 2.0 ** -24 + BLOCK
    for g, w in zip(ct.gated_feed_forward_backward(dy, st, need_dx=False), (None, *got[2:])):
        assert g is None if w is None else torch.equal(g, w)


@pytest.mark.parametrize("T,H,F,Ho", [(1100, 256, 1056, 128), (1100, 256, 1024, 128)])
def test_block_beyond_few_tokens_in_graphs(ct, dev, T, H, F, Ho):
    x, w1, w2, dy = make(T, H, F, Ho, 5, dev)
    sx, sdy = x.clone(), dy.clone()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            gy, gst = ct.gated_feed_forward_forward(sx, w1, w2)
            gd = ct.gated_feed_forward_backward(sdy, gst)
        graphs.append((g, (gy, *gd)))
    for k in range(4):
        nx, _, _, ndy = make(T, H, F, Ho, 30 + k, dev)
        sx.copy_(nx)
        sdy.copy_(ndy)
        ey, est = ct.gated_feed_forward_forward(nx, w1, w2)
        eager = (ey, *ct.gated_feed_forward_backward(ndy, est))
        for g, out in graphs:
            g.replay()
            again = ct.gated_feed_forward_backward(ndy, est)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, eager)) and all(torch.equal(a, b) for a, b in zip(again, eager[1:]))
