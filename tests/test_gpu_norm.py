"""Layer norm against its definition in 64 bits: forward, backward, MX-quantised; lengths from one element to rows that no workgroup
holds, odd widths, pitches and alignments, rows that are constant, far from zero or not finite."""
import pytest
import torch

import ffnutil as R

pytestmark = pytest.mark.gpu

bf16, f16, f32 = torch.bfloat16, torch.float16, torch.float32
HALF = {f32: 2.0 ** -24, bf16: 2.0 ** -8, f16: 2.0 ** -11}
LEAST = {f32: 0.0, bf16: 0.0, f16: 2.0 ** -25}          # half a step of the subnormal numbers
# Sums in 32 bits: at most 32 elements of a thread in sequence, 6 steps over lanes, 16 waves: 54 roundings of 2^-24 each, and a few
# operations around them (long rows: 1 + H / 1024 in the place of 32).
SUM = 2.0 ** -18
SIZES = [(1, 1), (3, 2), (1, 32), (3, 33), (5, 255), (2, 511), (70, 512), (9, 513), (33, 1000), (4, 1024), (4, 1025), (5, 2047), (130, 2048),
         (3, 2049), (5, 4096), (2, 5001), (600, 5120), (3, 8192), (2, 8193), (3, 16384), (2, 16390), (3, 32768), (2, 40001)]


def make(dev, rows, H, dtype, seed=0, std=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed * 7919 + rows * 31 + H)
    return (torch.randn((rows, H), generator=g) * std + mean).to(dtype).to(dev)


def vectors(dev, H, dtype, seed=1):
    g = torch.Generator().manual_seed(seed + H)
    return (1 + 0.2 * torch.randn(H, generator=g)).to(dtype).to(dev), (0.3 * torch.randn(H, generator=g)).to(dtype).to(dev)


def d64(t):
    return None if t is None else t.detach().cpu().double()


def stats(x, eps):
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    return mean, rstd


def forward(x, w, b, eps):
    """y, and what the sums' roundings can make of it: the mean is off by SUM of mean |x|, differences by that and their own rounding."""
    x, w, b = d64(x), d64(w), d64(b)
    mean, rstd = stats(x, eps)
    w = torch.ones(x.shape[-1]).double() if w is None else w
    b = torch.zeros(x.shape[-1]).double() if b is None else b
    y = (x - mean) * rstd * w + b
    off = 2 * SUM * (x.abs().mean(-1, keepdim=True) + 2.0 ** -4 * x.abs()) * rstd
    off = off * (1 + ((x - mean) * rstd).abs()) + SUM * ((x - mean) * rstd).abs()
    return y, off * w.abs() + 2.0 ** -23 * b.abs()


def near(got, want, off, dtype):
    got = d64(got)
    bound = off + HALF[dtype] * (want.abs() + off) + LEAST[dtype]
    bad = ~((got - want).abs() <= bound)
    assert not bool(bad.any()), (float((got - want).abs().max()), int(bad.sum()), bad.nonzero()[:3].tolist())


@pytest.mark.parametrize("dtype", [f32, bf16, f16], ids=str)
@pytest.mark.parametrize("rows,H", SIZES)
def test_forward(ct, dev, rows, H, dtype):
    x = make(dev, rows, H, dtype, 1, 2.0, 0.5)
    w, b = vectors(dev, H, dtype)
    y, off = forward(x, w, b, 1e-5)
    near(ct.layer_norm(x, w, b), y, off, dtype)
    got, mean, rstd = ct.layer_norm_forward(x, w, b)
    near(got, y, off, dtype)
    m, r = stats(d64(x), 1e-5)
    assert mean.dtype == rstd.dtype == f32 and mean.shape == (rows,)
    near(mean, m[:, 0], SUM * d64(x).abs().mean(-1), f32)
    # (sqrt and reciprocal: 2^-23 each; the variance as the sums, doubled by the mean's error where it is small)
    near(rstd, r[:, 0], r[:, 0] * (4 * SUM + r[:, 0] ** 2 * (2 * SUM * d64(x).abs().mean(-1)) ** 2 + 2.0 ** -20), f32)


@pytest.mark.parametrize("wt,bt", [(None, None), (f32, None), (None, bf16), (f32, f32), (bf16, f32), (f16, bf16)])
@pytest.mark.parametrize("H", [31, 640, 4100])
def test_parameters_of_any_type(ct, dev, H, wt, bt):
    x = make(dev, 7, H, bf16, 2)
    w, b = vectors(dev, H, f32)
    w, b = None if wt is None else w.to(wt), None if bt is None else b.to(bt)
    y, off = forward(x, w, b, 1e-6)
    near(ct.layer_norm(x, w, b, eps=1e-6), y, off, bf16)


@pytest.mark.parametrize("H", [1, 65, 512, 777, 4096, 9000])
@pytest.mark.parametrize("dtype", [f32, bf16], ids=str)
def test_views(ct, dev, H, dtype):
    wide = make(dev, 12, H + 9, dtype, 3)
    w, b = vectors(dev, H + 1, dtype)
    w, b = w[1:], b[1:]                                   # off 16-byte borders
    for x in (wide[:, 3:3 + H], wide[::3, 9:], wide[:1, :H].expand(5, H), wide[:, :H].reshape(2, 6, H), wide.T[:H].T, wide[:0, :H]):
        want = ct.layer_norm(x.contiguous(), w, b)
        got = ct.layer_norm(x, w, b)
        assert got.shape == x.shape
        # (the same rows; a piece is read at another alignment, not in another order)
        assert torch.equal(got, want)


def test_rows_far_from_zero(ct, dev):
    """Means of a thousand standard deviations: the variance is that of the differences."""
    for H in (100, 3000, 20000):
        x = make(dev, 4, H, f32, 4, 1.0, 1000.0)
        y, off = forward(x, None, None, 1e-5)
        near(ct.layer_norm(x), y, off, f32)
        assert float(off.max()) < 0.1


@pytest.mark.parametrize("H", [1, 64, 1000, 5000, 33000])
def test_rows_of_one_value(ct, dev, H):
    x = torch.full((3, H), 3.0, dtype=f32, device=dev)
    w, b = vectors(dev, H, f32)
    assert torch.equal(ct.layer_norm(x, w, b), b.expand(3, H))
    y, mean, rstd = ct.layer_norm_forward(x, w, b, eps=4.0)
    assert bool((mean == 3).all()) and bool((rstd == 0.5).all())


@pytest.mark.parametrize("H", [40, 3000])
def test_rows_that_are_not_finite_stay_apart(ct, dev, H):
    x = make(dev, 6, H, bf16, 5)
    want = ct.layer_norm(x)
    x[1, 3], x[2, H - 1], x[4, 0] = float("nan"), float("inf"), -float("inf")
    got = ct.layer_norm(x)
    assert bool(got[[1, 2, 4]].isnan().all()) and torch.equal(got[[0, 3, 5]], want[[0, 3, 5]])
    q, s = ct.layer_norm_quantize(x)
    wq, ws = ct.layer_norm_quantize(x[[0, 3, 5]].contiguous())
    assert torch.equal(q[[0, 3, 5]].view(torch.uint8), wq.view(torch.uint8)) and torch.equal(s[[0, 3, 5]].view(torch.uint8), ws.view(torch.uint8))


# ---- quantised ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2", "e2m1"])
@pytest.mark.parametrize("mode", ["floor", "ceil"])
@pytest.mark.parametrize("rows,H", [(1, 32), (3, 33), (5, 500), (9, 1056), (4, 2048), (3, 4127), (2, 8192), (2, 20000), (2, 33001)])
def test_quantized_is_the_quantisation_of_the_float_result(ct, dev, rows, H, mode, fmt):
    """Of fp32 rows the unrounded result can be had, by the same arithmetic: the codes are then the same to the bit."""
    x = make(dev, rows, H, f32, 6, 3.0, 1.0)
    w, b = vectors(dev, H, bf16)
    how = fmt if fmt == "e2m1" else R.ELEM[fmt]
    q, s = ct.layer_norm_quantize(x, w, b, how, scale_mode=mode)
    wq, ws = ct.block_quantize(ct.layer_norm(x, w, b), 32, how, scale_mode=mode)
    assert q.dtype == wq.dtype and q.shape == wq.shape and s.shape == ws.shape
    assert torch.equal(q.view(torch.uint8), wq.view(torch.uint8)) and torch.equal(s.view(torch.uint8), ws.view(torch.uint8))


@pytest.mark.parametrize("dtype", [bf16, f16], ids=str)
@pytest.mark.parametrize("rows,H", [(1, 4096), (70, 96), (33, 1000), (3, 5001), (2, 17000)])
def test_quantized_from_16_bits(ct, dev, rows, H, dtype):
    x = make(dev, rows, H, dtype, 7, 3.0)
    w, b = vectors(dev, H, dtype)
    y, off = forward(x, w, b, 1e-5)
    q, s = ct.layer_norm_quantize(x, w, b)
    y, off = (torch.nn.functional.pad(t, (0, -H % 32)) for t in (y, off))
    wq, ws = R.quantize(y)
    step = ws.repeat_interleave(32, -1)
    s64 = torch.ldexp(torch.ones_like(ws), s.cpu().view(torch.uint8).int() - 127)
    # a block whose largest element is that close to a power of two may have its neighbour's scale: half or twice
    top, slack = y.abs().view(rows, -1, 32).amax(-1), off.view(rows, -1, 32).amax(-1)
    border = torch.frexp(top - slack)[1] != torch.frexp(top + slack)[1]
    assert bool(((s64 == ws) | border).all())
    got = R.value(q, s)
    assert bool(((got - y).abs() <= off + R.HALF_E4M3 * (y.abs() + off) + step * 2.0 ** -9 + (y.abs() > 447 * step) * y.abs() / 8).all())
    assert bool((got[:, H:] == 0).all())
    x3 = x.view(1, rows, H)
    q3, s3 = ct.layer_norm_quantize(x3, w, b)
    assert q3.shape == (1, rows, y.shape[1]) and torch.equal(q3[0].view(torch.uint8), q.view(torch.uint8))


@pytest.mark.parametrize("dtype", [f32, bf16], ids=str)
@pytest.mark.parametrize("rows,H", [(33000, 40), (9001, 600), (5003, 1500), (3001, 4096), (1531, 8192), (1100, 16000), (1030, 17000)])
def test_more_rows_than_fit_at_once(ct, dev, rows, H, dtype):
    """Workgroups that take several rows, the last of them fewer: every row is what it is by itself, and the definition's."""
    x = make(dev, rows, H, dtype, 20, 2.0, 0.5)
    w, b = vectors(dev, H, dtype)
    y, mean, rstd = ct.layer_norm_forward(x, w, b)
    q, s = ct.layer_norm_quantize(x, w, b)
    for at in (slice(0, 5), slice(rows // 2, rows // 2 + 3), slice(rows - 2, rows)):
        part = ct.layer_norm_forward(x[at], w, b)
        assert torch.equal(part[0], y[at]) and torch.equal(part[1], mean[at]) and torch.equal(part[2], rstd[at])
        pq, ps = ct.layer_norm_quantize(x[at], w, b)
        assert torch.equal(pq.view(torch.uint8), q[at].view(torch.uint8)) and torch.equal(ps.view(torch.uint8), s[at].view(torch.uint8))
    some = torch.randperm(rows, generator=torch.Generator().manual_seed(1))[:1000]
    want, off = forward(x[some.to(dev)], w, b, 1e-5)
    near(y[some.to(dev)], want, off, dtype)


# ---- backward ---------------------------------------------------------------------------------------------------------------
def backward(dy, x, w, eps):
    dy, x, w = d64(dy), d64(x), d64(w)
    mean, rstd = stats(x, eps)
    xh = (x - mean) * rstd
    h = dy if w is None else dy * w
    c0, c1 = h.mean(-1, keepdim=True), (h * xh).mean(-1, keepdim=True)
    dx = rstd * (h - c0 - xh * c1)
    # xhat is off by what the forward pass allows
    dxh = 2 * SUM * (x.abs().mean(-1, keepdim=True) + 2.0 ** -4 * x.abs()) * rstd * (1 + xh.abs()) + SUM * xh.abs()
    size = h.abs() + h.abs().mean(-1, keepdim=True) + xh.abs() * (h * xh).abs().mean(-1, keepdim=True)
    off_dx = rstd * (2 * SUM * size + dxh * c1.abs() + xh.abs() * (h.abs() * dxh).mean(-1, keepdim=True)) + dx.abs() * 4 * SUM
    chain = x.shape[0] * 2.0 ** -24 + SUM                  # a column's sum: no more roundings than rows, and the parts'
    off_dw = chain * (dy * xh).abs().sum(0) + (dy.abs() * dxh).sum(0)
    return (dx, (dy * xh).sum(0), dy.sum(0)), (off_dx, off_dw, chain * dy.abs().sum(0))


@pytest.mark.parametrize("dtype", [f32, bf16, f16], ids=str)
@pytest.mark.parametrize("rows,H", SIZES + [(1000, 96), (5000, 40), (700, 2500), (300, 16384), (257, 17000)])
def test_backward(ct, dev, rows, H, dtype):
    x, dy = make(dev, rows, H, dtype, 8, 2.0, 0.5), make(dev, rows, H, dtype, 9, 0.5)
    w, b = vectors(dev, H, dtype)
    want, off = backward(dy, x, w, 1e-5)
    _, mean, rstd = ct.layer_norm_forward(x, w, b)
    got = ct.layer_norm_backward(dy, x, mean, rstd, w)
    for g, t, o in zip(got, want, off):
        near(g, t, o, dtype)
    again = ct.layer_norm_backward(dy, x, mean, rstd, w)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    for k in range(3):
        one = ct.layer_norm_backward(dy, x, mean, rstd, w, need_dx=k == 0, need_dweight=k == 1, need_dbias=k == 2)
        assert torch.equal(one[k], got[k]) and all(one[i] is None for i in range(3) if i != k)


@pytest.mark.parametrize("xt,wt,bt", [(bf16, f32, f32), (bf16, f32, bf16), (f32, bf16, None), (bf16, None, None), (f16, None, f32)])
def test_autograd(ct, dev, xt, wt, bt):
    rows, H = 77, 1100
    x, dy = make(dev, rows, H, xt, 10), make(dev, rows, H, xt, 11)
    w, b = vectors(dev, H, f32)
    w, b = None if wt is None else w.to(wt).requires_grad_(), None if bt is None else b.to(bt).requires_grad_()
    want, off = backward(dy, x, w, 1e-5)
    x.requires_grad_()
    y = ct.layer_norm(x.view(7, 11, H), w, b)
    y.backward(dy.view(7, 11, H))
    for t, g, o in zip((x, w, b), want, off):
        if t is not None:
            assert t.grad.dtype == t.dtype and t.grad.shape == t.shape
            near(t.grad, g, o, t.dtype)
    near(y.view(rows, H), *forward(x, w, b, 1e-5), xt)


def test_gradient_against_differences(ct, dev):
    x, dy = make(dev, 3, 50, f32, 12), make(dev, 3, 50, f32, 13)
    w, b = vectors(dev, 50, f32)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    ct.layer_norm(*leaves).backward(dy)
    for t in leaves:
        step = make(dev, t.numel(), 1, f32, 14).view(t.shape).cpu().double()
        at = [[d64(u) + s * 1e-4 * step if u is t else d64(u) for u in leaves] for s in (-1, 1)]
        lo, hi = ((forward(*a, 1e-5)[0] * d64(dy)).sum() for a in at)
        # (difference quotient: third derivatives times 1e-8; the gradient in 32 bits)
        assert abs(float((hi - lo) / 2e-4 - (d64(t.grad) * step).sum())) < 1e-4 * float((d64(t.grad).abs() * step.abs()).sum())


def test_only_some_gradients(ct, dev):
    x = make(dev, 5, 64, bf16, 15)
    w, b = vectors(dev, 64, bf16)
    w.requires_grad_()
    (ct.layer_norm(x, w, b) * 2).sum().backward()
    assert w.grad is not None and x.grad is None and b.grad is None
    with torch.no_grad():
        assert not ct.layer_norm(x, w, b).requires_grad
    y = ct.layer_norm(x.requires_grad_(), None, b)
    (g,) = torch.autograd.grad(y.float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        g.sum().backward()


def test_input_changed_before_the_backward_pass_is_noticed(ct, dev):
    x = make(dev, 5, 64, bf16, 16).requires_grad_()
    h = x * 1
    y = ct.layer_norm(h)
    h.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.float().sum().backward()


def test_streams_and_graphs(ct, dev):
    rows, H = 40, 3000
    x, dy = make(dev, rows, H, bf16, 17), make(dev, rows, H, bf16, 18)
    w, b = vectors(dev, H, bf16)

    def everything():
        y, mean, rstd = ct.layer_norm_forward(x, w, b)
        return (y, *ct.layer_norm_backward(dy, x, mean, rstd, w), *(t.view(torch.uint8) for t in ct.layer_norm_quantize(x, w, b)))

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
    for seed in (19, 20, 21):
        x.copy_(make(dev, rows, H, bf16, seed))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(held, everything()))
    leaf = x.clone().requires_grad_()
    refused = torch.cuda.CUDAGraph()
    with torch.cuda.graph(refused):
        with pytest.raises(RuntimeError, match="cannot be captured"):
            ct.layer_norm(leaf, w, b)
        keep = x + 1                                       # (a graph of something)


def test_rows_past_32_bit_offsets(ct, dev):
    H, pitch = 96, 1 << 24
    big = torch.zeros(140 * pitch, dtype=bf16, device=dev)  # 4.7 GB, rows 32 MB apart: the last begins past 2^31 elements
    x = big.as_strided((140, H), (pitch, 1))
    x.copy_(make(dev, 140, H, bf16, 22))
    dense = x.contiguous()
    assert torch.equal(ct.layer_norm(x), ct.layer_norm(dense))
    _, mean, rstd = ct.layer_norm_forward(dense)
    for a, c in zip(ct.layer_norm_backward(x, x, mean, rstd), ct.layer_norm_backward(dense, dense, mean, rstd)):
        assert torch.equal(a, c)


def test_no_rows(ct, dev):
    x = torch.empty((0, 64), dtype=bf16, device=dev, requires_grad=True)
    w = torch.ones(64, dtype=f32, device=dev, requires_grad=True)
    y = ct.layer_norm(x, w)
    y.sum().backward()
    assert y.shape == (0, 64) and x.grad.shape == (0, 64) and bool((w.grad == 0).all())
    q, s = ct.layer_norm_quantize(x.detach(), w.detach())
    assert q.shape == (0, 64) and s.shape == (0, 2)
