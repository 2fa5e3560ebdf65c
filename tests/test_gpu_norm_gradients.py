"""Gradients of layer norm where its backward pass can go wrong: rows whose mean times rstd is beyond the largest float in rows that do not
fill their threads, and gradients of weight and bias that are of different types."""
import pytest
import torch

from cutile_amd import norm
from test_gpu_norm import SUM, backward, d64, make, near, vectors

pytestmark = pytest.mark.gpu

bf16, f16, f32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [f32, bf16], ids=str)
@pytest.mark.parametrize("H", [1, 5, 100, 512, 600, 1000, 1500, 2500, 4097, 6001, 8192, 9000, 15999, 17001])
def test_mean_times_rstd_beyond_the_largest_float(ct, dev, H, dtype):
    """Rows of 2^100 and eps = 2^-80: every sum is exact, xhat is zero, rstd 2^40, and 2^140, which a lane without an element would make of the
    mean, is infinite."""
    rows = 7
    x = torch.full((rows, H), 2.0 ** 100, dtype=dtype, device=dev)
    x[3] = -x[3]
    dy = make(dev, rows, H, dtype, 21, 2.0 ** -45)
    w, b = vectors(dev, H, f32)
    y, mean, rstd = ct.layer_norm_forward(x, w, b, eps=2.0 ** -80)
    assert bool((mean.abs() == 2.0 ** 100).all()) and bool((rstd == 2.0 ** 40).all())
    near(y, d64(b).expand(rows, H), torch.zeros(1).double(), dtype)
    dx, dw, db = ct.layer_norm_backward(dy, x, mean, rstd, w)
    h = d64(dy) * d64(w)
    # (h and its mean: a product, the sum's roundings, a difference)
    near(dx, 2.0 ** 40 * (h - h.mean(-1, keepdim=True)), 2.0 ** 40 * 2 * SUM * (h.abs() + h.abs().mean(-1, keepdim=True)), dtype)
    assert bool((dw == 0).all())
    near(db, d64(dy).sum(0), SUM * d64(dy).abs().sum(0), f32)
    assert torch.equal(ct.layer_norm_backward(dy, x, mean, rstd, w, need_dweight=False, need_dbias=False)[0], dx)


@pytest.mark.parametrize("how,wt,bt", [(h, w, b) for h in ("x", "weight", "bias") for w, b in ((bf16, f32), (f16, f32), (f16, bf16), (f32, bf16), (None, f16), (f32, f32))
                                       if (h, w) != ("weight", None)])
def test_each_gradient_in_its_own_type(ct, dev, wt, bt, how):
    """Rows, weight or bias that lie apart take another way to the same kernels than contiguous ones: gradients are the same bits, and a bias's
    sum is rounded once, to the bias's type, whatever the weight's (sums here go to 1e5, beyond fp16's largest number)."""
    B, S, H = 10, 100, 300
    big = 100.0 if bt != f16 else 1.0
    dy = make(dev, B * S, H, f32, 31, 1.0, big).view(B, S, H)
    base = make(dev, S * B, H, f32, 32, 2.0, 0.5).view(S, B, H)
    w0, b0 = vectors(dev, H, f32)
    w0, b0 = None if wt is None else w0.to(wt), b0.to(bt)
    apart = lambda t: torch.stack((t, t), -1)[..., 0]  # noqa: E731

    def grads(strided):
        x = base.transpose(0, 1) if strided and how == "x" else base.transpose(0, 1).contiguous()
        w, b = w0, b0
        if strided and how == "weight":
            w = apart(w)
        if strided and how == "bias":
            b = apart(b)
        leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b)]
        assert not strided or not leaves[["x", "weight", "bias"].index(how)].is_contiguous()
        ct.layer_norm(*leaves).backward(dy)
        return [None if t is None else t.grad for t in leaves]

    want, off = backward(dy.reshape(-1, H), base.transpose(0, 1).reshape(-1, H), w0, 1e-5)
    plain, strided = grads(False), grads(True)
    for g, p, t, o, typ in zip(strided, plain, want, off, (f32, wt, bt)):
        if g is not None:
            assert g.dtype == typ and torch.equal(g, p)
            if typ != f16 or float(t.abs().max()) < 65000:
                near(g.reshape(t.shape), t, o, typ)
    assert bool(torch.isfinite(strided[2]).all())


def test_statistics_that_lie_apart(ct, dev, monkeypatch):
    """mean and rstd as columns of one tensor: the copies that are made of them are held until the kernel has been enqueued, so that nobody else on
    the stream gets their memory before."""
    x, dy = make(dev, 300, 700, bf16, 41, 2.0, 0.5), make(dev, 300, 700, bf16, 42)
    w, b = vectors(dev, 700, f32)
    _, mean, rstd = ct.layer_norm_forward(x, w, b)
    want = ct.layer_norm_backward(dy, x, mean, rstd, w)
    both = torch.stack((mean, rstd), -1)
    assert not both[:, 0].is_contiguous()
    real = norm._call

    def call(dev, f, *args):
        others = [torch.full((300,), float("nan"), device=dev) for _ in range(64)]
        real(dev, f, *args)
        del others

    monkeypatch.setattr(norm, "_call", call)
    got = ct.layer_norm_backward(dy, x, both[:, 0], both[:, 1], w)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
