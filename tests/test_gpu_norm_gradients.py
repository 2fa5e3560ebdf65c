"""Gradients of layer norm where its backward pass can go wrong: rows whose mean times rstd is beyond the largest float."""
import pytest
import torch

from test_gpu_norm import SUM, d64, make, near, vectors

pytestmark = pytest.mark.gpu

bf16, f32 = torch.bfloat16, torch.float32


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
