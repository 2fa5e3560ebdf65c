"""The block's autograd form in the ways a training program calls it, and what becomes of gradients that are not finite."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from test_gpu_ffn import make

pytestmark = pytest.mark.gpu
SIZES = [(9, 64, 96, 64), (130, 128, 64, 96), (1100, 128, 544, 96)]


def leaves(t):
    return [v.detach().clone().requires_grad_() for v in t]


@pytest.mark.parametrize("size", SIZES)
def test_recomputed_and_offloaded(ct, dev, size):
    """Activation checkpointing, of both kinds, and saved tensors that wait on the host give the same bits."""
    *w, dy = make(*size, 3, dev)
    a = leaves(w)
    y = ct.gated_feed_forward(*a)
    want = (y, *torch.autograd.grad(y, a, dy))
    for reentrant in (False, True):
        b = leaves(w)
        z = checkpoint(ct.gated_feed_forward, *b, use_reentrant=reentrant)
        z.backward(dy)
        assert all(torch.equal(p, q) for p, q in zip((z, *(t.grad for t in b)), want))
    b = leaves(w)
    with torch.autograd.graph.save_on_cpu():
        z = ct.gated_feed_forward(*b)
    assert all(torch.equal(p, q) for p, q in zip((z, *torch.autograd.grad(z, b, dy)), want))


@pytest.mark.parametrize("size", SIZES)
def test_in_front_of_and_behind_other_operators(ct, dev, size):
    """A residual around the block, hooks on its result and its input, a result that is written to in place, a frozen weight."""
    *w, dy = make(*size, 4, dev)
    seen = []
    x, w1, w2 = leaves(w)
    w1.requires_grad_(False)
    h = x * 2
    h.register_hook(lambda g: seen.append(g.clone()))
    y = ct.gated_feed_forward(h, w1, w2)
    y.mul_(0.5)
    y.backward(dy)
    plain, st = ct.gated_feed_forward_forward(w[0] * 2, w[1], w[2])
    dx, _, dw2 = ct.gated_feed_forward_backward(dy * 0.5, st)
    assert torch.equal(y, plain * 0.5) and torch.equal(seen[0], dx) and torch.equal(x.grad, dx * 2) and torch.equal(w2.grad, dw2) and w1.grad is None


@pytest.mark.parametrize("size", SIZES)
def test_backward_on_another_stream(ct, dev, size):
    """The forward pass on a side stream, gradients taken from the current one: autograd runs them where the forward pass ran."""
    *w, dy = make(*size, 5, dev)
    a = leaves(w)
    y = ct.gated_feed_forward(*a)
    want = (y, *torch.autograd.grad(y, a, dy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    b = leaves(w)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        z = ct.gated_feed_forward(*b)
    torch.cuda.current_stream().wait_stream(side)
    got = (z, *torch.autograd.grad(z, b, dy))
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("size", SIZES)
def test_gradients_that_are_not_finite(ct, dev, size):
    """A NaN of the gradient reaches its row of dx and every weight's gradient in both rules; an infinity is a NaN under the ceiling rule, and the
    largest number of its block's scale under the floor rule (finite)."""
    *w, dy = make(*size, 6, dev)
    row = size[0] // 2
    keep = [i for i in range(size[0]) if i != row]
    for mode in ("floor", "ceil"):
        _, st = ct.gated_feed_forward_forward(*w, scale_mode=mode)
        clean = ct.gated_feed_forward_backward(dy, st)
        for value in (float("nan"), float("inf"), float("-inf")):
            bad = dy.clone()
            bad[row, 33] = value
            dx, dw1, dw2 = ct.gated_feed_forward_backward(bad, st)
            if mode == "floor" and value == value:
                continue
            assert bool(dx[row].isnan().all()) and bool(dw1.isnan().any()) and bool(dw2[33].isnan().all())
            assert torch.equal(dx[keep], clean[0][keep])
