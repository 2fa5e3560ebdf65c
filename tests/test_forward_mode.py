"""Forward-mode differentiation: the differentiable operators have a backward pass alone.  An input with a tangent is refused, whether anything
requires a gradient or not: a result without its tangent would be taken for a constant."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import cutile_amd as ct


def operators(dev="cpu"):
    t = lambda *shape: torch.ones(shape, device=dev)  # noqa: E731
    return {"layer_norm": (ct.layer_norm, [t(4, 64), t(64), t(64)]),
            "linear": (ct.linear, [t(4, 64), t(96, 64), t(96), t(4, 96)]),
            "gated_feed_forward": (ct.gated_feed_forward, [t(4, 64), t(64, 64), t(64, 32)])}


CASES = [("layer_norm", 3), ("linear", 4), ("gated_feed_forward", 3)]


def refused(name, which, dev, grad):
    f, args = operators(dev)[name]
    if grad:
        args[0].requires_grad_()
    with fwd.dual_level():
        args[which] = fwd.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match=f"{name} has no forward-mode derivative"):
            f(*args)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name,which", [(n, i) for n, k in CASES for i in range(k)])
def test_a_tangent_is_refused(name, which, grad):
    refused(name, which, "cpu", grad)


@pytest.mark.parametrize("name", [n for n, _ in CASES])
def test_jvp_is_refused(name):
    f, args = operators()[name]
    with pytest.raises(RuntimeError):
        torch.func.jvp(f, tuple(args), tuple(torch.ones_like(t) for t in args))


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name,which", [(n, i) for n, k in CASES for i in range(k)])
def test_a_tangent_is_refused_on_the_gpu(dev, name, which, grad):
    refused(name, which, dev, grad)


@pytest.mark.gpu
@pytest.mark.parametrize("name", [n for n, _ in CASES])
def test_jvp_is_refused_and_plain_inputs_are_not(dev, name):
    f, args = operators(dev)[name]
    with pytest.raises(RuntimeError):
        torch.func.jvp(f, tuple(args), tuple(torch.ones_like(t) for t in args))
    want = f(*args)
    with fwd.dual_level():                               # a level alone changes nothing
        assert torch.equal(f(*args), want)
