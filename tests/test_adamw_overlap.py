"""What an AdamW step writes must not overlap what other workgroups of it read: refused before anything touches a device."""
import pytest
import torch

import cutile_amd as ct
from cutile_amd import _lib as L
from test_norm_adamw_validation import B, P, adam, one

OTHER = 1 << 16


@pytest.mark.parametrize("tensors,over", [
    ([one(grad=P)], {}),                                                    # a parameter that is its own gradient
    ([one(grad=P + 252)], {}),
    ([one(grad=P + 2048 - 252)], {}),                                       # the gradient's last number is the first moment's first
    ([one(grad=P + 3008 + 252)], {}),
    ([one(), one(at=8192, grad=P)], {}),                                    # of another tensor
    ([one(at=8192), one(grad=P + 8192 + 2048)], {}),
    ([one(copy=P + OTHER), one(at=8192, grad=P + OTHER)], {}),              # a copy in the place of another tensor's gradient
    ([one(copy=P + OTHER), one(at=8192, g=B, grad=P + OTHER + 126)], {}),
    ([one(at=8192, g=B, grad=P + OTHER - 126), one(copy=P + OTHER)], {}),
    ([one(grad=P + OTHER - 8000, n=2001, param=P + 100000, exp_avg=P + 120000, exp_avg_sq=P + 140000, copy=P + OTHER)], {}),
    ([one(small=True, grad=P + 3600)], dict(state_bits=8)),
    ([one(small=True, grad=P + 3248)], dict(state_bits=8)),           # (64 elements: two scales, from 3500 on)
    ([one()], dict(step_at=P)),
    ([one()], dict(step_at=P - 4)),
    ([one()], dict(lr_at=P + 2048 + 252)),
    ([one()], dict(scale_at=P + 3008)),
])
def test_what_is_written_is_read_by_nobody_else(tensors, over):
    assert adam(tensors, **over) == L.MX_ERR_INVALID and "must not overlap a gradient" in L.last_error(), L.last_error()


def test_the_first_kind_is_named_first():
    assert adam([one(), one()]) == L.MX_ERR_INVALID and "listed twice" in L.last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_neighbours_are_fine(ct, dev, bits):
    """Parameters, gradients, copies, step and rate one behind the other in one buffer and gradients that are the same are taken; what overlaps by
    an element is not, and nothing is written then."""
    n = 96
    room = torch.zeros(8 * n, device=dev)
    p, q, g = room[:n], room[n:2 * n], room[2 * n:3 * n]
    c = room[3 * n:3 * n + n // 2].view(torch.bfloat16)
    g.fill_(1.0)
    step, lr = room[3 * n + n // 2:3 * n + n // 2 + 2].view(torch.int64), room[4 * n:4 * n + 1]
    step.fill_(1)
    lr.fill_(0.5)
    s = [ct.adamw_state(p, bits), ct.adamw_state(q, bits)]
    ct.adamw_step([p, q], [g, g], s, step=step, lr=lr, weight_decay=0.0, copies=[c, None])
    # the first step is lr, to some sixteen roundings of 2^-24 (1 - b1, 1 - b2, their products and powers, a root, two quotients) and eps
    assert all(bool(((t + 0.5).abs() <= 2.0 ** -20).all()) for t in (p, q)) and bool((c == -0.5).all()) and bool((g == 1).all())
    for grads, copies in (([g, c[:n]], [c, None]), ([p, g], [None, None]), ([g, room[n - 1:2 * n - 1]], [None, None])):
        before = room.clone()
        with pytest.raises(ValueError, match="must not overlap a gradient"):
            ct.adamw_step([p, q], grads, s, step=1, copies=copies)
        assert torch.equal(room, before)
    with pytest.raises(ValueError, match="must not overlap a gradient"):
        ct.adamw_step([p, q], [g, g], s, step=step, lr=p[:1])
