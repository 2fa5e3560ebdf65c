"""Layer norm, linear layers and AdamW together, as a model has them: a pre-norm block trained by autograd, the same step captured into a
graph, and the block served on quantised operands."""
import pytest
import torch

import ffnutil as R
from oracle import mx_oracle as O
from test_gpu_ffn_elements import check_codes, sum_error
from test_gpu_linear import FLIPS, act64, d64, u8

pytestmark = pytest.mark.gpu

bf16, f32 = torch.bfloat16, torch.float32


def parameters(dev, H, F, seed, dtype=f32):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    p = dict(ln_w=1 + 0.1 * r(H), ln_b=0.1 * r(H), w1=r(F, H) * H ** -0.5, b1=0.1 * r(F), w2=r(H, F) * F ** -0.5, b2=0.1 * r(H))
    return {k: v.to(dtype).to(dev) for k, v in p.items()}


def rows(dev, T, H, seed, dtype):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((T, H), generator=g).to(dtype).to(dev), (torch.randn((T, H), generator=g) * 1e-2).to(dtype).to(dev)


def block(ct, x, p):
    return ct.linear(ct.linear(ct.layer_norm(x, p["ln_w"], p["ln_b"]), p["w1"], p["b1"], activation="gelu"), p["w2"], p["b2"], x)


def by_hand(ct, x, dy, p):
    """(everything on the way, gradients) without autograd."""
    h, mean, rstd = ct.layer_norm_forward(x, p["ln_w"], p["ln_b"])
    a, s1 = ct.linear_forward(h, p["w1"], p["b1"], activation="gelu")
    y, s2 = ct.linear_forward(a, p["w2"], p["b2"], x)
    da, dw2, db2 = ct.linear_backward(dy, s2)
    dh, dw1, db1 = ct.linear_backward(da, s1)
    dx, dln_w, dln_b = ct.layer_norm_backward(dh, x, mean, rstd, p["ln_w"])
    return (h, a, y, da, dh, dx), dict(ln_w=dln_w, ln_b=dln_b, w1=dw1, b1=db1, w2=dw2, b2=db2)


def near(got, want, tol):
    """The relative distance, with a result's own rounding."""
    assert R.rel(got, want) <= tol + {f32: 0.0, bf16: R.HALF_BF16}[got.dtype], R.rel(got, want)


@pytest.mark.parametrize("dtype", [f32, bf16])
@pytest.mark.parametrize("T,H,F", [(1, 64, 96), (60, 256, 1024), (700, 512, 2048), (1531, 256, 1056)])
def test_a_block_trained(ct, dev, T, H, F, dtype):
    p = {k: v.requires_grad_() for k, v in parameters(dev, H, F, 1, dtype).items()}
    x, dy = rows(dev, T, H, 2, dtype)
    x.requires_grad_()
    y = block(ct, x, p)
    grads = torch.autograd.grad(y, (x, *p.values()), dy)
    (h, a, y2, da, dh, dx), hand = by_hand(ct, x.detach(), dy, {k: v.detach() for k, v in p.items()})
    assert torch.equal(y, y2) and all(torch.equal(g, hand[k]) for k, g in zip(p, grads[1:]))
    assert torch.equal(grads[0], dx + dy) or torch.equal(grads[0], dy + dx)
    # each product from what the operator in front of it left, by the layer's definition
    q = {k: d64(v) for k, v in p.items()}
    how = ("e4m3", "floor")
    p1 = R.rows(d64(h), *how) @ R.rows(q["w1"], *how).T + q["b1"]
    near(a, act64(p1, "gelu")[0], 2.0 ** -14)
    near(y, R.rows(d64(a), *how) @ R.rows(q["w2"], *how).T + q["b2"] + d64(x), 2.0 ** -14)
    near(da, R.rows(d64(dy), *how) @ R.columns(q["w2"], *how).T, 2.0 ** -14)
    near(hand["w2"], R.columns(d64(dy), *how) @ R.columns(d64(a), *how).T, 2.0 ** -14)
    d = d64(da) * act64(R.bf16(p1), "gelu")[1]
    near(dh, R.rows(d, *how) @ R.columns(q["w1"], *how).T, FLIPS + 2.0 ** -14)
    near(hand["w1"], R.columns(d, *how) @ R.columns(d64(h), *how).T, FLIPS + 2.0 ** -14)
    # ... and the norm's against autograd in 64 bits
    leaves = [t.detach().cpu().double().requires_grad_() for t in (x, p["ln_w"], p["ln_b"])]
    n = torch.nn.functional.layer_norm(leaves[0], (H,), leaves[1], leaves[2], 1e-5)
    near(h, n.detach(), 2.0 ** -18)
    for g, t in zip((dx, hand["ln_w"], hand["ln_b"]), torch.autograd.grad(n, leaves, d64(dh))):
        near(g, t, 2.0 ** -16)


def test_beside_a_gated_block(ct, dev):
    """A norm in front of the gated feed-forward block, a linear layer behind it: gradients through all three."""
    T, H, F = 90, 256, 512
    x, dy = rows(dev, T, H, 3, bf16)
    p = parameters(dev, H, F, 4, bf16)
    g = torch.Generator().manual_seed(5)
    gate_up = (torch.randn((2 * F, H), generator=g) * H ** -0.5).to(bf16).to(dev)
    leaves = [t.requires_grad_() for t in (x, p["ln_w"], p["ln_b"], gate_up, p["w2"])]
    out = (torch.randn((H, H), generator=g) * H ** -0.5).to(bf16).to(dev).requires_grad_()
    y = ct.linear(ct.gated_feed_forward(ct.layer_norm(x, p["ln_w"], p["ln_b"]), gate_up, p["w2"]), out, None, x)
    got = torch.autograd.grad(y, (*leaves, out), dy)
    with torch.no_grad():
        h, mean, rstd = ct.layer_norm_forward(x, p["ln_w"], p["ln_b"])
        f, s = ct.gated_feed_forward_forward(h, gate_up, p["w2"])
        y2, s2 = ct.linear_forward(f, out, None, x)
        df, dout, none = ct.linear_backward(dy, s2)
        dh, dgu, dw2 = ct.gated_feed_forward_backward(df, s)
        dx, dlw, dlb = ct.layer_norm_backward(dh, x, mean, rstd, p["ln_w"])
    assert none is None and torch.equal(y, y2)
    for a, b in zip(got[1:], (dlw, dlb, dgu, dw2, dout)):
        assert torch.equal(a, b)
    assert torch.equal(got[0], dx + dy) or torch.equal(got[0], dy + dx)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("sizes", [((60, 256, 512),), ((700, 256, 1024), (33, 128, 256))])
def test_steps_in_graphs(ct, dev, sizes, bits):
    """Forward and backward passes and the optimizer's step in one graph (two graphs in turn), against the same steps eagerly."""
    def setup():
        out = []
        for k, (T, H, F) in enumerate(sizes):
            masters = parameters(dev, H, F, 10 + k)
            copies = {n: t.to(bf16) for n, t in masters.items()}
            x, dy = rows(dev, T, H, 20 + k, bf16)
            states = [ct.adamw_state(t, bits) for t in masters.values()]
            step, lr = torch.zeros(1, dtype=torch.int64, device=dev), torch.full((1,), 1e-3, device=dev)
            out.append((masters, copies, x, dy, states, step, lr))
        return out

    def step(s):
        masters, copies, x, dy, states, count, lr = s
        count.add_(1)
        _, g = by_hand(ct, x, dy, copies)
        ct.adamw_step(list(masters.values()), [g[n] for n in masters], states, step=count, lr=lr, weight_decay=0.1, seed=3, copies=list(copies.values()))

    eager, held = setup(), setup()
    graphs = []
    for s in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(s)
        graphs.append(g)
    for turn in range(4):
        for k, (s, e) in enumerate(zip(held, eager)):
            x, dy = rows(dev, *s[2].shape, 100 * turn + k, bf16)
            for t in (s, e):
                t[2].copy_(x)
                t[3].copy_(dy)
                t[6].fill_(1e-3 / (turn + 1))
            graphs[k].replay()
            step(e)
        torch.cuda.synchronize()
        for s, e in zip(held, eager):
            assert int(s[5]) == turn + 1
            for a, b in zip((*s[0].values(), *s[1].values()), (*e[0].values(), *e[1].values())):
                assert torch.equal(a, b) and bool(a.isfinite().all())
            for a, b in zip(s[4], e[4]):
                assert all(torch.equal(u8(p), u8(q)) for p, q in zip(a, b) if p is not None)
            assert all(torch.equal(c, m.to(bf16)) for c, m in zip(s[1].values(), s[0].values()))


@pytest.mark.parametrize("wf", ["e4m3", "e2m1"])
@pytest.mark.parametrize("T,H,F", [(1, 256, 1024), (20, 512, 2048), (130, 256, 1056), (1531, 512, 1056)])
def test_a_block_served(ct, dev, T, H, F, wf):
    """The norm's codes into the up projection, whose codes go into the down projection, with the residual stream."""
    p = parameters(dev, H, F, 30)
    x, _ = rows(dev, T, H, 31, bf16)
    fmt = {"e4m3": O.E4M3, "e2m1": O.E2M1}[wf]
    q = {k: ct.block_quantize(p[k], 32, dtype=torch.float8_e4m3fn if wf == "e4m3" else "e2m1", scale_mode="floor") for k in ("w1", "w2")}
    h, hs = ct.layer_norm_quantize(x, p["ln_w"], p["ln_b"])
    a, as_ = ct.block_scaled_linear(h, hs, *q["w1"], p["b1"], activation="gelu", w_format=wf, out_dtype=torch.float8_e4m3fn)
    y = ct.block_scaled_linear(a, as_, *q["w2"], p["b2"], x, w_format=wf)
    def de(c, s, f):
        c = u8(c).cpu().numpy()
        return O.dequantize(O.unpack_fp4(c) if f == O.E2M1 else c, u8(s).cpu().numpy(), f).double()

    W1, W2 = (de(*q[k], fmt) for k in ("w1", "w2"))
    Hq, Aq = de(h, hs, O.E4M3), de(a, as_, O.E4M3)
    # within the bounds of each operator's own tests, from the codes in front of it
    p1 = Hq @ W1.T + d64(p["b1"])
    want = act64(p1, "gelu")[0]
    check_codes(a, as_, want, 1.13 * (2 * sum_error(Hq, W1) + 2.0 ** -23 * p1.abs()) + 2.1e-6 * want.abs())
    want = Aq @ W2.T + d64(p["b2"]) + d64(x)
    err = 2 * sum_error(Aq, W2) + 2.0 ** -22 * (want.abs() + d64(x).abs() + d64(p["b2"]).abs())
    assert bool(((d64(y) - want).abs() <= err + R.HALF_BF16 * (want.abs() + err)).all())
    # the norm against block_quantize of the 64-bit norm: off where a number lies at a border alone
    n = torch.nn.functional.layer_norm(d64(x), (H,), d64(p["ln_w"]), d64(p["ln_b"]), 1e-5)
    assert R.rel(Hq, R.rows(n, "e4m3", "floor")) <= 2.0 ** -10
