"""AdamW over many tensors against the formula in 64 bits; states in 8 bits element by element, their random rounding by its chances."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

bf16, f32 = torch.bfloat16, torch.float32
HALF = {f32: 2.0 ** -24, bf16: 2.0 ** -8}
SIZES = [1, 2, 7, 31, 32, 33, 255, 1000, 4095, 4096, 4097, 12289, 0, 65]
HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1)


def tensors(dev, sizes, ptype, gtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    p = [torch.randn(n, generator=g).to(ptype).to(dev) for n in sizes]
    d = [(torch.randn(n, generator=g) * 10 ** float(torch.randn((), generator=g))).to(gtype).to(dev) for n in sizes]
    return p, d


def step64(p, g, m, v, step, lr, betas, eps, weight_decay, scale=1.0):
    b1, b2 = betas
    g = g * scale
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    return p * (1 - lr * weight_decay) - lr / (1 - b1 ** step) * m / (torch.sqrt(v / (1 - b2 ** step)) + eps), m, v


def d64(t):
    return t.detach().cpu().double()


def near(got, want, size, dtype=f32):
    """Within some operations of 2^-24 each of the terms' size, and one rounding to the type."""
    got = d64(got)
    bad = ~((got - want).abs() <= 2.0 ** -20 * size + HALF[dtype] * (want.abs() + 2.0 ** -20 * size))
    assert not bool(bad.any()), (float((got - want).abs().max()), int(bad.sum()))


@pytest.mark.parametrize("ptype,gtype", [(f32, f32), (f32, bf16), (bf16, bf16), (bf16, f32)], ids=str)
def test_states_in_32_bits(ct, dev, ptype, gtype):
    params, _ = tensors(dev, SIZES, ptype, gtype)
    states = [ct.adamw_state(p) for p in params]
    copies = [torch.zeros_like(p, dtype=bf16) if i % 2 else None for i, p in enumerate(params)]
    for step in (1, 2, 3):
        _, grads = tensors(dev, SIZES, ptype, gtype, step)
        before = [[d64(t) for t in (p, s.exp_avg, s.exp_avg_sq)] for p, s in zip(params, states)]
        ct.adamw_step(params, grads, states, step=step, copies=copies, **HYPER)
        for p, g, s, c, (p0, m0, v0) in zip(params, grads, states, copies, before):
            want, m, v = step64(p0, d64(g), m0, v0, step, **HYPER)
            near(s.exp_avg, m, 0.9 * m0.abs() + 0.1 * d64(g).abs())
            near(s.exp_avg_sq, v, v)
            update = HYPER["lr"] * (0.9 * m0.abs() + d64(g).abs()) / (1 - 0.9 ** step) / (torch.sqrt(v / (1 - 0.99 ** step)) + HYPER["eps"])
            near(p, want, p0.abs() + update, ptype)
            if c is not None:
                near(c, want, p0.abs() + update, bf16)


def test_many_tensors_of_mixed_types(ct, dev):
    """More than a launch holds, in an order that mixes the types; some without a gradient."""
    sizes = [(37 * i * i) % 5000 + 1 for i in range(150)]
    params, grads, states = [], [], []
    for i, n in enumerate(sizes):
        p, g = tensors(dev, [n], (f32, bf16)[i % 2], (f32, bf16)[i // 2 % 2], i)
        params += p
        grads += g if i % 11 else [None]
        states.append(ct.adamw_state(p[0]))
    before = [d64(p) for p in params]
    ct.adamw_step(tuple(params), tuple(grads), tuple(states), step=1, **HYPER)
    for p, g, s, p0 in zip(params, grads, states, before):
        if g is None:
            assert torch.equal(d64(p), p0) and bool((s.exp_avg == 0).all())
            continue
        want, m, v = step64(p0, d64(g), torch.zeros_like(p0), torch.zeros_like(p0), 1, **HYPER)
        near(s.exp_avg, m, d64(g).abs())
        near(p, want, p0.abs() + HYPER["lr"] * 2, p.dtype)


def test_views_off_alignment_and_gradients_of_other_strides(ct, dev):
    base = torch.randn(10007, generator=torch.Generator().manual_seed(1)).to(dev)
    for ptype in (f32, bf16):
        whole = base.to(ptype)
        p = whole[3:9004]
        g = torch.randn((9001, 2), generator=torch.Generator().manual_seed(2)).to(ptype).to(dev)[:, 1]
        s, p0, edge = ct.adamw_state(p), d64(p), (d64(whole[:3]), d64(whole[9004:]))
        ct.adamw_step([p], [g], [s], step=1, **HYPER)
        want, _, _ = step64(p0, d64(g), torch.zeros_like(p0), torch.zeros_like(p0), 1, **HYPER)
        near(p, want, p0.abs() + HYPER["lr"] * 2, ptype)
        assert torch.equal(d64(whole[:3]), edge[0]) and torch.equal(d64(whole[9004:]), edge[1])


def test_gradient_scale_zero_rate_and_tensors_in_the_place_of_numbers(ct, dev):
    (p,), (g,) = tensors(dev, [5000], f32, f32, 3)
    one = lambda v, t=f32: torch.tensor(v, dtype=t, device=dev)  # noqa: E731
    results = []
    for kw in (dict(step=7, lr=3e-3, grad_scale=0.25), dict(step=one(7, torch.int64), lr=one(3e-3), grad_scale=one(0.25)),
               dict(step=one([7], torch.int64), lr=3e-3, grad_scale=one([0.25])), dict(step=7, lr=one(3e-3), grad_scale=0.25)):
        q, s = p.clone(), ct.adamw_state(p)
        ct.adamw_step([q], [g], [s], betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1, **kw)
        results.append((q, s))
    want, m, v = step64(d64(p), d64(g), 0 * d64(p), 0 * d64(p), 7, 3e-3, (0.9, 0.999), 1e-8, 0.1, 0.25)
    for q, s in results:
        near(s.exp_avg, m, m.abs())
        near(q, want, d64(p).abs() + 3e-3 * 10)
    q, s = p.clone(), ct.adamw_state(p)
    ct.adamw_step([q], [g], [s], step=1, lr=0.0)
    assert torch.equal(q, p) and not bool((s.exp_avg == 0).all())


# ---- states in 8 bits ----------------------------------------------------------------------------------------------------------
M32 = 0xFFFFFFFF


def mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x9E3779B1) & M32
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & M32
    return x ^ (x >> 16)


def words(n, seed, step, index):
    key = mix(torch.tensor(seed & M32)) ^ (step & M32)
    key = mix(mix(mix(key) ^ index) ^ 0)
    return mix((key + torch.arange(n)) & M32)


def pad(x):
    return torch.nn.functional.pad(x, (0, -x.numel() % 32))


def store64(x, chance, root):
    b = pad(x).view(-1, 32)
    top = b.abs().amax(-1)
    f, e = torch.frexp(top)
    scale = torch.ldexp(torch.ones_like(top), torch.where(top > 0, e - 9 + (f > 0.875), -127).clamp(-127, 127))
    v = b.abs() / scale[:, None]
    step = torch.ldexp(torch.ones_like(v), (torch.frexp(v)[1] - 4).clamp(min=-9))
    place = v / step + pad(chance).view(-1, 32) / 65536
    q = (torch.floor(place) * step).clamp(max=448)
    if root:
        q = torch.where(b > 0, q.clamp(min=2.0 ** -9), q)
    return (torch.sign(b) * q).view(-1), scale, ((place - place.round()).abs() < 1e-4).view(-1)


def value(q, s):
    return d64(q.float()) * d64(s.float()).repeat_interleave(32)


@pytest.mark.parametrize("ptype,gtype", [(f32, f32), (bf16, bf16), (f32, bf16)], ids=str)
def test_states_in_8_bits(ct, dev, ptype, gtype):
    params, _ = tensors(dev, SIZES, ptype, gtype)
    states = [ct.adamw_state(p, 8) for p in params]
    for step in (1, 2, 1000):
        _, grads = tensors(dev, SIZES, ptype, gtype, step)
        before = [(d64(p), value(s.exp_avg, s.exp_avg_scale)[:p.numel()], value(s.exp_avg_sq, s.exp_avg_sq_scale)[:p.numel()]) for p, s in zip(params, states)]
        ct.adamw_step(params, grads, states, step=step, seed=77, **HYPER)
        for i, (p, g, s, (p0, m0, r0)) in enumerate(zip(params, grads, states, before)):
            if p.numel() == 0:
                continue
            want, m, v = step64(p0, d64(g), m0, r0 * r0, step, **HYPER)
            update = HYPER["lr"] * (0.9 * m0.abs() + d64(g).abs()) / (1 - 0.9 ** step) / (torch.sqrt(v / (1 - 0.99 ** step)) + HYPER["eps"])
            near(p, want, p0.abs() + update, ptype)
            w = words(p.numel(), 77, step, i)
            for got, scale, x, chance, root in ((s.exp_avg, s.exp_avg_scale, m, w & 0xFFFF, False), (s.exp_avg_sq, s.exp_avg_sq_scale, v.sqrt(), w >> 16, True)):
                q, sc, close = store64(x, chance, root)
                border = sc != store64(x * (1 - 1e-6), chance, root)[1]   # the scale may be the neighbour's
                border |= sc != store64(x * (1 + 1e-6), chance, root)[1]
                assert bool(((d64(scale.float()) == sc) | border).all())
                same = d64(got.float()) == q
                assert bool((same | close | border.repeat_interleave(32)).all()), (i, int((~same).sum()))
                assert bool((d64(got.float())[p.numel():] == 0).all())
                # few are that close to a border: 2e-4 of the places outside of border blocks.  (Whole blocks may have the neighbour's scale: 0.1
                # times a bf16 number is a border between two scales but for a rounding now and then, and a block is 1 / 8 of 255 elements.)
                assert int((~same & ~border.repeat_interleave(32)).sum()) <= 3 + 1e-3 * p.numel()


def test_random_rounding_has_the_right_mean(ct, dev):
    """Over seeds the mean of a stored root is the root: 512 draws, each off by less than a step (2^-3 of the value at most), so that
    the mean of 8192 elements' relative error has a deviation below 2^-3 / 2 / sqrt(512 * 8192)."""
    n, draws = 8192, 512
    g = (1 + torch.rand(n, generator=torch.Generator().manual_seed(5))).to(dev)
    total = torch.zeros(n, dtype=torch.float64)
    roots = torch.zeros(n, dtype=torch.float64)
    for seed in range(draws):
        s = ct.adamw_state(g, 8)
        ct.adamw_step([torch.zeros_like(g)], [g], [s], step=1, seed=seed, betas=(0.9, 0.99), weight_decay=0.0)
        total += value(s.exp_avg, s.exp_avg_scale)
        roots += value(s.exp_avg_sq, s.exp_avg_sq_scale)
    g = d64(g)
    for mean, want in ((total / draws, 0.1 * g), (roots / draws, 0.1 * g)):
        off = mean / want - 1
        assert abs(float(off.mean())) < 6 * 2.0 ** -4 / math.sqrt(draws * n) + 2.0 ** -17
        assert float(off.abs().max()) < 6 * 2.0 ** -4 / math.sqrt(draws) + 2.0 ** -16


def test_second_moment_moves(ct, dev):
    """A root ten times too small or too large comes to the gradients' size within some multiples of 1 / (1 - b2) steps."""
    n = 4096
    for factor in (0.1, 10.0):
        g = torch.full((n,), 1e-3, device=dev)
        p, s = torch.zeros(n, device=dev), ct.adamw_state(g, 8)
        ct.adamw_step([p], [g * factor * 10], [s], step=1, betas=(0.9, 0.99), lr=0.0)     # root: 0.1 * 10 * factor of it
        for step in range(2, 802):
            ct.adamw_step([p], [g], [s], step=step, betas=(0.9, 0.99), lr=0.0, seed=9)
        r = value(s.exp_avg_sq, s.exp_avg_sq_scale)
        assert 0.9 < float(r.mean()) / 1e-3 < 1.1


def test_root_above_zero_is_never_stored_as_zero(ct, dev):
    g = torch.full((64,), 1e-6, device=dev)
    g[0] = g[32] = 1e4
    s = ct.adamw_state(g, 8)
    for seed in range(20):
        ct.adamw_step([torch.zeros_like(g)], [g], [s], step=1, seed=seed)
        assert bool((s.exp_avg_sq.float() > 0).all())


def test_not_finite(ct, dev):
    for bits in (32, 8):
        p, g = torch.ones(96, device=dev), torch.full((96,), 0.5, device=dev)
        g[40], g[70] = float("nan"), float("inf")
        s = ct.adamw_state(p, bits)
        ct.adamw_step([p], [g], [s], step=1)
        bad = p.isnan().cpu()
        assert bool(bad[40]) and not bool(bad[:32].any()) and bool((p[:32] == p[0]).all())
        assert int(bad.sum()) <= 2                          # (inf / sqrt(inf) of the other one)
        m = s.exp_avg.float().cpu()
        assert bool(m[40].isnan()) and not bool(m[:32].isnan().any())


def test_same_arguments_same_bits(ct, dev):
    runs = []
    for _ in range(2):
        params, grads = tensors(dev, [5000, 333, 70000], bf16, bf16, 6)
        states = [ct.adamw_state(p, 8) for p in params]
        for step in (1, 2):
            ct.adamw_step(params, grads, states, step=step, seed=3)
        runs.append([t.view(torch.uint8) for s in states for t in s] + params)
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_captured_steps_go_on_counting(ct, dev):
    params, grads = tensors(dev, [3000, 50], f32, f32, 7)
    twin = [p.clone() for p in params]
    states, twins = ([ct.adamw_state(p, 8) for p in params] for _ in range(2))
    count, lr = torch.zeros((), dtype=torch.int64, device=dev), torch.tensor(1e-2, device=dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        count.add_(1)
        ct.adamw_step(params, grads, states, step=count, lr=lr, seed=4)
    for step in (1, 2, 3, 4):
        lr.fill_(1e-2 / step)
        graph.replay()
        torch.cuda.synchronize()
        ct.adamw_step(twin, grads, twins, step=count, lr=lr, seed=4)
        assert int(count) == step
        for a, b in zip(params + [t.view(torch.uint8) for s in states for t in s], twin + [t.view(torch.uint8) for s in twins for t in s]):
            assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ct.adamw_step(params, grads, states, step=5, seed=4)
    torch.cuda.current_stream().wait_stream(side)
    ct.adamw_step(twin, grads, twins, step=5, seed=4)
    assert all(torch.equal(a, b) for a, b in zip(params, twin))


def test_autograd_is_told(ct, dev):
    p = torch.randn(64, device=dev, requires_grad=True)
    y = (p * p).sum()
    ct.adamw_step([p], [torch.ones_like(p)], [ct.adamw_state(p)], step=1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_listed_twice(ct, dev):
    p = torch.zeros(64, device=dev)
    s, t = ct.adamw_state(p), ct.adamw_state(p)
    g = torch.ones_like(p)
    for params, states in (([p, p], [s, t]), ([p, p.clone()], [s, s]), ([p[:40], p[30:]], [ct.adamw_state(p[:40]), ct.adamw_state(p[30:])])):
        with pytest.raises(ValueError, match="overlap"):
            ct.adamw_step(params, [g[:q.numel()] for q in params], states, step=1)
    assert bool((p == 0).all())
    ct.adamw_step([p, p.clone()], [g, g], [s, t], step=1)   # one gradient for two is fine


def test_past_32_bits(ct, dev):
    n = (1 << 31) + 4097                                    # bf16: 4 GiB each of parameter and gradient, 8-bit states 4.3 GB
    p, g = torch.zeros(n, dtype=bf16, device=dev), torch.zeros(n, dtype=bf16, device=dev)
    g[-4200:] = 1.0
    g[:100] = -1.0
    s = ct.adamw_state(p, 8)
    ct.adamw_step([p], [g], [s], step=1, lr=0.5, weight_decay=0.0)
    assert bool((p[-4200:] == -0.5).all()) and bool((p[:100] == 0.5).all()) and bool((p[100:5000] == 0).all()) and bool((p[-10000:-4200] == 0).all())
    tail = s.exp_avg[-4200:].float() * s.exp_avg_scale.float().repeat_interleave(32)[-4200:]
    live = n % 32
    assert bool((tail[:-(32 - live)] > 0.09).all()) and bool((tail[-(32 - live):] == 0).all())
