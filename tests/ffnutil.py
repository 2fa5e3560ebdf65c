"""The gated feed-forward block in 64 bits, on the CPU: what the tests of its kernels compare with."""
from __future__ import annotations

import torch

EMAX = {"e4m3": 8, "e5m2": 15}
FMAX = {"e4m3": 448.0, "e5m2": 57344.0}
ELEM = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
# half a step relative to the value
HALF_E4M3, HALF_BF16 = 2.0 ** -4, 2.0 ** -8


def _grid(v, bits, least):
    """Nearest number of `bits` significant digits, the last worth at least 2^least; ties to even."""
    step = torch.ldexp(torch.ones_like(v), (torch.frexp(v)[1] - bits).clamp(min=least))
    return torch.round(v / step) * step


def quantize(x, fmt="e4m3", mode="floor"):
    """(element values, scales) of the MX quantisation of the last axis, a multiple of 32, of a float64 tensor."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    top = b.abs().amax(-1)
    if mode == "floor":
        e = torch.where(top > 0, torch.frexp(top)[1] - 1 - EMAX[fmt], -127)
    else:
        m, e = torch.frexp((top / 448.0).clamp(min=1e-12))
        e = torch.where(m == 0.5, e - 1, e)
    s = torch.ldexp(torch.ones_like(top), e.clamp(-127, 127))
    v = (b / s[..., None]).clamp(-FMAX[fmt], FMAX[fmt])
    return (_grid(v, 4, -9) if fmt == "e4m3" else _grid(v, 3, -16)).reshape(x.shape), s


def value(q, s):
    """Codes (or element values) and E8M0 scales -> float64."""
    s = s.cpu()
    if s.dtype != torch.float64:
        s = torch.ldexp(torch.ones(s.shape, dtype=torch.float64), s.view(torch.uint8).int() - 127)
    return q.cpu().double() * s.repeat_interleave(32, -1)


def rows(x, *how):
    return value(*quantize(x, *how))


def padded_t(x):
    """x^T with its last axis padded to a multiple of 32."""
    return torch.nn.functional.pad(x, (0, 0, 0, -x.shape[0] % 32)).T.contiguous()


def columns(x, *how):
    """x^T quantised along the rows of x."""
    return value(*quantize(padded_t(x), *how))


def bf16(x):
    return _grid(x, 8, -133)


def silu_mul(gu):
    g, u = gu.chunk(2, -1)
    return g * torch.sigmoid(g) * u


def silu_mul_backward(dh, gu):
    """(d[g|u], the activation)."""
    g, u = gu.chunk(2, -1)
    s = torch.sigmoid(g)
    return torch.cat((dh * u * s * (1 + g * (1 - s)), dh * g * s), -1), g * s * u


def block(x, w1, w2, dy, *how):
    """y, dx, dw1, dw2 of the block with every quantisation (`how`: format, rule) and bf16 rounding that belongs to its definition."""
    gu = bf16(rows(x, *how) @ rows(w1, *how).T)
    y = rows(silu_mul(gu), *how) @ rows(w2, *how).T
    dh = bf16(rows(dy, *how) @ columns(w2, *how).T)
    d, a = silu_mul_backward(dh, rows(gu, *how))
    return (y, rows(d, *how) @ columns(w1, *how).T, columns(d, *how) @ columns(x, *how).T,
            columns(dy, *how) @ columns(a, *how).T)


def block_unquantized(x, w1, w2):
    return silu_mul(x @ w1.T) @ w2.T


def rel(a, b):
    a, b = a.detach().cpu().double(), b.double()
    return float((a - b).norm() / b.norm().clamp(min=1e-300))
