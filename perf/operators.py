"""Measured calls of the gated feed-forward block that is trained in 8 bits, and of its parts.

A case is a dict of plain values; ``kind`` names the operator:

  both      ``block_quantize_both``: MX codes of a matrix along its rows and, transposed, along its columns
  gated     ``gated_block_scaled_matmul``: both projections, SiLU and the product with quantised operands
  backward  ``silu_and_mul_backward_quantize``: the activation's backward pass from an 8-bit checkpoint
  train     ``gated_feed_forward``: forward and backward of the whole block, from bf16 input and weights

Sizes are those of the benchmark and the tests (layers of 4096 x 14336 and 2048 x 7168, 8192 rows) and generic ones
around them.  In the formulas below ``Q`` is MX quantisation: blocks of 32 values share a power of two.
"""
import math
import pathlib
import sys

import torch

own = False

EMAX = {"e4m3": 8, "e5m2": 15}
LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
ELEM = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
SRC = {"bf16": torch.bfloat16, "f32": torch.float32, "f16": torch.float16}


def listed():
    return [
        # a short ragged batch of fp32 activations, checkpointed
        {"name": "both_333x4096_f32", "kind": "both", "rows": 333, "K": 4096, "src": "f32", "fmt": "e4m3", "mode": "floor"},
        # activations of a full prompt batch, or a square weight
        {"name": "both_8192_bf16", "kind": "both", "rows": 8192, "K": 8192, "src": "bf16", "fmt": "e4m3", "mode": "floor"},
        # gradients of an odd number of tokens in the wide-range format
        {"name": "both_1531x14336_e5m2", "kind": "both", "rows": 1531, "K": 14336, "src": "bf16", "fmt": "e5m2", "mode": "ceil"},
        # one token being decoded: the smallest call, latency counts
        {"name": "gated_m1_fp8", "kind": "gated", "M": 1, "K": 2048, "F": 7168, "w": "e4m3", "out": "bf16"},
        # a batch of 32 sequences being decoded, FP4 weights
        {"name": "gated_m32_fp4", "kind": "gated", "M": 32, "K": 8192, "F": 14336, "w": "e2m1", "out": "e4m3"},
        # a prompt of ragged length
        {"name": "gated_m1531_fp8", "kind": "gated", "M": 1531, "K": 4096, "F": 14336, "w": "e4m3", "out": "e4m3"},
        # a full prompt batch
        {"name": "gated_m8192_fp8", "kind": "gated", "M": 8192, "K": 4096, "F": 14336, "w": "e4m3", "out": "bf16"},
        # activation gradients of few tokens, ragged
        {"name": "backward_77x1408", "kind": "backward", "M": 77, "F": 1408},
        # activation gradients of a full batch
        {"name": "backward_4096x14336", "kind": "backward", "M": 4096, "F": 14336},
        # a training step of a small block on one token: launches and host work
        {"name": "train_1x1024x2048", "kind": "train", "T": 1, "H": 1024, "F": 2048},
        # a ragged micro-batch
        {"name": "train_1531x2048x7168", "kind": "train", "T": 1531, "H": 2048, "F": 7168},
        # the largest: a full batch through the large block
        {"name": "train_4096x4096x14336", "kind": "train", "T": 4096, "H": 4096, "F": 14336},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _log_mult(rng, lo, hi, m):
    return max(lo, _log(rng, lo, hi) // m * m)


def draw(rng):
    kind = rng.choice(["both", "gated", "gated", "backward", "train"])
    if kind == "both":
        return {"kind": kind, "rows": _log(rng, 1, 8192), "K": _log_mult(rng, 128, 14336, 32),
                "src": rng.choice(["bf16", "bf16", "f32", "f16"]), "fmt": rng.choice(["e4m3", "e4m3", "e5m2"]),
                "mode": rng.choice(["floor", "ceil"])}
    if kind == "gated":
        return {"kind": kind, "M": _log(rng, 1, 8192), "K": _log_mult(rng, 512, 4096, rng.choice([32, 128, 512])),
                "F": _log_mult(rng, 512, 14336, rng.choice([32, 64, 256])), "w": rng.choice(["e4m3", "e2m1"]),
                "out": rng.choice(["bf16", "e4m3"])}
    if kind == "backward":
        return {"kind": kind, "M": _log(rng, 1, 4096), "F": _log_mult(rng, 256, 14336, 32)}
    return {"kind": kind, "T": _log(rng, 1, 4096), "H": _log_mult(rng, 256, 4096, rng.choice([32, 128])),
            "F": _log_mult(rng, 512, 14336, rng.choice([32, 256]))}


class _Maker:
    """Random operands on the GPU, from the seed alone."""

    def __init__(self, seed):
        self.dev = torch.device("cuda:0")
        self.g = torch.Generator(device=self.dev).manual_seed(seed)

    def normal(self, shape, std=1.0, dtype=torch.float32):
        return torch.empty(shape, device=self.dev, dtype=dtype).normal_(0.0, std, generator=self.g)

    def codes(self, rows, K, fmt, exponent):
        """Elements and scales of a matrix that was quantised before: blocks whose largest value is near the format's,
        scales around 2^exponent."""
        scale = torch.randint(exponent + 126, exponent + 129, (rows, K // 32), generator=self.g, device=self.dev,
                              dtype=torch.uint8)
        if fmt == "e2m1":
            q = torch.randint(0, 256, (rows, K // 2), generator=self.g, device=self.dev, dtype=torch.uint8)
        else:
            q = self.normal((rows, K), 128.0).clamp(-448.0, 448.0).to(ELEM[fmt])
        return q, scale.view(torch.float8_e8m0fnu)


def prepare(case, seed):
    m = _Maker(seed)
    kind = case["kind"]
    s = {"case": dict(case)}
    if kind == "both":
        s["x"] = m.normal((case["rows"], case["K"]), 1.0, SRC[case["src"]])
    elif kind == "gated":
        s["a"], s["as"] = m.codes(case["M"], case["K"], "e4m3", -7)
        # weights around 1 / sqrt(K), so that gate and up are around one
        e = -7 - round(math.log2(case["K"]) / 2) if case["w"] == "e4m3" else -1 - round(math.log2(case["K"]) / 2)
        s["w"], s["ws"] = m.codes(2 * case["F"], case["K"], case["w"], e)
        s["e2m1"] = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=m.dev)
    elif kind == "backward":
        s["dh"] = m.normal((case["M"], case["F"]), 1e-3, torch.bfloat16)
        s["gu"], s["gus"] = m.codes(case["M"], 2 * case["F"], "e4m3", -7)
    else:
        T, H, F = case["T"], case["H"], case["F"]
        s["x"] = m.normal((T, H), 1.0, torch.bfloat16).requires_grad_()
        s["w1"] = m.normal((2 * F, H), 1.0 / math.sqrt(H), torch.bfloat16).requires_grad_()
        s["w2"] = m.normal((H, F), 1.0 / math.sqrt(F), torch.bfloat16).requires_grad_()
        s["dy"] = m.normal((T, H), 1e-3, torch.bfloat16)
    return s


def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    import cutile_amd as ct

    case = s["case"]
    if case["kind"] == "both":
        return ct.block_quantize_both(s["x"], ELEM[case["fmt"]], scale_mode=case["mode"])
    if case["kind"] == "gated":
        return ct.gated_block_scaled_matmul(s["a"], s["as"], s["w"], s["ws"], w_format=case["w"],
                                            out_dtype=torch.bfloat16 if case["out"] == "bf16" else torch.float8_e4m3fn)
    if case["kind"] == "backward":
        return ct.silu_and_mul_backward_quantize(s["dh"], s["gu"], s["gus"])
    y = ct.gated_feed_forward(s["x"], s["w1"], s["w2"])
    return (y, *torch.autograd.grad(y, (s["x"], s["w1"], s["w2"]), s["dy"]))


_PACKAGE = str(pathlib.Path(__file__).resolve().parent.parent / "cutile-python_amd")


# ---- the operators in elementary operations, 32 bits ------------------------------------------------------------------
def _power(e):
    """2^e for whole numbers e from -126 to 127, by its bits."""
    return ((e + 127) << 23).int().view(torch.float32)


def _quantize(x, fmt="e4m3", mode="floor"):
    """Q along the last axis (a multiple of 32): elements (8-bit floats) and scales (E8M0)."""
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    amax = b.abs().amax(-1)
    if mode == "floor":      # 2^(floor(log2 amax) - emax)
        e = torch.frexp(amax)[1] - 1 - EMAX[fmt]
    else:                    # 2^ceil(log2(amax / 448))
        f, e = torch.frexp((amax / 448.0).clamp(min=1e-12))
        e = torch.where(f == 0.5, e - 1, e)
    e = torch.where((amax == 0) & (mode == "floor"), -127, e).clamp(-127, 127)
    half = -e // 2           # 2^127 and 2^-127 in two steps
    v = b * _power(half).unsqueeze(-1) * _power(-e - half).unsqueeze(-1)
    q = v.clamp(-LARGEST[fmt], LARGEST[fmt]).to(ELEM[fmt]).reshape(x.shape)
    return q, (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _quantize_columns(x, fmt="e4m3", mode="floor"):
    """Q of x^T along the rows of x, which are padded with zeros to a multiple of 32."""
    return _quantize(torch.nn.functional.pad(x, (0, 0, 0, -x.shape[0] % 32)).T.contiguous(), fmt, mode)


def _value(q, scale):
    return (q.float().reshape(*scale.shape, 32) * scale.float().unsqueeze(-1)).reshape(q.shape)


def _row(x):
    return _value(*_quantize(x))


def _col(x):
    """What Q along the columns leaves of x, transposed."""
    return _value(*_quantize_columns(x))


def _weight(q, scale, fmt, table):
    if fmt != "e2m1":
        return _value(q, scale)
    v = torch.stack((table[(q & 15).int()], table[(q >> 4).int()]), -1)
    return _value(v.reshape(q.shape[0], -1), scale)


def _gate_up(a, w):
    """Both projections, in the precision of the activation between them."""
    return (a @ w.T).bfloat16().float().chunk(2, dim=1)


def _silu_backward(dh, g, u):
    s = 1.0 / (1.0 + torch.exp(-g))
    return torch.cat((dh * u * s * (1.0 + g * (1.0 - s)), dh * g * s), 1), g * s * u


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "both":
        x = s["x"].float()
        return (*_quantize(x, case["fmt"], case["mode"]), *_quantize_columns(x, case["fmt"], case["mode"]))
    if kind == "gated":
        g, u = _gate_up(_value(s["a"], s["as"]), _weight(s["w"], s["ws"], case["w"], s["e2m1"]))
        h = g / (1.0 + torch.exp(-g)) * u
        return h.bfloat16() if case["out"] == "bf16" else _quantize(h)
    if kind == "backward":
        d, a = _silu_backward(s["dh"].float(), *_value(s["gu"], s["gus"]).chunk(2, dim=1))
        return (*_quantize(d), *_quantize_columns(d), *_quantize_columns(a))
    with torch.no_grad():
        x, w1, w2, dy = (s[n].float() for n in ("x", "w1", "w2", "dy"))
        g, u = _gate_up(_row(x), _row(w1))
        y = _row(g / (1.0 + torch.exp(-g)) * u) @ _row(w2).T
        dh = (_row(dy) @ _col(w2).T).bfloat16().float()
        d, a = _silu_backward(dh, _row(g), _row(u))
        out = (y, _row(d) @ _col(w1).T, _col(d) @ _col(x).T, _col(dy) @ _col(a).T)
        return tuple(t.bfloat16() for t in out)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------
def work(case):
    mx = 1 + 1 / 32
    kind = case["kind"]
    if kind == "both":
        n, padded = case["rows"] * case["K"], -(-case["rows"] // 32) * 32 * case["K"]
        return {"bytes": n * (4 if case["src"] == "f32" else 2) + (n + padded) * mx, "flops": 4 * n}
    if kind == "gated":
        M, K, F = case["M"], case["K"], case["F"]
        w = (0.5 if case["w"] == "e2m1" else 1) + 1 / 32
        return {"bytes": M * K * mx + 2 * F * K * w + M * F * (2 if case["out"] == "bf16" else mx), "flops": 4 * M * F * K}
    if kind == "backward":
        M, F, P = case["M"], case["F"], -(-case["M"] // 32) * 32
        return {"bytes": M * F * (2 + 2 * mx + 2 * mx) + 3 * P * F * mx, "flops": 16 * M * F}
    T, H, F = case["T"], case["H"], case["F"]
    # x, dy, y, dx; both weights and their gradients, 16 bits each
    return {"bytes": 8 * T * H + 4 * 3 * H * F, "flops": 18 * T * H * F}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------------
def _two_to(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _round_to(v, bits, least):
    """v to the nearest number of `bits` significant binary digits whose last one is worth 2^least or more, ties to even."""
    step = _two_to(torch.clamp(torch.frexp(v)[1] - bits, min=least))
    return torch.round(v / step) * step


def _q64(x, fmt="e4m3", mode="floor"):
    """Element values and scales of Q along the last axis."""
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    top = torch.amax(torch.abs(b), -1)
    if mode == "floor":
        e = torch.where(top > 0, torch.frexp(top)[1] - 1.0 - EMAX[fmt], torch.full_like(top, -127.0))
    else:
        f, k = torch.frexp(torch.clamp((top / 448.0).float(), min=1e-12).double())
        e = k - (f == 0.5).double()
    scale = _two_to(torch.clamp(e, -127.0, 127.0))
    v = torch.clamp(b / scale[..., None], -LARGEST[fmt], LARGEST[fmt])
    v = _round_to(v, 4, -9) if fmt == "e4m3" else _round_to(v, 3, -16)
    return v.reshape(x.shape), scale


def _q64_columns(x, *how):
    rows = -(-x.shape[0] // 32) * 32
    t = torch.zeros((x.shape[1], rows), dtype=torch.float64, device=x.device)
    t[:, :x.shape[0]] = x.T
    return _q64(t, *how)


def _r64(x):
    v, scale = _q64(x)
    return v * scale.repeat_interleave(32, -1)


def _c64(x):
    v, scale = _q64_columns(x)
    return v * scale.repeat_interleave(32, -1)


def _half64(x):
    """The nearest bf16 numbers."""
    return _round_to(x, 8, -133)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "both":
        x = s["x"].double()
        return (*_q64(x, case["fmt"], case["mode"]), *_q64_columns(x, case["fmt"], case["mode"]))
    if kind == "gated":
        a = s["a"].double() * s["as"].double().repeat_interleave(32, -1)
        w = s["w"]
        if case["w"] == "e2m1":
            code = torch.stack((w % 16, w // 16), 2).reshape(w.shape[0], -1).long()
            e, m = (code // 2) % 4, code % 2
            v = torch.where(e == 0, m * 0.5, (1 + m * 0.5) * _two_to(e - 1))
            w = torch.where(code >= 8, -v, v)
        gu = _half64(a @ (w.double() * s["ws"].double().repeat_interleave(32, -1)).T)
        g, u = gu[:, :case["F"]], gu[:, case["F"]:]
        h = g * torch.sigmoid(g) * u
        return h if case["out"] == "bf16" else _q64(h)
    if kind == "backward":
        gu = s["gu"].double() * s["gus"].double().repeat_interleave(32, -1)
        g, u, dh = gu[:, :case["F"]], gu[:, case["F"]:], s["dh"].double()
        s = torch.sigmoid(g)
        d = torch.hstack((dh * u * (s + g * s * torch.sigmoid(-g)), dh * g * s))
        return (*_q64(d), *_q64_columns(d), *_q64_columns(u * g * s))
    with torch.no_grad():
        x, w1, w2, dy = (s[n].double() for n in ("x", "w1", "w2", "dy"))
        F = case["F"]
        gu = _half64(_r64(x) @ _r64(w1).T)
        h = gu[:, :F] * torch.sigmoid(gu[:, :F]) * gu[:, F:]
        y = _r64(h) @ _r64(w2).T
        dh = _half64(_r64(dy) @ _c64(w2).T)
        gu = _r64(gu)
        g, u, p = gu[:, :F], gu[:, F:], torch.sigmoid(gu[:, :F])
        d = torch.hstack((dh * u * (p + g * p * torch.sigmoid(-g)), dh * g * p))
        return y, _r64(d) @ _c64(w1).T, _c64(d) @ _c64(x).T, _c64(dy) @ _c64(u * g * p).T
