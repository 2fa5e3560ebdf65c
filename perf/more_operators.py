"""Measured calls of what stands around a block-scaled product in a model: the norm in front of it, bias, activation and residual
behind it, and the optimizer's step on the gradients that come of it.

A case is a dict of plain values; ``kind`` names the operator:

  norm_quantize  ``layer_norm_quantize``: layer norm whose result leaves as MX elements, ready for a product (serving)
  norm           ``layer_norm``: forward and backward pass, with the gradients of weight and bias
  linear         ``block_scaled_linear``: act(A @ W.T + bias) + residual with block-scaled operands (serving)
  train          ``linear``: forward and backward pass of the same from bf16 input and weights, every product block-scaled
  adamw          ``adamw_step``: one step over many tensors, states in 32 or in 8 bits

Sizes are those of the benchmark and the tests (layers of 4096 x 14336 and 2048 x 7168, 8192 rows) and generic ones around
them.  In the formulas below ``Q`` is MX quantisation: blocks of 32 values share a power of two.
"""
import math
import pathlib
import random
import sys

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "f16": torch.float16}
EPS = 1e-5
LR, BETA1, BETA2, ADAM_EPS, DECAY, STEP, SEED = 1e-3, 0.9, 0.999, 1e-8, 0.01, 1000, 20251


def listed():
    return [
        # one token being decoded, in front of a projection: latency
        {"name": "norm_quantize_1x4096", "kind": "norm_quantize", "rows": 1, "H": 4096, "src": "bf16"},
        # a prompt of ragged length
        {"name": "norm_quantize_1531x8192", "kind": "norm_quantize", "rows": 1531, "H": 8192, "src": "bf16"},
        # a training step's norm over an odd width, fp32 activations
        {"name": "norm_777x2047_f32", "kind": "norm", "rows": 777, "H": 2047, "src": "f32", "par": "f32"},
        # a training step's norm over a full batch
        {"name": "norm_16384x4096_bf16", "kind": "norm", "rows": 16384, "H": 4096, "src": "bf16", "par": "bf16"},
        # one token through an up projection: the weights are read once, latency counts
        {"name": "linear_m1_gelu", "kind": "linear", "M": 1, "K": 2048, "N": 8192, "w": "e4m3", "act": "gelu_tanh", "res": False, "out": "bf16"},
        # 32 sequences being decoded, FP4 weights, the result quantised for the next projection
        {"name": "linear_m32_fp4", "kind": "linear", "M": 32, "K": 4096, "N": 14336, "w": "e2m1", "act": "gelu", "res": False, "out": "e4m3"},
        # a down projection of a ragged prompt, added to the residual stream
        {"name": "linear_m1531_residual", "kind": "linear", "M": 1531, "K": 14336, "N": 4096, "w": "e4m3", "act": "none", "res": True, "out": "bf16"},
        # an up projection of a full prompt batch: the largest
        {"name": "linear_m8192_gelu", "kind": "linear", "M": 8192, "K": 4096, "N": 14336, "w": "e4m3", "act": "gelu", "res": False, "out": "e4m3"},
        # a training step of few tokens, ragged: launches and host work
        {"name": "train_77x1024x4096", "kind": "train", "T": 77, "K": 1024, "N": 4096, "act": "gelu_tanh", "res": False},
        # a training step's down projection with the residual, full batch
        {"name": "train_4096x14336x4096", "kind": "train", "T": 4096, "K": 14336, "N": 4096, "act": "silu", "res": True},
        # many small tensors (norms, biases, small projections): launches and host work
        {"name": "adamw_200_small", "kind": "adamw", "tensors": 200, "total": 1000003, "bits": 32, "par": "f32", "grad": "f32", "copy": False},
        # the weights of a 4096 x 14336 block with fp32 masters, bf16 gradients and copies, states in 8 bits
        {"name": "adamw_117m_8bit", "kind": "adamw", "tensors": 8, "total": 117440512, "bits": 8, "par": "f32", "grad": "bf16", "copy": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _log_mult(rng, lo, hi, m):
    return max(lo, _log(rng, lo, hi) // m * m)


def draw(rng):
    kind = rng.choice(["norm_quantize", "norm", "norm", "linear", "linear", "train", "adamw", "adamw"])
    if kind == "norm_quantize":
        return {"kind": kind, "rows": _log(rng, 1, 8192), "H": _log(rng, 32, 16384), "src": rng.choice(["bf16", "bf16", "f32", "f16"])}
    if kind == "norm":
        return {"kind": kind, "rows": _log(rng, 1, 16384), "H": _log(rng, 16, 8192), "src": rng.choice(["bf16", "bf16", "f32", "f16"]),
                "par": rng.choice(["bf16", "f32"])}
    act = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
    if kind == "linear":
        return {"kind": kind, "M": _log(rng, 1, 8192), "K": _log_mult(rng, 512, 4096, rng.choice([32, 128, 512])),
                "N": _log_mult(rng, 512, 14336, rng.choice([32, 64, 256])), "w": rng.choice(["e4m3", "e2m1"]), "act": act,
                "res": rng.random() < 0.4, "out": rng.choice(["bf16", "e4m3"])}
    if kind == "train":
        return {"kind": kind, "T": _log(rng, 1, 4096), "K": _log_mult(rng, 256, 14336, rng.choice([32, 128])),
                "N": _log_mult(rng, 256, 4096, rng.choice([32, 256])), "act": act, "res": rng.random() < 0.4}
    return {"kind": kind, "tensors": _log(rng, 1, 300), "total": _log(rng, 1000, 100000000), "bits": rng.choice([8, 32]),
            "par": rng.choice(["f32", "bf16"]), "grad": rng.choice(["f32", "bf16"]), "copy": rng.random() < 0.3}


class _Maker:
    """Random operands on the GPU, from the seed alone."""

    def __init__(self, seed):
        self.dev = torch.device("cuda:0")
        self.g = torch.Generator(device=self.dev).manual_seed(seed)

    def normal(self, shape, std=1.0, dtype=torch.float32, mean=0.0):
        return torch.empty(shape, device=self.dev, dtype=dtype).normal_(mean, std, generator=self.g)

    def scales(self, shape, exponent):
        """E8M0 scales around 2^exponent."""
        return torch.randint(exponent + 126, exponent + 129, shape, generator=self.g, device=self.dev,
                             dtype=torch.uint8).view(torch.float8_e8m0fnu)

    def codes(self, rows, K, fmt, exponent):
        """Elements and scales of a matrix that was quantised before: blocks whose largest value is near the format's."""
        if fmt == "e2m1":
            q = torch.randint(0, 256, (rows, K // 2), generator=self.g, device=self.dev, dtype=torch.uint8)
        else:
            q = self.normal((rows, K), 128.0).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
        return q, self.scales((rows, K // 32), exponent)


def _sizes(case):
    """Sizes of the optimizer's tensors: spread over a factor of some hundred, `total` in all but for rounding."""
    r = random.Random(case["total"])
    share = [math.exp(r.uniform(0.0, 6.0)) for _ in range(case["tensors"])]
    return [max(1, int(case["total"] * s / sum(share))) for s in share]


def prepare(case, seed):
    m = _Maker(seed)
    kind = case["kind"]
    s = {"case": dict(case)}
    if kind in ("norm_quantize", "norm"):
        H = case["H"]
        par = TYPES[case.get("par", "f32")]
        s["x"] = m.normal((case["rows"], H), 2.0, TYPES[case["src"]], mean=0.5)
        s["w"] = m.normal((H,), 0.2, par, mean=1.0)
        s["b"] = m.normal((H,), 0.1, par)
        if kind == "norm":
            s["dy"] = m.normal((case["rows"], H), 1e-2, TYPES[case["src"]])
            for n in ("x", "w", "b"):
                s[n].requires_grad_()
    elif kind == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        s["a"], s["as"] = m.codes(M, K, "e4m3", -7)
        # weights around 1 / sqrt(K), so that sums are around one
        e = -7 - round(math.log2(K) / 2) if case["w"] == "e4m3" else -1 - round(math.log2(K) / 2)
        s["w"], s["ws"] = m.codes(N, K, case["w"], e)
        s["bias"] = m.normal((N,), 0.2, torch.bfloat16)
        s["res"] = m.normal((M, N), 1.0, torch.bfloat16) if case["res"] else None
        s["e2m1"] = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=m.dev)
    elif kind == "train":
        T, K, N = case["T"], case["K"], case["N"]
        s["x"] = m.normal((T, K), 1.0, torch.bfloat16).requires_grad_()
        s["w"] = m.normal((N, K), 1.0 / math.sqrt(K), torch.bfloat16).requires_grad_()
        s["bias"] = m.normal((N,), 0.2, torch.bfloat16).requires_grad_()
        s["res"] = m.normal((T, N), 1.0, torch.bfloat16) if case["res"] else None
        s["dy"] = m.normal((T, N), 1e-3, torch.bfloat16)
    else:
        # one tensor behind the other in memory, each from a multiple of 128 elements on, zeros between them
        sizes = _sizes(case)
        first, at = [], 0
        for n in sizes:
            first.append(at)
            at += -(-n // 128) * 128
        count = torch.tensor([-(-n // 128) * 128 for n in sizes], device=m.dev)
        s["which"] = torch.arange(len(sizes), device=m.dev).repeat_interleave(count)   # tensor of each element
        s["inside"] = torch.arange(at, device=m.dev) - torch.tensor(first, device=m.dev)[s["which"]]
        live = s["inside"] < torch.tensor(sizes, device=m.dev)[s["which"]]
        s["p"] = (m.normal((at,), 0.02) * live).to(TYPES[case["par"]])
        s["g"] = (m.normal((at,), 1e-3) * live).to(TYPES[case["grad"]])
        if case["bits"] == 8:
            blocks = live.view(-1, 32).any(1)
            s["m"] = (m.normal((at,), 128.0).clamp(-448.0, 448.0) * live).to(torch.float8_e4m3fn)
            s["v"] = (m.normal((at,), 128.0).abs().clamp(1.0, 448.0) * live).to(torch.float8_e4m3fn)
            s["ms"], s["vs"] = ((m.scales((at // 32,), e).view(torch.uint8) * blocks).view(torch.float8_e8m0fnu) for e in (-19, -17))
        else:
            s["m"] = m.normal((at,), 3e-4) * live
            s["v"] = m.normal((at,), 1e-3).square() * live
            s["ms"] = s["vs"] = None
        s["copy"] = torch.zeros(at, dtype=torch.bfloat16, device=m.dev) if case["copy"] else None
        part = lambda t, k: [None if t is None else t[a // k:(a + n + k - 1) // k] for a, n in zip(first, sizes)]  # noqa: E731
        pad = lambda t: [t[a:a + -(-n // 32) * 32] if case["bits"] == 8 else t[a:a + n] for a, n in zip(first, sizes)]  # noqa: E731
        s["params"], s["grads"], s["copies"] = part(s["p"], 1), part(s["g"], 1), part(s["copy"], 1)
        s["states"] = list(zip(pad(s["m"]), pad(s["v"]), part(s["ms"], 32), part(s["vs"], 32)))
    return s


def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    import cutile_amd as ct

    case = s["case"]
    kind = case["kind"]
    if kind == "norm_quantize":
        return ct.layer_norm_quantize(s["x"], s["w"], s["b"], eps=EPS)
    if kind == "norm":
        y = ct.layer_norm(s["x"], s["w"], s["b"], eps=EPS)
        return (y, *torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"]))
    act = None if case.get("act") == "none" else case.get("act")
    if kind == "linear":
        return ct.block_scaled_linear(s["a"], s["as"], s["w"], s["ws"], s["bias"], s["res"], activation=act, w_format=case["w"],
                                      out_dtype=torch.bfloat16 if case["out"] == "bf16" else torch.float8_e4m3fn)
    if kind == "train":
        y = ct.linear(s["x"], s["w"], s["bias"], s["res"], activation=act)
        return (y, *torch.autograd.grad(y, (s["x"], s["w"], s["bias"]), s["dy"]))
    ct.adamw_step(s["params"], s["grads"], s["states"], step=STEP, lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS,
                  weight_decay=DECAY, seed=SEED, copies=s["copies"] if case["copy"] else None)
    return _adamw_outputs(s)


_PACKAGE = str(pathlib.Path(__file__).resolve().parent.parent / "cutile-python_amd")


def _adamw_outputs(s):
    return {n: s[n] for n in ("p", "m", "v", "ms", "vs", "copy") if s[n] is not None}


# ---- the operators in elementary operations, 32 bits ------------------------------------------------------------------
def _power(e):
    """2^e for whole numbers e from -126 to 127, by its bits."""
    return ((e + 127) << 23).int().view(torch.float32)


def _exponent(amax):
    """floor(log2 amax) - 8, at least -127: the power of two of an E4M3 block."""
    return torch.where(amax == 0, -127, torch.frexp(amax)[1] - 9).clamp(-127, 127)


def _down(b, e):
    """b / 2^e in two steps, so that each power of two is a number."""
    half = -e // 2
    return b * _power(half).unsqueeze(-1) * _power(-e - half).unsqueeze(-1)


def _byte(e):
    return (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _quantize(x):
    """Q along the last axis, zero-padded to a multiple of 32: E4M3 elements and E8M0 scales."""
    x = torch.nn.functional.pad(x, (0, -x.shape[-1] % 32))
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    e = _exponent(b.abs().amax(-1))
    return _down(b, e).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).reshape(x.shape), _byte(e)


def _value(q, scale):
    return (q.float().reshape(*scale.shape, 32) * scale.float().unsqueeze(-1)).reshape(q.shape)


def _row(x):
    return _value(*_quantize(x))


def _col(x):
    """What Q along the columns leaves of x, transposed (rows padded with zeros to a multiple of 32)."""
    return _value(*_quantize(x.T.contiguous()))


def _weight(q, scale, fmt, table):
    if fmt != "e2m1":
        return _value(q, scale)
    v = torch.stack((table[(q & 15).int()], table[(q >> 4).int()]), -1)
    return _value(v.reshape(q.shape[0], -1), scale)


def _tanh_argument(p):
    return 1.5957691216057308 * p * (1.0 + 0.044715 * p * p)


def _act(p, name):
    if name == "relu":
        return p.clamp(min=0.0)
    if name == "gelu":
        return 0.5 * p * torch.erfc(-p * 0.7071067811865476)
    if name == "gelu_tanh":
        return p / (1.0 + torch.exp(-_tanh_argument(p)))
    return p / (1.0 + torch.exp(-p)) if name == "silu" else p


def _slope(p, name):
    """The activation's derivative."""
    if name == "relu":
        return (p > 0).float()
    if name == "gelu":
        return 0.5 * torch.erfc(-p * 0.7071067811865476) + p * torch.exp(-0.5 * p * p) * 0.3989422804014327
    if name == "gelu_tanh":
        t = 1.0 / (1.0 + torch.exp(-_tanh_argument(p)))
        return t + p * t * (1.0 - t) * 1.5957691216057308 * (1.0 + 0.134145 * p * p)
    t = 1.0 / (1.0 + torch.exp(-p))
    return t + p * t * (1.0 - t)


def _normed(x):
    c = x - x.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(c.square().mean(-1, keepdim=True) + EPS)
    return c * rstd, rstd


def _mix(x):
    """32 bits to 32 bits, in int64."""
    x = x ^ (x >> 16)
    x = (x * 0x9E3779B1) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _words(s):
    """The 32 random bits of each element: of the seed, the step, the tensor's place in the list and the element's in the tensor."""
    key = _mix(_mix(torch.full_like(s["which"], SEED)) ^ STEP) ^ s["which"]
    key = _mix(_mix(key) ^ (s["inside"] >> 32))
    return _mix((key + s["inside"]) & 0xFFFFFFFF)


def _round_up_or_down(x, bits):
    """Magnitudes below 512 to E4M3, up with the chance that 16 random bits give; signs kept, 448 at most."""
    a = x.abs()
    tiny = torch.where(a < 0.015625, 0.015625, 0.0)   # (the grid below 2^-6 is that of 2^-6 .. 2^-5)
    a = (((a + tiny).view(torch.int32) + (bits << 4).int()) & -1048576).view(torch.float32).clamp(max=448.0) - tiny
    return torch.copysign(a, x)


def _store(value, bits, root):
    """An optimizer state as E4M3 elements and E8M0 scales; roots above zero are never stored as zero.  The scale is the least power of
    two that the block's largest element is at most 448 times of: one that ended at 448 could not grow from step to step."""
    b = value.view(-1, 32)
    amax = b.abs().amax(-1)
    f, e = torch.frexp(amax)
    e = torch.where(amax == 0, -127, e - 9 + (f > 0.875)).clamp(-127, 127)
    v = _round_up_or_down(_down(b, e), bits.view(-1, 32))
    if root:
        v = torch.where(b > 0, v.clamp(min=0.001953125), v)
    return v.to(torch.float8_e4m3fn).view(-1), _byte(e)


def _adamw(s):
    p, g = s["p"].float(), s["g"].float()
    small = s["case"]["bits"] == 8
    m = _value(s["m"], s["ms"]) if small else s["m"]
    v = _value(s["v"], s["vs"]).square() if small else s["v"]
    m = BETA1 * m + (1.0 - BETA1) * g
    v = BETA2 * v + (1.0 - BETA2) * g * g
    root = torch.sqrt(v)
    p = p * (1.0 - LR * DECAY) - LR / (1.0 - BETA1 ** STEP) * m / (root / math.sqrt(1.0 - BETA2 ** STEP) + ADAM_EPS)
    if small:
        bits = _words(s)
        (m, ms), (v, vs) = _store(m, bits & 0xFFFF, False), _store(root, bits >> 16, True)
        s["ms"].copy_(ms)
        s["vs"].copy_(vs)
    for n, t in (("p", p), ("m", m), ("v", v)):
        s[n].copy_(t)
    if s["copy"] is not None:
        s["copy"].copy_(p)
    return _adamw_outputs(s)


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    with torch.no_grad():
        if kind == "adamw":
            return _adamw(s)
        if kind in ("norm_quantize", "norm"):
            x, w, b = (s[n].float() for n in ("x", "w", "b"))
            hat, rstd = _normed(x)
            y = hat * w + b
            if kind == "norm_quantize":
                return _quantize(y)
            dy = s["dy"].float()
            h = dy * w
            dx = rstd * (h - h.mean(-1, keepdim=True) - hat * (h * hat).mean(-1, keepdim=True))
            out = (y, dx, (dy * hat).sum(0), dy.sum(0))
            return tuple(t.to(s[n].dtype) for t, n in zip(out, ("x", "x", "w", "b")))
        res = 0.0 if s["res"] is None else s["res"].float()
        if kind == "linear":
            p = _value(s["a"], s["as"]) @ _weight(s["w"], s["ws"], case["w"], s["e2m1"]).T + s["bias"].float()
            y = _act(p, case["act"]) + res
            return y.bfloat16() if case["out"] == "bf16" else _quantize(y)
        x, w, dy = (s[n].float() for n in ("x", "w", "dy"))
        p = _row(x) @ _row(w).T + s["bias"].float()
        d = dy if case["act"] == "none" else dy * _slope(p.bfloat16().float(), case["act"])
        out = (_act(p, case["act"]) + res, _row(d) @ _col(w).T, _col(d) @ _col(x).T, d.sum(0))
        return tuple(t.bfloat16() for t in out)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------
def _bytes(name):
    return 4 if name == "f32" else 2


def work(case):
    mx = 1 + 1 / 32
    kind = case["kind"]
    if kind == "norm_quantize":
        n = case["rows"] * case["H"]
        return {"bytes": n * (_bytes(case["src"]) + mx) + 8 * case["H"], "flops": 8 * n}
    if kind == "norm":   # x, y; x, dy, dx
        n = case["rows"] * case["H"]
        return {"bytes": 5 * n * _bytes(case["src"]) + 4 * case["H"] * _bytes(case["par"]), "flops": 20 * n}
    if kind == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        w = (0.5 if case["w"] == "e2m1" else 1) + 1 / 32
        return {"bytes": M * K * mx + N * K * w + M * N * ((2 if case["out"] == "bf16" else mx) + (2 if case["res"] else 0)),
                "flops": 2 * M * N * K}
    if kind == "train":   # x, dx; y, dy, residual; w, dw: 16 bits each
        T, K, N = case["T"], case["K"], case["N"]
        return {"bytes": 4 * T * K + (6 if case["res"] else 4) * T * N + 4 * N * K, "flops": 6 * T * K * N}
    n = sum(_sizes(case))
    state = 4 * mx if case["bits"] == 8 else 16
    return {"bytes": n * (2 * _bytes(case["par"]) + _bytes(case["grad"]) + state + (2 if case["copy"] else 0)), "flops": 16 * n}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------------
def _two_to(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _steps(v, bits, least):
    """The distance of neighbours around v among numbers of `bits` significant digits whose last is worth 2^least or more."""
    return _two_to(torch.clamp(torch.frexp(v)[1] - bits, min=least))


def _nearest(v, bits, least):
    step = _steps(v, bits, least)
    return torch.round(v / step) * step


def _scale64(b):
    top = torch.amax(torch.abs(b), -1)
    return _two_to(torch.clamp(torch.where(top > 0, torch.frexp(top)[1] - 9.0, torch.full_like(top, -127.0)), -127.0, 127.0))


def _q64(x):
    """Element values and scales of Q along the last axis."""
    n = -(-x.shape[-1] // 32) * 32
    full = torch.zeros((*x.shape[:-1], n), dtype=torch.float64, device=x.device)
    full[..., :x.shape[-1]] = x
    b = full.reshape(*x.shape[:-1], n // 32, 32)
    scale = _scale64(b)
    return _nearest(torch.clamp(b / scale[..., None], -448.0, 448.0), 4, -9).reshape(full.shape), scale


def _r64(x):
    v, scale = _q64(x)
    return v * scale.repeat_interleave(32, -1)


def _c64(x):
    return _r64(x.T)


def _act64(p, name):
    """The activation and its derivative."""
    if name == "none":
        return p, torch.ones_like(p)
    if name == "relu":
        return torch.relu(p), torch.where(p > 0, 1.0, 0.0).double()
    if name == "silu":
        t = torch.sigmoid(p)
        return p * t, t * (1 + p * torch.sigmoid(-p))
    if name == "gelu":
        t = torch.special.ndtr(p)
        return p * t, t + p * torch.exp(-p * p / 2) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (p + 0.044715 * p ** 3))
    return 0.5 * p * (1 + t), 0.5 * (1 + t) + 0.5 * p * (1 - t * t) * c * (1 + 3 * 0.044715 * p * p)


def _hash64(x):
    """The random words' mixing step with products of 16-bit halves."""
    def times(a, k):
        return ((a % 65536) * k + ((a // 65536 * (k % 65536)) % 65536) * 65536) % 4294967296

    x = torch.bitwise_xor(x, x // 65536)
    x = times(x, 2654435761)
    x = torch.bitwise_xor(x, x // 32768)
    x = times(x, 3144134277)
    return torch.bitwise_xor(x, x // 65536)


def _state64(value, chance, root):
    b = value.reshape(-1, 32)
    top = torch.amax(torch.abs(b), -1)
    scale = _two_to(torch.clamp(torch.where(top > 0, torch.ceil(torch.log2(top / 448)), torch.full_like(top, -127.0)), -127.0, 127.0))
    scale = torch.where(top > 448 * scale, 2 * scale, scale)   # (a logarithm rounded down to a whole number)
    v = torch.abs(b) / scale[:, None]
    step = _steps(v, 4, -9)
    v = torch.clamp(torch.floor(v / step + chance.reshape(-1, 32) / 65536) * step, max=448.0)
    if root:
        v = torch.maximum(v, torch.where(b > 0, 2.0 ** -9, 0.0).double())
    return (torch.sign(b) * v).reshape(-1), scale


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    with torch.no_grad():
        if kind in ("norm_quantize", "norm"):
            x, w, b = (s[n].double() for n in ("x", "w", "b"))
            var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
            rstd = torch.rsqrt(var + EPS)
            hat = (x - mean) * rstd
            y = hat * w + b
            if kind == "norm_quantize":
                return _q64(y)
            dy = s["dy"].double()
            h, H = dy * w, x.shape[-1]
            dx = rstd / H * (H * h - h.sum(-1, keepdim=True) - hat * (h * hat).sum(-1, keepdim=True))
            return y, dx, (dy * hat).sum(0), dy.sum(0)
        if kind == "adamw":
            p, g = s["p"].double(), s["g"].double()
            small = case["bits"] == 8
            m = s["m"].double() * (s["ms"].double().repeat_interleave(32) if small else 1.0)
            v = (s["v"].double() * s["vs"].double().repeat_interleave(32)) ** 2 if small else s["v"].double()
            m = BETA1 * m + (1 - BETA1) * g
            v = BETA2 * v + (1 - BETA2) * g ** 2
            hat = (m / (1 - BETA1 ** STEP)) / ((v / (1 - BETA2 ** STEP)).sqrt() + ADAM_EPS)
            out = {"p": p - LR * DECAY * p - LR * hat, "m": m, "v": v}
            if small:
                key = _hash64(torch.bitwise_xor(_hash64(torch.full_like(s["which"], SEED)), torch.full_like(s["which"], STEP)))
                key = _hash64(torch.bitwise_xor(_hash64(torch.bitwise_xor(key, s["which"])), s["inside"] // 4294967296))
                word = _hash64((key + s["inside"]) % 4294967296)
                out["m"], out["ms"] = _state64(m, word % 65536, False)
                out["v"], out["vs"] = _state64(v.sqrt(), word // 65536, True)
            if s["copy"] is not None:
                out["copy"] = out["p"]
            return out
        res = 0.0 if s["res"] is None else s["res"].double()
        if kind == "linear":
            a = s["a"].double() * s["as"].double().repeat_interleave(32, -1)
            w = s["w"]
            if case["w"] == "e2m1":
                code = torch.stack((w % 16, w // 16), 2).reshape(w.shape[0], -1).long()
                e, f = (code // 2) % 4, code % 2
                v = torch.where(e == 0, f * 0.5, (1 + f * 0.5) * _two_to(e - 1))
                w = torch.where(code >= 8, -v, v)
            p = a @ (w.double() * s["ws"].double().repeat_interleave(32, -1)).T + s["bias"].double()
            y = _act64(p, case["act"])[0] + res
            return y if case["out"] == "bf16" else _q64(y)
        x, w, dy = (s[n].double() for n in ("x", "w", "dy"))
        p = _r64(x) @ _r64(w).T + s["bias"].double()
        d = dy * _act64(_nearest(p, 8, -133), case["act"])[1]
        return _act64(p, case["act"])[0] + res, _r64(d) @ _c64(w).T, _c64(d) @ _c64(x).T, d.sum(0)
