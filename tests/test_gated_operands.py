"""Operands of the gated product at the ends of what it takes: an empty sum, packed scales that are not where they have to be."""
import ctypes

import pytest
import torch

from cutile_amd import _lib as L
from mxutil import randn_operand
from oracle import mx_oracle as O
from test_ffn_validation import P, d, refs

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def test_workspace_of_an_empty_sum():
    """The query names what the call asks for, at K = 0 as elsewhere."""
    lib = L.lib()
    M, F = 40, 64
    need = lib.mx_gated_gemm_workspace_bytes(M, F, 0, None)
    assert need >= M * 2 * F * 2 and lib.mx_gated_gemm_workspace_bytes(M, F, -32, None) == 0
    good = dict(A=d(L.MX_E4M3, M, 0), As=d(L.MX_E8M0, M, 0), W=d(L.MX_E4M3, 2 * F, 0), Ws=d(L.MX_E8M0, 2 * F, 0),
                out=d(L.MX_E4M3, M, F), out_s=d(L.MX_E8M0, M, F // 32), gu=None, gus=None, mode=1, opts=None, ws=P, ws_bytes=need - 1)
    assert lib.mx_gated_gemm(*refs(good.values()), None) == L.MX_ERR_WORKSPACE and f"workspace of {need} bytes" in L.last_error()


@pytest.mark.parametrize("operand", ["A_scale", "W_scale"])
@pytest.mark.parametrize("kernel,M", [(L.MX_KERNEL_MFMA_PINGPONG, 300), (L.MX_KERNEL_AUTO, 4000), (L.MX_KERNEL_MFMA_128x128, 300)])
def test_packed_scales_that_are_not_aligned(kernel, M, operand):
    """Refused by every kernel that reads them, before anything is enqueued."""
    K, F = 512, 2048
    o = L.MxGemmOpts(struct_size=32, kernel=kernel, block_size=32, a_scale_layout=L.MX_SCALE_NATIVE, b_scale_layout=L.MX_SCALE_NATIVE)
    lib = L.lib()
    need = lib.mx_gated_gemm_workspace_bytes(M, F, K, ctypes.byref(o))
    at = {"A_scale": 0, "W_scale": 0, operand: 4}
    args = [d(L.MX_E4M3, M, K), d(L.MX_E8M0, M, K // 32, ptr=P + at["A_scale"]), d(L.MX_E4M3, 2 * F, K), d(L.MX_E8M0, 2 * F, K // 32, ptr=P + at["W_scale"]),
            d(L.MX_BF16, M, F), None, None, None, 1, ctypes.byref(o), P, need]
    assert lib.mx_gated_gemm(*refs(args), None) == L.MX_ERR_LAYOUT and "16-byte aligned" in L.last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 40, 300])
@pytest.mark.parametrize("out", [torch.bfloat16, E4M3, torch.float8_e5m2])
def test_an_empty_sum(ct, dev, M, out):
    """Zeros, as block_scaled_matmul gives, and their quantisation."""
    F = 64
    a, w = (torch.empty((n, 0), dtype=torch.uint8, device=dev) for n in (M, 2 * F))
    s = [t.view(E8M0) for t in (a, w)]
    got = ct.gated_block_scaled_matmul(a.view(E4M3), s[0], w.view(E4M3), s[1], out_dtype=out, checkpoint=True)
    gu = torch.zeros((M, 2 * F), dtype=torch.bfloat16, device=dev)
    want = (gu[:, :F],) if out == torch.bfloat16 else ct.silu_and_mul_quantize(gu, out, scale_mode="floor")
    want = (*want, *ct.block_quantize(gu, 32, E4M3, scale_mode="floor"))
    assert len(got) == len(want)
    for x, y in zip(got, want):
        assert x.dtype == y.dtype and torch.equal(x.view(torch.uint8), y.contiguous().view(torch.uint8))
    assert torch.equal(ct.block_scaled_matmul(a.view(E4M3), s[0], w.view(E4M3).T, s[1].T, out_dtype=torch.bfloat16), gu)
