"""Every kernel that the fused product can launch, each at the sizes of least work that reach it, with bias, an activation
and the residual, in place too, both output types, and its last rows and columns whole tiles or not: against 64-bit
arithmetic. And addresses beyond 2^31 elements.

Tolerance: (k + 1) roundings of 2^-24 of the absolute sum whatever the order, an activation's slope of at most 1.13 and its
own evaluation within 2^-20 (1 + |y|), and one rounding each for the residual and the outputs (f32 2^-24, bf16 2^-8)."""
import math

import pytest
import torch

from glm53f_forward import ffi
from oracle import lin_oracle as lo

import fused_dispatch as fd
import harness as hs
from harness import ptr

pytestmark = pytest.mark.gpu
DEV = hs.DEV
CASES = sorted(fd.cheapest().items(), key=str)


def check(got, x, w, b, r, act, f32_out):
    want, a = lo.gemm(x, w, b, act, r)
    y = want - r.double()
    step = 2.0 ** -24 if f32_out else 2.0 ** -8
    tol = 1.13 * (x.shape[1] + 1) * 2.0 ** -24 * a + 2.0 ** -20 * (1 + y.abs()) + 2.0 ** -24 * (want.abs() + y.abs()) + step * want.abs()
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"{float((err / tol).max()):.2f} of the tolerance"


@pytest.mark.parametrize("kernel,size", CASES, ids=["-".join(str(int(v) if isinstance(v, bool) else v) for v in k) for k, _ in CASES])
def test_kernel(kernel, size):
    assert fd.kernel_of(*size[:3], 1, size[3]) == kernel
    for f32_out, in_place in ((False, True), (True, False), (True, True)):
        print(f"{kernel} {size} f32 {f32_out} in place {in_place}", flush=True)
        run(*size, f32_out, in_place)


def run(rows, n, k, aligned, f32_out, in_place):
    shift = 0 if aligned else 1
    gen = torch.Generator().manual_seed(rows + n + k)
    kind = torch.float32 if f32_out else torch.bfloat16
    x, w = torch.randn(rows, k, generator=gen).bfloat16(), (torch.randn(n, k, generator=gen) * k ** -0.5).bfloat16()
    b, r = torch.randn(n, generator=gen).bfloat16(), torch.randn(rows, n, generator=gen).to(kind)
    d_x, d_w = (torch.full((shift + t.shape[0] * (k + 8),), math.nan, dtype=torch.bfloat16, device=DEV) for t in (x, w))
    for d, t in ((d_x, x), (d_w, w)):
        d[shift:].view(t.shape[0], k + 8)[:, :k] = t.to(DEV)
    ldo = n + 8
    d_r = torch.full((rows, ldo), math.nan, dtype=kind, device=DEV)
    d_r[:, :n] = r.to(DEV)
    d_o = d_r if in_place else torch.full((rows, ldo), math.nan, dtype=kind, device=DEV)
    d_b = b.to(DEV)
    assert ffi.glm53f_fwd_gemm_bf16_fused(ptr(d_x, shift), k + 8, 0, ptr(d_w, shift), k + 8, 0, 1, rows, n, k, ptr(d_b), 0, 2, ptr(d_r), ldo, 0,
                                          ptr(d_o), int(f32_out), ldo, 0, None) == 0
    hs.sync()
    got = d_o.cpu()
    assert bool(got[:, n:].isnan().all()), "wrote behind the rows"
    check(got[:, :n], x, w, b, r, 2, f32_out)


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("f32_out", [False, True])
@pytest.mark.parametrize("kind_of_kernel,rows,stride", [("tile", 300, (1 << 23) + 8), ("stream", 40, (1 << 26) + 8)])
def test_rows_beyond_31_bits(kind_of_kernel, rows, stride, shift, f32_out):
    """Rows of x, of the residual and of the outputs further than 2^31 elements apart (2.5e9 and 2.6e9)."""
    n, k = 64, 128
    assert fd.kernel_of(rows, n, k, 1, shift == 0)[0] == kind_of_kernel
    gen = torch.Generator().manual_seed(shift)
    kind = torch.float32 if f32_out else torch.bfloat16
    x, w = torch.randn(rows, k, generator=gen).bfloat16(), torch.randn(n, k, generator=gen).bfloat16()
    b, r = torch.randn(n, generator=gen).bfloat16(), torch.randn(rows, n, generator=gen).to(kind)
    big = torch.empty(shift + (rows - 1) * stride + k, dtype=torch.bfloat16, device=DEV)
    out = torch.empty((rows - 1) * stride + n + 8, dtype=kind, device=DEV)
    torch.as_strided(big, (rows, k), (stride, 1), shift).copy_(x.to(DEV))
    torch.as_strided(out, (rows, n + 8), (stride, 1)).fill_(7.0)
    torch.as_strided(out, (rows, n), (stride, 1)).copy_(r.to(DEV))
    d_w, d_b = w.to(DEV), b.to(DEV)
    assert ffi.glm53f_fwd_gemm_bf16_fused(ptr(big, shift), stride, 0, ptr(d_w), k, 0, 1, rows, n, k, ptr(d_b), 0, 0, ptr(out), stride, 0,
                                          ptr(out), int(f32_out), stride, 0, None) == 0
    hs.sync()
    got = torch.as_strided(out, (rows, n + 8), (stride, 1)).cpu()
    assert bool((got[:, n:] == 7).all()), "wrote behind the rows"
    check(got[:, :n], x, w, b, r, 0, f32_out)
