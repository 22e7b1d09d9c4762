"""The fused product where k is a multiple of 128 that the waves of a workgroup cannot share in equal whole chunks, and thin
products of 65 to 256 rows on both sides of the length from which they stream their weights: against 64-bit arithmetic,
with k columns of NaN behind the rows and outputs' neighbours held.

Tolerance: (k + 1) roundings of 2^-24 of the absolute sum whatever the order, an activation's slope of at most 1.13 and its
own evaluation within 2^-20 (1 + |y|), and one rounding each for the residual and the outputs (f32)."""
import math

import pytest
import torch

from glm53f_forward import ffi
from oracle import lin_oracle as lo

import harness as hs
from harness import ptr

pytestmark = pytest.mark.gpu
DEV = hs.DEV


def product(rows, n, k, pad, seed, groups=1, act=2):
    gen = torch.Generator().manual_seed(seed)
    ld = k + pad
    x = torch.full((groups, rows, ld), math.nan, dtype=torch.bfloat16)
    w = torch.full((groups, n, ld), math.nan, dtype=torch.bfloat16)
    x[..., :k] = torch.randn(groups, rows, k, generator=gen).bfloat16()
    w[..., :k] = (torch.randn(groups, n, k, generator=gen) * k ** -0.5).bfloat16()
    b, r = torch.randn(groups, n, generator=gen).bfloat16(), torch.randn(groups, rows, n, generator=gen)
    d_x, d_w, d_b, d_r = x.to(DEV), w.to(DEV), b.to(DEV), r.to(DEV)
    out = torch.full((groups * rows * n + 64,), 7.0, device=DEV)
    assert ffi.glm53f_fwd_gemm_bf16_fused(ptr(d_x), ld, rows * ld, ptr(d_w), ld, n * ld, groups, rows, n, k, ptr(d_b), n, act, ptr(d_r), n,
                                          rows * n, ptr(out), 1, n, rows * n, None) == 0
    hs.sync()
    got = out.cpu().double()
    assert bool((got[groups * rows * n:] == 7).all()), "wrote behind the outputs"
    for g in range(groups):
        want, a = lo.gemm(x[g, :, :k], w[g, :, :k], b[g], act, r[g])
        y = want - r[g].double()
        tol = 1.13 * (k + 1) * 2.0 ** -24 * a + 2.0 ** -20 * (1 + y.abs()) + 2 * 2.0 ** -24 * (want.abs() + y.abs())
        err = (got[g * rows * n:(g + 1) * rows * n].reshape(rows, n) - want).abs()
        assert bool((err <= tol).all()), f"group {g}: {float((err / tol).max()):.2f} of the tolerance"


@pytest.mark.parametrize("k", [640, 896, 1152, 1536, 2560, 5248, 11008])
def test_k_of_whole_chunks_but_no_equal_shares(k):
    for rows, n in ((1, 1024), (16, 4096), (17, 208), (33, 1040), (64, 4112), (40, 8208)):
        print(f"{rows} rows {k} -> {n}", flush=True)
        product(rows, n, k, 8, rows + k)


@pytest.mark.parametrize("k", [8, 136, 384, 504, 512, 520, 640, 1152, 2176])
def test_thin_products_of_more_rows(k):
    for rows, n in ((65, 512), (100, 1024), (200, 2048), (256, 1024), (129, 333)):
        print(f"{rows} rows {k} -> {n}", flush=True)
        product(rows, n, k, 8, rows + k)


@pytest.mark.parametrize("rows", [7, 50, 90])
def test_groups_of_such_products(rows):
    product(rows, 160, 1152, 8, rows, groups=3, act=5)
