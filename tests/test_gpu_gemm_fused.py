"""The matrix product with bias, activation and residual (glm53f_fwd_gemm_bf16_fused) through the C ABI against 64-bit
arithmetic: sizes of whole tiles and of none, one row to thousands, groups, strides and alignments, every activation,
both output types, the residual in place.

Tolerances. The products are exact in f32; a sum of k of them and the bias is off by at most (k + 1) roundings of 2^-24
of the absolute sum `a`, whatever the order (tiles and waves only shorten the chains). An activation's slope is at most
1.13, its own evaluation within 16 roundings of 1 + |y|; the residual's addition is one rounding, a stored bf16 value
one of 2^-8."""
import math

import pytest
import torch

from glm53f_forward import ffi
from oracle import lin_oracle as lo

import harness as hs
from harness import ptr

pytestmark = pytest.mark.gpu
DEV = hs.DEV
ACTS = ("none", "relu", "silu", "gelu", "gelu_tanh", "sigmoid")


def run(groups, rows, n, k, act="none", bias=True, residual=True, f32_out=False, pad=0, shift=0, in_place=False, seed=1, sigma=1.0,
        stream=None):
    gen = torch.Generator().manual_seed(seed)
    kind = torch.float32 if f32_out else torch.bfloat16

    def dev(shape, ld, scale, dtype=torch.bfloat16, fill=math.nan):
        host = (torch.randn(*shape, generator=gen) * scale).to(dtype)
        flat = torch.full((shift + math.prod(shape[:-1]) * ld,), fill, dtype=dtype)
        flat[shift:].view(*shape[:-1], ld)[..., :shape[-1]] = host
        return host, flat.to(DEV)

    ldx, ldw, ldo = k + pad, k + pad, n + pad
    x, d_x = dev((groups, rows, k), ldx, sigma)
    w, d_w = dev((groups, n, k), ldw, k ** -0.5)
    b, d_b = dev((groups, n), n + pad, 0.5) if bias else (None, None)
    r, d_r = dev((groups, rows, n), ldo, 1.0, kind, 7.0) if residual else (None, None)
    if in_place:
        d_o = d_r
    else:
        d_o = torch.full((shift + groups * rows * ldo,), 7.0, dtype=kind, device=DEV)
    at = lambda t: None if t is None else ptr(t, shift)  # noqa: E731
    rc = ffi.glm53f_fwd_gemm_bf16_fused(at(d_x), ldx, rows * ldx, at(d_w), ldw, n * ldw, groups, rows, n, k, at(d_b), n + pad,
                                        ACTS.index(act), at(d_r), ldo, rows * ldo, at(d_o), int(f32_out), ldo, rows * ldo, stream)
    assert rc == 0, rc
    hs.sync()
    flat = d_o.float().cpu()
    got = flat[shift:].view(groups, rows, ldo)
    assert bool((flat[:shift] == 7).all()) and bool((got[..., n:] == 7).all()), "wrote outside the rows"
    for g in range(groups):
        want, a = lo.gemm(x[g], w[g], None if b is None else b[g], ACTS.index(act), None if r is None else r[g])
        mid = want - (0 if r is None else r[g].double())
        tol = 1.13 * (k + 1) * 2.0 ** -24 * a + 2.0 ** -24 * want.abs() + 1e-30
        if act not in ("none", "relu"):
            tol = tol + 16 * 2.0 ** -24 * (1 + mid.abs())
        if not f32_out:
            tol = tol + 2.0 ** -8 * want.abs()
        err = (got[g, :, :n].double() - want).abs()
        assert bool((err <= tol).all()), f"group {g}: {float((err / tol).max()):.2f} of the tolerance"
    return got[..., :n]


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 33, 64, 65, 127, 128, 129, 200, 256, 257, 384, 520, 1025])
@pytest.mark.parametrize("n,k", [(256, 512), (4112, 1024), (1999, 1001), (48, 8192), (300, 136)])
def test_rows_and_sizes(rows, n, k):
    print(f"rows {rows} n {n} k {k}", flush=True)
    run(1, rows, n, k, "silu", f32_out=rows % 2 == 0, seed=rows + n)


@pytest.mark.parametrize("n,k", [(1, 1), (1, 8), (7, 3), (16, 128), (17, 127), (64, 64), (24640, 4096), (4096, 8192), (8192, 128)])
def test_the_smallest_sizes_and_the_layers(n, k):
    for rows in (1, 3, 16, 70):
        print(f"rows {rows} n {n} k {k}", flush=True)
        run(1, rows, n, k, "none", f32_out=True, seed=n)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("f32_out", [False, True])
@pytest.mark.parametrize("rows", [5, 48, 150, 300])
def test_activations(act, f32_out, rows):
    run(1, rows, 272, 256, act, f32_out=f32_out, seed=3, sigma=3.0)


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows", [9, 100])
def test_parts_of_the_epilogue(bias, residual, rows):
    run(1, rows, 160, 384, "gelu", bias, residual, seed=5)


@pytest.mark.parametrize("rows", [1, 20, 90, 260])
@pytest.mark.parametrize("pad,shift", [(8, 0), (8, 8), (1, 0), (0, 1), (6, 2), (3, 5)])
def test_strides_and_alignments(rows, pad, shift):
    for f32_out in (False, True):
        run(1, rows, 144, 256, "relu", pad=pad, shift=shift, f32_out=f32_out, seed=7)


@pytest.mark.parametrize("rows", [3, 40, 130, 300])
def test_groups(rows):
    run(3, rows, 272, 384, "sigmoid", seed=9)
    run(2, rows, 33, 50, "none", seed=10, pad=3)


@pytest.mark.parametrize("rows", [4, 64, 300])
@pytest.mark.parametrize("f32_out", [False, True])
def test_the_residual_stream_in_place(rows, f32_out):
    run(1, rows, 512, 256, "none", f32_out=f32_out, in_place=True, seed=11)


@pytest.mark.parametrize("rows", [2, 40, 128, 400])
def test_broadcast_groups_and_a_shared_input(rows):
    """Group strides of 0: one x, one weight or one bias for all groups."""
    gen = torch.Generator().manual_seed(13)
    n, k, groups = 96, 128, 3
    x, w = torch.randn(rows, k, generator=gen).bfloat16(), (torch.randn(groups, n, k, generator=gen) * 0.1).bfloat16()
    b = torch.randn(n, generator=gen).bfloat16()
    d_x, d_w, d_b = x.to(DEV), w.to(DEV), b.to(DEV)
    out = torch.zeros(groups, rows, n, device=DEV)
    assert ffi.glm53f_fwd_gemm_bf16_fused(ptr(d_x), k, 0, ptr(d_w), k, n * k, groups, rows, n, k, ptr(d_b), 0, 0, None, 0, 0,
                                          ptr(out), 1, n, rows * n, None) == 0
    hs.sync()
    for g in range(groups):
        want, a = lo.gemm(x, w[g], b, 0, None)
        assert bool(((out[g].cpu().double() - want).abs() <= (k + 2) * 2.0 ** -24 * a).all())


def test_extreme_values_pass_the_activations():
    """Infinite and huge pre-activations give what the formula's limits are, and a NaN row stays in its row."""
    n, k = 64, 128
    for rows in (4, 80):
        for act in range(6):
            x = torch.zeros(rows, k, dtype=torch.bfloat16)
            x[0, 0], x[1, 0], x[2, 0] = 1e30, -1e30, math.nan
            w = torch.zeros(n, k, dtype=torch.bfloat16)
            w[:, 0] = 1e5
            d_x, d_w = x.to(DEV), w.to(DEV)
            out = torch.zeros(rows, n, device=DEV)
            assert ffi.glm53f_fwd_gemm_bf16_fused(ptr(d_x), k, 0, ptr(d_w), k, 0, 1, rows, n, k, None, 0, act, None, 0, 0, ptr(out), 1,
                                                  n, 0, None) == 0
            hs.sync()
            o = out.cpu()
            high = x[0, 0].float() * w[0, 0].float()
            assert bool((o[0] == (1.0 if act == 5 else high)).all()), act
            low = {0: -high, 1: 0.0, 2: 0.0, 3: 0.0, 4: 0.0, 5: 0.0}[act]
            assert bool((o[1] == low).all()), act
            # max(NaN, 0) is the one activation that may drop a NaN; this one keeps it
            assert bool(o[2].isnan().all()), act
            assert bool((o[3] == (0.5 if act == 5 else 0.0)).all()), act


def test_offsets_past_32_bits():
    rows, n, k = 70, 32, 64
    stride = 1 << 25                              # 70 rows span 2.3e9 elements
    gen = torch.Generator().manual_seed(17)
    x, w = torch.randn(rows, k, generator=gen).bfloat16(), torch.randn(n, k, generator=gen).bfloat16()
    big = torch.zeros((rows - 1) * stride + k, dtype=torch.bfloat16, device=DEV)
    out = torch.zeros((rows - 1) * stride + n, dtype=torch.bfloat16, device=DEV)
    torch.as_strided(big, (rows, k), (stride, 1)).copy_(x.to(DEV))
    d_w = w.to(DEV)
    want, a = lo.gemm(x, w, None, 0, None)
    for m in (rows, 5):
        first = rows - m
        assert ffi.glm53f_fwd_gemm_bf16_fused(ptr(big), stride, 0, ptr(d_w), k, 0, 1, rows, n, k, None, 0, 0, None, 0, 0, ptr(out), 0,
                                              stride, 0, None) == 0
        hs.sync()
        got = torch.as_strided(out, (rows, n), (stride, 1)).float().cpu().double()
        assert bool(((got - want).abs()[first:] <= (2.0 ** -8 * want.abs() + (k + 1) * 2.0 ** -24 * a)[first:]).all())


def test_a_captured_product_replays_like_eager_products():
    gen = torch.Generator().manual_seed(19)
    n, k = 256, 512
    w = (torch.randn(n, k, generator=gen) * 0.05).bfloat16().to(DEV)
    for rows in (1, 48, 300):
        x = torch.randn(rows, k, generator=gen).bfloat16().to(DEV)
        streams = [torch.zeros(rows, n, dtype=torch.bfloat16, device=DEV) for _ in range(2)]

        def step(h, stream):                      # the residual stream in place: every call adds once more
            assert ffi.glm53f_fwd_gemm_bf16_fused(ptr(x), k, 0, ptr(w), k, 0, 1, rows, n, k, None, 0, 2, ptr(h), n, 0, ptr(h), 0, n, 0,
                                                  stream) == 0

        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(streams[0], torch.cuda.current_stream().cuda_stream)
        for replay in range(1, 4):
            graph.replay()
            step(streams[1], None)
            assert math.isfinite(torch.randn(1 << 16, device=DEV).sum().item())
            hs.sync()
            assert torch.equal(streams[0], streams[1]), f"{rows} rows, replay {replay}"


def test_no_rows_is_no_launch():
    assert ffi.glm53f_fwd_gemm_bf16_fused(None, 8, 0, None, 8, 0, 1, 0, 8, 8, None, 0, 0, None, 0, 0, None, 0, 8, 0, None) == 0


@pytest.mark.parametrize("rows,n,k", [(65, 203, 128), (300, 203, 192), (513, 1001, 64), (1025, 4099, 256), (2100, 8190, 64), (300, 7, 128), (70, 3, 128)])
@pytest.mark.parametrize("f32_out", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
def test_residual_rows_whose_stride_is_longer_than_they_are(rows, n, k, f32_out, in_place):
    """Aligned rows of x, w and the residual, n of no multiple: what the residual's tile is asked for early ends at the rows'
    ends. The columns behind are NaN in the residual and stay what they are in the outputs."""
    gen = torch.Generator().manual_seed(rows + n)
    kind, ld = (torch.float32 if f32_out else torch.bfloat16), (n + 15) // 8 * 8
    x, w = torch.randn(rows, k, generator=gen).bfloat16(), (torch.randn(n, k, generator=gen) * k ** -0.5).bfloat16()
    res = torch.full((rows, ld), math.nan, dtype=kind)
    res[:, :n] = torch.randn(rows, n, generator=gen).to(kind)
    d_x, d_w, d_r = x.to(DEV), w.to(DEV), res.to(DEV)
    d_o = d_r if in_place else torch.full((rows, ld), math.nan, dtype=kind, device=DEV)
    assert ffi.glm53f_fwd_gemm_bf16_fused(ptr(d_x), k, 0, ptr(d_w), k, 0, 1, rows, n, k, None, 0, 0, ptr(d_r), ld, 0, ptr(d_o), int(f32_out),
                                          ld, 0, None) == 0
    hs.sync()
    got = d_o.cpu().double()
    want, a = lo.gemm(x, w, None, 0, res[:, :n])
    tol = 1.13 * (k + 1) * 2.0 ** -24 * a + 2.0 ** -24 * want.abs() + 1e-30 + (0 if f32_out else 2.0 ** -8 * want.abs())
    assert bool(((got[:, :n] - want).abs() <= tol).all()) and bool(got[:, n:].isnan().all())


@pytest.mark.parametrize("rows,n,k", [(100, 2000, 8), (200, 4096, 264), (300, 4096, 72), (400, 2500, 1000), (513, 4096, 4104), (1025, 4096, 200),
                                      (2049, 4096, 328), (4096, 4096, 72), (130, 77, 136)])
@pytest.mark.parametrize("groups", [1, 2])
def test_aligned_rows_whose_k_is_no_whole_step(rows, n, k, groups):
    """Every tile's shape with k a multiple of 8 and no more; NaN in the eight columns behind k, which no product may reach."""
    if groups == 2 and rows > 600:
        rows = rows // 8 + 1
    run(groups, rows, n, k, "none", f32_out=True, pad=8, seed=k)
    run(groups, rows, n, k, "silu", residual=False, seed=k + 1)
