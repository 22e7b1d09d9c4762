"""Linear attention with one decay per head where the terms of an output cancel: the chunked form's outputs are held to
f32 rounding of their terms, not to the outputs' own rounding.

Every request has one key that is not zero, another one each, so that no sum over the keys rounds: row t's output is
scale q_t e^(g t) (e^g S + k_0 v_0) with the states S chosen so that the bracket is a 2^-14th of its terms or nothing.
Tolerance: what is left are the decays (exp of a rounded argument of at most 2: four roundings each), their products
with the scale, the score, the state's sum and the three partial sums of each: at most 24 roundings of 2^-24 of the terms'
absolute values, and the output's own, 2^-8 of itself."""
import pytest
import torch

from glm53f_lin import ffi
from oracle import lin_oracle as lo

import harness as hs
from harness import ptr

pytestmark = pytest.mark.gpu
DEV = hs.DEV


@pytest.mark.parametrize("form", ["chain", "prefill"])
@pytest.mark.parametrize("bf16_state", [False, True])
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 128), (128, 64), (64, 64)])
def test_outputs_whose_terms_cancel(form, bf16_state, dk, dv):
    for rows, read_only in ((1, True), (20, True), (32, False), (40, False)):
        for shift in (0, 1):
            print(f"{form} bf16 {bf16_state} {dk} {dv}: {rows} rows, shift {shift}", flush=True)
            run(form, bf16_state, dk, dv, rows, read_only, shift)


def run(form, bf16_state, dk, dv, rows, read_only, shift):
    heads, batch, scale = 2, dk, 0.0921
    gen = torch.Generator().manual_seed(dk + dv + rows)
    g = torch.tensor([0.0, 0.0] if bf16_state else [-0.05, -0.011])
    q, k = torch.zeros(batch, rows, heads, dk), torch.zeros(batch, rows, heads, dk)
    key = torch.arange(batch)
    q[key, :, :, key] = torch.rand(batch, rows, heads, generator=gen) + 0.5
    k[key, 0, :, key] = 1.0
    v = torch.randn(batch, rows, heads, dv, generator=gen)
    q, k, v = q.bfloat16(), k.bfloat16(), v.bfloat16()
    near = 1 + (0 if bf16_state else 2.0 ** -14) * torch.randn(batch, heads, dv, generator=gen).double()
    state = torch.zeros(batch, heads, dv, dk, dtype=torch.float64)
    state[key, :, :, key] = -v[:, 0].double() * torch.exp(-g.double())[:, None] * near
    state = state.to(torch.bfloat16 if bf16_state else torch.float32)

    width = (2 * dk + dv) * heads
    rows_buf = torch.zeros(shift + batch * rows * width, dtype=torch.bfloat16)
    rows_buf[shift:] = torch.cat([x.reshape(batch * rows, -1) for x in (q, k, v)], 1).flatten()
    d_rows, d_state, d_g = rows_buf.to(DEV), state.to(DEV), g.to(DEV)
    off = torch.arange(batch, dtype=torch.int64, device=DEV) * (heads * dv * dk)
    cu = torch.arange(batch + 1, dtype=torch.int32, device=DEV) * rows
    out = torch.zeros(batch * rows, heads * dv, dtype=torch.bfloat16, device=DEV)
    base = ptr(d_rows, shift)
    args = (base, width, base + 2 * heads * dk, width, base + 4 * heads * dk, width, ptr(d_g), scale, ptr(d_state),
            None if read_only else ptr(d_state), ptr(off), ptr(out), heads * dv)
    name = f"glm53f_lin_{form}_batch" + ("_bf16state" if bf16_state else "")
    lead = (heads, heads, dk, dv, batch, ptr(cu))
    assert (getattr(ffi, name)(*lead, *args, None) if form == "chain" else getattr(ffi, name)(*lead, rows, *args, None, 0, None)) == 0
    hs.sync()
    got = out.cpu().double().reshape(batch, rows, heads, dv)
    for b in range(0, batch, 3):
        o, _, ao, _ = lo.attention(q[b], k[b], v[b], g, scale, state[b])
        tol = 2.0 ** -8 * o.abs() + 24 * 2.0 ** -24 * ao + 1e-30
        worst = float(((got[b] - o).abs() / tol).max())
        assert worst <= 1, f"request {b}: {worst:.2f} of the tolerance"
