"""Linear attention with one decay per head, a prompt whose keys and values are larger than the caches behind the L2: rows and states of some heads against the recurrence in 64 bits, all others finite, and what
lies around the rows as it was.

Tolerances as for any prompt: R rows bring at most R roundings of 2^-24 to a state's entry, a read-out key_dim more and the
chunks' sums 48, all of the sum of the terms' absolute values; an output's own rounding is 2^-8 of itself."""
import math

import pytest
import torch

from glm53f_lin import ffi
from oracle import lin_oracle as lo

import harness as hs
from harness import ptr

pytestmark = pytest.mark.gpu
DEV = hs.DEV


@pytest.mark.parametrize("shift", [0, 1])
def test_a_prompt_larger_than_the_caches(shift):
    heads, d, rows = 64, 128, 6301
    assert rows * heads * d * 2 * 2 > 192 << 20
    gen = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, 3 * heads * d, generator=gen).bfloat16()
    width = 3 * heads * d + (0 if shift == 0 else 3)
    d_x = torch.full((shift + rows * width,), math.nan, dtype=torch.bfloat16, device=DEV)
    d_x[shift:].view(rows, width)[:, :3 * heads * d] = x.to(DEV)
    state = torch.randn(heads, d, d, generator=gen)
    g = -torch.rand(heads, generator=gen) * 0.02
    d_state, d_g = state.to(DEV), g.to(DEV)
    off, cu = torch.zeros(1, dtype=torch.int64, device=DEV), torch.tensor([0, rows], dtype=torch.int32, device=DEV)
    ld = heads * d + 8
    out = torch.full((rows + 2, ld), 7.0, dtype=torch.bfloat16, device=DEV)
    need = ffi.glm53f_lin_prefill_workspace_bytes(heads, d, d, 1, rows)
    assert need > 0
    ws = torch.full((need,), 255, dtype=torch.uint8, device=DEV)
    base = ptr(d_x, shift)
    assert ffi.glm53f_lin_prefill_batch(heads, heads, d, d, 1, ptr(cu), rows, base, width, base + 2 * heads * d, width, base + 4 * heads * d,
                                        width, ptr(d_g), 0.09, ptr(d_state), ptr(d_state), ptr(off), ptr(out, ld), ld, ptr(ws), need, None) == 0
    hs.sync()
    got = out.cpu().double()
    assert bool((got[0] == 7).all()) and bool((got[-1] == 7).all()) and bool((got[1:-1, heads * d:] == 7).all())
    got = got[1:-1, :heads * d].reshape(rows, heads, d)
    assert bool(torch.isfinite(got).all()) and bool(torch.isfinite(d_state).all())
    some = [0, 29, 63]
    q, k, v = (x[:, i * heads * d:(i + 1) * heads * d].reshape(rows, heads, d)[:, some] for i in range(3))
    s, a = state[some], state[some].abs()
    for first in range(0, rows, 700):                    # the oracle keeps every row's state
        last = min(first + 700, rows)
        part = [t[first:last] for t in (q, k, v)]
        o, st, _, _ = lo.attention(*part, g[some], 0.09, s)
        ao, ast, _, _ = lo.attention(*(t.abs() for t in part), g[some], 0.09, a)       # every term's absolute value
        err = (got[first:last, some] - o).abs()
        tol = 2.0 ** -8 * o.abs() + (last + d + 48) * 2.0 ** -24 * ao
        assert bool((err <= tol).all()), f"rows from {first}: {float((err / tol).max()):.2f} of the tolerance"
        s, a = st[-1], ast[-1]
    err, tol = (d_state.cpu().double()[some] - s).abs(), (rows + 16) * 2.0 ** -24 * a
    assert bool((err <= tol).all()), f"states: {float((err / tol).max()):.2f} of the tolerance"
