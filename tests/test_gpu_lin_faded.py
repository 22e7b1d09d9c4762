"""Linear attention with one decay per head: a value that is not finite reaches every later row of its request, also those
that the decay leaves nothing of it to (0 times an infinity or a NaN is NaN), and none before it."""
import math

import pytest
import torch

from glm53f_lin import ffi

import harness as hs
from harness import ptr

pytestmark = pytest.mark.gpu
DEV = hs.DEV


@pytest.mark.parametrize("form", ["chain", "prefill"])
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("value", [math.inf, math.nan])
@pytest.mark.parametrize("rows,at,write", [(32, 3, False), (32, 20, True), (70, 40, True)])
@pytest.mark.parametrize("shift", [0, 1])
def test_what_is_not_finite_outlives_its_decay(form, what, value, rows, at, write, shift):
    heads, d = 3, 128
    gen = torch.Generator().manual_seed(rows + at)
    x = torch.randn(rows, 3, heads, d, generator=gen).bfloat16()
    x[at, 1 if what == "k" else 2, :, :] = value
    buf = torch.zeros(shift + x.numel(), dtype=torch.bfloat16)
    buf[shift:] = x.flatten()
    d_x, state = buf.to(DEV), torch.randn(heads, d, d, generator=gen).to(DEV)
    g = torch.tensor([-0.1, -60.0, -math.inf], device=DEV)
    off, cu = torch.zeros(1, dtype=torch.int64, device=DEV), torch.tensor([0, rows], dtype=torch.int32, device=DEV)
    out = torch.zeros(rows, heads * d, dtype=torch.bfloat16, device=DEV)
    width, base = 3 * heads * d, ptr(d_x, shift)
    args = (base, width, base + 2 * heads * d, width, base + 4 * heads * d, width, ptr(g), 0.1, ptr(state), ptr(state) if write else None,
            ptr(off), ptr(out), heads * d)
    if form == "chain":
        assert ffi.glm53f_lin_chain_batch(heads, heads, d, d, 1, ptr(cu), *args, None) == 0
    else:
        assert ffi.glm53f_lin_prefill_batch(heads, heads, d, d, 1, ptr(cu), rows, *args, None, 0, None) == 0
    hs.sync()
    got = torch.isfinite(out.cpu().float())
    assert bool(got[:at].all()), "an earlier row"
    assert not bool(got[at:].any()), "a later row is finite"
    if write:
        assert not bool(torch.isfinite(state).any()), "the state"
