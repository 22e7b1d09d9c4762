"""Linear attention with one decay per head (include/ext/glm53f_lin.h) through the C ABI against the recurrence in 64
bits: both forms, both state types, every head size, shared heads of q and k, lengths from none to many chunks, strides
and alignments, decays from "nothing is remembered" to "nothing is forgotten", the commit of accepted rows, and what a
call leaves alone.

Tolerances. Every term of a sum is an exact product of bf16 values times powers of the decay; R rows bring at most R
roundings to a state's entry and a read-out adds key_dim more, each 2^-24 of the sum of the terms' absolute values (the
oracle's `abs` results); the chunked form takes the decay's powers from exp, whose argument is rounded once (2^-24 of
g n, at most 0.4 of it after the factor exp(g n)), which the constant covers. The chunked form's read-outs pass through
pairs of bf16 values: two roundings of 2^-17 of their terms. A stored bf16 value is off by 2^-8 of itself more, a state
read as bf16 not at all."""
import math

import pytest
import torch

from glm53f_lin import ffi
from oracle import lin_oracle as lo

import harness as hs
from harness import ptr

pytestmark = pytest.mark.gpu
DEV = hs.DEV

SHAPES = [(4, 4, 128, 128), (6, 2, 128, 128), (3, 1, 64, 128), (4, 2, 128, 64), (5, 5, 64, 64)]


class Problem:
    """Requests of `lens` rows over a pool of states. The projection rows hold q | k | v with `pad` columns of NaN behind
    them and start `shift` elements into their buffer; rows that belong to no request, and slots that belong to none, are
    NaN too. The outputs lie `shift` elements into a buffer of sevens, with rows before and behind the requests'."""

    def __init__(self, shape, lens, bf16_state, seed, pad=0, shift=0, decay=None, sigma=1.0):
        self.heads, self.qk, self.dk, self.dv = self.shape = shape
        self.lens, self.bf16, self.scale = list(lens), bf16_state, shape[2] ** -0.5
        self.ahead, self.behind = 2, 3            # rows that belong to no request
        gen = torch.Generator().manual_seed(seed)
        total = sum(self.lens)
        self.total, self.pad, self.shift = total, pad, shift
        rnd = lambda *s: (torch.randn(*s, generator=gen) * sigma).to(torch.bfloat16)  # noqa: E731
        self.q, self.k = rnd(total, self.qk, self.dk), rnd(total, self.qk, self.dk)
        self.v = rnd(total, self.heads, self.dv)
        self.width = 2 * self.qk * self.dk + self.heads * self.dv
        self.stride = self.width + pad
        rows = torch.full((self.ahead + total + self.behind, self.stride), math.nan, dtype=torch.bfloat16)
        rows[self.ahead:self.ahead + total, :self.width] = torch.cat([self.q.flatten(1), self.k.flatten(1), self.v.flatten(1)], 1)
        self.rows = torch.full((shift + rows.numel(),), math.nan, dtype=torch.bfloat16)
        self.rows[shift:] = rows.flatten()
        self.rows = self.rows.to(DEV)
        self.g = decay if decay is not None else -torch.rand(self.heads, generator=gen) * 0.3
        self.d_g = self.g.float().to(DEV)
        self.kind = torch.bfloat16 if bf16_state else torch.float32
        self.slots = len(self.lens) + 2
        order = torch.randperm(self.slots, generator=gen)[:len(self.lens)].tolist()
        self.order = order
        n = self.heads * self.dv * self.dk
        pool = torch.full((self.slots, n), math.nan)
        for s in order:
            pool[s] = torch.randn(n, generator=gen) * 0.5
        self.pool = pool.to(self.kind)
        self.off = torch.tensor([s * n for s in order], dtype=torch.int64, device=DEV)
        cu = [self.ahead]
        for m in self.lens:
            cu.append(cu[-1] + m)
        self.cu = torch.tensor(cu, dtype=torch.int32, device=DEV)
        self.out_stride = self.heads * self.dv + pad
        self.out = torch.full((shift + (self.ahead + total + self.behind) * self.out_stride,), 7.0, dtype=torch.bfloat16, device=DEV)

    def fn(self, name):
        return getattr(ffi, f"glm53f_lin_{name}_batch" + ("_bf16state" if self.bf16 else ""))

    def row_args(self):
        base = ptr(self.rows, self.shift)
        k, v = base + 2 * self.qk * self.dk, base + 4 * self.qk * self.dk
        return (base, self.stride, k, self.stride, v, self.stride, ptr(self.d_g), self.scale)

    def call(self, form, state_in, state_out, max_rows=None, stream=None, workspace=None):
        tail = (ptr(state_in), None if state_out is None else ptr(state_out), ptr(self.off), ptr(self.out, self.shift), self.out_stride)
        if form == "chain":
            return self.fn("chain")(*self.shape, len(self.lens), ptr(self.cu), *self.row_args(), *tail, stream)
        most = max(self.lens, default=0) if max_rows is None else max_rows
        need = ffi.glm53f_lin_prefill_workspace_bytes(self.heads, self.dk, self.dv, len(self.lens), most)
        if workspace is None:
            workspace = torch.full((need,), 255, dtype=torch.uint8, device=DEV)       # NaN bits
        return self.fn("prefill")(*self.shape, len(self.lens), ptr(self.cu), most, *self.row_args(), *tail,
                                  ptr(workspace) if need else None, need, stream)

    def advance(self, keep, state_in, state_out, stream=None):
        base = ptr(self.rows, self.shift)
        k, v = base + 2 * self.qk * self.dk, base + 4 * self.qk * self.dk
        return self.fn("advance")(*self.shape, 1, len(self.lens), ptr(self.cu), ptr(keep), k, self.stride, 0, v, self.stride, 0,
                                  ptr(self.d_g), ptr(state_in), ptr(state_out), 0, ptr(self.off), stream)

    def out_rows(self):
        """The requests' rows; checks that nothing else was written."""
        flat = self.out.float().cpu()
        assert bool((flat[:self.shift] == 7).all())
        rows = flat[self.shift:].reshape(-1, self.out_stride)
        assert bool((rows[:self.ahead] == 7).all()) and bool((rows[self.ahead + self.total:] == 7).all())
        assert bool((rows[:, self.heads * self.dv:] == 7).all())
        return rows[self.ahead:self.ahead + self.total, :self.heads * self.dv].reshape(self.total, self.heads, self.dv).double()

    def oracle(self, b, rows=None):
        lo_row = sum(self.lens[:b])
        hi = lo_row + (self.lens[b] if rows is None else rows)
        state = self.pool[self.order[b]].reshape(self.heads, self.dv, self.dk)
        return lo.attention(self.q[lo_row:hi], self.k[lo_row:hi], self.v[lo_row:hi], self.g, self.scale, state)

    def state_of(self, pool, b):
        return pool[self.order[b]].reshape(self.heads, self.dv, self.dk)


def within(got, want, tol, what):
    err = (got - want).abs()
    worst = float((err / tol).max()) if err.numel() else 0.0
    assert bool((err <= tol).all()), f"{what}: {worst:.2f} of the tolerance"


def check_outputs(p, form, label, rows_of=None):
    out = p.out_rows()
    for b, n in enumerate(p.lens):
        first = sum(p.lens[:b])
        n = n if rows_of is None else min(n, rows_of)
        o, _, ao, _ = p.oracle(b)
        tol = 2.0 ** -8 * o.abs() + ((n + p.dk + 16) * 2.0 ** -24 + (2.0 ** -16 if form == "prefill" else 0)) * ao + 1e-30
        within(out[first:first + n], o[:n], tol[:n], f"{label}, request {b}")


def check_states(p, pool, label, kept=None):
    pool = pool.cpu().double()
    for b, n in enumerate(p.lens):
        n = n if kept is None else kept[b]
        _, s, _, a = p.oracle(b)
        tol = (n + 16) * 2.0 ** -24 * a[n] + (2.0 ** -8 * s[n].abs() if p.bf16 else 0) + 1e-30
        if n == 0:
            assert torch.equal(p.state_of(pool, b), s[0]), f"{label}, request {b}: moved without rows"
        else:
            within(p.state_of(pool, b), s[n], tol, f"{label}, state of request {b}")
    for s in range(p.slots):
        if s not in p.order:
            assert bool(pool[s].isnan().all()), f"{label}: wrote slot {s}"


LENS = {"chain": [[1], [1, 1, 1, 1, 1], [3, 0, 1, 8], [17, 2]],
        "prefill": [[1], [2, 1, 16, 0, 7], [64, 65, 63], [15, 33, 100], [0, 257], [777]]}


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("bf16_state", [False, True])
@pytest.mark.parametrize("form", ["chain", "prefill"])
@pytest.mark.parametrize("in_place", [True, False])
def test_outputs_and_states_of_batches(shape, bf16_state, form, in_place):
    for i, lens in enumerate(LENS[form]):
        p = Problem(shape, lens, bf16_state, seed=100 + i)
        print(f"{form} {shape} {lens} bf16 {bf16_state} in place {in_place}", flush=True)
        pool = p.pool.to(DEV)
        after = pool if in_place else torch.full_like(pool, math.nan)
        assert p.call(form, pool, after) == 0
        hs.sync()
        check_outputs(p, form, f"{lens}")
        check_states(p, after, f"{lens}")
        if not in_place:
            assert torch.equal(hs_bits(pool), hs_bits(p.pool.to(DEV))), "the states read were written"


def hs_bits(t):
    return t.contiguous().view(torch.int32 if t.element_size() == 4 else torch.int16)


@pytest.mark.parametrize("form", ["chain", "prefill"])
@pytest.mark.parametrize("pad,shift", [(8, 8), (3, 0), (8, 1), (5, 7), (4, 2)])
@pytest.mark.parametrize("shape", [(6, 2, 128, 128), (3, 1, 64, 64)])
def test_strides_and_alignments(form, pad, shift, shape):
    p = Problem(shape, [1, 5, 40] if form == "prefill" else [1, 5], False, seed=7, pad=pad, shift=shift)
    pool = p.pool.to(DEV)
    assert p.call(form, pool, pool) == 0
    hs.sync()
    check_outputs(p, form, "strides")
    check_states(p, pool, "strides")
    if form == "chain":
        q = Problem(shape, [1, 5], False, seed=7)
        other = q.pool.to(DEV)
        assert q.call(form, other, other) == 0
        hs.sync()
        assert torch.equal(hs_bits(other), hs_bits(pool)) and torch.equal(q.out_rows(), p.out_rows())


@pytest.mark.parametrize("form", ["chain", "prefill"])
@pytest.mark.parametrize("bf16_state", [False, True])
def test_decays_from_nothing_remembered_to_nothing_forgotten(form, bf16_state):
    g = torch.tensor([-math.inf, 0.0, -1e-4, -0.7, -20.0, -200.0])
    lens = [1, 4, 9] if form == "chain" else [1, 4, 150]
    p = Problem((6, 6, 128, 128), lens, bf16_state, seed=11, decay=g)
    pool = p.pool.to(DEV)
    assert p.call(form, pool, pool) == 0
    hs.sync()
    check_outputs(p, form, "decays")
    check_states(p, pool, "decays")


@pytest.mark.parametrize("form", ["chain", "prefill"])
@pytest.mark.parametrize("sigma", [1e-12, 1e8])
def test_magnitudes_far_from_one(form, sigma):
    """bf16 rows of any magnitude that the products' f32 range holds."""
    p = Problem((4, 4, 128, 128), [5, 70] if form == "prefill" else [5], False, seed=13, sigma=sigma)
    p.pool = p.pool * (sigma * sigma)
    pool = p.pool.to(DEV)
    assert p.call(form, pool, pool) == 0
    hs.sync()
    check_outputs(p, form, "magnitudes")
    check_states(p, pool, "magnitudes")


@pytest.mark.parametrize("form", ["chain", "prefill"])
def test_a_verify_window_leaves_the_states_alone(form):
    p = Problem((6, 2, 128, 128), [3, 1, 16, 0, 9], True, seed=17)
    pool = p.pool.to(DEV)
    assert p.call(form, pool, None) == 0
    hs.sync()
    check_outputs(p, form, "verify")
    assert torch.equal(hs_bits(pool), hs_bits(p.pool.to(DEV)))


@pytest.mark.parametrize("shape", [(6, 2, 128, 128), (64, 64, 128, 128), (3, 1, 64, 64)])
def test_a_window_has_the_bits_of_single_rows_with_f32_states(shape):
    p = Problem(shape, [6, 2, 11], False, seed=19)
    pool, serial = p.pool.to(DEV), p.pool.to(DEV)
    assert p.call("chain", pool, pool) == 0
    hs.sync()
    want = p.out_rows()
    starts = p.cu.cpu().tolist()
    for t in range(max(p.lens)):
        alive = [b for b, n in enumerate(p.lens) if n > t]
        for b in alive:
            one = torch.tensor([starts[b] + t, starts[b] + t + 1], dtype=torch.int32, device=DEV)
            off = p.off[b:b + 1].contiguous()
            assert p.fn("chain")(*p.shape, 1, ptr(one), *p.row_args(), ptr(serial), ptr(serial), ptr(off), ptr(p.out), p.out_stride,
                                 None) == 0
    hs.sync()
    assert torch.equal(hs_bits(serial), hs_bits(pool)) and torch.equal(p.out_rows(), want)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("bf16_state", [False, True])
def test_the_commit_of_accepted_rows(shape, bf16_state):
    lens, keep = [4, 1, 16, 0, 9, 5], [4, 0, 7, 3, -2, 50]         # out of range counts are taken to the nearer end
    kept = [max(0, min(a, b)) for a, b in zip(lens, keep)]
    p = Problem(shape, lens, bf16_state, seed=23)
    pool, other = p.pool.to(DEV), p.pool.to(DEV)
    d_keep = torch.tensor(keep, dtype=torch.int32, device=DEV)
    assert p.advance(d_keep, pool, pool) == 0
    copy = torch.full_like(pool, math.nan)
    assert p.advance(d_keep, other, copy) == 0
    hs.sync()
    check_states(p, pool, "commit", kept)
    assert torch.equal(hs_bits(copy[p.order]), hs_bits(pool[p.order]))
    # the bits of the chain over the same rows
    short = Problem(shape, lens, bf16_state, seed=23)
    cu = short.cu.cpu().tolist()
    for b, n in enumerate(kept):
        one = torch.tensor([cu[b], cu[b] + n], dtype=torch.int32, device=DEV)
        off = short.off[b:b + 1].contiguous()
        assert short.fn("chain")(*short.shape, 1, ptr(one), *short.row_args(), ptr(other), ptr(other), ptr(off), ptr(short.out),
                                 short.out_stride, None) == 0
    hs.sync()
    assert torch.equal(hs_bits(other[p.order]), hs_bits(pool[p.order]))


def test_the_commit_of_all_layers_in_one_launch():
    layers, lens, keep = 3, [4, 6, 1], [2, 6, 0]
    ps = [Problem((4, 2, 128, 64), lens, True, seed=31 + i) for i in range(layers)]
    d_keep = torch.tensor(keep, dtype=torch.int32, device=DEV)
    one = ps[0]
    rows = torch.stack([p.rows for p in ps])
    g = torch.stack([p.d_g for p in ps])
    arena = torch.stack([p.pool for p in ps]).to(DEV)
    arena[:, [s for s in range(one.slots) if s not in one.order]] = math.nan
    base = ptr(rows)
    off = one.off
    for p in ps:                                  # the layers share the slots
        p.pool = torch.stack([p.pool[p.order[one.order.index(s)]] if s in one.order else torch.full_like(p.pool[0], math.nan)
                              for s in range(one.slots)])
        p.order = one.order
    arena = torch.stack([p.pool for p in ps]).to(DEV)
    qk = 2 * one.qk * one.dk
    assert ffi.glm53f_lin_advance_batch_bf16state(*one.shape, layers, len(lens), ptr(one.cu), ptr(d_keep), base + qk, one.stride,
                                                  rows.stride(0), base + 2 * qk, one.stride, rows.stride(0), ptr(g), ptr(arena),
                                                  ptr(arena), arena.stride(0), ptr(off), None) == 0
    hs.sync()
    for layer, p in enumerate(ps):
        check_states(p, arena[layer], f"layer {layer}", keep)


def test_rows_beyond_max_rows_are_left_out():
    p = Problem((4, 4, 128, 128), [5, 90, 20], False, seed=37)
    pool = p.pool.to(DEV)
    assert p.call("prefill", pool, pool, max_rows=20) == 0
    hs.sync()
    out = p.out_rows()
    for b, first in enumerate((0, 5, 95)):
        n = min(p.lens[b], 20)
        o, s, ao, a = p.oracle(b)
        within(out[first:first + n], o[:n], 2.0 ** -8 * o[:n].abs() + 2.0 ** -15 * ao[:n], f"request {b}")
        within(p.state_of(pool.cpu().double(), b), s[n], 36 * 2.0 ** -24 * a[n], f"state {b}")
    assert bool((out[25:95] == 7).all())


@pytest.mark.parametrize("bf16_state", [False, True])
def test_a_long_prompt_in_segments_agrees_with_one_pass(bf16_state):
    """Few heads and many rows: the sequence is cut over the GPU and joined."""
    p = Problem((3, 3, 128, 128), [5000, 0, 1237], bf16_state, seed=41, decay=torch.tensor([-1e-3, -0.05, 0.0]))
    pool = p.pool.to(DEV)
    assert p.call("prefill", pool, pool) == 0
    hs.sync()
    check_outputs(p, "prefill", "long")
    check_states(p, pool, "long")


def test_offsets_past_32_bits():
    """A pool of states and a row buffer whose far ends lie beyond 2^31 elements."""
    heads, dk, dv = 2, 64, 64
    n = heads * dk * dv
    far = (1 << 31) + 8 * 1000
    pool = torch.zeros(far + n, dtype=torch.bfloat16, device=DEV)
    gen = torch.Generator().manual_seed(43)
    state = torch.randn(heads, dv, dk, generator=gen).to(torch.bfloat16)
    pool[far:] = state.flatten().to(DEV)
    off = torch.tensor([far], dtype=torch.int64, device=DEV)
    stride, rows = (1 << 30) + 8, 3
    buf = torch.zeros(2 * stride + 3 * heads * dk, dtype=torch.bfloat16, device=DEV)
    parts = torch.randn(rows, 3 * heads * dk, generator=gen).to(torch.bfloat16)
    for t in range(rows):
        buf[t * stride:t * stride + parts.shape[1]] = parts[t].to(DEV)
    cu = torch.tensor([0, rows], dtype=torch.int32, device=DEV)
    g = torch.tensor([-0.1, -0.5], device=DEV)
    q, k, v = (parts[:, i * heads * dk:(i + 1) * heads * dk].reshape(rows, heads, dk) for i in range(3))
    o, s, ao, a = lo.attention(q, k, v, g.cpu(), 0.5, state)
    out = torch.zeros(rows, heads * dv, dtype=torch.bfloat16, device=DEV)
    base = ptr(buf)
    for form in ("chain", "prefill"):
        pool[far:] = state.flatten().to(DEV)
        rows_args = (base, stride, base + 2 * heads * dk, stride, base + 4 * heads * dk, stride, ptr(g), 0.5, ptr(pool), ptr(pool), ptr(off),
                     ptr(out), heads * dv)
        if form == "chain":
            assert ffi.glm53f_lin_chain_batch_bf16state(heads, heads, dk, dv, 1, ptr(cu), *rows_args, None) == 0
        else:
            assert ffi.glm53f_lin_prefill_batch_bf16state(heads, heads, dk, dv, 1, ptr(cu), rows, *rows_args, None, 0, None) == 0
        hs.sync()
        got = out.float().cpu().double().reshape(rows, heads, dv)
        within(got, o, 2.0 ** -8 * o.abs() + 2.0 ** -15 * ao, form)
        within(pool[far:].float().cpu().double().reshape(heads, dv, dk), s[-1], 2.0 ** -8 * s[-1].abs() + 2.0 ** -19 * a[-1], form)


def test_a_captured_round_replays_like_eager_rounds():
    """Prompt, decode window and commit recorded once; `keep` is rewritten between the replays."""
    lens = [3, 1, 16]
    keeps = [[3, 0, 5], [1, 1, 16], [0, 0, 0]]

    def buffers():
        p, long = Problem((4, 2, 128, 128), lens, False, seed=51), Problem((4, 2, 128, 128), [900], False, seed=52)
        need = ffi.glm53f_lin_prefill_workspace_bytes(4, 128, 128, 1, 900)
        return dict(p=p, long=long, pool=p.pool.to(DEV), long_pool=long.pool.to(DEV), keep=torch.zeros(3, dtype=torch.int32, device=DEV),
                    ws=torch.zeros(max(need, 1), dtype=torch.uint8, device=DEV))

    def step(b, stream):
        assert b["long"].call("prefill", b["long_pool"], b["long_pool"], stream=stream, workspace=b["ws"]) == 0
        assert b["p"].call("prefill", b["pool"], None, stream=stream) == 0
        assert b["p"].advance(b["keep"], b["pool"], b["pool"], stream=stream) == 0
        assert b["p"].call("chain", b["pool"], b["pool"], stream=stream) == 0

    g, e = buffers(), buffers()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(g, torch.cuda.current_stream().cuda_stream)
    for replay, keep in enumerate(keeps, 1):
        for b in (g, e):
            b["keep"].copy_(torch.tensor(keep, dtype=torch.int32))
        graph.replay()
        step(e, None)
        assert math.isfinite(torch.randn(1 << 16, device=DEV).sum().item())
        hs.sync()
        for name in ("pool", "long_pool"):
            assert torch.equal(hs_bits(g[name]), hs_bits(e[name])), f"{name} after replay {replay}"
        assert torch.equal(g["p"].out, e["p"].out) and torch.equal(g["long"].out, e["long"].out), f"outputs of replay {replay}"


def test_two_calls_on_two_streams():
    ps = [Problem((4, 4, 128, 128), [400, 3], False, seed=61 + i) for i in range(2)]
    pools = [p.pool.to(DEV) for p in ps]
    streams = [torch.cuda.Stream() for _ in ps]
    hs.sync()
    for p, pool, s in zip(ps, pools, streams):
        with torch.cuda.stream(s):
            assert p.call("prefill", pool, pool, stream=s.cuda_stream) == 0
            assert p.call("chain", pool, None, stream=s.cuda_stream) == 0
    hs.sync()
    for p, pool in zip(ps, pools):
        check_states(p, pool, "streams")


def test_bits_do_not_depend_on_the_requests_beside():
    """A decode row's state and output alone and in a large batch (which cuts the heads more coarsely)."""
    p = Problem((64, 64, 128, 128), [1] * 12, False, seed=71)
    pool, alone = p.pool.to(DEV), p.pool.to(DEV)
    assert p.call("chain", pool, pool) == 0
    hs.sync()
    want = p.out_rows()
    cu = p.cu.cpu().tolist()
    for b in range(12):
        one = torch.tensor([cu[b], cu[b] + 1], dtype=torch.int32, device=DEV)
        off = p.off[b:b + 1].contiguous()
        assert ffi.glm53f_lin_chain_batch(*p.shape, 1, ptr(one), *p.row_args(), ptr(alone), ptr(alone), ptr(off), ptr(p.out), p.out_stride,
                                          None) == 0
    hs.sync()
    assert torch.equal(hs_bits(alone), hs_bits(pool)) and torch.equal(p.out_rows(), want)


@pytest.mark.parametrize("form", ["prefill", "chain"])
@pytest.mark.parametrize("shape", [(4, 2, 128, 128), (3, 1, 64, 64), (2, 2, 128, 64), (2, 1, 64, 128)])
@pytest.mark.parametrize("what", ["v", "k", "q"])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_a_value_that_is_not_finite_reaches_no_earlier_row(form, shape, what, value):
    """Planted in one row of a prompt of several chunks (and segments), and in the last rows of a short one: the rows before
    it, the other heads and requests are right as without it; the rows that the recurrence carries it to are not finite."""
    lens, shift = [700, 5, 40], 0 if value > 0 else 1
    clean, bad = (Problem(shape, lens, False, seed=91, shift=shift) for _ in range(2))
    heads, qk, dk, dv = shape
    group, col = heads // qk, {"q": 0, "k": qk * dk, "v": 2 * qk * dk}[what]
    head, lane = (heads - 1, dv - 3) if what == "v" else (qk - 1, dk - 5)
    rows = [(0, 333), (0, 699), (1, 3), (2, 0)] if what == "q" else [(0, 333), (1, 3), (2, 39)]
    first = [0, 700, 705]
    plant = bad.rows.cpu()
    at = lambda r: shift + (bad.ahead + r) * bad.stride + col + head * (dv if what == "v" else dk) + lane  # noqa: E731
    for b, t in rows:
        plant[at(first[b] + t)] = value
    bad.rows.copy_(plant)
    for p in (clean, bad):
        pool = p.pool.to(DEV)
        need = ffi.glm53f_lin_prefill_workspace_bytes(*(shape[0], dk, dv), 3, 700)
        ws = torch.zeros(max(need, 16), dtype=torch.uint8, device=DEV)
        assert (p.call(form, pool, pool, workspace=ws) if form == "prefill" else p.call(form, pool, pool)) == 0
    hs.sync()
    want, got = (p.out_rows().reshape(745, heads, dv) for p in (clean, bad))
    touched = torch.zeros(745, heads, dv, dtype=torch.bool)
    for b, t in rows:
        r, end = first[b] + t, first[b] + lens[b]
        if what == "v":
            touched[r:end, head, lane] = True
        elif what == "k":
            touched[r:end, head * group:(head + 1) * group] = True
        else:
            touched[r, head * group:(head + 1) * group] = True
    assert bool(torch.isfinite(want).all())
    for b, n in enumerate(lens):
        here, free = slice(first[b], first[b] + n), ~touched[first[b]:first[b] + n]
        o, _, ao, _ = clean.oracle(b)
        tol = 2.0 ** -8 * o.abs() + ((n + dk + 16) * 2.0 ** -24 + (2.0 ** -16 if form == "prefill" else 0)) * ao + 1e-30
        within(got[here][free], o[free], tol[free], f"what it cannot reach of request {b}")
    assert not bool(torch.isfinite(got[touched]).any()), "a row that it reaches is finite"


@pytest.mark.parametrize("form", ["prefill", "chain"])
def test_windows_of_one_state(form):
    """Several windows behind the same state (drafts of one prompt): nothing is written, so the regions may be the same."""
    p = Problem((4, 2, 128, 128), [5, 5, 16], False, seed=97)
    p.off[1:] = p.off[0]
    pool = p.pool.to(DEV)
    assert p.call(form, pool, None) == 0
    hs.sync()
    slot = p.pool[p.order[0]]
    state = slot.reshape(4, 128, 128)
    at = 0
    for m in p.lens:
        o, _, ao, _ = lo.attention(p.q[at:at + m], p.k[at:at + m], p.v[at:at + m], p.g, p.scale, state)
        got = p.out_rows().reshape(-1, 4, 128)[at:at + m].double()
        within(got, o, 2.0 ** -8 * o.abs() + (2.0 ** -15 + (m + 144) * 2.0 ** -24) * ao, form)
        at += m
    assert torch.equal(pool[p.order[0]].cpu(), slot)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("bf16_state", [False, True])
@pytest.mark.parametrize("pad,shift", [(0, 0), (8, 8), (3, 1)])
@pytest.mark.parametrize("lens", [[1, 16, 0, 5, 32], [7, 33, 2]])
def test_windows_that_only_read_their_states(shape, bf16_state, pad, shift, lens):
    """Windows of one chunk (no state is written) in every head size, and one that is a row longer."""
    p = Problem(shape, lens, bf16_state, seed=101, pad=pad, shift=shift)
    pool = p.pool.to(DEV)
    assert p.call("prefill", pool, None) == 0
    hs.sync()
    check_outputs(p, "prefill", f"windows {lens}")
    assert torch.equal(hs_bits(pool), hs_bits(p.pool.to(DEV)))


@pytest.mark.parametrize("bf16_state", [False, True])
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_a_draft_that_is_not_finite_leaves_the_rows_before_it(bf16_state, value):
    """An infinity or a NaN in v of a window's later row: the rows before it, which may be accepted, are right."""
    clean, bad = (Problem((4, 2, 128, 128), [16, 9, 30], bf16_state, seed=103) for _ in range(2))
    row, head, lane = 11, 2, 77
    at = (bad.ahead + row) * bad.stride + 2 * 2 * 128 + head * 128 + lane
    bad.rows[at] = value
    for p in (clean, bad):
        assert p.call("prefill", p.pool.to(DEV), None) == 0
    hs.sync()
    got = bad.out_rows()
    reached = got[row:16, head, lane]
    assert not bool(torch.isfinite(reached).any())
    for b, n in enumerate(clean.lens):
        first = sum(clean.lens[:b])
        o, _, ao, _ = clean.oracle(b)
        here = got[first:first + n].clone()
        if b == 0:
            here[row:, head, lane] = o[row:, head, lane]
        within(here, o, 2.0 ** -8 * o.abs() + ((n + 144) * 2.0 ** -24 + 2.0 ** -16) * ao + 1e-30, f"request {b}")
