"""Probabilities of logits and the verification of drafted tokens (include/ext/glm53f_spec.h) through the C ABI against
64-bit models.

Tolerances. A probability is exp(z) / sum with z = (x - top) / T <= 0: z takes up to four roundings, each 2^-24 of |z|,
the exponential two of its own, the sum of the segments' at most 2^-24 for every addition of a chain of 64 (a thread's
share) + 32 (joins), and the product one: 2^-24 (4 |z| + 112) of the probability. The accepted counts and the tokens are
whole numbers: equal."""
import math

import pytest
import torch

from glm53f_kda import ffi as kda
from glm53f_spec import ffi
from oracle import lin_oracle as lo

import harness as hs
from harness import ptr

pytestmark = pytest.mark.gpu
DEV = hs.DEV


def spec_probs(logits, temperature, pad=0, shift=0, in_place=False, stream=None):
    """logits [m][vocab] on the host -> f32 probabilities on the host."""
    rows, vocab = logits.shape
    ld = vocab + pad
    buf = torch.full((shift + rows * ld,), 7.0, dtype=logits.dtype)
    buf[shift:].view(rows, ld)[:, :vocab] = logits
    buf = buf.to(DEV)
    out = buf if in_place else torch.full((shift + rows * ld,), 7.0, device=DEV)
    need = ffi.glm53f_spec_probs_workspace_bytes(rows, vocab)
    ws = torch.full((need,), 255, dtype=torch.uint8, device=DEV)
    d_t = None if temperature is None else temperature.float().to(DEV)
    assert ffi.glm53f_spec_probs(rows, vocab, ptr(buf, shift), int(logits.dtype == torch.float32), ld, ptr(d_t), ptr(out, shift), ld,
                                 ptr(ws), need, stream) == 0
    hs.sync()
    flat = out.cpu()
    got = flat[shift:].view(rows, ld)
    assert bool((flat[:shift] == 7).all()) and bool((got[:, vocab:] == 7).all()), "wrote outside the rows"
    return got[:, :vocab]


def check_probs(logits, temperature, **kw):
    got = spec_probs(logits, temperature, **kw).double()
    t = torch.ones(len(logits)) if temperature is None else temperature
    want = lo.probs(logits, t)
    x = logits.double()
    z = ((x - x.amax(1, keepdim=True)) / t.double()[:, None]).abs()
    tol = 2.0 ** -24 * (4 * z + 112) * want + 2.0 ** -126
    tol = torch.where(want == 0, 2.0 ** -126, tol)
    err = (got - want).abs()
    assert bool((err <= tol).all()), f"{float((err / tol).max()):.2f} of the tolerance"


@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 4096, 4097, 50001, 151936])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 5])
def test_probabilities(vocab, kind, rows):
    gen = torch.Generator().manual_seed(vocab + rows)
    x = (torch.randn(rows, vocab, generator=gen) * 4).to(kind)
    check_probs(x, None)
    check_probs(x, torch.rand(rows, generator=gen) * 2 + 0.1)


def test_probabilities_of_many_rows():
    gen = torch.Generator().manual_seed(1)
    check_probs(torch.randn(300, 9001, generator=gen).bfloat16(), torch.rand(300, generator=gen) + 0.2)


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pad,shift", [(8, 0), (1, 0), (0, 1), (5, 3), (4, 2)])
def test_probabilities_strides_alignments_and_in_place(kind, pad, shift):
    gen = torch.Generator().manual_seed(2)
    x = (torch.randn(3, 5003, generator=gen) * 3).to(kind)
    check_probs(x, torch.tensor([0.5, 1.0, 2.0]), pad=pad, shift=shift)
    if kind == torch.float32:
        check_probs(x, torch.tensor([0.5, 1.0, 2.0]), pad=pad, shift=shift, in_place=True)


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_probabilities_of_masked_rows(kind):
    low = torch.finfo(kind).min
    x = torch.full((8, 6000), -math.inf, dtype=kind)
    x[1, 5999] = -3.0                             # one entry left, in the last segment
    x[2, 17] = low                                # the type's lowest value and nothing else
    x[3, :] = low                                 # all masked by the lowest value: uniform
    x[4, ::2] = 1.0                               # half of the row
    x[5, 100:200] = torch.finfo(kind).max         # differences overflow
    x[5, 0] = low
    x[6, 4096:] = 0.5                             # the first segment is empty
    want = lo.probs(x, torch.ones(8))             # row 0 and row 7: nothing left, all zeros
    for t in (torch.ones(8), torch.full((8,), 1e-30), torch.full((8,), 1e-42)):
        got = spec_probs(x, t).double()
        assert bool(((got - want).abs() <= 2.0 ** -24 * 112 * want).all()), float((got - want).abs().max())


def test_probabilities_with_nan_and_infinity():
    x = torch.zeros(4, 5000)
    x[0, 4500], x[1, 3], x[3, 1] = math.nan, math.inf, math.nan
    x[3, 2:] = -math.inf
    got = spec_probs(x, None)
    assert bool(got[0].isnan().all()) and bool(got[1].isnan().all()) and bool(got[3].isnan().all())
    assert bool((got[2] == spec_probs(torch.zeros(1, 5000), None)[0]).all())


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_greedy_rows(kind):
    x = torch.randn(6, 9000, generator=torch.Generator().manual_seed(3)).to(kind)
    x[0, 8000] = x[0, 300] = 50.0                 # equal ones: the lowest index
    x[1, 4096] = 60.0
    x[2, :] = -math.inf
    x[3, 7] = math.nan
    x[4, 5] = math.inf
    t = torch.tensor([0.0, 0.0, 0.0, 0.0, 0.0, -1.0])
    got = spec_probs(x, t).double()
    assert torch.equal(got, lo.probs(x, t))


# ---------------------------------------------------------------------------------------------------------------

class Round:
    def __init__(self, lens, vocab, seed, draft=True, pad=0, shift=0, near=0.5):
        gen = torch.Generator().manual_seed(seed)
        self.lens, self.vocab = lens, vocab
        n = sum(lens)
        z = torch.randn(n, vocab, generator=gen) * 2
        self.target = torch.softmax(z, 1)
        self.draft = torch.softmax(z + near * torch.randn(n, vocab, generator=gen), 1) if draft else None
        source = self.draft if draft else self.target
        self.tokens = torch.multinomial(source, 1, generator=gen).flatten().to(torch.int32) if n else torch.zeros(0, dtype=torch.int32)
        self.uniform = torch.rand(n, generator=gen)
        self.pad, self.shift = pad, shift

    def run(self, stream=None, ahead=0):
        def dev(t):
            ld = self.vocab + self.pad
            flat = torch.full((self.shift + (ahead + len(t) + 1) * ld,), math.nan)
            flat[self.shift:].view(-1, ld)[ahead:ahead + len(t), :self.vocab] = t
            return flat.to(DEV), ld

        batch = len(self.lens)
        cu = torch.tensor([ahead + sum(self.lens[:i]) for i in range(batch + 1)], dtype=torch.int32, device=DEV)
        fill = torch.zeros(ahead)
        tokens = torch.cat([fill.to(torch.int32), self.tokens]).to(DEV)
        uniform = torch.cat([fill, self.uniform]).to(DEV)
        p, ldp = dev(self.target)
        q, ldq = dev(self.draft) if self.draft is not None else (None, 0)
        keep, token = (torch.full((batch + 1,), -7, dtype=torch.int32, device=DEV) for _ in range(2))
        need = ffi.glm53f_spec_accept_workspace_bytes(batch, self.vocab)
        ws = torch.full((need,), 255, dtype=torch.uint8, device=DEV)
        assert ffi.glm53f_spec_accept(batch, self.vocab, ptr(cu), ptr(tokens), ptr(p, self.shift), ldp,
                                      None if q is None else ptr(q, self.shift), ldq, ptr(uniform), ptr(keep), ptr(token), ptr(ws), need,
                                      stream) == 0
        hs.sync()
        assert keep[batch].item() == -7 and token[batch].item() == -7
        return keep[:batch].tolist(), token[:batch].tolist()

    def want(self):
        keep, token = [], []
        for b, n in enumerate(self.lens):
            lo_row = sum(self.lens[:b])
            s = slice(lo_row, lo_row + n)
            k, t = lo.accept(self.tokens[s], self.target[s], None if self.draft is None else self.draft[s], self.uniform[s])
            keep.append(k)
            token.append(t)
        return keep, token


@pytest.mark.parametrize("vocab", [1, 5, 255, 4096, 4100, 32000, 151936])
@pytest.mark.parametrize("draft", [True, False])
def test_accepted_counts_and_next_tokens(vocab, draft):
    lens = [1, 5, 0, 9, 2, 16] if vocab < 100000 else [1, 5, 0, 4]
    for seed in range(4 if vocab < 100000 else 2):
        r = Round(lens, vocab, seed=seed, draft=draft)
        got, want = r.run(), r.want()
        print(f"vocab {vocab} draft {draft} seed {seed}: keep {got[0]}, next {got[1]}", flush=True)
        assert got == want


def test_windows_longer_than_a_wave():
    r = Round([150, 65, 64, 1], 40, seed=5, near=0.0)
    r.uniform[1:149] = 0.0                        # accepted but for the last one
    r.uniform[149] = 0.999999
    r.draft[149] = 0.0
    r.draft[149, int(r.tokens[149])] = 1.0
    got = r.run()
    assert got == r.want() and got[0][0] >= 149


@pytest.mark.parametrize("pad,shift,ahead", [(0, 0, 3), (3, 0, 0), (8, 1, 2), (5, 2, 1)])
def test_strides_and_rows_ahead(pad, shift, ahead):
    r = Round([3, 6, 1], 9001, seed=6, pad=pad, shift=shift)
    assert r.run(ahead=ahead) == r.want()


def test_the_ends_of_the_random_numbers():
    for u in (0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, math.nan):
        r = Round([4, 1, 7], 5000, seed=7)
        r.uniform[[0, 4, 5]] = u
        got = r.run()
        assert got[0] == r.want()[0]
        if u < 1:
            assert got == r.want()
        else:                                     # nothing exceeds the edge: the last entry that has a weight
            assert all(0 <= t < 5000 for t in got[1])


def test_drafts_that_can_only_be_accepted_or_rejected():
    r = Round([5, 5, 5, 5], 300, seed=8)
    r.draft[5:10] = r.target[4:9].clone()         # the draft is the target of the row before: always accepted
    r.target[10:15, :] = 0                        # no probability: rejected at once, and nothing to draw from
    r.tokens[16], r.tokens[17] = -1, 300          # outside the vocabulary
    got = r.run()
    assert got == r.want()
    assert got[0][1] == 5 and got[0][2] == 1 and got[1][2] == -1 and got[0][3] == 1
    sure = Round([3, 3], 300, seed=9, draft=False)
    sure.target[0] = 0
    sure.target[0, int(sure.tokens[1])] = 1.0     # certain on both sides
    sure.tokens[4] = 301                          # outside: nothing is taken out of the row
    assert sure.run() == sure.want()


def test_a_residual_that_is_empty_takes_the_target():
    r = Round([2, 2], 6000, seed=10)
    r.draft[1] = 1.0                              # over the target everywhere
    r.uniform[1] = 0.9999
    got = r.run()
    assert got == r.want() and got[0][0] == 1 and got[1][0] >= 0


def test_weights_that_are_no_numbers_count_as_nothing():
    r = Round([3, 2], 5000, seed=11)
    r.target[0, 10:20] = math.nan
    r.target[1, 30] = math.inf
    r.target[2, 40:] = -1.0
    r.draft[1, 50] = math.nan
    r.draft[2, 60] = math.inf
    assert r.run() == r.want()


def test_the_lowest_token_of_those_that_carry_the_edge():
    """One-hot rows, also at the ends of segments: the token itself whatever the random number."""
    for at in (0, 4095, 4096, 8191, 8999):
        r = Round([1], 9000, seed=12)
        r.target[0] = 0
        r.target[0, at] = 1.0
        for u in (0.0, 0.5, 0.9999999):
            r.uniform[0] = u
            assert r.run() == ([1], [at])


def test_a_round_from_logits_to_a_committed_kda_state():
    """Probabilities, verification and the commit by selection on one stream, with nothing read back in between."""
    heads, vocab, lens, slots = 2, 1000, [4, 1, 3], 3
    gen = torch.Generator().manual_seed(13)
    total = sum(lens)
    logits = (torch.randn(total, vocab, generator=gen) * 2).to(torch.bfloat16).to(DEV)
    tokens = torch.randint(0, vocab, (total,), generator=gen).to(torch.int32)
    tokens[1:3] = logits[:2].float().argmax(1).cpu().to(torch.int32)
    uniform = torch.full((total,), 1e-6)
    cu = torch.tensor([0, 4, 5, 8], dtype=torch.int32, device=DEV)
    n = heads * 128 * 128
    ckpt = torch.randn(total * n, generator=gen).to(torch.bfloat16).to(DEV)
    pool = torch.zeros(slots * n, dtype=torch.bfloat16, device=DEV)
    off = torch.tensor([n, 0, 2 * n], dtype=torch.int64, device=DEV)
    probs = torch.zeros(total, vocab, device=DEV)
    keep, token = torch.zeros(3, dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
    d_tokens, d_uniform = tokens.to(DEV), uniform.to(DEV)
    ws1 = torch.zeros(ffi.glm53f_spec_probs_workspace_bytes(total, vocab), dtype=torch.uint8, device=DEV)
    ws2 = torch.zeros(ffi.glm53f_spec_accept_workspace_bytes(3, vocab), dtype=torch.uint8, device=DEV)

    def step(stream):
        assert ffi.glm53f_spec_probs(total, vocab, ptr(logits), 0, vocab, None, ptr(probs), vocab, ptr(ws1), ws1.numel(), stream) == 0
        assert ffi.glm53f_spec_accept(3, vocab, ptr(cu), ptr(d_tokens), ptr(probs), vocab, None, 0, ptr(d_uniform), ptr(keep), ptr(token),
                                      ptr(ws2), ws2.numel(), stream) == 0
        assert kda.glm53f_kda_select_batch_bf16state(heads, 1, 3, ptr(cu), ptr(keep), ptr(ckpt), ckpt.numel(), ptr(pool), pool.numel(),
                                                     ptr(off), stream) == 0

    step(None)
    hs.sync()
    kept = keep.tolist()
    assert kept[0] >= 3 and kept[1] == 1
    want = [lo.accept(tokens[a:b], probs[a:b].cpu(), None, uniform[a:b]) for a, b in ((0, 4), (4, 5), (5, 8))]
    assert [w[0] for w in want] == kept and [w[1] for w in want] == token.tolist()
    for b, (slot, first) in enumerate(((1, 0), (0, 4), (2, 5))):
        row = first + kept[b] - 1
        assert torch.equal(pool[slot * n:(slot + 1) * n], ckpt[row * n:(row + 1) * n])
    # recorded once and replayed with other random numbers
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(torch.cuda.current_stream().cuda_stream)
    for replay in range(3):
        d_uniform.copy_(torch.rand(total, generator=gen))
        graph.replay()
        hs.sync()
        a = (keep.tolist(), token.tolist(), probs.clone(), pool.clone())
        step(None)
        hs.sync()
        assert a[0] == keep.tolist() and a[1] == token.tolist() and torch.equal(a[2], probs) and torch.equal(a[3], pool), replay


def test_probabilities_of_more_rows_than_the_caches_hold():
    """The rows go in parts; each part's rows, the last one's too, come out as by themselves (a row's sums do not depend on
    the rows beside it while the number of rows leaves the cut alone)."""
    rows, vocab = 700, 90001
    gen = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randn(rows, vocab, generator=gen, device=DEV) * 3
    t = torch.rand(rows, generator=gen, device=DEV) + 0.3
    out = torch.zeros(rows, vocab, device=DEV)
    need = ffi.glm53f_spec_probs_workspace_bytes(rows, vocab)
    ws = torch.zeros(need, dtype=torch.uint8, device=DEV)
    assert ffi.glm53f_spec_probs(rows, vocab, ptr(x), 1, vocab, ptr(t), ptr(out), vocab, ptr(ws), need, None) == 0
    for at in (0, 333, 699):
        want = torch.softmax(x[at].double() / t[at].double(), 0)
        assert bool(((out[at].double() - want).abs() <= 2.0 ** -24 * (4 * 60 + 112) * want + 2.0 ** -126).all()), at
    part = torch.zeros(100, vocab, device=DEV)
    assert ffi.glm53f_spec_probs(100, vocab, ptr(x[600:]), 1, vocab, ptr(t[600:]), ptr(part), vocab, ptr(ws), need, None) == 0
    hs.sync()
    assert torch.equal(part, out[600:])


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_an_infinite_temperature_is_uniform(kind):
    gen = torch.Generator().manual_seed(8)
    x = (torch.randn(3, 4999, generator=gen) * 30).to(kind)
    x[1, 7:90] = -math.inf
    x[2] = -math.inf
    got = spec_probs(x, torch.full((3,), math.inf)).double()
    left = (x > -math.inf).double()
    want = left / left.sum(1, keepdim=True).clamp(min=1)
    assert bool(((got - want).abs() <= 2.0 ** -24 * 112 * want).all())
    got = spec_probs(x, torch.tensor([3e38, 1e-45, 1.0]))
    assert bool(((got[0].double() - 1 / 4999).abs() <= 2.0 ** -24 * 112).all())
    assert int(got[1].argmax()) == int(x[1].float().argmax()) and abs(float(got[1].sum()) - 1) < 1e-6 and bool((got[2] == 0).all())
