"""A speculative engine's steps with the operators of include/ext run together, as they would be used: two layers of
linear attention, each a projection with bias, the attention, the output projection added to the residual stream in
place and a feed-forward pair with an activation; the LM head in f32, the probabilities, the verification and the commit
of both layers by the counts on the device. First a ragged prompt, then verify rounds.

Every stage is checked against 64-bit arithmetic on the stage's own inputs as they lie on the device, with the stage's
own tolerance (derived in the operators' tests: terms' roundings of 2^-24 of the absolute sums, pairs of bf16 values of
2^-17 in the chunked read-outs, one rounding of 2^-8 per stored bf16 value); counts and tokens are equal."""
import pytest
import torch

from glm53f_forward import ffi as fwd
from glm53f_lin import ffi as lin
from glm53f_spec import ffi as spec
from oracle import lin_oracle as lo

import harness as hs
from harness import ptr

pytestmark = pytest.mark.gpu
DEV = hs.DEV
LAYERS, HIDDEN, INNER, VOCAB = 2, 160, 208, 1003
HEADS, QK, DK, DV = 4, 2, 64, 128
WIDTH, STATE = 2 * QK * DK + HEADS * DV, HEADS * DV * DK
SLOTS, BATCH, ROWS = 4, 3, 640
GELU_TANH = 4


class Engine:
    """Weights, states of SLOTS requests ([layer][slot]) and buffers for one step of at most ROWS rows."""

    def __init__(self, seed):
        gen = torch.Generator().manual_seed(seed)
        w = lambda n, k: (torch.randn(n, k, generator=gen) * k ** -0.5).bfloat16().to(DEV)  # noqa: E731
        self.qkv = [w(WIDTH, HIDDEN) for _ in range(LAYERS)]
        self.bias = [(torch.randn(WIDTH, generator=gen) * 0.1).bfloat16().to(DEV) for _ in range(LAYERS)]
        self.o = [w(HIDDEN, HEADS * DV) for _ in range(LAYERS)]
        self.up = [w(INNER, HIDDEN) for _ in range(LAYERS)]
        self.down = [w(HIDDEN, INNER) for _ in range(LAYERS)]
        self.head = w(VOCAB, HIDDEN) * 4
        self.decay = (-torch.rand(LAYERS, HEADS, generator=gen) * 0.2).to(DEV)
        self.pool = (torch.randn(LAYERS, SLOTS, STATE, generator=gen) * 0.3).to(DEV)
        self.x = torch.zeros(ROWS, HIDDEN, dtype=torch.bfloat16, device=DEV)
        self.rows = torch.zeros(LAYERS, ROWS, WIDTH, dtype=torch.bfloat16, device=DEV)
        self.att = torch.zeros(ROWS, HEADS * DV, dtype=torch.bfloat16, device=DEV)
        self.mid = torch.zeros(ROWS, INNER, dtype=torch.bfloat16, device=DEV)
        self.logits = torch.zeros(ROWS, VOCAB, device=DEV)
        self.probs = torch.zeros(ROWS, VOCAB, device=DEV)
        self.keep, self.next = (torch.zeros(BATCH, dtype=torch.int32, device=DEV) for _ in range(2))
        self.tokens = torch.zeros(ROWS, dtype=torch.int32, device=DEV)
        self.uniform = torch.zeros(ROWS, device=DEV)
        self.off = torch.tensor([2 * STATE, 0, 3 * STATE], dtype=torch.int64, device=DEV)
        self.cu = torch.zeros(BATCH + 1, dtype=torch.int32, device=DEV)
        most = max([lin.glm53f_lin_prefill_workspace_bytes(HEADS, DK, DV, b, r) for b in (1, 2, 3) for r in range(0, ROWS + 1, 64)])
        self.lin_ws = torch.zeros(max(most, 16), dtype=torch.uint8, device=DEV)
        need = max(spec.glm53f_spec_probs_workspace_bytes(ROWS, VOCAB), spec.glm53f_spec_accept_workspace_bytes(BATCH, VOCAB))
        self.spec_ws = torch.zeros(need, dtype=torch.uint8, device=DEV)

    def project(self, x, w, rows, out, stream, bias=None, act=0, residual=None):
        n, k = w.shape
        assert fwd.glm53f_fwd_gemm_bf16_fused(ptr(x), k, 0, ptr(w), k, 0, 1, rows, n, k, None if bias is None else ptr(bias), 0, act,
                                              None if residual is None else ptr(residual), n, 0, ptr(out), int(out.dtype == torch.float32),
                                              n, 0, stream) == 0

    def attend(self, layer, longest, prompt, stream):
        r = ptr(self.rows[layer])
        pool = ptr(self.pool[layer])
        assert lin.glm53f_lin_prefill_batch(HEADS, QK, DK, DV, BATCH, ptr(self.cu), longest, r, WIDTH, r + 2 * QK * DK, WIDTH,
                                            r + 4 * QK * DK, WIDTH, ptr(self.decay[layer]), DK ** -0.5, pool, pool if prompt else None,
                                            ptr(self.off), ptr(self.att), HEADS * DV, ptr(self.lin_ws), self.lin_ws.numel(), stream) == 0

    def forward(self, rows, longest, prompt, stream, watch=lambda *a: None):
        """`watch(name, layer)` is called behind every stage (checks; not while a graph is captured)."""
        for i in range(LAYERS):
            self.project(self.x, self.qkv[i], rows, self.rows[i], stream, bias=self.bias[i])
            watch("qkv", i)
            self.attend(i, longest, prompt, stream)
            watch("attention", i)
            self.project(self.att, self.o[i], rows, self.x, stream, residual=self.x)
            watch("o", i)
            self.project(self.x, self.up[i], rows, self.mid, stream, act=GELU_TANH)
            watch("up", i)
            self.project(self.mid, self.down[i], rows, self.x, stream, residual=self.x)
            watch("down", i)

    def verify(self, rows, stream):
        self.project(self.x, self.head, rows, self.logits, stream)
        assert spec.glm53f_spec_probs(rows, VOCAB, ptr(self.logits), 1, VOCAB, None, ptr(self.probs), VOCAB, ptr(self.spec_ws),
                                      self.spec_ws.numel(), stream) == 0
        assert spec.glm53f_spec_accept(BATCH, VOCAB, ptr(self.cu), ptr(self.tokens), ptr(self.probs), VOCAB, None, 0, ptr(self.uniform),
                                       ptr(self.keep), ptr(self.next), ptr(self.spec_ws), self.spec_ws.numel(), stream) == 0

    def commit(self, stream):
        r = ptr(self.rows)
        assert lin.glm53f_lin_advance_batch(HEADS, QK, DK, DV, LAYERS, BATCH, ptr(self.cu), ptr(self.keep), r + 2 * QK * DK, WIDTH,
                                            ROWS * WIDTH, r + 4 * QK * DK, WIDTH, ROWS * WIDTH, ptr(self.decay), ptr(self.pool),
                                            ptr(self.pool), SLOTS * STATE, ptr(self.off), stream) == 0

    def round(self, rows, longest, stream):
        self.forward(rows, longest, False, stream)
        self.verify(rows, stream)
        self.commit(stream)


def host(t):
    hs.sync()
    return t.float().cpu().double()


def within(got, want, tol, what):
    err = (got - want).abs()
    assert bool((err <= tol).all()), f"{what}: {float((err / tol).max()):.2f} of the tolerance"


class Watch:
    """Checks every stage of a forward pass against 64-bit arithmetic on what the stage read."""

    def __init__(self, e, lens, prompt):
        self.e, self.lens, self.rows, self.prompt = e, lens, sum(lens), prompt
        self.x, self.before = host(e.x[:self.rows]), host(e.pool)

    def gemm(self, x, w, bias, act, residual, got, what):
        want, a = lo.gemm(x, host(w), None if bias is None else host(bias), act, residual)
        mid = want if residual is None else want - residual
        tol = 1.13 * (x.shape[1] + 1) * 2.0 ** -24 * a + 2.0 ** -24 * want.abs() + 1e-30 + 2.0 ** -8 * want.abs()
        within(got, want, tol + (16 * 2.0 ** -24 * (1 + mid.abs()) if act else 0), what)

    def __call__(self, name, i):
        e, n = self.e, self.rows
        if name == "qkv":
            self.gemm(self.x, e.qkv[i], e.bias[i], 0, None, host(e.rows[i, :n]), f"qkv {i}")
        elif name == "attention":
            rows, att, pool = host(e.rows[i, :n]), host(e.att[:n]), host(e.pool[i])
            at = 0
            for b, m in enumerate(self.lens):
                r = rows[at:at + m]
                slot = int(e.off[b]) // STATE
                q, k = (r[:, j * QK * DK:(j + 1) * QK * DK].reshape(m, QK, DK) for j in (0, 1))
                o, s, ao, a = lo.attention(q, k, r[:, 2 * QK * DK:].reshape(m, HEADS, DV), e.decay[i].cpu(), DK ** -0.5,
                                           self.before[i, slot].reshape(HEADS, DV, DK))
                within(att[at:at + m].reshape(m, HEADS, DV), o, 2.0 ** -8 * o.abs() + (2.0 ** -15 + (m + DK + 16) * 2.0 ** -24) * ao, f"attention {i} {b}")
                want = s[-1] if self.prompt else s[0]
                within(pool[slot].reshape(HEADS, DV, DK), want, (m + 32) * 2.0 ** -24 * a[-1] + 1e-30, f"state {i} {b}")
                at += m
            assert torch.equal(pool[1], self.before[i, 1]), "a slot of no request was written"
        elif name in ("o", "down"):
            src, w = (e.att, e.o) if name == "o" else (e.mid, e.down)
            got = host(e.x[:n])
            self.gemm(host(src[:n]), w[i], None, 0, self.x, got, f"{name} {i}")
            self.x = got
        else:
            self.gemm(self.x, e.up[i], None, GELU_TANH, None, host(e.mid[:n]), f"up {i}")


def test_a_prompt_and_verify_rounds():
    gen = torch.Generator().manual_seed(3)
    e = Engine(1)

    def inputs(lens):
        n = sum(lens)
        e.x[:n] = torch.randn(n, HIDDEN, generator=gen).bfloat16().to(DEV)
        e.x[n:] = 0
        e.cu.copy_(torch.tensor([sum(lens[:b]) for b in range(BATCH + 1)], dtype=torch.int32))
        return n

    lens = [570, 1, 67]                                  # segments, one row, a ragged tail
    n = inputs(lens)
    e.forward(n, max(lens), True, None, Watch(e, lens, True))
    for round_, lens in enumerate(([5, 1, 9], [1, 4, 0], [16, 16, 16])):
        n = inputs(lens)
        before = host(e.pool)
        e.forward(n, max(lens), False, None, Watch(e, lens, False))
        # drafts: what the target likes best, up to a row of each window (one pass to know it)
        e.verify(n, None)
        hs.sync()
        probs, logits = e.probs[:n].cpu(), e.logits[:n].cpu()
        tokens = torch.randint(0, VOCAB, (n,), generator=gen).to(torch.int32)
        at = 0
        for m in lens:
            good = max(0, (m * 2) // 3)
            tokens[at + 1:at + good] = probs[at:at + max(good - 1, 0)].argmax(1).int()
            at += m
        uniform = torch.rand(n, generator=gen) * 0.01
        e.tokens[:n], e.uniform[:n] = tokens.to(DEV), uniform.to(DEV)
        e.verify(n, None)
        hs.sync()
        x, want_x = host(e.x[:n]), None
        want_x, a = lo.gemm(x, host(e.head), None, 0, None)
        within(logits.double(), want_x, (HIDDEN + 2) * 2.0 ** -24 * a + 1e-30, "logits")
        want_p = lo.probs(logits, torch.ones(n))
        z = (logits.double() - logits.double().amax(1, keepdim=True)).abs()
        within(e.probs[:n].cpu().double(), want_p, 2.0 ** -24 * (4 * z + 112) * want_p + 2.0 ** -126, "probabilities")
        at, kept = 0, e.keep.tolist()
        for b, m in enumerate(lens):
            want = lo.accept(tokens[at:at + m], e.probs[at:at + m].cpu(), None, uniform[at:at + m])
            assert (kept[b], int(e.next[b])) == want, f"round {round_} request {b}"
            assert kept[b] >= (m * 2) // 3 or m == 0
            at += m
        e.commit(None)
        hs.sync()
        after = host(e.pool)
        for i in range(LAYERS):
            at = 0
            for b, m in enumerate(lens):
                r, slot = host(e.rows[i, at:at + kept[b]]), int(e.off[b]) // STATE
                q, k = (r[:, j * QK * DK:(j + 1) * QK * DK].reshape(kept[b], QK, DK) for j in (0, 1))
                _, s, _, a = lo.attention(q, k, r[:, 2 * QK * DK:].reshape(kept[b], HEADS, DV), e.decay[i].cpu(), 1.0,
                                          before[i, slot].reshape(HEADS, DV, DK))
                within(after[i, slot].reshape(HEADS, DV, DK), s[-1], (m + 16) * 2.0 ** -24 * a[-1] + 1e-30, f"commit {i} {b}")
                at += m
            assert torch.equal(after[i, 1], before[i, 1])


def test_a_captured_round_of_the_whole_chain():
    """One verify round in a graph, replayed with other hidden rows, drafts and window lengths: every result has the bits of
    the eager round on a second engine."""
    gen = torch.Generator().manual_seed(9)
    g, e = Engine(4), Engine(4)
    n, longest = 30, 16
    e.cu.copy_(torch.tensor([0, 10, 20, 30], dtype=torch.int32)), g.cu.copy_(e.cu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g.round(n, longest, torch.cuda.current_stream().cuda_stream)
    for replay, cu in enumerate(([0, 10, 20, 30], [0, 1, 17, 30], [0, 0, 16, 30])):
        x = torch.randn(n, HIDDEN, generator=gen).bfloat16()
        tokens, uniform = torch.randint(0, VOCAB, (n,), generator=gen).int(), torch.rand(n, generator=gen) * 1e-3
        for t in (g, e):
            t.x[:n], t.tokens[:n], t.uniform[:n] = x.to(DEV), tokens.to(DEV), uniform.to(DEV)
            t.cu.copy_(torch.tensor(cu, dtype=torch.int32))
        graph.replay()
        e.round(n, longest, None)
        hs.sync()
        for name in ("x", "rows", "att", "probs", "keep", "next", "pool"):
            assert torch.equal(getattr(g, name), getattr(e, name)), f"{name} of replay {replay}"
