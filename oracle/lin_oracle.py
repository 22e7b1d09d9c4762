"""Plain 64-bit models of linear attention with one decay per head, of the matrix product with its epilogue, of softmax
rows and of the verification of drafted tokens, on the CPU, for the tests of include/ext. Each follows the operator's
formula row by row; the attention also returns the sums of the terms' absolute values, which f32 errors are counted by.
"""
import math

import torch


def attention(q, k, v, log_decay, scale, state):
    """One request: q, k [R][qk_heads][dk], v [R][heads][dv], state [heads][dv][dk] -> outputs [R][heads][dv], the state
    behind every row [R + 1][heads][dv][dk], and both once more with every term's absolute value."""
    heads = v.shape[1]
    q, k = (x.double().repeat_interleave(heads // x.shape[1], 1) for x in (q, k))
    v, s = v.double(), state.double()
    a = s.abs()
    fade = torch.exp(log_decay.double())[:, None, None]
    outs, abs_outs, states, abs_states = [], [], [s], [a]
    for t in range(v.shape[0]):
        s = fade * s + v[t][:, :, None] * k[t][:, None, :]
        a = fade * a + v[t].abs()[:, :, None] * k[t].abs()[:, None, :]
        outs.append(scale * (s * q[t][:, None, :]).sum(-1))
        abs_outs.append(abs(scale) * (a * q[t].abs()[:, None, :]).sum(-1))
        states.append(s)
        abs_states.append(a)
    empty = torch.zeros(0, heads, v.shape[2], dtype=torch.float64)
    pack = lambda x: torch.stack(x) if x else empty  # noqa: E731
    return pack(outs), torch.stack(states), pack(abs_outs), torch.stack(abs_states)


def activate(y, act):
    return [lambda z: z, lambda z: z.clamp(min=0), lambda z: z * torch.sigmoid(z),
            lambda z: z * 0.5 * torch.erfc(-z / math.sqrt(2)),
            lambda z: z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)), torch.sigmoid][act](y)


def gemm(x, w, bias, act, residual):
    """One group: x [m][k], w [n][k] -> the result, and the absolute sums of the products and the bias."""
    y, a = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
    if bias is not None:
        y, a = y + bias.double(), a + bias.double().abs()
    y = activate(y, act)
    return (y if residual is None else y + residual.double()), a


def probs(logits, temperature):
    """Rows [m][vocab] with a temperature each; a temperature that is not above 0 takes the greatest logit alone."""
    out = torch.zeros(logits.shape, dtype=torch.float64)
    for r, row in enumerate(logits.double()):
        t = float(temperature[r])
        if not t > 0:
            known = torch.where(row.isnan(), -math.inf, row)
            if known.max() > -math.inf:
                out[r, int((known == known.max()).nonzero()[0])] = 1.0
        elif not bool((row == -math.inf).all()):
            z = (row - row.max()) / t
            out[r] = torch.exp(z) / torch.exp(z).sum()
    return out


def accept(tokens, target, draft, uniform):
    """One request's window: tokens [n], target and draft [n][vocab] (draft None: certain drafts), uniform [n] -> the kept
    rows and the next token."""
    def clean(x):
        x = x.double()
        return torch.where((x > 0) & (x < math.inf), x, 0.0)

    n = len(tokens)
    if n == 0:
        return 0, -1
    vocab, kept, rejected = target.shape[1], n, False
    for i in range(1, n):
        x = int(tokens[i])
        ok = 0 <= x < vocab
        if ok:
            q = float(clean(draft[i])[x]) if draft is not None else 1.0
            ok = float(uniform[i]) * q < float(clean(target[i - 1])[x])
        if not ok:
            kept, rejected = i, True
            break
    p = clean(target[kept - 1])
    w = p
    if rejected and draft is not None:
        w = (p - clean(draft[kept])).clamp(min=0)
    elif rejected and 0 <= int(tokens[kept]) < vocab:
        w = p.clone()
        w[int(tokens[kept])] = 0
    if float(w.sum()) == 0 and rejected:
        w = p
    total = torch.cumsum(w, 0)
    if float(total[-1]) == 0:
        return kept, -1
    over = (total > float(uniform[0]) * float(total[-1])).nonzero()
    return kept, int(over[0]) if len(over) else int((w > 0).nonzero()[-1])
