"""The operators around a speculative round of a linear-attention layer, each in its plain form and as this library's
call: linear attention with one decay per head (prompt, decode, verify and commit), the projections' matrix product with
its epilogue, the probabilities of the LM head's logits, and the verification of drafted tokens.

Real use: a serving engine. Prompts run through the chunked form, decode steps of some slots through the recurrent one,
a verify window is read without touching the states and committed by the accepted counts, the projections run with
1 to some thousand rows, and the LM head's logits become probabilities that the drafted tokens are judged by.
"""
import math
import random

import torch

own = False

DEV = "cuda"
ACTS = ("none", "relu", "silu", "gelu", "gelu_tanh", "sigmoid")


# ---------------------------------------------------------------------------------------------------- the cases

def listed():
    lin = {"op": "lin", "qk_heads": 0, "dk": 128, "dv": 128, "ragged": False}
    gemm = {"op": "gemm", "groups": 1, "bias": False, "act": "none", "residual": False, "out_f32": False}
    return [
        # one long prompt of a 64-head layer, states kept in f32
        {**lin, "name": "prompt_1x8192", "mode": "prefill", "heads": 64, "batch": 1, "rows": 8192, "bf16_state": False},
        # prompts of several users in one pass, lengths from none to odd, shared q and k heads, narrow keys, bf16 states
        {**lin, "name": "prompts_ragged", "mode": "prefill", "heads": 32, "qk_heads": 8, "dk": 64, "batch": 9, "rows": 1801,
         "ragged": True, "bf16_state": True},
        # a decode step of sixteen slots, states updated in place
        {**lin, "name": "decode_16", "mode": "decode", "heads": 64, "batch": 16, "rows": 1, "bf16_state": True},
        # one user alone: the smallest decode step
        {**lin, "name": "decode_1", "mode": "decode", "heads": 64, "batch": 1, "rows": 1, "bf16_state": False},
        # a verify round of 48 slots with windows of up to sixteen rows, and the commit of what was accepted
        {**lin, "name": "verify_48x16", "mode": "verify", "heads": 64, "batch": 48, "rows": 16, "ragged": True,
         "bf16_state": True},
        # the input projection of a decode step of sixteen slots, with bias and SiLU
        {**gemm, "name": "project_16", "rows": 16, "n": 24640, "k": 4096, "bias": True, "act": "silu"},
        # the output projection of a prompt's segment onto the residual stream
        {**gemm, "name": "project_2048", "rows": 2048, "n": 4096, "k": 8192, "bias": True, "residual": True},
        # sizes that are no multiple of anything
        {**gemm, "name": "project_odd", "rows": 333, "n": 1999, "k": 1001, "bias": True, "act": "gelu", "residual": True,
         "out_f32": True},
        # one row of the LM head's logits
        {"op": "probs", "name": "probs_1", "rows": 1, "vocab": 151936, "logits_f32": False, "temperature": 0.8},
        # all windows' logits of a verify round
        {"op": "probs", "name": "probs_384", "rows": 384, "vocab": 151936, "logits_f32": True, "temperature": 1.0},
        # one user's five rows, drafted by a model
        {"op": "accept", "name": "accept_1", "batch": 1, "rows": 5, "vocab": 151936, "ragged": False, "draft": True},
        # 64 users, windows of one to nine rows
        {"op": "accept", "name": "accept_64", "batch": 64, "rows": 9, "vocab": 151936, "ragged": True, "draft": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(("lin", "lin", "lin", "gemm", "gemm", "probs", "accept"))
    if op == "lin":
        mode = rng.choice(("prefill", "prefill", "decode", "verify"))
        heads = rng.choice((4, 8, 12, 16, 24, 32, 48, 64))
        divisors = [d for d in range(1, heads + 1) if heads % d == 0]
        case = {"op": "lin", "mode": mode, "heads": heads, "qk_heads": rng.choice((0, rng.choice(divisors))),
                "dk": rng.choice((64, 128, 128)), "dv": rng.choice((64, 128, 128)), "bf16_state": rng.random() < 0.5,
                "ragged": rng.random() < 0.6}
        if mode == "prefill":
            rows = _log_int(rng, 17, 8192)
            most = max(1, min(64, 8192 * 64 // (rows * heads)))
            return {**case, "rows": rows, "batch": _log_int(rng, 1, most)}
        if mode == "decode":
            return {**case, "rows": 1, "ragged": False, "batch": _log_int(rng, 1, 48)}
        return {**case, "rows": rng.randint(2, 16), "batch": _log_int(rng, 1, 48)}
    if op == "gemm":
        rows, groups = _log_int(rng, 1, 2048), rng.choice((1, 1, 1, 2, 3))
        n, k = _log_int(rng, 16, 24640), _log_int(rng, 64, 8192)
        if rng.random() < 0.6:                        # most weights have sizes of whole tiles
            n, k = max(16, n // 16 * 16), max(128, k // 128 * 128)
        while rows * n * k * groups > 2048 * 4096 * 8192:
            n = max(16, n // 32 * 16)
        return {"op": "gemm", "rows": rows, "n": n, "k": k, "groups": groups, "bias": rng.random() < 0.5,
                "act": rng.choice(ACTS), "residual": rng.random() < 0.5, "out_f32": rng.random() < 0.4}
    vocab = rng.choice((151936, 32000, 50001, _log_int(rng, 256, 151936)))
    if op == "probs":
        return {"op": "probs", "rows": _log_int(rng, 1, 384), "vocab": vocab, "logits_f32": rng.random() < 0.5,
                "temperature": round(rng.uniform(0.3, 1.5), 3)}
    return {"op": "accept", "batch": _log_int(rng, 1, 64), "rows": rng.randint(1, 9), "vocab": vocab,
            "ragged": rng.random() < 0.5, "draft": rng.random() < 0.7}


def _lengths(case):
    """Rows of each request: all `rows`, or spread from none to `rows` with the longest among them (a window has one at
    least)."""
    if not case["ragged"]:
        return [case["rows"]] * case["batch"]
    r = random.Random(case["rows"] * 1000003 + case["batch"])
    low = 0 if case.get("mode") == "prefill" else 1
    lens = [r.randint(low, case["rows"]) for _ in range(case["batch"])]
    lens[r.randrange(case["batch"])] = case["rows"]
    return lens


# ---------------------------------------------------------------------------------------------------- the inputs

def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 11)

    def normal(*shape, scale=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32) * scale).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device=DEV, dtype=torch.float32)

    def starts(lens):
        return torch.tensor([0] + [sum(lens[:i + 1]) for i in range(len(lens))], dtype=torch.int32, device=DEV)

    s = {"case": case, "stream": torch.cuda.current_stream().cuda_stream}
    if case["op"] == "lin":
        lens, heads, dk, dv = _lengths(case), case["heads"], case["dk"], case["dv"]
        qk_heads, total, batch = case["qk_heads"] or heads, max(1, sum(lens)), case["batch"]
        # the projection's rows hold q | k | v side by side
        s["qkv"] = normal(total, 2 * qk_heads * dk + heads * dv)
        s["qkv"][:, :2 * qk_heads * dk] *= dk ** -0.25
        s["cu_rows"], s["total"] = starts(lens), total
        # decays of about two rows to some hundred rows, as slopes over the heads
        s["log_decay"] = -torch.exp2(-8.0 * torch.arange(1, heads + 1, device=DEV, dtype=torch.float32) / heads) * 0.7
        slots = batch + 1
        s["state"] = normal(slots, heads, dv, dk, scale=0.5, dtype=torch.bfloat16 if case["bf16_state"] else torch.float32)
        order = list(range(slots))
        random.Random(batch).shuffle(order)
        s["slots"] = torch.tensor(order[:batch], dtype=torch.int64, device=DEV)
        s["state_off"] = s["slots"] * (heads * dv * dk)
        s["out"] = torch.zeros(total, heads * dv, dtype=torch.bfloat16, device=DEV)
        # accepted counts of a verify round, from one to all rows of a window
        lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
        s["keep"] = torch.minimum(1 + (uniform(batch) * lengths).to(torch.int32), lengths)
        s["workspace"] = torch.empty(_lin_workspace(case), dtype=torch.uint8, device=DEV)
    elif case["op"] == "gemm":
        groups, rows, n, k = case["groups"], case["rows"], case["n"], case["k"]
        s["x"], s["w"] = normal(groups, rows, k), normal(groups, n, k, scale=k ** -0.5)
        kind = torch.float32 if case["out_f32"] else torch.bfloat16
        s["bias"] = normal(groups, n, scale=0.3) if case["bias"] else None
        s["residual"] = normal(groups, rows, n, dtype=kind) if case["residual"] else None
        s["out"] = torch.zeros(groups, rows, n, dtype=kind, device=DEV)
    elif case["op"] == "probs":
        rows, vocab = case["rows"], case["vocab"]
        s["logits"] = normal(rows, vocab, scale=2.5, dtype=torch.float32 if case["logits_f32"] else torch.bfloat16)
        s["temperature"] = torch.full((rows,), case["temperature"], dtype=torch.float32, device=DEV)
        s["probs"] = torch.zeros(rows, vocab, dtype=torch.float32, device=DEV)
        s["workspace"] = torch.empty(_SPEC_WORKSPACE, dtype=torch.uint8, device=DEV)
    else:
        lens, vocab = _lengths(case), case["vocab"]
        total, batch = sum(lens), case["batch"]
        # a draft model that is near the target; its tokens are drawn from its own probabilities
        z = normal(total, vocab, scale=2.5, dtype=torch.float32)
        s["target"] = torch.softmax(z, dim=1)
        zq = z + normal(total, vocab, scale=0.7, dtype=torch.float32)
        gumbel = -torch.log(-torch.log(uniform(total, vocab).clamp_(1e-12, 1 - 1e-7)))
        s["tokens"] = torch.argmax(zq + gumbel, dim=1).to(torch.int32)
        s["draft"] = torch.softmax(zq, dim=1) if case["draft"] else None
        del z, zq, gumbel
        s["uniform"] = uniform(total)
        s["cu_rows"] = starts(lens)
        s["keep"] = torch.zeros(batch, dtype=torch.int32, device=DEV)
        s["next"] = torch.zeros(batch, dtype=torch.int32, device=DEV)
        s["workspace"] = torch.empty(_SPEC_WORKSPACE, dtype=torch.uint8, device=DEV)
    return s


# What a program that serves these sizes sets aside once: partial results of the longest rows and prompts.
_SPEC_WORKSPACE = 1 << 20


def _lin_workspace(case):
    if case["mode"] != "prefill":
        return 0
    return 1 << 28


# ---------------------------------------------------------------------------------------------------- one pass

def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state)
    return _PLAIN[op](state)


def _plain_lin(s):
    case = s["case"]
    old = s["state"].index_select(0, s["slots"]).float()
    lens = s["cu_rows"][1:] - s["cu_rows"][:-1]
    out, after = _lin_formula(s, old, lens)
    s["out"].copy_(out)
    if case["mode"] == "verify":
        after = _lin_formula(s, old, s["keep"])[1]
    s["state"].index_copy_(0, s["slots"], after.to(s["state"].dtype))
    return {"out": s["out"], "state": s["state"]}


def _lin_formula(s, old, lens):
    """The first lens[b] rows of every request, in chunks of 64: inside a chunk the scores q k^T times the decay between
    the two rows, across chunks the state at the chunk's start; all of it as products over all chunks at once."""
    case = s["case"]
    heads, dk, dv = case["heads"], case["dk"], case["dv"]
    qk_heads, batch, total = case["qk_heads"] or heads, case["batch"], s["total"]
    size = min(64, case["rows"])
    chunks = -(-case["rows"] // size)
    g = s["log_decay"]
    t = torch.arange(chunks * size, device=DEV)
    live = t[None, :] < lens[:, None]
    at = torch.where(live, s["cu_rows"][:-1, None] + t[None, :], 0).long()
    qkv = s["qkv"].float()[at] * live[:, :, None]

    def split(x, n, d):
        x = x.reshape(batch, chunks, size, n, d).permute(0, 3, 1, 2, 4)
        return x.repeat_interleave(heads // n, dim=1)

    q = split(qkv[:, :, :qk_heads * dk], qk_heads, dk)
    k = split(qkv[:, :, qk_heads * dk:2 * qk_heads * dk], qk_heads, dk)
    v = split(qkv[:, :, 2 * qk_heads * dk:], heads, dv)
    i = torch.arange(size, device=DEV, dtype=torch.float32)
    gap = i[:, None] - i[None, :]
    decay = torch.exp(g[:, None, None] * gap.clamp(min=0)) * (gap >= 0)
    out = ((q @ k.transpose(-1, -2)) * decay[None, :, None]) @ v
    # the state at every chunk's start: the chunks before it, decayed by the rows between
    tail = torch.exp(g[:, None] * (size - 1 - i))[None, :, None, :, None]
    added = ((v * tail).transpose(-1, -2) @ k).reshape(batch, heads, chunks, dv * dk)
    n = torch.arange(chunks, device=DEV, dtype=torch.float32)
    gap = n[:, None] - 1 - n[None, :]
    mix = torch.exp(g[:, None, None] * (gap.clamp(min=0) * size)) * (gap >= 0)
    start = (mix @ added).reshape(batch, heads, chunks, dv, dk)
    start = start + torch.exp(g[:, None] * (n * size))[None, :, :, None, None] * old[:, :, None]
    out = out + torch.exp(g[:, None] * (i + 1))[None, :, None, :, None] * (q @ start.transpose(-1, -2))
    out = (out * dk ** -0.5).permute(0, 2, 3, 1, 4).reshape(batch, chunks * size, heads * dv)
    row = torch.arange(total, device=DEV)
    request = torch.searchsorted(s["cu_rows"][1:].long(), row, right=True).clamp(max=batch - 1)
    out = out[request, row - s["cu_rows"].long()[request]]
    # the state behind the last row
    left = (lens[:, None] - 1 - t[None, :]).clamp(min=0).float()
    weight = torch.exp(g[None, :, None] * left[:, None, :]).reshape(batch, heads, chunks, size, 1)
    kept = (v * weight * live.reshape(batch, 1, chunks, size, 1)).reshape(batch, heads, chunks * size, dv)
    after = kept.transpose(-1, -2) @ k.reshape(batch, heads, chunks * size, dk)
    return out, after + torch.exp(g[None, :] * lens[:, None].float())[:, :, None, None] * old


def _activate(y, act):
    if act == "relu":
        return y.clamp(min=0)
    if act == "silu":
        return y / (1 + torch.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-y))
    return y


def _plain_gemm(s):
    y = s["x"].float() @ s["w"].float().transpose(-1, -2)
    if s["bias"] is not None:
        y = y + s["bias"].float()[:, None, :]
    y = _activate(y, s["case"]["act"])
    if s["residual"] is not None:
        y = s["residual"].float() + y
    s["out"].copy_(y)
    return s["out"]


def _plain_probs(s):
    z = s["logits"].float() / s["temperature"][:, None]
    e = torch.exp(z - z.amax(dim=1, keepdim=True))
    torch.div(e, e.sum(dim=1, keepdim=True), out=s["probs"])
    return s["probs"]


def _plain_accept(s):
    batch, rows = s["case"]["batch"], s["case"]["rows"]
    first = s["cu_rows"][:-1].long()
    lens = s["cu_rows"][1:].long() - first
    i = torch.arange(1, rows, device=DEV)
    drafted = i[None, :] < lens[:, None]
    row = torch.where(drafted, first[:, None] + i[None, :], first[:, None] + 0 * i[None, :])
    token = s["tokens"].long()[row]
    before = torch.where(drafted, row - 1, row)
    p = s["target"][before, token].double()
    q = s["draft"][row, token].double() if s["draft"] is not None else torch.ones_like(p)
    yes = drafted & (s["uniform"].double()[row] * q < p)
    accepted = torch.cumprod(yes.long(), dim=1).sum(dim=1)
    last = first + accepted
    weight = s["target"][last].double()
    judged = (first + torch.minimum(accepted + 1, lens - 1))
    rejected = (accepted + 1 < lens)[:, None]
    if s["draft"] is not None:
        weight = torch.where(rejected, (weight - s["draft"][judged].double()).clamp(min=0), weight)
    else:
        x = torch.arange(s["case"]["vocab"], device=DEV)[None, :] == s["tokens"].long()[judged][:, None]
        weight = torch.where(rejected & x, 0.0, weight)
    total = torch.cumsum(weight, dim=1)
    edge = s["uniform"].double()[first] * total[:, -1]
    s["next"].copy_((total <= edge[:, None]).sum(dim=1))
    s["keep"].copy_(accepted + 1)
    return {"keep": s["keep"], "next": s["next"]}


_PLAIN = {"lin": _plain_lin, "gemm": _plain_gemm, "probs": _plain_probs, "accept": _plain_accept}


# ------------------------------------------------------------------------------------------- this library's calls

def _bindings():
    import os
    import sys
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "glm53f-afd_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from glm53f_forward import ffi as fwd
    from glm53f_lin import ffi as lin
    from glm53f_spec import ffi as spec
    return lin.lib(), fwd.lib(), spec.lib()


_libs = None


def _lib(which):
    global _libs
    if _libs is None:
        _libs = _bindings()
    return _libs[which]


def _done(rc):
    if rc != 0:
        raise RuntimeError(f"the call returned {rc}")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _own_lin(s):
    case, lib = s["case"], _lib(0)
    heads, dk, dv = case["heads"], case["dk"], case["dv"]
    qk_heads = case["qk_heads"] or heads
    width = 2 * qk_heads * dk + heads * dv
    q = s["qkv"].data_ptr()
    k, v = q + 2 * qk_heads * dk, q + 4 * qk_heads * dk
    shape = (heads, qk_heads, dk, dv)
    state, offs, cu = s["state"].data_ptr(), s["state_off"].data_ptr(), s["cu_rows"].data_ptr()
    rows = (q, width, k, width, v, width, s["log_decay"].data_ptr(), dk ** -0.5)
    out = (s["out"].data_ptr(), heads * dv)
    bf16 = case["bf16_state"]
    if case["mode"] == "prefill":
        call = lib.glm53f_lin_prefill_batch_bf16state if bf16 else lib.glm53f_lin_prefill_batch
        ws = s["workspace"]
        _done(call(*shape, case["batch"], cu, case["rows"], *rows, state, state, offs, *out, ws.data_ptr(), ws.numel(), s["stream"]))
    elif case["mode"] == "decode":
        call = lib.glm53f_lin_chain_batch_bf16state if bf16 else lib.glm53f_lin_chain_batch
        _done(call(*shape, case["batch"], cu, *rows, state, state, offs, *out, s["stream"]))
    else:
        # the window's outputs without a new state, then the accepted rows of it
        call = lib.glm53f_lin_prefill_batch_bf16state if bf16 else lib.glm53f_lin_prefill_batch
        _done(call(*shape, case["batch"], cu, case["rows"], *rows, state, None, offs, *out, None, 0, s["stream"]))
        call = lib.glm53f_lin_advance_batch_bf16state if bf16 else lib.glm53f_lin_advance_batch
        _done(call(*shape, 1, case["batch"], cu, s["keep"].data_ptr(), k, width, 0, v, width, 0, s["log_decay"].data_ptr(),
                   state, state, 0, offs, s["stream"]))
    return {"out": s["out"], "state": s["state"]}


def _own_gemm(s):
    case = s["case"]
    rows, n, k = case["rows"], case["n"], case["k"]
    _done(_lib(1).glm53f_fwd_gemm_bf16_fused(
        s["x"].data_ptr(), k, rows * k, s["w"].data_ptr(), k, n * k, case["groups"], rows, n, k, _ptr(s["bias"]), n,
        ACTS.index(case["act"]), _ptr(s["residual"]), n, rows * n, s["out"].data_ptr(), int(case["out_f32"]), n, rows * n,
        s["stream"]))
    return s["out"]


def _own_probs(s):
    case, ws = s["case"], s["workspace"]
    _done(_lib(2).glm53f_spec_probs(case["rows"], case["vocab"], s["logits"].data_ptr(), int(case["logits_f32"]), case["vocab"],
                                    s["temperature"].data_ptr(), s["probs"].data_ptr(), case["vocab"], ws.data_ptr(), ws.numel(),
                                    s["stream"]))
    return s["probs"]


def _own_accept(s):
    case, ws = s["case"], s["workspace"]
    _done(_lib(2).glm53f_spec_accept(case["batch"], case["vocab"], s["cu_rows"].data_ptr(), s["tokens"].data_ptr(),
                                     s["target"].data_ptr(), case["vocab"], _ptr(s["draft"]), case["vocab"],
                                     s["uniform"].data_ptr(), s["keep"].data_ptr(), s["next"].data_ptr(), ws.data_ptr(),
                                     ws.numel(), s["stream"]))
    return {"keep": s["keep"], "next": s["next"]}


_OWN = {"lin": _own_lin, "gemm": _own_gemm, "probs": _own_probs, "accept": _own_accept}


# ---------------------------------------------------------------------------------------------------- the measure

def work(case):
    if case["op"] == "lin":
        lens, heads, dk, dv = _lengths(case), case["heads"], case["dk"], case["dv"]
        qk_heads, rows = case["qk_heads"] or heads, sum(_lengths(case))
        states = case["batch"] * heads * dk * dv * (2 if case["bf16_state"] else 4)
        return {"bytes": rows * (2 * qk_heads * dk + 2 * heads * dv) * 2 + 2 * states, "flops": 4 * rows * heads * dk * dv}
    if case["op"] == "gemm":
        groups, rows, n, k = case["groups"], case["rows"], case["n"], case["k"]
        cell = 4 if case["out_f32"] else 2
        moved = 2 * (rows * k + n * k) + cell * rows * n * (2 if case["residual"] else 1) + (2 * n if case["bias"] else 0)
        return {"bytes": groups * moved, "flops": 2 * groups * rows * n * k}
    if case["op"] == "probs":
        return {"bytes": case["rows"] * case["vocab"] * (8 if case["logits_f32"] else 6), "flops": 4 * case["rows"] * case["vocab"]}
    rows = 2 if case["draft"] else 1                   # the next token's row of the target, and of the draft
    return {"bytes": case["batch"] * case["vocab"] * 4 * rows, "flops": 3 * case["batch"] * case["vocab"]}


def exact(case, seed):
    if case["op"] == "accept":
        return None                                    # whole numbers
    s = prepare(case, seed)
    if case["op"] == "lin":
        return _exact_lin(s)
    if case["op"] == "gemm":
        y = torch.stack([x.double() @ w.double().t() for x, w in zip(s["x"], s["w"])])
        if s["bias"] is not None:
            y += s["bias"].double().unsqueeze(1)
        y = {"none": lambda v: v, "relu": torch.relu, "silu": lambda v: v * torch.sigmoid(v),
             "gelu": lambda v: v * 0.5 * torch.erfc(-v / math.sqrt(2)), "sigmoid": torch.sigmoid,
             "gelu_tanh": lambda v: v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))}[case["act"]](y)
        return y if s["residual"] is None else y + s["residual"].double()
    rows = [torch.softmax(z.double() / t.double(), 0) for z, t in zip(s["logits"], s["temperature"])]
    return torch.stack(rows)


def _exact_lin(s):
    """The recurrence itself, row by row, in 64 bits."""
    case = s["case"]
    heads, dk, dv = case["heads"], case["dk"], case["dv"]
    qk_heads, lens = case["qk_heads"] or heads, _lengths(case)
    state = s["state"].double()
    cur = state[s["slots"]]
    fade = torch.exp(s["log_decay"].double())[None, :, None, None]
    stop = s["keep"] if case["mode"] == "verify" else s["cu_rows"].diff()
    kept = cur.clone()
    out = torch.zeros(s["total"], heads, dv, dtype=torch.float64, device=DEV)
    first = s["cu_rows"][:-1].long()
    count = s["cu_rows"].diff()
    order = sorted(set(lens), reverse=True)
    groups = {n: torch.tensor([b for b, m in enumerate(lens) if m >= n], device=DEV) for n in order}
    for t in range(max(lens)):
        who = groups[min(n for n in order if n > t)]
        row = first[who] + t
        x = s["qkv"][row].double()
        q = x[:, :qk_heads * dk].reshape(-1, qk_heads, dk).repeat_interleave(heads // qk_heads, 1)
        k = x[:, qk_heads * dk:2 * qk_heads * dk].reshape(-1, qk_heads, dk).repeat_interleave(heads // qk_heads, 1)
        v = x[:, 2 * qk_heads * dk:].reshape(-1, heads, dv)
        new = cur[who] * fade + v.unsqueeze(-1) * k.unsqueeze(-2)
        cur[who] = new
        out[row] = (new @ q.unsqueeze(-1)).squeeze(-1) / math.sqrt(dk)
        if case["mode"] == "verify":
            kept[who] = torch.where((stop[who] > t)[:, None, None, None], new, kept[who])
    state[s["slots"]] = kept if case["mode"] == "verify" else cur
    return {"out": out.reshape(s["total"], heads * dv), "state": state}
