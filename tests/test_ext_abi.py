"""The headers under include/ext as a boundary (C99 on their own, every entry point exported and bound with its number of
arguments) and everything that the host rejects. No launch: runs without a GPU."""
import glob
import os
import re
import subprocess

import pytest

from glm53f_forward import ffi as fwd
from glm53f_lin import ffi as lin
from glm53f_spec import ffi as spec

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EXT = os.path.join(ROOT, "include", "ext")


def declarations(name):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(EXT, name)).read(), flags=re.S)
    return {m.group(1): len(m.group(2).split(","))
            for m in re.finditer(r"\bint(?:32|64)_t\s+(glm53f_\w+)\s*\(([^;]*?)\)\s*;", text, flags=re.S)}


@pytest.mark.parametrize("header,ffi,count", [("glm53f_lin.h", lin, 7), ("glm53f_spec.h", spec, 4), ("glm53f_fwd_gemm.h", fwd, 1)])
def test_every_entry_point_is_exported_and_bound(header, ffi, count):
    decl = declarations(header)
    assert len(decl) == count and set(decl) <= set(ffi.PROTOTYPES)
    lib = ffi.lib()
    for name, nargs in decl.items():
        assert hasattr(lib, name), name
        assert len(ffi.PROTOTYPES[name][1]) == nargs, name


def test_the_headers_are_plain_c():
    headers = sorted(glob.glob(os.path.join(EXT, "*.h")))
    assert len(headers) == 3
    for h in headers:
        r = subprocess.run(["gcc", "-std=c99", "-Wall", "-Wextra", "-Werror", "-fsyntax-only", "-x", "c", h],
                           capture_output=True, text=True)
        assert r.returncode == 0, r.stderr
    names = sorted(n for h in headers for n in declarations(os.path.basename(h)))
    prog = "".join(f'#include "ext/{os.path.basename(h)}"\n' for h in headers)
    prog += "int main(void) {\n  const void* p[] = {" + ", ".join(f"(const void*){n}" for n in names) + "};\n  return p[0] == 0;\n}\n"
    lib_dir = os.path.join(ROOT, "glm53f-afd_amd", "csrc")
    r = subprocess.run(["gcc", "-std=gnu99", "-x", "c", "-", "-I", os.path.join(ROOT, "include"), "-L", lib_dir, "-lglm53f_kda",
                        "-L/opt/rocm/lib", "-lamdhip64", "-Wl,-rpath," + lib_dir, "-Wl,-rpath,/opt/rocm/lib", "-o", "/dev/null"],
                       input=prog, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


A = 1 << 20                                       # an aligned address that nothing dereferences on the host


def lin_call(form, **kw):
    a = dict(heads=4, qk=2, dk=128, dv=128, layers=1, batch=2, cu=A, keep=A, most=100, q=A, qs=256, k=A, ks=256, kl=0, v=A, vs=512, vl=0,
             g=A, scale=1.0, si=A, so=A, sl=0, off=A, out=A, os=512, ws=None, wb=0)
    a.update(kw)
    shape = (a["heads"], a["qk"], a["dk"], a["dv"])
    if form == "advance":
        return [f(*shape, a["layers"], a["batch"], a["cu"], a["keep"], a["k"], a["ks"], a["kl"], a["v"], a["vs"], a["vl"], a["g"],
                  a["si"], a["so"], a["sl"], a["off"], None)
                for f in (lin.glm53f_lin_advance_batch, lin.glm53f_lin_advance_batch_bf16state)]
    rows = (a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["g"], a["scale"], a["si"], a["so"], a["off"], a["out"], a["os"])
    if form == "chain":
        return [f(*shape, a["batch"], a["cu"], *rows, None) for f in (lin.glm53f_lin_chain_batch, lin.glm53f_lin_chain_batch_bf16state)]
    return [f(*shape, a["batch"], a["cu"], a["most"], *rows, a["ws"], a["wb"], None)
            for f in (lin.glm53f_lin_prefill_batch, lin.glm53f_lin_prefill_batch_bf16state)]


SHAPE = [dict(heads=0), dict(heads=70000), dict(qk=0), dict(qk=3), dict(qk=8), dict(dk=96), dict(dv=32), dict(dk=256), dict(batch=0),
         dict(batch=70000)]
ROWS = [dict(cu=None), dict(k=None), dict(v=None), dict(g=None), dict(si=None), dict(off=None), dict(ks=255), dict(vs=511), dict(ks=-256),
        dict(k=A + 1), dict(v=A + 1), dict(si=A + 8), dict(so=A + 2), dict(off=A + 4), dict(cu=A + 2), dict(g=A + 2)]


@pytest.mark.parametrize("bad", SHAPE + ROWS + [dict(q=None), dict(out=None), dict(qs=255), dict(os=511), dict(q=A + 1), dict(out=A + 1)])
@pytest.mark.parametrize("form", ["chain", "prefill"])
def test_attention_rejects(form, bad):
    assert lin_call(form, **bad) == [1, 1]


def test_prefill_rejects_its_own():
    assert lin_call("prefill", most=-1) == [1, 1]
    need = lin.glm53f_lin_prefill_workspace_bytes(4, 128, 128, 2, 1 << 20)
    if need > 0:
        for bad in (dict(ws=None, wb=need), dict(ws=A, wb=need - 1), dict(ws=A + 8, wb=need)):
            assert lin_call("prefill", most=1 << 20, **bad) == [1, 1]
    for bad in ((0, 128, 128, 1, 1), (4, 32, 128, 1, 1), (4, 128, 96, 1, 1), (4, 128, 128, 0, 1), (4, 128, 128, 1, -1)):
        assert lin.glm53f_lin_prefill_workspace_bytes(*bad) == -1
    assert lin.glm53f_lin_prefill_workspace_bytes(64, 128, 128, 48, 16) == 0


@pytest.mark.parametrize("bad", SHAPE + ROWS + [dict(keep=None), dict(keep=A + 1), dict(so=None), dict(layers=0), dict(layers=2, sl=0),
                                                dict(layers=2, sl=9), dict(layers=2, sl=8, kl=-1), dict(layers=2, sl=8, vl=-1)])
def test_commit_rejects(bad):
    assert lin_call("advance", **bad) == [1, 1]


def gemm_call(**kw):
    a = dict(x=A, ldx=64, xg=0, w=A, ldw=64, wg=0, groups=1, rows=4, n=32, k=64, b=A, bg=0, act=0, r=2 * A, ldr=32, rg=0, o=3 * A, f32=0,
             ldo=32, og=0)
    a.update(kw)
    return fwd.glm53f_fwd_gemm_bf16_fused(a["x"], a["ldx"], a["xg"], a["w"], a["ldw"], a["wg"], a["groups"], a["rows"], a["n"], a["k"],
                                          a["b"], a["bg"], a["act"], a["r"], a["ldr"], a["rg"], a["o"], a["f32"], a["ldo"], a["og"], None)


@pytest.mark.parametrize("bad", [dict(groups=0), dict(groups=70000), dict(rows=-1), dict(n=0), dict(k=0), dict(act=-1), dict(act=6),
                                 dict(x=None), dict(w=None), dict(o=None), dict(ldx=63), dict(ldw=63), dict(ldo=31), dict(ldr=31),
                                 dict(xg=-1), dict(wg=-1), dict(og=-1), dict(rg=-1), dict(bg=-1), dict(x=A + 1), dict(w=A + 1),
                                 dict(b=A + 1), dict(o=A + 1), dict(r=A + 1), dict(f32=1, o=A + 2), dict(f32=1, r=A + 2),
                                 dict(r=A, o=A, ldr=40), dict(r=A, o=A, groups=2, rg=128, og=256)])
def test_product_rejects(bad):
    assert gemm_call(**bad) == 1


def probs_call(**kw):
    a = dict(rows=4, vocab=100, x=A, f32=1, ldl=100, t=None, p=2 * A, ldp=100, ws=A, wb=1 << 20)
    a.update(kw)
    return spec.glm53f_spec_probs(a["rows"], a["vocab"], a["x"], a["f32"], a["ldl"], a["t"], a["p"], a["ldp"], a["ws"], a["wb"], None)


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(rows=70000), dict(vocab=0), dict(x=None), dict(p=None), dict(ws=None), dict(ldl=99),
                                 dict(ldp=99), dict(x=A + 2), dict(f32=0, x=A + 1), dict(p=A + 2), dict(t=A + 2), dict(ws=A + 8),
                                 dict(wb=1), dict(p=A, f32=0), dict(p=A, ldp=128)])
def test_probabilities_reject(bad):
    assert probs_call(**bad) == 1


def accept_call(**kw):
    a = dict(batch=2, vocab=100, cu=A, tok=A, p=A, ps=100, q=A, qs=100, u=A, keep=A, next=A, ws=A, wb=1 << 20)
    a.update(kw)
    return spec.glm53f_spec_accept(a["batch"], a["vocab"], a["cu"], a["tok"], a["p"], a["ps"], a["q"], a["qs"], a["u"], a["keep"],
                                   a["next"], a["ws"], a["wb"], None)


@pytest.mark.parametrize("bad", [dict(batch=-1), dict(batch=70000), dict(vocab=0), dict(cu=None), dict(tok=None), dict(p=None), dict(u=None),
                                 dict(keep=None), dict(next=None), dict(ws=None), dict(ps=99), dict(qs=99), dict(cu=A + 2), dict(tok=A + 1),
                                 dict(p=A + 2), dict(q=A + 2), dict(u=A + 1), dict(keep=A + 3), dict(next=A + 2), dict(ws=A + 8), dict(wb=8)])
def test_verification_rejects(bad):
    assert accept_call(**bad) == 1


def test_workspaces_and_empty_calls():
    assert spec.glm53f_spec_probs_workspace_bytes(-1, 5) == spec.glm53f_spec_probs_workspace_bytes(1, 0) == -1
    assert spec.glm53f_spec_accept_workspace_bytes(-1, 5) == spec.glm53f_spec_accept_workspace_bytes(1, 0) == -1
    assert spec.glm53f_spec_probs_workspace_bytes(3, 151936) > 0 < spec.glm53f_spec_accept_workspace_bytes(3, 151936)
    assert probs_call(rows=0, x=None, p=None, ws=None) == 0 and accept_call(batch=0, cu=None, ws=None) == 0
    assert gemm_call(rows=0, x=None, o=None) == 0


def test_a_vocabulary_past_its_bound_is_rejected():
    big = (1 << 30) + 1
    assert probs_call(vocab=big, ldl=big, ldp=big, wb=1 << 40) == 1 and accept_call(vocab=big, ps=big, qs=big, wb=1 << 40) == 1
    assert spec.glm53f_spec_probs_workspace_bytes(1, big) == spec.glm53f_spec_accept_workspace_bytes(1, big) == -1
    assert spec.glm53f_spec_probs_workspace_bytes(65536, 8) == spec.glm53f_spec_accept_workspace_bytes(65536, 8) == -1


@pytest.mark.parametrize("vocab", [1, 4096, 4097, 151936, 2_100_000])
def test_a_workspace_serves_fewer_rows_too(vocab):
    sizes = [spec.glm53f_spec_probs_workspace_bytes(r, vocab) for r in range(0, 700)]
    assert sizes == sorted(sizes) and sizes[0] == 0
    for rows, size in enumerate(sizes):
        assert size >= rows * -(-vocab // 4096) * 16


@pytest.mark.parametrize("heads,dk,dv", [(1, 64, 64), (16, 128, 128), (48, 64, 128), (300, 128, 64)])
def test_the_documented_bound_of_the_chunked_forms_workspace(heads, dk, dv):
    for batch in list(range(1, 70)) + [511, 512, 600]:
        for rows in (0, 1, 256, 257, 512, 700, 4096, 8191, 100_000, 1 << 30):
            need = lin.glm53f_lin_prefill_workspace_bytes(heads, dk, dv, batch, rows)
            assert 0 <= need <= min(1535, heads * batch * -(-rows // 256)) * dk * dv * 4
            if rows <= 256:
                assert need == 0


def test_the_gemms_python_wrapper():
    from glm53f_forward import gemm
    w = gemm.Bf16Mat(A, 32, 64, 64)
    with pytest.raises(gemm.GemmError):
        gemm.Gemm.fused(A, 64, 0, w, 4, gemm.Epilogue(act="swish"), A, 32, 0, False)
    with pytest.raises(gemm.GemmError):
        gemm.Gemm.fused(A, 63, 0, w, 4, gemm.Epilogue(act="silu"), A, 32, 0, False)
    gemm.Gemm.fused(A, 64, 0, w, 0, gemm.Epilogue(act="silu"), A, 32, 0, False)       # no rows: no launch
    assert gemm.ACTIVATIONS.index("gelu_tanh") == 4 and gemm.ACTIVATIONS.index("sigmoid") == 5


@pytest.mark.parametrize("bad", [dict(rows=(1 << 30) + 1), dict(n=(1 << 30) + 1, ldo=1 << 31, ldr=1 << 31), dict(k=(1 << 30) + 1, ldx=1 << 31, ldw=1 << 31)])
def test_a_product_past_its_bounds_is_rejected(bad):
    assert gemm_call(**bad) == 1
