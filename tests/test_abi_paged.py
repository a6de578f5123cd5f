"""Refusals of the operators over a K/V cache in pages and of draft_verify, before anything is enqueued (no GPU needed), their
sizes, and calls with nothing to do."""
import ctypes

import pytest

from test_abi_attn import WS

G4 = 1 << 32  # the buffers of a call lie 4 GiB apart
B, PAGES, MOST, NKVH, ROWS = 3, 50, 8, 4, 64
KB, VB = 4 * 64 * 272, 4 * 64 * 144


class KV:
    """Stands for ops.KvPages over addresses."""

    def __init__(self, k=G4, v=2 * G4, table=3 * G4, n_seqs=B, max_pages=MOST, n_pages=PAGES, nkvh=NKVH, rows=ROWS, type=2):
        from qwen27_engine_amd._lib import KvPagesC

        self.c = KvPagesC(k, v, table, n_seqs, max_pages, n_pages, nkvh, rows, type)
        self.ref = ctypes.addressof(self.c)


T = 10
SIZES = {"k": PAGES * KB, "v": PAGES * VB, "table": B * MOST * 4, "pos": B * 4, "cu": B * 4 + 4}
PREP = dict(SIZES, qg=T * 24 * 2048, kx=T * NKVH * 1024, vx=T * NKVH * 1024, qw=1024, kw=1024, qn=T * 24 * 1024, rope3=T * 12, rdelta=B * 4)
ATTN = dict(SIZES, qn=T * 24 * 1024, o=T * 24 * 1024, lse=T * 24 * 4, ws=1000)
READ = {"k": PAGES * KB, "v": PAGES * VB, "table": B * MOST * 4, "start": B * 4, "count": B * 4, "ko": B * NKVH * 100 * 1024,
        "vo": B * NKVH * 100 * 1024}
V = 5000
VERIFY = {"p": T * V * 4, "q": T * V * 4, "ids": T * 4, "u": T * 4, "u_last": B * 4, "cu": B * 4 + 4, "out": T * 4, "path": T * 4,
          "n_path": B * 4, "pos": B * 4, "ws": 16}
PLACES = {n: (i + 1) * G4 for i, n in enumerate(["k", "v", "table", "pos", "cu", "qg", "kx", "vx", "qw", "kw", "qn", "rope3", "rdelta", "o",
                                                 "lse", "ws", "start", "count", "ko", "vo", "p", "q", "ids", "u", "u_last", "out", "path",
                                                 "n_path"])}


def prep(ops, kv=None, nqh=24, tokens=T, **at):
    a = PLACES | at
    kv = KV(**({"k": a["k"], "v": a["v"], "table": a["table"]} | (kv or {})))
    ops.attn_prep_paged(a["qg"], a["kx"], a["vx"], a["qw"], a["kw"], a["qn"], kv, a["pos"], a["cu"], tokens, 1e-6, 0.6, nqh, 0, a["rope3"],
                      a["rdelta"])


def attn(ops, kv=None, nqh=24, tokens=T, most=4, ws_bytes=1 << 30, **at):
    a = PLACES | at
    kv = KV(**({"k": a["k"], "v": a["v"], "table": a["table"]} | (kv or {})))
    ops.attn_paged(a["qn"], kv, a["pos"], a["cu"], tokens, most, 0.0625, nqh, a["o"], WS(ws_bytes, a["ws"]), 0, a["lse"])


def read(ops, kv=None, n_out=100, type=0, **at):
    from qwen27_engine_amd._lib import check, lib

    a = PLACES | at
    kv = KV(**({"k": a["k"], "v": a["v"], "table": a["table"]} | (kv or {})))
    check(lib().q27h_kv_pages_read(kv.ref, a["start"], a["count"], n_out, type, a["ko"], a["vo"], None))


def verify(ops, n_seqs=B, tokens=T, vocab=V, parent=None, ldp=V, ldq=V, ws_bytes=1 << 30, **at):
    from qwen27_engine_amd._lib import check, lib

    a = PLACES | at
    check(lib().q27h_draft_verify(a["p"], ldp, a["q"], ldq, a["ids"], parent, a["u"], a["u_last"], a["cu"], n_seqs, tokens, vocab, a["out"],
                                  a["path"], a["n_path"], a["pos"], a["ws"], ws_bytes, None))


def accept(ops, kv=None, layers=2, tokens=T, other=None, **at):
    """Two layers, the second one's pages 100 places on; `other`: what it has of its own."""
    from qwen27_engine_amd._lib import KvPagesC, check, lib

    a = PLACES | at
    one = {"k": a["k"], "v": a["v"], "table": a["table"]} | (kv or {})
    two = one | {"k": 101 * G4, "v": 102 * G4} | (other or {})
    hs = [KV(**one), KV(**two)]
    c = (KvPagesC * 2)(*(h.c for h in hs))
    check(lib().q27h_kv_accept_paged(c if layers else None, layers, a["pos"], a["cu"], a["path"], a["n_path"], tokens, None))


def refused(q27, call, code, needle, **args):
    with pytest.raises(q27.Q27Error) as ei:
        call(q27.ops, **args)
    assert ei.value.code == code and needle in str(ei.value)


@pytest.mark.parametrize("call", [prep, attn, read])
@pytest.mark.parametrize("bad,code,needle", [
    (dict(type=3), -1, "unknown type"), (dict(type=-1), -1, "unknown type"), (dict(rows=48), -1, "power of two"),
    (dict(rows=16), -1, "power of two"), (dict(rows=0), -1, "power of two"), (dict(rows=131072), -1, "power of two"),
    (dict(nkvh=0), -1, "bad sizes"), (dict(nkvh=5000), -1, "bad sizes"), (dict(n_seqs=-1), -1, "bad sizes"),
    (dict(max_pages=1 << 25), -1, "bad sizes"), (dict(n_pages=-1), -1, "bad sizes"), (dict(k=None), -4, "null pointer"),
    (dict(v=None), -4, "null pointer"), (dict(table=None), -4, "null pointer"), (dict(k=G4 + 8), -4, "alignment"),
    (dict(v=2 * G4 + 4), -4, "alignment"), (dict(table=3 * G4 + 2), -4, "alignment")])
def test_bad_handles(q27, call, bad, code, needle):
    refused(q27, call, code, needle, kv=bad)


@pytest.mark.parametrize("call,args,code,needle", [
    (prep, dict(tokens=-1), -1, "bad shape"), (prep, dict(nqh=0), -1, "bad shape"), (prep, dict(nqh=5000), -1, "bad shape"),
    (prep, dict(cu=None), -1, "one token for each"), (prep, dict(tokens=2 ** 31 // 64), -1, "too many tokens"),
    (attn, dict(tokens=-1), -1, "bad shape"), (attn, dict(most=0), -1, "bad shape"), (attn, dict(most=65), -1, "bad shape"),
    (attn, dict(nqh=25), -1, "bad shape"), (attn, dict(nqh=0), -1, "bad shape"), (attn, dict(cu=None), -1, "one token for each"),
    (attn, dict(kv=dict(n_seqs=1 << 20, max_pages=1 << 14)), -1, "too many rows"),
    (attn, dict(kv=dict(n_seqs=1 << 20, max_pages=1)), -1, "too many query rows"),
    (attn, dict(tokens=1 << 20), -1, "too many query rows"),
    (attn, dict(ws_bytes=1000), -4, "workspace too small"), (attn, dict(ws=0), -4, "workspace too small"),
    (read, dict(n_out=-1), -1, "bad n_out"), (read, dict(type=3), -1, "bad n_out"), (read, dict(type=-1), -1, "bad n_out"),
    (read, dict(n_out=1 << 29, kv=dict(n_seqs=1 << 10)), -1, "too many rows"),
    (verify, dict(n_seqs=-1), -1, "bad shape"), (verify, dict(tokens=-1), -1, "bad shape"), (verify, dict(vocab=0), -1, "bad shape"),
    (verify, dict(vocab=(1 << 24) + 1, ldp=1 << 25, ldq=1 << 25), -1, "bad shape"), (verify, dict(ldp=V - 1), -1, "row stride"),
    (verify, dict(ldq=V - 1), -1, "row stride"), (verify, dict(ldp=1 << 29), -1, "row stride"),
    (verify, dict(n_seqs=1 << 23), -1, "too many sequences"), (verify, dict(parent=50 * G4), -4, "exclude each other"),
    (verify, dict(ws_bytes=8), -4, "workspace too small"),
])
def test_bad_shapes(q27, call, args, code, needle):
    refused(q27, call, code, needle, **args)


def cases(call, sizes, unless):
    return [(call, n) for n in sizes if n not in unless]


@pytest.mark.parametrize("call,name", cases(prep, PREP, ("cu", "rope3", "rdelta", "k", "v", "table")) +
                         cases(attn, ATTN, ("cu", "lse", "k", "v", "table", "ws")) + [(read, "count")] +
                         cases(verify, VERIFY, ("q", "pos", "ws")))
def test_null_pointers(q27, call, name):
    refused(q27, call, -4, "null pointer", **{name: None})


@pytest.mark.parametrize("call,name", cases(prep, PREP, ("k", "v", "table")) + cases(attn, ATTN, ("k", "v", "table")) +
                         cases(read, READ, ("k", "v", "table")) + cases(verify, VERIFY, ()))
def test_alignment(q27, call, name):
    refused(q27, call, -4, "alignment", **{name: PLACES[name] + 2})
    if name in ("qg", "kx", "vx", "qw", "kw", "qn", "o", "ko", "vo", "ws"):
        refused(q27, call, -4, "alignment", **{name: PLACES[name] + 8})


def pairs(call, outs, sizes):
    return [(call, a, b, sizes[b]) for a in outs for b in sizes if a != b]


@pytest.mark.parametrize("call,out,other,size", pairs(prep, ["qn", "k", "v"], PREP) + pairs(attn, ["o", "lse", "ws"], ATTN) +
                         pairs(read, ["ko", "vo"], READ) + pairs(verify, ["out", "path", "n_path", "pos", "ws"], VERIFY))
def test_overlaps(q27, call, out, other, size):
    refused(q27, call, -4, "overlap", **{out: PLACES[other] + (size - 1) // 16 * 16})  # its last 16 bytes


def test_nothing_to_do(q27):
    o = q27.ops
    none = dict(k=None, v=None, table=None, n_seqs=0, max_pages=0, n_pages=0)
    prep(o, kv=none)
    prep(o, tokens=0)
    attn(o, kv=none)
    attn(o, tokens=0)
    read(o, kv=none)
    read(o, n_out=0)
    read(o, ko=None, vo=None)
    verify(o, n_seqs=0)


def test_sizes(q27):
    o = q27.ops
    assert o.kv_page_bytes(4, 64, o.KV_F16, False) == o.kv_page_bytes(4, 64, o.KV_F16, True) == 4 * 64 * 512
    assert o.kv_page_bytes(4, 64, o.KV_Q8, True) == o.kv_page_bytes(4, 64, o.KV_Q8_Q4, False) == KB
    assert o.kv_page_bytes(4, 64, o.KV_Q8_Q4, True) == VB
    assert o.kv_page_bytes(4, 64, 3, True) == o.kv_page_bytes(0, 64, 1, True) == o.kv_page_bytes(4, -1, 1, True) == 0
    assert o.attn_paged_ws_bytes(KV(), 10, 4, 24) > 0
    assert o.attn_paged_ws_bytes(KV(), 0, 4, 24) == o.attn_paged_ws_bytes(KV(rows=48), 10, 4, 24) == 0
    assert o.attn_paged_ws_bytes(KV(), 10, 65, 24) == o.attn_paged_ws_bytes(KV(), 10, 4, 25) == 0
    assert o.draft_verify_ws_bytes(3, 248320) >= 3 * 61 * 16
    assert o.draft_verify_ws_bytes(0, 10) == o.draft_verify_ws_bytes(1, 0) == o.draft_verify_ws_bytes(1, (1 << 24) + 1) == 0


def test_a_handle_needs_a_whole_table(q27):
    import torch

    k, v = torch.zeros(2 * KB, dtype=torch.uint8), torch.zeros(3 * VB, dtype=torch.uint8)
    kv = q27.ops.KvPages(k, v, torch.zeros(3, 8, dtype=torch.int32), 4, 64, q27.ops.KV_Q8_Q4)
    assert (kv.c.n_pages, kv.c.n_seqs, kv.c.max_pages) == (2, 3, 8)
    for table in (torch.zeros(3, 8, dtype=torch.int64), torch.zeros(8, 3, dtype=torch.int32).t(), torch.zeros(24, dtype=torch.int32)):
        with pytest.raises(ValueError):
            q27.ops.KvPages(k, v, table, 4, 64, q27.ops.KV_Q8_Q4)


def test_a_handle_refuses_other_numbers_and_pages_apart(q27):
    import torch

    k, v, table = torch.zeros(2, KB, dtype=torch.uint8), torch.zeros(2, VB, dtype=torch.uint8), torch.zeros(3, 8, dtype=torch.int32)
    for bad in ((k, v, table.float()), (k.t(), v, table), (k, v[:, ::2], table)):
        with pytest.raises(ValueError):
            q27.ops.KvPages(*bad, 4, 64, q27.ops.KV_Q8_Q4)


ACCEPT = dict(SIZES, path=T * 4, n_path=B * 4)


@pytest.mark.parametrize("args,code,needle", [
    (dict(tokens=-1), -1, "bad shape"), (dict(layers=-1), -1, "bad shape"), (dict(kv=dict(rows=48)), -1, "power of two"),
    (dict(kv=dict(k=None)), -4, "null pointer"), (dict(other=dict(v=None)), -4, "null pointer"),
    (dict(kv=dict(n_seqs=40000)), -1, "too many sequences"), (dict(other=dict(type=1)), -4, "different"),
    (dict(other=dict(n_seqs=2)), -4, "different"), (dict(other=dict(max_pages=9)), -4, "different"),
    (dict(other=dict(n_pages=49)), -4, "different"), (dict(other=dict(nkvh=2)), -4, "different"),
    (dict(other=dict(rows=32)), -4, "different"), (dict(other=dict(table=4 * G4)), -4, "different"),
    (dict(other=dict(k=G4 + 16)), -4, "overlap"), (dict(other=dict(v=G4)), -4, "overlap"),
    (dict(other=dict(k=101 * G4, v=101 * G4 + PAGES * KB - 16)), -4, "overlap")] +
    [({n: None}, -4, "null pointer") for n in ("pos", "cu", "path", "n_path")] +
    [({n: PLACES[n] + 2}, -4, "alignment") for n in ("pos", "cu", "path", "n_path")] +
    [({o: PLACES[n] + (ACCEPT[n] - 1) // 16 * 16}, -4, "overlap") for o in ("k", "v") for n in ACCEPT if n != o])
def test_accept_refusals(q27, args, code, needle):
    refused(q27, accept, code, needle, **args)


def test_accept_with_nothing_to_do(q27):
    accept(q27.ops, layers=0)
    accept(q27.ops, tokens=0)
    accept(q27.ops, kv=dict(k=None, v=None, table=None, n_seqs=0, max_pages=0, n_pages=0), other=dict(k=None, v=None))


def attn_of_trees(ops, tree, **at):
    a = PLACES | at
    ops.attn_paged(a["qn"], KV(), a["pos"], a["cu"], T, 4, 0.0625, 24, a["o"], WS(1 << 30, a["ws"]), 0, a["lse"], tree)


def test_masks_are_checked(q27):
    refused(q27, attn_of_trees, -4, "alignment", tree=60 * G4 + 4)
    for out in ("o", "lse", "ws"):
        refused(q27, attn_of_trees, -4, "overlap", tree=60 * G4, **{out: 60 * G4 + T * 8 - 16})


def test_cpp_header_forwards(tmp_path):
    """include/q27/attn.h: every function compiles in a caller, and a refusal arrives as an exception."""
    import os
    import subprocess

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    lib = os.path.join(root, "qwen27-engine_amd", "lib")
    src, exe = tmp_path / "caller.cpp", tmp_path / "caller"
    src.write_text(r'''
#include <cstdio>
#include "q27/attn.h"
void step(const float* x, const q27::KvPages& kv, int* pos, const int* cu, int* out, float* o, float* lse, void* ws, size_t n,
          hipStream_t s) {
  q27::attn_prep_paged(x, x, x, x, x, o, kv, pos, cu, 9, 1e-6f, 0.6f, 24, s, nullptr, pos);
  q27::attn_paged(x, kv, pos, cu, 9, 4, 0.0625f, 24, o, ws, n, s, lse);
  q27::kv_pages_read(kv, nullptr, pos, 100, Q27H_F16, ws, ws, s);
  q27::draft_verify(x, 100, x, 100, pos, nullptr, x, x, cu, 3, 9, 100, out, out, out, ws, n, s, pos);
  q27::kv_accept_paged(&kv, 1, pos, cu, out, out, 9, s);
  q27::attn_paged(x, kv, pos, cu, 9, 4, 0.0625f, 24, o, ws, n, s, lse, (const uint64_t*)out);
}
int main(int argc, char**) {
  q27::KvPages kv = {nullptr, nullptr, nullptr, 3, 8, 50, 4, 64, Q27H_KV_Q8_Q4};
  if (argc > 9) step(nullptr, kv, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 0, nullptr);
  size_t n = q27::kv_page_bytes(4, 64, kv.type, true) + q27::attn_paged_ws_bytes(kv, 9, 4, 24) + q27::draft_verify_ws_bytes(3, 100);
  try {
    q27::attn_paged(nullptr, kv, nullptr, nullptr, 9, 4, 1.0f, 24, nullptr, nullptr, 0, nullptr);
  } catch (const std::runtime_error& e) {
    std::printf("%d %s\n", n > 0, e.what());
    return 0;
  }
  return 1;
}
''')
    subprocess.run(["/opt/rocm/llvm/bin/clang++", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    f"-I{root}/include", str(src), f"-L{lib}", "-lq27h", "-L/opt/rocm/lib", "-lamdhip64", f"-Wl,-rpath,{lib}",
                    "-Wl,-rpath,/opt/rocm/lib", "-o", str(exe)], check=True, capture_output=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=60).stdout
    assert out.startswith("1 ") and "null pointer" in out


def test_header_is_c(tmp_path):
    import os
    import subprocess

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "caller.c"
    src.write_text('#include "q27h.h"\nint main(void) { q27h_kv_pages kv = {0}; return q27h_kv_pages_read(&kv, 0, 0, 0, Q27H_F32, 0, 0, 0) == 0; }\n')
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", f"-I{root}/include", "-c", str(src), "-o", str(tmp_path / "o")], check=True)
