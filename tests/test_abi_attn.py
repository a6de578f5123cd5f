"""Refusals of the operators over the K/V cache, before anything is enqueued (no GPU needed), their workspace sizes, and
calls with nothing to do."""
import pytest

FAKE = 1 << 20   # an aligned address that no call below may touch
BIG = 1 << 40


class WS:
    """Stands for a workspace tensor."""

    def __init__(self, n, at=BIG):
        self.n, self.at = n, at

    def numel(self):
        return self.n

    def element_size(self):
        return 1

    def data_ptr(self):
        return self.at


F, W = FAKE, WS(1 << 34)


def tree(o, qn=F, k=F, v=F, pos0=F, T=4, nqh=24, nkvh=4, n_ctx=4096, out=F << 4, ws=W):
    o.attn_tree(qn, k, v, pos0, None, T, 0.0625, nqh, nkvh, n_ctx, True, out, ws, 0)


def weights(o, qn=F, lse=F, k=F, T=4, nqh=24, nkvh=4, n_ctx=4096, acc=F):
    o.attn_weights(qn, lse, k, F, None, T, 0.0625, nqh, nkvh, n_ctx, True, acc, 0)


def evict(o, k=1 << 32, v=2 << 32, acc=3 << 32, keep=64, first=4, last=16, ko=4 << 32, vo=5 << 32, ao=6 << 32, n_out=128,
          nkvh=4, n_ctx=4096, ws=W):
    o.kv_evict(k, v, acc, F, keep, first, last, ko, vo, ao, n_out, None, nkvh, n_ctx, True, ws, 0)


def accept(o, caches=(F, 2 * F), accs=(), T=4, nkvh=4, n_ctx=64, path=F):
    o.kv_accept(list(caches), list(accs), F, path, F, T, nkvh, n_ctx, True, 0)


def bounds(o, k=F, T=4, nkvh=4, n_ctx=4096, kb=F):
    o.kv_block_bounds(k, F, T, nkvh, n_ctx, True, kb, 0)


def select(o, qn=F, kb=F, T=4, nqh=24, nkvh=4, n_ctx=4096, nsel=16, first=1, last=2, ws=W):
    o.attn_select(qn, kb, F, T, nqh, nkvh, n_ctx, nsel, first, last, F, ws, 0)


def blocks(o, qn=F, T=4, nsel=16, nqh=24, nkvh=4, n_ctx=4096, out=F << 4, ws=W):
    o.attn_blocks(qn, F, F, F, F, T, nsel, 0.0625, nqh, nkvh, n_ctx, True, out, ws, 0)


@pytest.mark.parametrize("call,code,needle", [
    (lambda o: tree(o, T=65), -1, "0..64"),
    (lambda o: tree(o, T=-1), -1, "0..64"),
    (lambda o: tree(o, nqh=25), -1, "bad shape"),
    (lambda o: tree(o, nkvh=0), -1, "bad shape"),
    (lambda o: tree(o, n_ctx=0), -1, "bad shape"),
    (lambda o: tree(o, qn=None), -4, "null pointer"),
    (lambda o: tree(o, pos0=None), -4, "null pointer"),
    (lambda o: tree(o, k=F + 8), -4, "alignment"),
    (lambda o: tree(o, out=F + 4), -4, "alignment"),
    (lambda o: tree(o, ws=WS(1000)), -4, "workspace too small"),
    (lambda o: tree(o, ws=None), -4, "workspace too small"),
    (lambda o: tree(o, ws=WS(1 << 34, BIG + 8)), -4, "alignment"),
    (lambda o: tree(o, out=F + 1024), -4, "o overlaps qn"),
    (lambda o: blocks(o, out=F + 1024), -4, "o overlaps qn"),
    (lambda o: weights(o, T=65), -1, "0..64"),
    (lambda o: weights(o, nqh=23), -1, "bad shape"),
    (lambda o: weights(o, lse=None), -4, "null pointer"),
    (lambda o: weights(o, acc=None), -4, "null pointer"),
    (lambda o: weights(o, k=F + 4), -4, "alignment"),
    (lambda o: evict(o, keep=0), -1, "keep >= 1"),
    (lambda o: evict(o, first=-1), -1, "first + last"),
    (lambda o: evict(o, first=50, last=15), -1, "first + last"),
    (lambda o: evict(o, keep=200), -1, "n_ctx_out"),
    (lambda o: evict(o, keep=5000, n_out=8192), -1, "n_ctx_out"),
    (lambda o: evict(o, nkvh=0), -1, "bad shape"),
    (lambda o: evict(o, acc=None), -4, "null pointer"),
    (lambda o: evict(o, ko=(4 << 32) + 8), -4, "alignment"),
    (lambda o: evict(o, ws=WS(100)), -4, "workspace too small"),
    (lambda o: evict(o, ko=1 << 32), -4, "overlap"),                              # K in place, the others not
    (lambda o: evict(o, ko=1 << 32, vo=2 << 32, ao=3 << 32), -4, "overlap"),      # in place with another context
    (lambda o: evict(o, vo=(1 << 32) + 4096), -4, "overlap"),
    (lambda o: evict(o, ao=(3 << 32) + 16), -4, "overlap"),
    (lambda o: evict(o, vo=4 << 32), -4, "overlap"),
    (lambda o: o.kv_evict_pos(F, F, 0, 0), -1, "keep >= 1"),
    (lambda o: o.kv_evict_pos(None, F, 4, 0), -4, "null pointer"),
    (lambda o: accept(o, T=65), -1, "0..64"),
    (lambda o: accept(o, nkvh=0), -1, "bad shape"),
    (lambda o: accept(o, path=None), -4, "null pointer"),
    (lambda o: accept(o, caches=(F, None)), -4, "null pointer"),
    (lambda o: accept(o, caches=(F, F + 8)), -4, "alignment"),
    (lambda o: accept(o, accs=(None,)), -4, "null pointer"),
    (lambda o: accept(o, caches=(F, 2 * F, F)), -4, "overlap"),                   # a cache twice
    (lambda o: accept(o, caches=(F, F + 4096)), -4, "overlap"),
    (lambda o: accept(o, accs=(F + 4096,)), -4, "overlap"),
    (lambda o: accept(o, caches=(2 * F,), accs=(F, F + 4)), -4, "overlap"),
    (lambda o: bounds(o, T=-1), -1, "bad shape"),
    (lambda o: bounds(o, n_ctx=0), -1, "bad shape"),
    (lambda o: bounds(o, kb=None), -4, "null pointer"),
    (lambda o: bounds(o, kb=F + 4), -4, "alignment"),
    (lambda o: select(o, nqh=68), -1, "at most 16"),
    (lambda o: select(o, nsel=2), -1, "first + last"),
    (lambda o: select(o, last=0), -1, "last >= 1"),
    (lambda o: select(o, first=-1), -1, "first >= 0"),
    (lambda o: select(o, n_ctx=1024001), -1, "1024000"),
    (lambda o: select(o, T=1 << 30), -1, "T too large"),
    (lambda o: select(o, kb=None), -4, "null pointer"),
    (lambda o: select(o, ws=WS(100)), -4, "workspace too small"),
    (lambda o: blocks(o, nqh=68), -1, "at most 16"),
    (lambda o: blocks(o, nsel=0), -1, "bad shape"),
    (lambda o: blocks(o, T=1 << 30), -1, "too large"),
    (lambda o: blocks(o, qn=None), -4, "null pointer"),
    (lambda o: blocks(o, qn=F + 4), -4, "alignment"),
    (lambda o: blocks(o, ws=WS(64)), -4, "workspace too small"),
])
def test_refused_before_launch(q27, call, code, needle):
    with pytest.raises(q27.Q27Error) as ei:
        call(q27.ops)
    assert ei.value.code == code
    assert needle in str(ei.value)


def test_no_tokens_is_no_work(q27):
    o = q27.ops
    tree(o, T=0), weights(o, T=0), accept(o, T=0), accept(o, caches=()), bounds(o, T=0), select(o, T=0), blocks(o, T=0)


def test_workspace_sizes(q27):
    o = q27.ops
    assert o.attn_tree_ws_bytes(65, 24, 4, 4096) == 0 and o.attn_tree_ws_bytes(4, 25, 4, 4096) == 0
    # parts: [row][split] of 256 values and two statistics; 32 rows of context are one split at the most
    assert o.attn_tree_ws_bytes(1, 24, 4, 32) == 0
    for T in (1, 4, 64):
        assert o.attn_tree_ws_bytes(T, 24, 4, 180224) % (T * 24 * 258 * 4) == 0
    assert o.kv_block_bytes(4, 180224) == 4 * 2816 * 516 and o.kv_block_bytes(2, 65) == 2 * 2 * 516
    assert o.attn_select_ws_bytes(5, 4, 129) == 5 * 4 * 3 * 4
    assert o.attn_blocks_ws_bytes(1027, 24, 4, 32) == 0 and o.attn_blocks_ws_bytes(1, 24, 4, 64) > 0
    assert o.kv_evict_ws_bytes(4, 4096, 64, True, True) >= o.kv_evict_ws_bytes(4, 4096, 64, True, False) + 2 * 4 * 64 * 272


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
void step(const float* qn, void* k, void* v, int* pos0, const uint64_t* tree, float* o, float* lse, float* acc, void* kb, int* idx,
          void* ws, size_t n, hipStream_t s) {
  q27::attn_tree(qn, k, v, pos0, tree, 4, 0.0625f, 24, 4, 4096, true, o, ws, n, s, lse);
  q27::attn_weights(qn, lse, k, pos0, tree, 4, 0.0625f, 24, 4, 4096, true, acc, s, tree);
  q27::kv_evict(k, v, acc, pos0, 1024, 4, 64, k, v, acc, 4096, nullptr, 4, 4096, true, ws, n, s);
  q27::kv_evict_pos(pos0, idx, 1024, s);
  void* caches[2] = {k, v};
  q27::kv_accept(caches, 2, &acc, 1, pos0, idx, idx, 4, 4, 4096, true, s);
  q27::kv_block_bounds(k, pos0, 4, 4, 4096, true, kb, s);
  q27::attn_select(qn, kb, pos0, 4, 24, 4, 4096, 32, 1, 2, idx, ws, n, s);
  q27::attn_blocks(qn, k, v, pos0, idx, 4, 32, 0.0625f, 24, 4, 4096, true, o, ws, n, s, lse);
}
int main(int argc, char**) {
  if (argc > 9) step(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 0, nullptr);
  size_t n = q27::attn_tree_ws_bytes(4, 24, 4, 4096) + q27::kv_evict_ws_bytes(4, 4096, 64, true, false) +
             q27::kv_block_bytes(4, 4096) + q27::attn_select_ws_bytes(4, 4, 4096) + q27::attn_blocks_ws_bytes(4, 24, 4, 32);
  try {
    q27::attn_tree(nullptr, nullptr, nullptr, nullptr, nullptr, 65, 1.0f, 24, 4, 4096, true, nullptr, nullptr, 0, nullptr);
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
    assert out.startswith("1 ") and "T must be 0..64" in out
