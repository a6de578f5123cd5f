"""attn_paged and kv_accept_paged with token offsets that do not rise or lie outside 0 .. T: they are cut to rise within it, each
sequence has the tokens that are left, and no byte but theirs is written, inside the arrays or around them."""
import numpy as np
import pytest

import pagedref as P
from test_gpu_attn import G, SCALE, near  # noqa: F401
from test_gpu_paged import TYPES, handle
from test_gpu_paged_trees import pools_of

pytestmark = pytest.mark.gpu
T = 8


def tokens(cu):
    """(first, behind the last) token of each sequence."""
    out = []
    for a, b in zip(cu, cu[1:]):
        a = min(max(a, 0), T)
        out.append((a, min(max(b, a), T)))
    return out


def guarded(G, x):  # noqa: F811
    """x on the GPU between bytes of 0x5A, and whether they still are."""
    import torch

    n = x.numel() * x.element_size() if hasattr(x, "numel") else x.nbytes
    buf = G.full((n + 8192,), 0x5A, torch.uint8)
    mid = buf[4096:4096 + n]
    mid.copy_(x.view(torch.uint8).view(-1) if hasattr(x, "numel") else G.up(x.reshape(-1).view(np.uint8)))
    return mid, lambda: bool(np.all(G.down(buf[:4096]) == 0x5A) and np.all(G.down(buf[4096 + n:]) == 0x5A))


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("most", [2, 8])
@pytest.mark.parametrize("cu", [[0, 5, 3, 9], [-4, 2, 2, 100], [3, 3, 3, 3], [7, 1, 0, -1], [-2 ** 31, 3, 2 ** 31 - 1, 5]])
def test_attn(G, cu, most, type):  # noqa: F811
    import torch

    r = np.random.default_rng(8)
    pos = [50, 9, 20]
    kp, vp, table = P.make_pages(r, pos, [8, 8, 8], 32, 4, type)
    q = r.standard_normal((T, 24, 256)).astype(np.float32)
    kv = handle(G, kp, vp, table, type)
    (o, o_whole), (lse, lse_whole) = (guarded(G, np.full(s, 7, np.float32)) for s in ((T, 24, 256), (T, 24)))
    o, lse = o.view(torch.float32).view(T, 24, 256), lse.view(torch.float32).view(T, 24)
    ws, ws_whole = guarded(G, G.ws(G.ops.attn_paged_ws_bytes(kv, T, most, 24)))
    G.ops.attn_paged(G.up(q), kv, G.i32(*pos), G.i32(*cu), T, most, SCALE, 24, o, ws, lse=lse)
    assert o_whole() and lse_whole() and ws_whole()
    o, lse = G.down(o), G.down(lse)
    of = [[] for _ in range(T)]  # the sequences that have each token
    for b, (c0, c1) in enumerate(tokens(cu)):
        for t in range(c0, min(c1, c0 + most)):
            of[t].append(b)
    for b, (c0, c1) in enumerate(tokens(cu)):
        n = min(c1 - c0, most)
        if n:
            on = [t for t in range(c0, c0 + n) if of[t] == [b]]
            eo, el, bo, bl = P.attend(q[c0:c0 + n], kp, vp, table[b:b + 1], pos[b:b + 1], [n], SCALE)
            at = [t - c0 for t in on]
            near(o[on], eo[at], bo[at], "o")
            near(lse[on], el[at], bl[at], "lse")
    none = [t for t in range(T) if not of[t]]
    assert np.all(o[none] == 7) and np.all(lse[none] == 7)


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("cu", [[0, 9, 3, 20], [-5, 3, 6, 100], [8, 1, 0, -1], [0, 6, 2, 8], [-2 ** 31, 5, 2 ** 31 - 1, 0]])
@pytest.mark.parametrize("pos,n_path", [([9, 7, 40], [4, 3, 5]), ([2 ** 31 - 1, 6, -2 ** 31], [-2 ** 31, 100, 2 ** 31 - 1])])
def test_accept(G, pos, n_path, cu, type):  # noqa: F811
    r = np.random.default_rng(1)
    table = np.array([[0, 1], [2, 3], [4, 5]], np.int32)
    d = G.up(table)
    layers = pools_of(r, 2, 6, 2, 32, type)
    pools, kvs = [], []
    for k, v in layers:
        pair = [guarded(G, x.buf) for x in (k, v)]
        kvs.append(G.ops.KvPages(*(x.view(6, -1) for x, _ in pair), d, 2, 32, type))
        pools += [(pool, x, whole) for pool, (x, whole) in zip((k, v), pair)]
    path = np.array([0, 2, 1, 0, 2, 2, 1, -1], np.int32)
    G.ops.kv_accept_paged(kvs, G.i32(*pos), G.i32(*cu), G.up(path), G.i32(*n_path), T)
    for pool, x, whole in pools:
        assert whole()
        for b, (c0, c1) in enumerate(tokens(cu)):
            P.accept(pool, table[b:b + 1], pos[b:b + 1], [c0, c1], path, n_path[b:b + 1])
        assert np.array_equal(G.down(x).reshape(pool.buf.shape), pool.buf)
