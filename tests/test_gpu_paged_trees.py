"""Trees of drafts over a K/V cache in pages on the GPU: attn_paged with masks (within the bounds of tests/attnref.py),
kv_accept_paged (byte for byte), and a step of a batch of trees, eager and in a HIP graph."""
import numpy as np
import pytest

import cfgdata as cd
import pagedref as P
from test_gpu_attn import G, SCALE, near  # noqa: F401
from test_gpu_paged import TYPES, handle, prep_inputs, probabilities

pytestmark = pytest.mark.gpu


def random_tree(r, n):
    """A parent for each token (-1 for the first), and the ancestors of each with itself as a mask."""
    parent = np.array([-1] + [int(r.integers(max(0, t - 4), t)) for t in range(1, n)], np.int32)
    mask = np.zeros(n, np.uint64)
    for t in range(n):
        mask[t] = np.uint64(1 << t) | (mask[parent[t]] if t else np.uint64(0))
    return parent, mask


def attn(G, q, kv, pos, cu, most, nqh, tree):  # noqa: F811
    T = q.shape[0]
    o, lse = G.full((T, nqh, 256), 7.0), G.full((T, nqh), 7.0)
    d = None if tree is None else G.up(np.asarray(tree, np.uint64).view(np.int64))
    G.ops.attn_paged(q, kv, pos, cu, T, most, SCALE, nqh, o, G.ws(G.ops.attn_paged_ws_bytes(kv, T, most, nqh)), lse=lse, tree=d)
    return G.down(o), G.down(lse)


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("kind", ["tree", "any bits", "none"])
@pytest.mark.parametrize("pos,new,page,nqh,nkvh", [
    ([0], [1], 32, 24, 4), ([40, 31, 0], [2, 1, 2], 32, 24, 4), ([63, 500, 7], [12, 0, 5], 64, 24, 4), ([20, 100], [64, 33], 64, 24, 4),
    ([6000, 90], [4, 6], 64, 24, 4), ([77, 1], [16, 3], 256, 7, 7), ([33], [40], 32, 24, 1)])
def test_masks(G, pos, new, page, nqh, nkvh, kind, type):  # noqa: F811
    """Ancestors; bits of any kind, those of tokens that do not exist among them; and no new token seen at all."""
    r = np.random.default_rng(sum(pos) + 3 * sum(new) + nqh)
    kp, vp, table = P.make_pages(r, pos, new, page, nkvh, type)
    T = sum(new)
    q = (r.standard_normal((T, nqh, 256)) * 1.5).astype(np.float32)
    if kind == "tree":
        tree = np.concatenate([random_tree(r, n)[1] for n in new if n])
    else:
        tree = r.integers(0, 2 ** 64, T, dtype=np.uint64) if kind == "any bits" else np.zeros(T, np.uint64)
    o, lse = attn(G, G.up(q), handle(G, kp, vp, table, type), G.i32(*pos), G.up(P.cu_of(new)), max(new), nqh, tree)
    eo, el, bo, bl = P.attend(q, kp, vp, table, pos, new, SCALE, tree)
    near(o, eo, bo, "o")
    seen = np.isfinite(el)
    assert np.array_equal(seen, lse != -np.inf)
    near(lse[seen], el[seen], bl[seen], "lse")
    if kind == "none":
        assert not seen[[b == 0 for b, n in zip(pos, new) for _ in range(n)]].any()


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("T", [1, 2, 4, 40])
def test_a_chain_s_mask_is_no_mask(G, T, type):  # noqa: F811
    r = np.random.default_rng(T)
    pos, new = [300, 17, 5000], [T, max(1, T - 1), T]
    kp, vp, table = P.make_pages(r, pos, new, 64, 4, type)
    q = G.up(r.standard_normal((sum(new), 24, 256)).astype(np.float32))
    tree = np.concatenate([[(2 << t) - 1 for t in range(n)] for n in new]).astype(np.uint64)
    got = [attn(G, q, handle(G, kp, vp, table, type), G.i32(*pos), G.up(P.cu_of(new)), T, 24, m) for m in (None, tree)]
    for a, b in zip(*got):
        assert np.array_equal(a.view(np.uint8), b.view(np.uint8))


@pytest.mark.parametrize("type", TYPES)
def test_rows_of_other_branches_may_hold_anything(G, type):  # noqa: F811
    """NaN and infinities in the rows of tokens that a token does not see do not reach it."""
    r = np.random.default_rng(3)
    pos, new, nqh, nkvh = [70, 30], [9, 5], 24, 4
    kp, vp, table = P.make_pages(r, pos, new, 32, nkvh, type)
    q = r.standard_normal((sum(new), nqh, 256)).astype(np.float32)
    tree = np.concatenate([np.full(n, 0b10101, np.uint64) for n in new])
    want = P.attend(q, kp, vp, table, pos, new, SCALE, tree)
    for b in range(2):
        for t in (1, 3):
            j = pos[b] + t
            for pool, x in ((kp, np.nan), (vp, np.inf)):
                row = (table[b, j // 32], slice(None), j % 32)
                (pool.codes if pool.scales is None else pool.scales)[row] = np.full(
                    (nkvh, 256 if pool.scales is None else 8), x, np.float16).view(np.uint8)
    o, lse = attn(G, G.up(q), handle(G, kp, vp, table, type), G.i32(*pos), G.up(P.cu_of(new)), 9, nqh, tree)
    near(o, want[0], want[2], "o")
    near(lse, want[1], want[3], "lse")


def pools_of(r, n_layers, n_pages, nkvh, page, type):
    out = []
    for _ in range(n_layers):
        pair = [P.Pool(n_pages, nkvh, page, P.bits_of(type, v), 0) for v in (False, True)]
        for p in pair:
            p.buf[:] = r.integers(0, 256, p.buf.shape)
        out.append(pair)
    return out


def accept(G, layers, table, type, pos, cu, path, n_path):  # noqa: F811
    """Runs kv_accept_paged and holds every byte of every pool to the plain form."""
    d = G.up(table)
    kvs = [G.ops.KvPages(G.up(k.buf), G.up(v.buf), d, k.nkvh, k.page, type) for k, v in layers]
    G.ops.kv_accept_paged(G.ops.kv_layers(kvs), G.i32(*pos), G.i32(*cu), G.up(np.asarray(path, np.int32)), G.i32(*n_path), len(path))
    for (k, v), kv in zip(layers, kvs):
        for pool, x in ((k, kv.k), (v, kv.v)):
            P.accept(pool, table, pos, cu, path, n_path)
            assert np.array_equal(G.down(x), pool.buf)


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("n_layers,nkvh,page", [(1, 4, 32), (3, 1, 64), (2, 7, 128), (33, 2, 32)])
def test_accept(G, n_layers, nkvh, page, type):  # noqa: F811
    """Prefixes, paths across pages, of 64 tokens, of none, in any order, with entries that are no tokens and counts past the
    tokens; sequences before row 0, behind the last page, and with a page that is none."""
    r = np.random.default_rng(nkvh)
    new = [4, 12, 64, 0, 70, 5, 9, 6, 12, 8]
    base = [10, page - 5, 2 * page - 30, 3, page, 50, -4, 3 * page, 2 * page - 6, 7]
    most = 4
    paths = [[0, 1, 2], [0, 2, 5, 11, 7], list(r.permutation(64)), [], list(range(0, 64, 3)), [0, 3, 9, 1], [0, 6, 7, 8], [0, 4, 5],
             [0, 3, 4, 8, 9, 11], [0, -1, 2]]
    n_path = [len(p) for p in paths]
    n_path[9] = 20  # more than its tokens
    cu = P.cu_of(new)
    path = np.full(sum(new), -1, np.int32)
    for b, p in enumerate(paths):
        path[cu[b]:cu[b] + len(p)] = p
    table = r.permutation(len(new) * most).reshape(len(new), most).astype(np.int32)
    table[8, 2] = len(new) * most  # none
    table[7, 3] = -1
    layers = pools_of(r, n_layers, len(new) * most, nkvh, page, type)
    accept(G, layers, table, type, [b + n for b, n in zip(base, n_path)], [int(x) for x in cu], path, n_path)


@pytest.mark.parametrize("type", TYPES)
def test_accept_with_bad_offsets_stays_inside(G, type):  # noqa: F811
    r = np.random.default_rng(1)
    layers = pools_of(r, 1, 6, 2, 32, type)
    table = np.array([[0, 1], [2, 3], [4, 5]], np.int32)
    for cu in ([0, 9, 3, 20], [-5, 2, 2, 100], [8, 1, 0, -1]):
        kv = [G.ops.KvPages(G.up(k.buf), G.up(v.buf), G.up(table), 2, 32, type) for k, v in layers]
        G.ops.kv_accept_paged(kv, G.i32(2 ** 31 - 1, 7, -2 ** 31), G.i32(*cu), G.up(r.integers(-9, 9, 8).astype(np.int32)),
                              G.i32(-2 ** 31, 3, 2 ** 31 - 1), 8)
        G.down(kv[0].k)


@pytest.mark.parametrize("type", TYPES)
def test_a_step_of_a_batch_of_trees(G, oracle, type):  # noqa: F811
    """Rows written, attended to by their masks, trees verified, their paths moved, and the next token of each sequence: eager, and
    in a HIP graph that is replayed with eager work between."""
    import torch

    r = np.random.default_rng(21)
    o = G.ops
    B, nqh, nkvh, page, V, old, new = 3, 24, 4, 32, 301, [200, 26, 64], [7, 12, 4]
    cu, T = P.cu_of(new), sum(new)
    kp, vp, table = P.make_pages(r, old, [n + 1 for n in new], page, nkvh, type)
    qg, kx, vx, qw, kw = prep_inputs(r, T, nqh, nkvh)
    trees = [random_tree(r, n) for n in new]
    parent, mask = (np.concatenate([t[i] for t in trees]) for i in (0, 1))
    depth = np.zeros(T, np.int32)
    p = probabilities(r, T, V, 9)
    ids = np.zeros(T, np.int32)
    for b in range(B):
        for t in range(1, new[b]):
            depth[cu[b] + t] = depth[cu[b] + parent[cu[b] + t]] + 1
            ids[cu[b] + t] = np.argsort(-p[cu[b] + parent[cu[b] + t]])[t % 3]
    rope3 = np.stack([np.concatenate([old[b] + depth[cu[b]:cu[b + 1]] for b in range(B)])] * 3, 1).astype(np.int32)
    u, ul = np.full(T, 0.15, np.float32), r.random(B).astype(np.float32)
    k0, v0 = G.up(kp.buf), G.up(vp.buf)
    kv = o.KvPages(k0.clone(), v0.clone(), G.up(table), nkvh, page, type)
    layers = o.kv_layers([kv])
    d = [G.up(x) for x in (qg, kx, vx, qw, kw, p, ids, parent, u, ul, rope3)]
    dmask = G.up(mask.view(np.int64))
    pos, start, dcu = G.i32(*old), G.i32(*old), G.up(cu)
    qn, out, q1, o1 = G.full((T, nqh, 256), 0.0), G.full((T, nqh, 256), 0.0), G.full((B, nqh, 256), 0.0), G.full((B, nqh, 256), 0.0)
    tok, path, n_path = G.i32(*[0] * T), G.i32(*[0] * T), G.i32(*[0] * B)
    ws = G.ws(max(o.attn_paged_ws_bytes(kv, T, 12, nqh), o.attn_paged_ws_bytes(kv, B, 1, nqh), o.draft_verify_ws_bytes(B, V)))

    def drafts():
        o.attn_prep_paged(*d[:5], qn, kv, pos, dcu, T, 1e-6, cd.THETA_SCALE, nqh, rope3=d[10])
        o.attn_paged(qn, kv, pos, dcu, T, 12, SCALE, nqh, out, ws, tree=dmask)

    def step():
        drafts()
        o.draft_verify(d[5], None, d[6], d[7], d[8], d[9], dcu, B, V, tok, path, n_path, ws, pos=pos)
        o.kv_accept_paged(layers, pos, dcu, path, n_path, T)
        o.attn_prep_paged(*d[:5], q1, kv, pos, None, B, 1e-6, cd.THETA_SCALE, nqh)
        o.attn_paged(q1, kv, pos, None, B, 1, SCALE, nqh, o1, ws)

    def reset():
        kv.k.copy_(k0), kv.v.copy_(v0), pos.copy_(start)
        for x in (qn, out, q1, o1, tok, path, n_path):
            x.zero_()

    def results():
        return [G.down(x).copy() for x in (qn, out, q1, o1, tok, path, n_path, pos, kv.k, kv.v)]

    reset()
    step()
    eager = results()
    reset()
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        step()
    for _ in range(3):
        reset()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(results(), eager):
            assert np.array_equal(a.view(np.uint8), b.view(np.uint8))

    want = P.verify(p, None, ids, parent, u, ul, cu, V, *(np.zeros(n, np.int32) for n in (T, T, B)), np.array(old, np.int32))
    for a, x in zip(eager[4:8], want):
        assert np.array_equal(a, x)
    assert any(list(eager[5][cu[b]:cu[b] + eager[6][b]]) != list(range(eager[6][b])) for b in range(B))  # a branch was taken
    # the drafts' rows as they were written, what their masks saw, and where the paths' rows lie then
    reset()
    drafts()
    kp.buf[:], vp.buf[:] = G.down(kv.k), G.down(kv.v)
    eo, _, bo, _ = P.attend(eager[0], kp, vp, table, old, new, SCALE, mask)
    near(eager[1], eo, bo, "the drafts")
    for pool in (kp, vp):
        P.accept(pool, table, eager[7], cu, eager[5], eager[6])
    at = [int(x) for x in eager[7]]
    for pool, x in ((kp, eager[8]), (vp, eager[9])):
        now = P.Pool(len(x), nkvh, page, pool.bits, 0)
        now.buf[:] = x
        for b in range(B):
            assert np.array_equal(pool.values(table[b], at[b])[0], now.values(table[b], at[b])[0])
        pool.buf[:] = x
    eo, _, bo, _ = P.attend(eager[2], kp, vp, table, at, [1] * B, SCALE)
    near(eager[3], eo, bo, "the next token")
