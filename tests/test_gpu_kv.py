"""Keeping the K/V cache on the GPU: eviction by accumulated weight and the move of an accepted path, bit for bit; and the
operators over the cache together, as a program runs them, in one HIP graph."""
import numpy as np
import pytest

import attnref as R
import cfgdata as cd
from conftest import assert_bits_equal
from test_gpu_attn import G, SCALE, near  # noqa: F401

pytestmark = pytest.mark.gpu


def rows_of(buf, nkvh, n_ctx, q8):
    """[nkvh][n_ctx][bytes of a row, scales behind the codes]."""
    if not q8:
        return buf.reshape(nkvh, n_ctx, 512)
    m = nkvh * n_ctx * 256
    return np.concatenate([buf[:m].reshape(nkvh, n_ctx, 256), buf[m:].reshape(nkvh, n_ctx, 16)], 2)


def evict(G, k, v, acc, pos0, keep, first, last, nkvh, n_ctx, q8, n_out=None, with_kept=True):  # noqa: F811
    """Outputs of kv_evict as numpy; n_out None: in place."""
    import torch

    dk, dv, da = G.up(k), G.up(v), G.up(acc)
    if n_out is None:
        ko, vo, ao, n_out, in_place = dk, dv, da, n_ctx, True
    else:
        nb = G.ops.kv_cache_bytes(nkvh, n_out, q8)
        ko, vo = (torch.full((nb,), 0xAB, dtype=torch.uint8, device=dk.device) for _ in range(2))
        ao, in_place = G.full((nkvh, n_out), -7.0), False
    kept = G.full((nkvh, keep), 99, dtype=torch.int32) if with_kept else None
    G.ops.kv_evict(dk, dv, da, G.i32(pos0), keep, first, last, ko, vo, ao, n_out, kept, nkvh, n_ctx, q8,
                   G.ws(G.ops.kv_evict_ws_bytes(nkvh, n_ctx, keep, q8, in_place)))
    return [G.down(x) for x in (ko, vo, ao)] + [None if kept is None else G.down(kept)]


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("n_ctx,pos0,keep,first,last,kind", [
    (1, 1, 1, 0, 0, "random"), (1, 0, 1, 1, 0, "random"), (300, 200, 64, 4, 16, "random"), (300, 300, 1, 0, 0, "random"), (300, 250, 40, 20, 20, "random"), (300, 250, 249, 4, 16, "random"),
    (300, 250, 250, 4, 16, "random"), (300, 60, 100, 4, 16, "random"), (300, 0, 10, 1, 1, "random"), (300, 500, 17, 3, 5, "random"),
    (5000, 4999, 700, 0, 0, "equal"), (5000, 4999, 700, 4, 64, "few"), (5000, 4800, 1000, 4, 64, "odd"), (9000, 8999, 4100, 4, 64, "close"),
    (32768, 32768, 5000, 4, 64, "random"), (33000, 32990, 9000, 4, 64, "close"), (33000, 20000, 300, 4, 64, "odd"),
    (33000, 33000, 300, 0, 0, "equal"), (33000, 25000, 30000, 4, 64, "random"), (33000, 32999, 32998, 4, 64, "few"),
    (33000, 33000, 64, 32, 32, "random")])
def test_evict(G, n_ctx, pos0, keep, first, last, kind, in_place, q8):  # noqa: F811
    r = np.random.default_rng(n_ctx + pos0 + keep)
    nkvh, n = 2, min(pos0, n_ctx)
    k, v = (r.integers(0, 256, nkvh * n_ctx * (272 if q8 else 512)).astype(np.uint8) for _ in range(2))
    acc = np.exp(2 * r.standard_normal((nkvh, n_ctx))).astype(np.float32)
    if kind == "equal":
        acc[:] = 0.25
    elif kind == "few":
        acc = r.integers(0, 4, acc.shape).astype(np.float32)
    elif kind == "odd":  # zeros of both signs, infinities, NaN, negative and subnormal weights
        acc = r.choice(np.array([0.0, -0.0, np.inf, -np.inf, np.nan, -1.0, 1e-42, 2.0], np.float32), acc.shape)
    elif kind == "close":  # neighbours in the last bit
        acc = (np.float32(1.0).view(np.int32) + r.integers(0, 3000, acc.shape).astype(np.int32)).view(np.float32)
    n_out = None if in_place else keep + 37
    ko, vo, ao, kept = evict(G, k, v, acc, pos0, keep, first, last, nkvh, n_ctx, q8, n_out)
    want = R.kept_rows(acc, n, keep, first, last)
    assert np.array_equal(kept, want)
    m = min(n, keep)
    for got, src, what in ((ko, k, "K"), (vo, v, "V")):
        a, b = rows_of(got, nkvh, n_out or n_ctx, q8), rows_of(src, nkvh, n_ctx, q8)
        for kh in range(nkvh):
            assert np.array_equal(a[kh, :m], b[kh, want[kh, :m]]), what
            rest = b[kh, m:] if in_place else np.full_like(a[kh, m:], 0xAB)
            assert np.array_equal(a[kh, m:], rest), f"{what} behind the kept rows"
    for kh in range(nkvh):
        assert_bits_equal(ao[kh, :m], acc[kh, want[kh, :m]], "acc")
        assert_bits_equal(ao[kh, m:], acc[kh, m:] if in_place else np.full(n_out - m, -7, np.float32), "acc behind the kept rows")
    again = evict(G, k, v, acc, pos0, keep, first, last, nkvh, n_ctx, q8, n_out, with_kept=False)
    assert np.array_equal(again[0], ko) and np.array_equal(again[1], vo)


def test_evict_pos(G):  # noqa: F811
    for n, rd, keep in ((100, 7, 40), (40, 7, 40), (10, -3, 40)):
        pos, rdelta = G.i32(n), G.i32(rd)
        G.ops.kv_evict_pos(pos, rdelta, keep)
        m = min(n, keep)
        assert G.down(pos)[0] == m and G.down(rdelta)[0] == rd - (n - m)
        assert m - G.down(rdelta)[0] == n - rd  # the next token's rotary position
        pos = G.i32(n)
        G.ops.kv_evict_pos(pos, None, keep)
        assert G.down(pos)[0] == m


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("T,pos0,path,n_path", [
    (4, 20, [0, 1, 2, 3], 4), (4, 20, [1, 3, 0, 0], 2), (64, 100, list(range(0, 64, 2)) + [0] * 32, 32), (64, 64, list(range(64)), 64),
    (5, 20, [2, 4, 1, 0, 3], 5), (5, 20, [1, 7, 2, 3, 4], 5), (5, 20, [-1, 1, 2, 3, 4], 5), (5, 20, [1, 2, 3, 4, 0], 0),
    (5, 20, [1, 2, 3, 4, 0], -3), (5, 20, [1, 1, 1, 2, 2], 9), (6, 197, [1, 2, 3, 5, 0, 0], 4), (6, -2, [1, 3, 4, 5, 0, 0], 4)])
def test_accept(G, T, pos0, path, n_path, q8):  # noqa: F811
    r = np.random.default_rng(T + pos0)
    nkvh, n_ctx, row = 3, 200, 272 if q8 else 512
    caches = [r.integers(0, 256, nkvh * n_ctx * row).astype(np.uint8) for _ in range(3)]
    accs = [r.standard_normal((nkvh, n_ctx)).astype(np.float32) for _ in range(2)]
    dc, da = [G.up(c) for c in caches], [G.up(a) for a in accs]
    G.ops.kv_accept(dc, da, G.i32(pos0), G.i32(*path), G.i32(n_path), T, nkvh, n_ctx, q8)
    moves = []
    for i in range(min(max(n_path, 0), T)):
        if not 0 <= path[i] < T:
            break
        if 0 <= pos0 + path[i] < n_ctx and 0 <= pos0 + i < n_ctx:
            moves.append((pos0 + path[i], pos0 + i))
    for got, src in zip(dc, caches):
        want = rows_of(src, nkvh, n_ctx, q8).copy()
        for a, b in moves:
            want[:, b] = rows_of(src, nkvh, n_ctx, q8)[:, a]
        assert np.array_equal(rows_of(G.down(got), nkvh, n_ctx, q8), want)
    for got, src in zip(da, accs):
        want = src.copy()
        for a, b in moves:
            want[:, b] = src[:, a]
        assert_bits_equal(G.down(got), want, "acc")


@pytest.mark.parametrize("q8,n_ctx", [(True, 3200000), (False, 1600000)])
def test_far_rows(G, q8, n_ctx):  # noqa: F811
    """The last head's last rows of a cache of more than 2^31 bytes: moved by kv_accept and kv_evict, bounded, chosen,
    attended to and weighed. All rows before them are zeros."""
    import torch

    r = np.random.default_rng(4)
    nkvh, tail = 4, 300
    pos0, row = n_ctx - tail, 272 if q8 else 512
    rest = [R.make_cache(r, 1, tail, q8) for _ in range(2)]
    bufs = []
    for x in rest:
        buf = torch.zeros(nkvh * n_ctx * row, dtype=torch.uint8, device="cuda:0")
        if q8:
            buf[(nkvh * n_ctx - tail) * 256:nkvh * n_ctx * 256] = G.up(x[:tail * 256])
            buf[-tail * 16:] = G.up(x[tail * 256:])
        else:
            buf[-tail * 512:] = G.up(x)
        bufs.append(buf)

    def rows(buf, a, b):  # of the last head
        if not q8:
            return G.down(buf[((nkvh - 1) * n_ctx + a) * 512:][:(b - a) * 512]).reshape(-1, 512)
        codes = buf[((nkvh - 1) * n_ctx + a) * 256:][:(b - a) * 256]
        scales = buf[nkvh * n_ctx * 256 + ((nkvh - 1) * n_ctx + a) * 16:][:(b - a) * 16]
        return np.concatenate([G.down(codes).reshape(-1, 256), G.down(scales).reshape(-1, 16)], 1)

    src = [rows(b, pos0, n_ctx) for b in bufs]
    kv = [R.values(x, 1, tail, q8) for x in rest]
    q = r.standard_normal((1, nkvh, 256)).astype(np.float32)
    # the tail's blocks alone
    idx = np.full((1, nkvh, 8), -1, np.int32)
    b0 = -(-pos0 // 64)
    idx[0, nkvh - 1, :3] = [b0, b0 + 2, b0 + 1]
    o, lse = G.blocks(G.up(q), bufs[0], bufs[1], G.i32(n_ctx - 1), G.up(idx), 1, 8, nkvh, nkvh, n_ctx, q8)
    at = 64 * b0 - pos0
    seen = np.zeros((1, tail), bool)
    seen[0, at:at + 192] = True
    eo, el, bo, bl = R.attend(q[:, -1:], kv[0], kv[1], seen, SCALE)
    near(G.down(o)[:, -1:], eo, bo, "o")
    near(G.down(lse)[:, -1:], el, bl, "lse")
    # their weights, by the blocks' lse
    acc = torch.zeros((nkvh, n_ctx), device="cuda:0")
    G.ops.attn_weights(G.up(q), lse, bufs[0], G.i32(n_ctx - 1), None, 1, SCALE, nkvh, nkvh, n_ctx, q8, acc,
                       rows=G.u64([1]))
    s = SCALE * (kv[0][0, at:at + 192] @ q[0, -1].astype(np.float64))
    ds = SCALE * (np.abs(kv[0][0, at:at + 192]) @ np.abs(q[0, -1].astype(np.float64))) * (2.0 ** -21 + 16 * 2.0 ** -23)
    p = np.exp(s - np.float64(G.down(lse)[0, -1]))
    near(G.down(acc[-1, pos0 + at:pos0 + at + 192]), p, p * (ds + (np.abs(s) + 10) * 2.0 ** -22 + 2.0 ** -22), "acc")
    # bounds of the tail's blocks
    kb = torch.zeros(G.ops.kv_block_bytes(nkvh, n_ctx), dtype=torch.uint8, device="cuda:0")
    G.ops.kv_block_bounds(bufs[0], G.i32(64 * b0), n_ctx - 64 * b0, nkvh, n_ctx, q8, kb)
    nblk = -(-n_ctx // 64)
    lo = G.down(kb[:nkvh * nblk * 256].view(torch.int8).view(nkvh, nblk, 256)[-1, b0:b0 + 3])
    d = G.down(kb[2 * nkvh * nblk * 256:].view(torch.float32).view(nkvh, nblk)[-1, b0:b0 + 3])
    for i in range(3):
        x = kv[0][0, at + 64 * i:at + 64 * (i + 1)]
        assert d[i] == np.float32(np.float32(np.abs(x).max()) / np.float32(127))
        # a code is off by half a step and the three roundings of x * (1 / d)
        assert np.all(np.abs(lo[i] - x.min(0) / np.float64(d[i])) <= 0.5 + 127 * 3 * 2.0 ** -24)
    # a path of the tail
    G.ops.kv_accept(bufs, [acc], G.i32(pos0 + 100), G.i32(3, 50, 60, *[0] * 61), G.i32(3), 64, nkvh, n_ctx, q8)
    for x in src:
        x[100:103] = x[[103, 150, 160]]
    for b, x in zip(bufs, src):
        assert np.array_equal(rows(b, pos0, n_ctx), x)
    # the tail and the first rows stay
    acc.zero_()
    ws = G.ws(G.ops.kv_evict_ws_bytes(nkvh, n_ctx, 400, q8, True))
    kept = G.full((nkvh, 400), 0, dtype=torch.int32)
    G.ops.kv_evict(bufs[0], bufs[1], acc, G.i32(n_ctx), 400, 50, tail, bufs[0], bufs[1], acc, n_ctx, kept, nkvh, n_ctx, q8, ws)
    assert np.array_equal(G.down(kept)[-1], np.r_[np.arange(100), pos0 + np.arange(tail)])
    for b, x in zip(bufs, src):
        assert np.array_equal(rows(b, 100, 400), x) and np.array_equal(rows(b, pos0, n_ctx), x)


def test_accept_of_many_arrays(G):  # noqa: F811
    """More caches and weight arrays than one launch takes."""
    import torch

    nkvh, n_ctx, T = 1, 8, 4
    caches = [torch.full((n_ctx * 512,), i, dtype=torch.uint8, device="cuda:0") for i in range(150)]
    accs = [torch.arange(n_ctx, dtype=torch.float32, device="cuda:0") + i for i in range(70)]
    for c in caches:
        c.view(n_ctx, 512)[5] = 255 - c[0]
    G.ops.kv_accept(G.ops.kv_pointers(caches), G.ops.kv_pointers(accs), G.i32(2), G.i32(3, 0, 0, 0), G.i32(1), T, nkvh, n_ctx, False)
    for i, c in enumerate(caches):
        x = G.down(c).reshape(n_ctx, 512)
        assert np.all(x[[2, 5]] == 255 - i) and np.all(x[[0, 1, 3, 4, 6, 7]] == i)
    for i, a in enumerate(accs):
        assert np.array_equal(G.down(a), np.array([0, 1, 5, 3, 4, 5, 6, 7], np.float32) + i)


@pytest.mark.parametrize("q8", [True, False])
def test_a_program_of_them(G, oracle, q8):  # noqa: F811
    """attn_prep writes a tree of drafts, attn_tree reads it, attn_weights adds up, kv_accept moves the path, kv_evict and
    kv_evict_pos make room, and the next token is written, read sparsely and densely: recorded in one graph and replayed
    three times from the same state with eager work between; every replay gives the eager run's bits, and those agree with
    the plain forms."""
    import torch

    r = np.random.default_rng(21)
    T, n, n_ctx, nqh, nkvh, keep, first, last, nsel = 6, 200, 512, cd.NQH, cd.NKVH, 150, 4, 32, 2
    o = G.ops
    k0, v0 = (R.make_cache(r, nkvh, n_ctx, q8) for _ in range(2))
    acc0 = r.uniform(0, 2, (nkvh, n_ctx)).astype(np.float32)
    qg, kx, vx = (r.standard_normal(s).astype(np.float32) for s in ((T, nqh, 512), (T, nkvh, 256), (T, nkvh, 256)))
    qw, kw = (1 + 0.1 * r.standard_normal(256)).astype(np.float32), (1 + 0.1 * r.standard_normal(256)).astype(np.float32)
    tree = R.random_tree(r, T)
    depth = np.array([bin(int(m)).count("1") - 1 for m in tree], np.int32)
    rope3 = np.repeat((n + depth)[:, None], 3, 1).astype(np.int32)
    t = max(range(T), key=lambda i: (depth[i], i))  # the deepest branch is accepted
    path = [u for u in range(T) if (int(tree[t]) >> u) & 1]
    taken = len(path)
    d = {"qg": G.up(qg), "kx": G.up(kx), "vx": G.up(vx), "qw": G.up(qw), "kw": G.up(kw), "tree": G.u64(tree), "rope3": G.up(rope3)}
    dpath = G.i32(*(path + [0] * (T - taken)))
    dn, rows = G.i32(taken), G.u64([sum(1 << u for u in path)])
    pos0, rdelta = G.i32(n), G.i32(0)
    k, v, acc = G.up(k0), G.up(v0), G.up(acc0)
    qn, out, lse = G.full((T, nqh, 256), 0.0), G.full((T, nqh, 256), 0.0), G.full((T, nqh), 0.0)
    q1, o1, o2 = (G.full((1, nqh, 256), 0.0) for _ in range(3))
    kept, idx = G.full((nkvh, keep), 0, torch.int32), G.full((1, nkvh, nsel), 0, torch.int32)
    after = G.i32(n + taken)
    kb = G.ws(o.kv_block_bytes(nkvh, n_ctx))
    zero = G.i32(0)
    ws = G.ws(max(o.attn_tree_ws_bytes(T, nqh, nkvh, n_ctx), o.attn_tree_ws_bytes(1, nqh, nkvh, n_ctx),
                  o.attn_select_ws_bytes(1, nkvh, n_ctx), o.attn_blocks_ws_bytes(1, nqh, nkvh, nsel),
                  o.kv_evict_ws_bytes(nkvh, n_ctx, keep, q8, True)))

    def step():
        o.attn_prep(d["qg"], d["kx"], d["vx"], d["qw"], d["kw"], qn, k, v, pos0, T, 1e-6, cd.THETA_SCALE, nqh, nkvh, n_ctx, q8,
                    rope3=d["rope3"])
        o.attn_tree(qn, k, v, pos0, d["tree"], T, SCALE, nqh, nkvh, n_ctx, q8, out, ws, lse=lse)
        o.attn_weights(qn, lse, k, pos0, d["tree"], T, SCALE, nqh, nkvh, n_ctx, q8, acc, rows=rows)
        o.kv_accept([k, v], [acc], pos0, dpath, dn, T, nkvh, n_ctx, q8)
        pos0.copy_(after)
        o.kv_evict(k, v, acc, pos0, keep, first, last, k, v, acc, n_ctx, kept, nkvh, n_ctx, q8, ws)
        o.kv_evict_pos(pos0, rdelta, keep)
        o.attn_prep(d["qg"], d["kx"], d["vx"], d["qw"], d["kw"], q1, k, v, pos0, 1, 1e-6, cd.THETA_SCALE, nqh, nkvh, n_ctx, q8,
                    rdelta=rdelta)
        o.kv_block_bounds(k, zero, keep + 1, nkvh, n_ctx, q8, kb)
        o.attn_select(q1, kb, pos0, 1, nqh, nkvh, n_ctx, nsel, 0, 1, idx, ws)
        o.attn_blocks(q1, k, v, pos0, idx, 1, nsel, SCALE, nqh, nkvh, n_ctx, q8, o1, ws)
        o.attn_tree(q1, k, v, pos0, None, 1, SCALE, nqh, nkvh, n_ctx, q8, o2, ws)

    state = {"k": (k, G.up(k0)), "v": (v, G.up(v0)), "acc": (acc, G.up(acc0)), "pos0": (pos0, G.i32(n)), "rdelta": (rdelta, G.i32(0))}

    def reset():
        for a, b in state.values():
            a.copy_(b)
        for x in (out, lse, o1, o2):
            x.zero_()

    def results():
        return {w: G.down(x).copy() for w, x in (("out", out), ("lse", lse), ("k", k), ("v", v), ("acc", acc), ("kept", kept),
                                                   ("idx", idx), ("o1", o1), ("o2", o2), ("pos0", pos0), ("rdelta", rdelta), ("q1", q1),
                                                   ("qn", qn))}

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
        got = results()
        for w in eager:
            assert np.array_equal(got[w].view(np.uint8), eager[w].view(np.uint8)), w

    # the plain forms, from the library's own qn and cache rows (attn_prep is tested elsewhere)
    import numpy.testing as npt
    kc, vc = k0.copy(), v0.copy()
    qn_e = oracle.attn_prep(qg.reshape(-1), kx.reshape(-1), vx.reshape(-1), qw, kw, kc, vc, n, T, 1e-6, cd.THETA_SCALE, nqh, nkvh,
                            n_ctx, q8, rope3=rope3)
    npt.assert_array_equal(eager["qn"].reshape(-1), qn_e)
    K, V = (R.values(x, nkvh, n_ctx, q8) for x in (kc, vc))
    vis = R.visible(T, n, n_ctx, tree)
    eo, el, bo, bl = R.attend(eager["qn"], K, V, vis, SCALE)
    near(eager["out"], eo, bo, "out")
    near(eager["lse"], el, bl, "lse")
    w, wb = R.weights(eager["qn"], eager["lse"], K, vis, SCALE, sum(1 << u for u in path), acc0, n, T)
    w[:, n:n + taken], wb[:, n:n + taken] = w[:, [n + u for u in path]], wb[:, [n + u for u in path]]
    total = n + taken
    kept_e = eager["kept"]
    assert np.all(np.diff(kept_e, axis=1) > 0) and eager["pos0"][0] == keep and eager["rdelta"][0] == keep - total
    for kh in range(nkvh):  # no row left out is heavier than a kept one of the middle, beyond the bounds of the weights
        mid = np.arange(first, total - last)
        inn = np.isin(mid, kept_e[kh])
        assert inn.sum() == keep - first - last
        low = (w - wb)[kh, mid[~inn]].max()
        assert np.all((w + wb)[kh, mid[inn]] >= low)
        near(eager["acc"][kh, :keep], w[kh, kept_e[kh]], wb[kh, kept_e[kh]], "acc")
    Kn, Vn = (R.values(eager[x], nkvh, n_ctx, q8) for x in "kv")
    for kh in range(nkvh):
        src = np.array([n + path[j - n] if n <= j < total else j for j in kept_e[kh]])
        npt.assert_array_equal(Kn[kh, :keep], K[kh, src])
        npt.assert_array_equal(Vn[kh, :keep], V[kh, src])
    eo, _, bo, _ = R.attend(eager["q1"], Kn, Vn, R.visible(1, keep, n_ctx, None), SCALE)
    near(eager["o2"], eo, bo, "dense")
    lo, hi, dd = R.bounds(Kn, keep + 1)
    assert np.array_equal(eager["idx"], R.select(eager["q1"], lo, hi, dd, keep, n_ctx, nsel, 0, 1))
    eo, _, bo, _ = R.attend(eager["q1"], Kn, Vn, R.block_visible(1, keep, n_ctx, eager["idx"].astype(np.int64)), SCALE)
    near(eager["o1"], eo, bo, "sparse")
