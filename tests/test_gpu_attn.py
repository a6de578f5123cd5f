"""Attention over the K/V cache on the GPU: trees of drafted tokens, weights per cache row, blocks chosen per token; against
plain 64-bit forms (tests/attnref.py), whose error bounds are derived there. Memory that no call may read holds NaN."""
import numpy as np
import pytest

import attnref as R
from conftest import assert_bits_equal

pytestmark = pytest.mark.gpu
SCALE = 1 / 16


@pytest.fixture(scope="module")
def G(dev, q27):
    import torch

    class H:
        ops = q27.ops

        def up(self, a):
            return torch.from_numpy(np.ascontiguousarray(a)).to(dev)

        def i32(self, *v):
            return torch.tensor(v, dtype=torch.int32, device=dev)

        def u64(self, v):
            return self.up(np.asarray(v, np.uint64).view(np.int64))

        def full(self, shape, value, dtype=torch.float32):
            return torch.full(shape, value, dtype=dtype, device=dev)

        def ws(self, n):
            return torch.full((n,), 0xFF, dtype=torch.uint8, device=dev) if n else None  # NaN wherever it is not written

        def down(self, t):
            torch.cuda.synchronize()
            return t.cpu().numpy()

        def tree(self, q, k, v, pos0, tree, T, nqh, nkvh, n_ctx, q8, scale=SCALE):
            o, lse = self.full((T, nqh, 256), 7.0), self.full((T, nqh), 7.0)
            ws = self.ws(self.ops.attn_tree_ws_bytes(T, nqh, nkvh, n_ctx))
            self.ops.attn_tree(q, k, v, pos0, tree, T, scale, nqh, nkvh, n_ctx, q8, o, ws, lse=lse)
            return o, lse

        def blocks(self, q, k, v, pos0, idx, T, nsel, nqh, nkvh, n_ctx, q8, scale=SCALE):
            o, lse = self.full((T, nqh, 256), 7.0), self.full((T, nqh), 7.0)
            ws = self.ws(self.ops.attn_blocks_ws_bytes(T, nqh, nkvh, nsel))
            self.ops.attn_blocks(q, k, v, pos0, idx, T, nsel, scale, nqh, nkvh, n_ctx, q8, o, ws, lse=lse)
            return o, lse

    return H()


def near(got, want, bound, what):
    off = np.abs(got.astype(np.float64) - want)
    assert np.all(off <= bound), f"{what}: off by {(off - bound).max():.3g} over a bound of {bound.max():.3g}"


# (T, rows before, n_ctx, query heads, kv heads, tree)
TREES = [
    (1, 0, 1, 24, 4, None),          # a cache of one row
    (2, 0, 1, 6, 6, "random"),
    (1, 0, 40, 24, 4, None),         # the very first token sees itself alone
    (1, 1, 40, 24, 4, None),
    (1, 31, 64, 4, 4, None),         # a tile of 32 rows, exactly
    (1, 32, 64, 24, 4, None),
    (1, 33, 64, 7, 1, None),
    (1, 700, 1000, 24, 4, None),     # several splits, a ragged last tile
    (4, 127, 256, 24, 4, None),      # a chain over a tile's border
    (3, 250, 251, 24, 4, None),      # tokens 1 and 2 have no row of their own in the cache
    (2, 64, 64, 6, 2, None),         # the cache is full: no drafted row exists
    (3, -2, 40, 24, 4, None),        # rows -2 and -1 do not exist
    (5, 0, 64, 24, 4, "empty"),      # no context, and tokens that see nothing at all
    (5, 61, 90, 24, 4, "empty"),
    (6, 95, 128, 16, 2, "random"),   # group of 8: three row tiles
    (11, 300, 400, 24, 4, "random"),  # five row tiles, the last of 2 rows
    (64, 65, 140, 24, 4, "random"),  # the widest tree
    (64, 513, 577, 1, 1, "random"),
    (17, 40, 64, 48, 2, "high"),     # mask bits of tokens that are none
    (27, 300, 400, 24, 4, "random"),  # eleven row tiles
    (45, 700, 1000, 24, 4, "random"),  # seventeen
]


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("T,pos0,n_ctx,nqh,nkvh,kind", TREES)
def test_tree(G, T, pos0, n_ctx, nqh, nkvh, kind, q8):
    r = np.random.default_rng(hash((T, pos0 + 5, n_ctx, nqh)) % 2**32)
    tree = None
    if kind:
        tree = R.random_tree(r, T, empty=(1, 3) if kind == "empty" else ())
        if kind == "high":
            tree = tree | np.uint64((1 << 63) | (1 << 40))
    end = min(max(pos0 + T, 0), n_ctx)
    k = R.make_cache(r, nkvh, n_ctx, q8, garbage_from=end)
    v = R.make_cache(r, nkvh, n_ctx, q8, garbage_from=end)
    q = (r.standard_normal((T, nqh, 256)) * 1.5).astype(np.float32)
    o, lse = G.tree(G.up(q), G.up(k), G.up(v), G.i32(pos0), None if tree is None else G.u64(tree), T, nqh, nkvh, n_ctx, q8)
    vis = R.visible(T, pos0, n_ctx, None if tree is None else tree & np.uint64((1 << T) - 1))
    eo, el, bo, bl = R.attend(q, R.values(k, nkvh, n_ctx, q8), R.values(v, nkvh, n_ctx, q8), vis, SCALE)
    near(G.down(o), eo, bo, "o")
    got = G.down(lse)
    seen = np.isfinite(el)
    assert np.array_equal(seen, got != -np.inf)
    near(got[seen], el[seen], bl[seen], "lse")


@pytest.mark.parametrize("q8", [True, False])
def test_tree_of_odd_values(G, q8):
    """Very large and very small queries, V scales (or values) from the smallest to the largest f16, rows that are all zero,
    scores that rise from row to row, so that every tile moves the softmax's reference."""
    r = np.random.default_rng(11)
    T, pos0, n_ctx, nqh, nkvh = 8, 500, 520, 8, 1
    k, v = R.values(R.make_cache(r, 1, n_ctx, False), 1, n_ctx, False), r.standard_normal((1, n_ctx, 256))
    k[0, :, 0] = np.linspace(0, 40, n_ctx)       # rising scores for queries along channel 0
    v[0] *= 2.0 ** r.integers(-23, 14, (n_ctx, 1))
    v[0, 100:140] = 0
    if q8:
        def enc(x):
            b = x.reshape(1, n_ctx, 8, 32)
            d = (np.abs(b).max(-1) / 127).astype(np.float16)
            with np.errstate(divide="ignore", invalid="ignore"):
                c = np.where(d[..., None] > 0, np.rint(b / d[..., None].astype(np.float64)), 0)
            return R.join_q8(np.clip(c, -127, 127).astype(np.int8).reshape(1, n_ctx, 256), d)
        k, v = enc(k), enc(v)
    else:
        k, v = (x.astype(np.float16).reshape(-1).view(np.uint8) for x in (k, v))
    q = r.standard_normal((T, nqh, 256)).astype(np.float32)
    q[0] *= 1e-30
    q[1] *= 1e-6
    q[2] *= 100
    q[3] = 0
    q[4, :, 0] = 300
    q[5, :, 0] = -300
    q[6, :, 1:] = 0
    o, lse = G.tree(G.up(q), G.up(k), G.up(v), G.i32(pos0), None, T, nqh, nkvh, n_ctx, q8)
    vis = R.visible(T, pos0, n_ctx, None)
    eo, el, bo, bl = R.attend(q, R.values(k, 1, n_ctx, q8), R.values(v, 1, n_ctx, q8), vis, SCALE)
    # V spans 2^37 here: a weight times a scale below 2^-36 of the largest product is lost in its second f16 term
    big = np.abs(R.values(v, 1, n_ctx, q8)).max()
    near(G.down(o), eo, bo + big * 2.0 ** -36 * n_ctx, "o")
    near(G.down(lse), el, bl, "lse")


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("where", ["k", "v"])
def test_odd_drafted_rows_reach_only_those_that_see_them(G, where, bad, q8):
    """Token 1's K or V row is not finite; tokens 1 and 3 see it, 0, 2 and 4 do not."""
    r = np.random.default_rng(5)
    T, pos0, n_ctx, nqh, nkvh = 5, 40, 64, 24, 4
    bufs = {w: R.make_cache(r, nkvh, n_ctx, q8, garbage_from=45) for w in "kv"}
    tree = np.array([1, 2, 4, 0b1010, 0b10101], np.uint64)
    clean = {w: b.copy() for w, b in bufs.items()}
    if q8:
        R.split_q8(bufs[where], nkvh, n_ctx)[1][:, pos0 + 1, 3] = bad
    else:
        bufs[where].view(np.float16).reshape(nkvh, n_ctx, 256)[:, pos0 + 1, 100] = bad
    q = r.standard_normal((T, nqh, 256)).astype(np.float32)
    run = lambda b: [G.down(x) for x in G.tree(G.up(q), G.up(b["k"]), G.up(b["v"]), G.i32(pos0), G.u64(tree), T, nqh, nkvh,  # noqa: E731
                                                n_ctx, q8)]
    (o, lse), (eo, elze) = run(bufs), run(clean)
    for t in (0, 2, 4):
        assert_bits_equal(o[t], eo[t], f"o of token {t}")
        assert_bits_equal(lse[t], elze[t], f"lse of token {t}")
    if where == "v":
        dims = slice(96, 128) if q8 else slice(100, 101)
        # codes may be 0, and 0 times infinity is NaN: not finite either way
        assert not np.isfinite(o[[1, 3]][..., dims]).any()
        rest = np.ones(256, bool)
        rest[dims] = False
        assert np.isfinite(o[[1, 3]][..., rest]).all()
    elif np.isnan(bad):
        assert np.isnan(o[[1, 3]]).all()


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("T", [5, 12])
def test_large_drafted_rows_do_not_coarsen_those_that_do_not_see_them(G, T, q8):
    """Token 1's V row is 2^30 times as large as the others; only tokens 1 and 3 see it."""
    r = np.random.default_rng(6)
    pos0, n_ctx, nqh, nkvh = 40, 64, 24, 4
    k, v = R.make_cache(r, nkvh, n_ctx, q8), R.make_cache(r, nkvh, n_ctx, q8, std=2.0 ** -10)
    tree = np.array([1 << t for t in range(T)], np.uint64)
    tree[3] |= np.uint64(2)
    big = v.copy()
    if q8:
        R.split_q8(big, nkvh, n_ctx)[1][:, pos0 + 1] = 20000
    else:
        big.view(np.float16).reshape(nkvh, n_ctx, 256)[:, pos0 + 1] *= np.float16(1024)
        big.view(np.float16).reshape(nkvh, n_ctx, 256)[:, pos0 + 1] *= np.float16(1024)
    q = r.standard_normal((T, nqh, 256)).astype(np.float32)
    run = lambda v: [G.down(x) for x in G.tree(G.up(q), G.up(k), G.up(v), G.i32(pos0), G.u64(tree), T, nqh, nkvh,  # noqa: E731
                                                n_ctx, q8)]
    (o, lse), (eo, elze) = run(big), run(v)
    others = [t for t in range(T) if t not in (1, 3)]
    assert_bits_equal(o[others], eo[others], "o")
    assert_bits_equal(lse, elze, "lse")
    assert (np.abs(o[1]) > 100 * np.abs(eo[1])).any()


@pytest.mark.parametrize("T,nqh", [(1, 24), (4, 24), (12, 24)])
def test_tree_of_blocks_of_different_size(G, T, nqh):
    """q8_0: the scales of a V row's 8 blocks span 2^28."""
    r = np.random.default_rng(8)
    pos0, n_ctx, nkvh = 300, 320, 4
    k, (c, d) = R.make_cache(r, nkvh, n_ctx, True), R.split_q8(R.make_cache(r, nkvh, n_ctx, True, std=64), nkvh, n_ctx)
    d = (d.astype(np.float32) * 2.0 ** (6 - 4 * np.arange(8))).astype(np.float16)
    v = R.join_q8(c, d)
    q = r.standard_normal((T, nqh, 256)).astype(np.float32)
    o, _ = G.tree(G.up(q), G.up(k), G.up(v), G.i32(pos0), None, T, nqh, nkvh, n_ctx, True)
    eo, _, bo, _ = R.attend(q, R.values(k, nkvh, n_ctx, True), R.values(v, nkvh, n_ctx, True), R.visible(T, pos0, n_ctx, None), SCALE)
    # a scale enters as a half relative to its row's largest, cut off: below 2^-14 of that by 2^-24 of it (f < 2 largest, so
    # 2^-23), times a code of at most 127; the weights sum to 1. A product with it rounds to a half again, 2^-25 of f
    # whatever its size, twice (both terms).
    near(G.down(o), eo, bo + d.astype(np.float64).max() * 127 * (2.0 ** -23 + 2 * 2.0 ** -24), "o")


@pytest.mark.parametrize("q8", [True, False])
def test_tree_is_the_same_alone_and_among_others(G, q8):
    """A token's result depends on its mask alone, bit for bit, and two calls at once on two streams do not disturb each
    other."""
    import torch

    r = np.random.default_rng(3)
    T, pos0, n_ctx, nqh, nkvh = 4, 1000, 1100, 24, 4
    k, v = (G.up(R.make_cache(r, nkvh, n_ctx, q8)) for _ in range(2))
    q = G.up(r.standard_normal((T, nqh, 256)).astype(np.float32))
    pos = G.i32(pos0)
    first = G.tree(q, k, v, pos, None, T, nqh, nkvh, n_ctx, q8)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append([G.tree(q, k, v, pos, None, T, nqh, nkvh, n_ctx, q8) for _ in range(5)])
    torch.cuda.synchronize()
    for many in outs:
        for o, lse in many:
            assert_bits_equal(G.down(o), G.down(first[0]), "o")
            assert_bits_equal(G.down(lse), G.down(first[1]), "lse")


@pytest.mark.parametrize("q8,n_ctx", [(True, 3200000), (False, 1600000)])
def test_far_rows_of_a_long_cache(G, q8, n_ctx):
    """Heads whose rows begin behind 2^31 bytes (q8: 2^31 bytes of codes, scales behind them), and the last rows of the
    context; the rows between are zeros, whose scores are 0."""
    import torch

    r = np.random.default_rng(8)
    nkvh = nqh = 4
    n, near_ = n_ctx - 1, 300
    row = 272 if q8 else 512
    bufs, vals = [], []
    for _ in range(2):
        buf = torch.zeros(nkvh * n_ctx * row, dtype=torch.uint8, device="cuda:0")
        x = r.integers(-60, 60, (nkvh, near_, 256)).astype(np.int8)
        if q8:
            codes = buf[:nkvh * n_ctx * 256].view(torch.int8).view(nkvh, n_ctx, 256)
            buf[nkvh * n_ctx * 256:].view(torch.float16).fill_(1 / 32)
            codes[:, -near_:] = G.up(x)
            vals.append(x.astype(np.float64) / 32)
        else:
            buf.view(torch.float16).view(nkvh, n_ctx, 256)[:, -near_:] = G.up((x / 32).astype(np.float16))
            vals.append((x / 32).astype(np.float16).astype(np.float64))
        bufs.append(buf)
    q = r.standard_normal((1, nqh, 256)).astype(np.float32)
    o, lse = (G.down(x)[0] for x in G.tree(G.up(q), bufs[0], bufs[1], G.i32(n), None, 1, nqh, nkvh, n_ctx, q8))
    for h in range(nqh):
        s = SCALE * (vals[0][h] @ q[0, h].astype(np.float64))
        m = max(0.0, s.max())
        p, zero = np.exp(s - m), np.exp(-m) * (n_ctx - near_)
        total = p.sum() + zero
        ds = SCALE * (np.abs(vals[0][h]) @ np.abs(q[0, h].astype(np.float64))).max() * (2.0 ** -21 + 16 * 2.0 ** -23)
        rel = 2 * (ds + 2.0 ** -20) + 2 * np.sqrt(n_ctx) * 2.0 ** -23
        near(o[h], p @ vals[1][h] / total, rel * (p @ np.abs(vals[1][h])) / total, "o")
        near(lse[h], m + np.log(total), np.float64(rel + 2.0 ** -20), "lse")


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("T,pos0,n_ctx,nqh,nkvh,rows", [
    (1, 0, 1, 24, 4, None), (1, 0, 40, 24, 4, None), (1, 33, 64, 24, 4, None), (4, 700, 1000, 24, 4, 0b1011), (5, 62, 65, 7, 1, None),
    (12, 95, 128, 16, 2, 0b100000000001), (64, 100, 200, 24, 4, None), (64, 130, 194, 6, 2, 1 << 63 | 5), (3, 50, 64, 24, 4, 0),
    (3, -1, 64, 24, 4, None), (27, 300, 400, 24, 4, 0x5ffffff), (9, 70, 200, 16, 1, None)])
def test_weights(G, T, pos0, n_ctx, nqh, nkvh, rows, q8):
    r = np.random.default_rng(T * 1000 + pos0 + 7)
    end = min(pos0 + T, n_ctx)
    k = R.make_cache(r, nkvh, n_ctx, q8, garbage_from=end)
    v = R.make_cache(r, nkvh, n_ctx, q8, garbage_from=end)
    q = (r.standard_normal((T, nqh, 256)) * 1.5).astype(np.float32)
    tree = R.random_tree(r, T)
    dq, dk, dt, pos = G.up(q), G.up(k), G.u64(tree), G.i32(pos0)
    _, lse = G.tree(dq, dk, G.up(v), pos, dt, T, nqh, nkvh, n_ctx, q8)
    acc = r.uniform(0, 3, (nkvh, n_ctx)).astype(np.float32)
    outs = []
    for _ in range(2):
        d = G.up(acc)
        G.ops.attn_weights(dq, lse, dk, pos, dt, T, SCALE, nqh, nkvh, n_ctx, q8, d, rows=None if rows is None else G.u64([rows]))
        outs.append(G.down(d))
    assert_bits_equal(outs[0], outs[1], "acc twice")
    vis = R.visible(T, pos0, n_ctx, tree)
    want, bound = R.weights(q, G.down(lse), R.values(k, nkvh, n_ctx, q8), vis, SCALE, (1 << 64) - 1 if rows is None else rows, acc,
                            pos0, T)
    near(outs[0], want, bound, "acc")
    assert_bits_equal(outs[0][:, max(end, 0):], acc[:, max(end, 0):], "rows behind the last")
    if rows is None and pos0 >= 0:  # the weights that one token gives are one per query head
        gained = (outs[0] - np.where(np.arange(n_ctx) < pos0, acc, 0))[:, :end].sum()
        assert abs(gained - T * nqh) < 1e-3 * T * nqh


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("n_ctx,pos0,T", [(64, 0, 1), (100, 0, 100), (130, 63, 2), (130, 64, 1), (300, 100, 77), (300, 250, 90),
                                          (200, -5, 20)])
def test_block_bounds(G, n_ctx, pos0, T, q8):
    r = np.random.default_rng(n_ctx + pos0 + T)
    nkvh, end, begin = 3, min(pos0 + T, n_ctx), max(pos0, 0)
    k = R.make_cache(r, nkvh, n_ctx, q8, garbage_from=end)
    if q8:
        R.split_q8(k, nkvh, n_ctx)[1][1, begin:end] = 0  # a head of zeros
    nblk = -(-n_ctx // 64)
    kb = G.full((G.ops.kv_block_bytes(nkvh, n_ctx),), 0x55, dtype=__import__("torch").uint8)
    G.ops.kv_block_bounds(G.up(k), G.i32(pos0), T, nkvh, n_ctx, q8, kb)
    got, m = G.down(kb), nkvh * nblk * 256
    lo, hi, d = R.bounds(R.values(k, nkvh, n_ctx, q8), end)
    b0, b1 = begin // 64, -(-end // 64)
    for what, x, want in (("lo", got[:m].view(np.int8).reshape(nkvh, nblk, 256), lo),
                          ("hi", got[m:2 * m].view(np.int8).reshape(nkvh, nblk, 256), hi),
                          ("d", got[2 * m:].view(np.float32).reshape(nkvh, nblk), d)):
        assert_bits_equal(x[:, b0:b1], want[:, b0:b1], what)
        assert np.all(np.ascontiguousarray(np.delete(x, np.s_[b0:b1], 1)).view(np.uint8) == 0x55), f"{what} of other blocks"


@pytest.mark.parametrize("T,pos0,n_ctx,nqh,nkvh,nsel,first,last", [
    (1, 0, 64, 24, 4, 4, 1, 2), (1, 2000, 4096, 24, 4, 8, 1, 2), (3, 639, 1000, 7, 1, 5, 0, 1), (70, 1000, 1200, 24, 4, 6, 1, 3),
    (5, 700, 900, 16, 1, 12, 12 - 1, 1), (9, 500, 700, 4, 4, 3, 0, 1), (33, 900, 933, 16, 2, 10, 2, 2), (2, 510, 512, 6, 2, 8, 0, 1),
    (2, 511, 512, 6, 2, 7, 0, 1), (4, -2, 128, 24, 4, 2, 0, 1), (1, 70000, 70400, 8, 2, 64, 1, 4)])
def test_select(G, T, pos0, n_ctx, nqh, nkvh, nsel, first, last):
    r = np.random.default_rng(T + pos0 + nsel)
    end = min(pos0 + T, n_ctx)
    k = R.make_cache(r, nkvh, n_ctx, False)
    kv = R.values(k, nkvh, n_ctx, False)
    if end > 640:  # equal blocks: equal scores, the lower one is taken
        kv[:, 320:384] = kv[:, 128:192]
        kv[:, 448:512] = kv[:, 128:192]
        kv[:, 192] = np.nan  # and one that has to be read
        k = kv.astype(np.float16).reshape(-1).view(np.uint8)
    q = r.standard_normal((T, nqh, 256)).astype(np.float32)
    q[0, 0] = 0
    if T > 1:
        q[1, nqh - 1, 5] = np.inf
    kb = G.ws(G.ops.kv_block_bytes(nkvh, n_ctx))
    G.ops.kv_block_bounds(G.up(k), G.i32(0), max(end, 1), nkvh, n_ctx, False, kb)
    idx = G.full((T, nkvh, nsel), 99, dtype=__import__("torch").int32)
    G.ops.attn_select(G.up(q), kb, G.i32(pos0), T, nqh, nkvh, n_ctx, nsel, first, last, idx,
                      G.ws(G.ops.attn_select_ws_bytes(T, nkvh, n_ctx)))
    lo, hi, d = R.bounds(kv, max(end, 1))
    want = R.select(q, lo, hi, d, pos0, n_ctx, nsel, first, last)
    assert np.array_equal(G.down(idx), want)


@pytest.mark.parametrize("n_ctx", [1024000, 958000])
def test_select_of_the_longest_context(G, n_ctx):
    """The bounds are written as they are; every block but the fixed ones is told apart by its scale."""
    r = np.random.default_rng(n_ctx)
    nblk, nsel, first, last = -(-n_ctx // 64), 40, 1, 2
    one = r.integers(1, 128, 256).astype(np.int8)
    d = r.permutation(nblk).astype(np.float32) + 1
    kb = np.concatenate([np.tile(one, nblk).view(np.uint8), np.tile(one, nblk).view(np.uint8), d.view(np.uint8)])
    q = np.abs(r.standard_normal((1, 2, 256))).astype(np.float32)  # scores: a positive constant times d
    idx = G.full((1, 1, nsel), 99, dtype=__import__("torch").int32)
    G.ops.attn_select(G.up(q), G.up(kb), G.i32(n_ctx - 1), 1, 2, 1, n_ctx, nsel, first, last, idx,
                      G.ws(G.ops.attn_select_ws_bytes(1, 1, n_ctx)))
    mid = first + np.argsort(-d[first:nblk - last])[:nsel - first - last]
    assert G.down(idx)[0, 0].tolist() == sorted([0, *mid.tolist(), nblk - 2, nblk - 1])


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("T,pos0,n_ctx,nqh,nkvh,nsel", [(1, 0, 1, 24, 4, 2), (1, 0, 40, 24, 4, 1), (1, 1000, 1100, 24, 4, 9), (3, 62, 70, 7, 1, 2),
                                                        (40, 300, 340, 16, 2, 4), (300, 20, 320, 6, 2, 3), (2, 200, 201, 16, 1, 5)])
def test_blocks(G, T, pos0, n_ctx, nqh, nkvh, nsel, q8):
    """Lists in any order, with entries that are no blocks, blocks behind the token, a block twice, and empty lists."""
    r = np.random.default_rng(T * 7 + pos0)
    end = min(pos0 + T, n_ctx)
    k, v = (R.make_cache(r, nkvh, n_ctx, q8, garbage_from=end) for _ in range(2))
    q = (r.standard_normal((T, nqh, 256)) * 1.5).astype(np.float32)
    idx = r.integers(-2, -(-n_ctx // 64) + 2, (T, nkvh, nsel)).astype(np.int32)
    idx[0, 0] = (pos0 // 64)
    if T > 1:
        idx[1] = -1
        idx[1, 0, 0] = np.iinfo(np.int32).max
    o, lse = G.blocks(G.up(q), G.up(k), G.up(v), G.i32(pos0), G.up(idx), T, nsel, nqh, nkvh, n_ctx, q8)
    vis = R.block_visible(T, pos0, n_ctx, idx.astype(np.int64))
    eo, el, bo, bl = R.attend(q, R.values(k, nkvh, n_ctx, q8), R.values(v, nkvh, n_ctx, q8), vis, SCALE)
    near(G.down(o), eo, bo, "o")
    seen, got = np.isfinite(el), G.down(lse)
    assert np.array_equal(seen, got != -np.inf)
    near(got[seen], el[seen], bl[seen], "lse")
