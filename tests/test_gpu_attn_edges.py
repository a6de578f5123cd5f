"""Attention over the K/V cache on the GPU where it can go wrong and tests/test_gpu_attn.py does not look, against a plain
64-bit form: query values far below their row's largest, V rows of very different size, values that are not finite, lists
of any numbers."""
import numpy as np
import pytest

import attnref as R
from test_gpu_attn import G, SCALE, near  # noqa: F401

pytestmark = pytest.mark.gpu


def cache(x, q8):
    """The bytes of a cache of the values x [nkvh][n_ctx][256] (rounded to what it holds)."""
    if not q8:
        return x.astype(np.float16).reshape(-1).view(np.uint8)
    b = x.reshape(*x.shape[:2], 8, 32)
    d = (np.abs(b).max(-1) / 127).astype(np.float16)
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where(d[..., None] > 0, np.rint(b / d[..., None].astype(np.float64)), 0)
    return R.join_q8(np.clip(c, -127, 127).astype(np.int8).reshape(x.shape), d)


def score_bound(q, k, s, scale):
    """q [..][256], k [n][256], s [..][n] = scale q k: how far a score may be off. As in R.attend; but a query value may
    also lose 2^-38 of the largest of its row, where its second f16 term is subnormal."""
    a = np.abs(k)
    return scale * (np.abs(q) @ a.T * (2.0 ** -21 + 16 * 2.0 ** -23) + 2.0 ** -38 * np.abs(q).max(-1, keepdims=True) * a.sum(1)) \
        + np.abs(s) * 2.0 ** -23


def attend(q, k, v, vis, q8, scale=SCALE):
    """o, lse and the bounds of their errors, as R.attend's, but with each row's weight off by its own score's error.
    q [T][nqh][256]; k, v [nkvh][n_ctx][256]; vis [T][n_ctx].

    lost: what the weights' two f16 terms lose where the second is subnormal. A weight is cut off to 2^-24 where the largest
    of its query row lies at 2^12 or above, so it loses 2^-36 of the largest, and at most itself. q8_0: it is cut off as p f
    in units of which the largest p f holds 2^12 or more, f the power of two above the row's largest scale m (f <= 2 m);
    the products with the scales round to halves three times more, 2^-25 each where they are subnormal. So a row adds less
    than 2.5 * 2^-24 * 2^-12 * 127 * 2 max(p m) < 2^-33 * 127 max(p m) wrongly, and at most 127 p m; 127 m is taken as
    the largest value of the row, which is so where a code of that block is 127 (as here)."""
    T, nqh, _ = q.shape
    nkvh, g, n = k.shape[0], nqh // k.shape[0], vis.shape[1]
    q = q.astype(np.float64).reshape(T, nkvh, g, 256)
    o, bo = np.zeros((2, T, nkvh, g, 256))
    lse, bl = np.zeros((2, T, nkvh, g))
    none = ~vis.any(1)
    for kh in range(nkvh):
        s = scale * (q[:, kh] @ k[kh].T)
        e = score_bound(q[:, kh], k[kh], s, scale) + 2.0 ** -22 + 2.0 ** -21  # the exponential, a weight's two terms
        s = np.where(vis[:, None], s, -np.inf)
        m = np.where(none[:, None], 0, s.max(-1))
        p = np.exp(s - m[..., None])
        total = np.where(none[:, None], 1, p.sum(-1))
        with np.errstate(divide="ignore"):
            lse[:, kh] = np.where(none[:, None], -np.inf, m + np.log(total))
        p /= total[..., None]
        common = 2 * np.sqrt(n) * 2.0 ** -23 + 2.0 ** -22
        off, mean = p * e, p @ np.abs(v[kh])
        o[:, kh] = p @ v[kh]
        if q8:
            most = p * np.abs(v[kh]).max(1)
            lost = np.minimum(most, 2.0 ** -33 * most.max(-1, keepdims=True)).sum(-1, keepdims=True)
        else:
            lost = np.minimum(p, 2.0 ** -36 * p.max(-1, keepdims=True)) @ np.abs(v[kh])
        bo[:, kh] = off @ np.abs(v[kh]) + (off.sum(-1, keepdims=True) + common) * mean + lost
        bl[:, kh] = off.sum(-1) + common + np.abs(np.where(none[:, None], 0, lse[:, kh])) * 2.0 ** -22
    shape = (T, nqh)
    return o.reshape(*shape, 256), lse.reshape(shape), bo.reshape(*shape, 256), bl.reshape(shape)


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("T", [1, 4, 8, 12, 27])
def test_query_values_far_below_the_largest(G, T, q8):  # noqa: F811
    """One value of q is 2^22 times the others, where K is small; the scores come from the others, where K is large."""
    r = np.random.default_rng(23)
    pos0, n_ctx, nqh, nkvh = 100, 140, 24, 4
    k, v = r.standard_normal((nkvh, n_ctx, 256)) * 1000, r.standard_normal((nkvh, n_ctx, 256))
    k[:, :, :32] *= 2.0 ** -20
    k, v = cache(k, q8), cache(v, q8)
    q = (r.standard_normal((T, nqh, 256)) * 2.0 ** -18).astype(np.float32)
    q[:, :, 0] = 16
    dq, dk, dv, pos = G.up(q), G.up(k), G.up(v), G.i32(pos0)
    o, lse = G.tree(dq, dk, dv, pos, None, T, nqh, nkvh, n_ctx, q8)
    acc = G.full((nkvh, n_ctx), 0.0)
    G.ops.attn_weights(dq, lse, dk, pos, None, T, SCALE, nqh, nkvh, n_ctx, q8, acc)
    idx = np.tile(np.arange(3, dtype=np.int32), (T, nkvh, 1))
    bo_, bl_ = G.blocks(dq, dk, dv, pos, G.up(idx), T, 3, nqh, nkvh, n_ctx, q8)
    vis = R.visible(T, pos0, n_ctx, None)
    k, v = R.values(k, nkvh, n_ctx, q8), R.values(v, nkvh, n_ctx, q8)
    eo, el, bo, bl = attend(q, k, v, vis, q8)
    lse = G.down(lse)
    near(G.down(o), eo, bo, "o")
    near(lse, el, bl, "lse")
    near(G.down(bo_), eo, bo, "o of blocks")
    near(G.down(bl_), el, bl, "lse of blocks")
    want, off = np.zeros((2, nkvh, n_ctx))
    for t in range(T):
        for h in range(nqh):
            kh, qd = h // 6, q[t, h].astype(np.float64)
            s = SCALE * (k[kh] @ qd)
            p = np.where(vis[t], np.exp(s - np.float64(lse[t, h])), 0)
            want[kh] += p
            off[kh] += p * (score_bound(qd, k[kh], s, SCALE) + (np.abs(s) + abs(lse[t, h])) * 2.0 ** -22 + 2.0 ** -22)
    near(G.down(acc), want, off + want * 2.0 ** -22, "acc")


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("where", ["full", "drafted"])
@pytest.mark.parametrize("T,nqh", [(1, 24), (4, 24), (8, 24), (12, 24), (20, 24)])
def test_a_large_row_of_little_weight(G, T, nqh, where, q8):  # noqa: F811
    """Every token sees one V row 2^26 (f16: 2^20) times as large as the others with 2^-69 of their weight: it gives next
    to nothing, and the others keep their precision. full: in a tile that all tokens see whole; drafted: the first drafted
    row, in the tile of the draft."""
    r = np.random.default_rng(17)
    pos0, n_ctx, nkvh = 70, 100, 4
    j = 3 if where == "full" else pos0
    k, v = r.standard_normal((nkvh, n_ctx, 256)), r.standard_normal((nkvh, n_ctx, 256)) * 2.0 ** -9
    k[:, :, :32] = 0
    k[:, j, 0] = -16  # times 48 and the scale: a score of -48
    v[:, j] *= 2.0 ** (26 if q8 else 20)
    k, v = cache(k, q8), cache(v, q8)
    q = r.standard_normal((T, nqh, 256)).astype(np.float32)
    q[:, :, 0] = 48
    vis = R.visible(T, pos0, n_ctx, None)
    k64, v64 = R.values(k, nkvh, n_ctx, q8), R.values(v, nkvh, n_ctx, q8)
    assert np.isfinite(v64).all()
    eo, el, bo, bl = attend(q, k64, v64, vis, q8)
    dq, dk, dv, pos = G.up(q), G.up(k), G.up(v), G.i32(pos0)
    o, lse = G.tree(dq, dk, dv, pos, None, T, nqh, nkvh, n_ctx, q8)
    near(G.down(o), eo, bo, "o")
    near(G.down(lse), el, bl, "lse")
    o, lse = G.blocks(dq, dk, dv, pos, G.up(np.tile(np.arange(2, dtype=np.int32), (T, nkvh, 1))), T, 2, nqh, nkvh, n_ctx, q8)
    near(G.down(o), eo, bo, "o of blocks")
    near(G.down(lse), el, bl, "lse of blocks")


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("T,g,nkvh,n", [(1, 6, 4, 20000), (4, 6, 64, 2000), (40, 2, 64, 1500)])
def test_a_large_row_whose_weight_shrinks(G, T, g, nkvh, n, q8):  # noqa: F811
    """The scores rise by 60 over the rows that a wave walks, and the first rows' values are the largest: whatever unit they
    were summed in, the last rows, which have all the weight, keep their precision."""
    r = np.random.default_rng(29)
    n_ctx, nqh = n + T, nkvh * g
    k, v = (r.standard_normal((nkvh, n_ctx, 256), dtype=np.float32) for _ in range(2))
    k[:, :, :32] = 0
    step = 20000 / 256 if T == 1 else n / 4  # rows of a split at the most: the scores rise within each
    at = np.arange(n_ctx) % step / step
    k[:, :, 0] = 16 * at
    v *= (2.0 ** np.where(at < 0.1, 12 if q8 else 8, -10))[:, None].astype(np.float32)
    k, v = cache(k, q8), cache(v, q8)
    q = r.standard_normal((T, nqh, 256)).astype(np.float32)
    q[:, :, 0] = 60
    eo, el, bo, bl = attend(q, R.values(k, nkvh, n_ctx, q8), R.values(v, nkvh, n_ctx, q8), R.visible(T, n, n_ctx, None), q8)
    o, lse = G.tree(G.up(q), G.up(k), G.up(v), G.i32(n), None, T, nqh, nkvh, n_ctx, q8)
    near(G.down(o), eo, bo, "o")
    near(G.down(lse), el, bl, "lse")


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("score", [-48, -192])
@pytest.mark.parametrize("where", ["full", "beside the draft", "drafted"])
@pytest.mark.parametrize("T", [1, 4, 8, 12])
def test_values_that_are_not_finite_reach_all_that_see_them(G, T, where, score, bad, q8):  # noqa: F811
    """However little the row's weight (2^-69; none in float32), and wherever the row lies: in a tile that all see whole, in
    the tile of the draft before it, or drafted and seen by every other token."""
    r = np.random.default_rng(31)
    pos0, n_ctx, nqh, nkvh = 70, 100, 24, 4
    j = {"full": 3, "beside the draft": pos0 - 1, "drafted": pos0}[where]
    k, v = r.standard_normal((nkvh, n_ctx, 256)), r.standard_normal((nkvh, n_ctx, 256))
    k[:, :, :32] = 0
    k[:, j, 0] = -16
    k, v = cache(k, q8), cache(v, q8)
    q = r.standard_normal((T, nqh, 256)).astype(np.float32)
    q[:, :, 0] = -score
    tree = np.array([1 << t | (t % 2 == 0) for t in range(T)], np.uint64)
    vis = R.visible(T, pos0, n_ctx, tree)
    eo, el, bo, bl = attend(q, R.values(k, nkvh, n_ctx, q8), R.values(v, nkvh, n_ctx, q8), vis, q8)
    if q8:
        R.split_q8(v, nkvh, n_ctx)[1][:, j, 3] = bad
    else:
        v.view(np.float16).reshape(nkvh, n_ctx, 256)[:, j, 100] = bad
    dims = np.zeros(256, bool)
    dims[slice(96, 128) if q8 else 100] = True
    dq, dk, dv, pos = G.up(q), G.up(k), G.up(v), G.i32(pos0)
    o, lse = (G.down(x) for x in G.tree(dq, dk, dv, pos, G.u64(tree), T, nqh, nkvh, n_ctx, q8))
    near(lse, el, bl, "lse")
    hit = vis[:, j]
    assert not np.isfinite(o[hit][..., dims]).any()
    near(o[..., ~dims], eo[..., ~dims], bo[..., ~dims], "o of the other channels")
    # a channel whose own row is left out differs by next to nothing from one that holds a finite value there
    near(o[~hit], eo[~hit], bo[~hit], "o of the tokens that do not see the row")
    if where != "drafted":
        idx = G.up(np.tile(np.arange(2, dtype=np.int32), (T, nkvh, 1)))
        o = G.down(G.blocks(dq, dk, dv, pos, idx, T, 2, nqh, nkvh, n_ctx, q8)[0])
        assert not np.isfinite(o[..., dims]).any() and np.isfinite(o[..., ~dims]).all()


@pytest.mark.parametrize("q8", [True, False])
def test_entries_that_are_no_block_whatever_their_number(G, q8):  # noqa: F811
    """Among them numbers whose product with the block's 64 rows is a row of the context again in 32 bits."""
    r = np.random.default_rng(37)
    pos0, n_ctx, nqh, nkvh = 200, 260, 24, 4
    k, v = (R.make_cache(r, nkvh, n_ctx, q8, garbage_from=pos0 + 1) for _ in range(2))
    q = r.standard_normal((1, nqh, 256)).astype(np.float32)
    odd = [2 ** 25, 2 ** 25 + 1, 2 ** 26, 2 ** 26 + 1, 2 ** 26 + 3, 2 ** 31 - 1, -2 ** 31, -2 ** 31 + 1, -2 ** 26, -2 ** 26 + 2, -1, 4, 5]
    idx = np.array(odd + [1] + odd + [3], np.int32)
    vis = np.zeros((1, n_ctx), bool)
    vis[:, 64:128] = vis[:, 192:pos0 + 1] = True
    eo, el, bo, bl = attend(q, *(np.nan_to_num(R.values(x, nkvh, n_ctx, q8)) for x in (k, v)), vis, q8)
    o, lse = G.blocks(G.up(q), G.up(k), G.up(v), G.i32(pos0), G.up(np.tile(idx, (1, nkvh, 1))), 1, len(idx), nqh, nkvh, n_ctx, q8)
    near(G.down(o), eo, bo, "o")
    near(G.down(lse), el, bl, "lse")


@pytest.mark.parametrize("bad", [np.inf, np.nan])
@pytest.mark.parametrize("j", [3, 69, 70])
@pytest.mark.parametrize("T", [1, 4, 8, 12])
def test_a_row_without_a_finite_scale(G, T, j, bad):  # noqa: F811
    """q8_0: none of a V row's scales is finite. Row 70 is drafted and seen by every other token, the others by all."""
    r = np.random.default_rng(47)
    pos0, n_ctx, nqh, nkvh = 70, 100, 24, 4
    k, v = (R.make_cache(r, nkvh, n_ctx, True) for _ in range(2))
    R.split_q8(v, nkvh, n_ctx)[0][:, :, ::32] = 127
    q = r.standard_normal((T, nqh, 256)).astype(np.float32)
    tree = np.array([1 << t | (t % 2 == 0) for t in range(T)], np.uint64)
    vis = R.visible(T, pos0, n_ctx, tree)
    eo, el, bo, bl = attend(q, R.values(k, nkvh, n_ctx, True), R.values(v, nkvh, n_ctx, True), vis, True)
    R.split_q8(v, nkvh, n_ctx)[1][:, j] = bad
    o, lse = (G.down(x) for x in G.tree(G.up(q), G.up(k), G.up(v), G.i32(pos0), G.u64(tree), T, nqh, nkvh, n_ctx, True))
    hit = vis[:, j]
    near(lse, el, bl, "lse")
    assert not np.isfinite(o[hit]).any()
    near(o[~hit], eo[~hit], bo[~hit], "o")


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("T", [2, 4, 8, 12])
def test_a_query_that_is_not_finite(G, T, bad, q8):  # noqa: F811
    """One head of one token: its results are NaN, all others keep their bits."""
    r = np.random.default_rng(53)
    pos0, n_ctx, nqh, nkvh = 70, 100, 24, 4
    k, v = (G.up(R.make_cache(r, nkvh, n_ctx, q8)) for _ in range(2))
    q = r.standard_normal((T, nqh, 256)).astype(np.float32)
    run = lambda q: [G.down(x) for x in G.tree(G.up(q), k, v, G.i32(pos0), None, T, nqh, nkvh, n_ctx, q8)]  # noqa: E731
    want = run(q)
    q[1, 7, 100] = bad
    got = run(q)
    for x, y in zip(got, want):
        assert np.isnan(x[1, 7]).all()
        x[1, 7] = y[1, 7]
        assert (x.view(np.int32) == y.view(np.int32)).all()
