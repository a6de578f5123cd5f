"""Attention over the K/V cache on the GPU with many tiles of cache rows to a workgroup, where the kernels' pipelines run: LDS
buffers and staged registers taken in turn, the softmax's reference and the unit of the outputs moved from tile to tile,
whole tiles before those of the draft; and that a token's result does not depend on the others'. Against a plain 64-bit
form."""
import numpy as np
import pytest

import attnref as R
from conftest import assert_bits_equal
from test_gpu_attn import G, SCALE, near  # noqa: F401
from test_gpu_attn_edges import attend, score_bound

pytestmark = pytest.mark.gpu


def rows_of_cache(r, nkvh, n_ctx, q8, end, spread):
    """K whose first channel rises by 40 over the rows, V whose rows' sizes differ by up to 2^spread; NaN from `end` on."""
    k, v = (R.make_cache(r, nkvh, n_ctx, q8, garbage_from=end) for _ in range(2))
    rise, size = np.linspace(0, 40, n_ctx), 2.0 ** r.integers(-spread, 1, n_ctx)
    if q8:
        c, d = R.split_q8(k, nkvh, n_ctx)
        d[:, :, 0] = 40 / 127
        c[:, :, :32] = 0
        c[:, :, 0] = np.rint(rise / 40 * 127)
        d[:, end:] = np.nan
        R.split_q8(v, nkvh, n_ctx)[1][:] *= size[None, :, None].astype(np.float16)
        R.split_q8(v, nkvh, n_ctx)[0][:, :, ::32] = 127  # every block's scale is that of a code of 127
    else:
        k.view(np.float16).reshape(nkvh, n_ctx, 256)[:, :end, 0] = rise[:end]
        v.view(np.float16).reshape(nkvh, n_ctx, 256)[:] *= size[None, :, None].astype(np.float16)
    return k, v


def queries(r, T, nqh):
    """Scores that rise with the rows, fall, or do neither."""
    q = r.standard_normal((T, nqh, 256)).astype(np.float32)
    q[:, :, 0] = np.array([0, 12, -12, 3], np.float32)[r.integers(0, 4, (T, nqh))]
    return q


# tokens, query heads of a kv head, kv heads, rows before, context, row tiles of 16 query rows. The many kv heads leave few
# splits of the rows for each, so that a workgroup walks many tiles.
WIDE = [(48, 1, 64, 2430, 2500, 3), (64, 1, 64, 2395, 2459, 4), (40, 2, 64, 1501, 1541, 5), (64, 2, 64, 1470, 1600, 8),
        (64, 3, 16, 3203, 3300, 12)]
NARROW = [(20, 1, 128, 905, 930, 2), (5, 6, 128, 1100, 1105, 2), (4, 4, 256, 1157, 1200, 1)]


def splits_at_most(G, T, nqh, nkvh, n_ctx):  # noqa: F811
    """Of attn_tree: its workspace holds 258 floats a query row and split."""
    return max(1, G.ops.attn_tree_ws_bytes(T, nqh, nkvh, n_ctx) // (T * nqh * 258 * 4))


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("T,g,nkvh,pos0,n_ctx,row_tiles", WIDE + NARROW)
def test_tree_over_many_tiles(G, T, g, nkvh, pos0, n_ctx, row_tiles, q8):  # noqa: F811
    """Two drafted rows' values are not finite besides: the tokens that see them get that, the others their results."""
    assert -(-T * g // 16) == row_tiles
    nqh, end = nkvh * g, pos0 + T
    per = -(-end // 32) // splits_at_most(G, T, nqh, nkvh, n_ctx)
    assert per >= (9 if row_tiles > 2 else 12), "too few tiles to a workgroup (narrow: four waves share them)"
    r = np.random.default_rng(T + pos0)
    k, v = rows_of_cache(r, nkvh, n_ctx, q8, end, 12)
    q, tree = queries(r, T, nqh), R.random_tree(r, T, empty=(0,))
    vis = R.visible(T, pos0, n_ctx, tree)
    eo, el, bo, bl = attend(q, *(np.nan_to_num(R.values(x, nkvh, n_ctx, q8)) for x in (k, v)), vis, q8)
    dims = np.zeros(256, bool)
    hit = np.zeros(T, bool)
    for t, bad in ((1, np.inf), (T - 2, np.nan)):
        if q8:
            R.split_q8(v, nkvh, n_ctx)[1][:, pos0 + t, 3] = bad
        else:
            v.view(np.float16).reshape(nkvh, n_ctx, 256)[:, pos0 + t, 100] = bad
        hit |= vis[:, pos0 + t]
    dims[slice(96, 128) if q8 else 100] = True
    o, lse = (G.down(x) for x in G.tree(G.up(q), G.up(k), G.up(v), G.i32(pos0), G.u64(tree), T, nqh, nkvh, n_ctx, q8))
    near(lse, el, bl, "lse")
    near(o[..., ~dims], eo[..., ~dims], bo[..., ~dims], "o")
    near(o[~hit], eo[~hit], bo[~hit], "o of the tokens that see no odd row")
    assert hit.any() and not hit.all() and not np.isfinite(o[hit][..., dims]).any()


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("T,nqh,nkvh,pos0,n_ctx", [(4, 24, 4, 1000, 1100), (2, 24, 4, 3000, 3100), (10, 24, 4, 700, 800), (20, 24, 4, 500, 600),
                                                   (64, 128, 64, 700, 764)])
def test_a_token_does_not_depend_on_the_others(G, T, nqh, nkvh, pos0, n_ctx, q8):  # noqa: F811
    """The same number of tokens with other queries and masks beside it: bit for bit the same o and lse. The others' scores
    are eight times as large, so that their softmax moves its reference where this token's does not."""
    r = np.random.default_rng(41)
    k, v = rows_of_cache(r, nkvh, n_ctx, q8, pos0 + T, 12)
    q, tree = queries(r, T, nqh), R.random_tree(r, T)
    q[:, :, 0] = 3
    dk, dv, pos = G.up(k), G.up(v), G.i32(pos0)
    run = lambda q, tree: [G.down(x) for x in G.tree(G.up(q), dk, dv, pos, G.u64(tree), T, nqh, nkvh, n_ctx, q8)]  # noqa: E731
    o, lse = run(q, tree)
    for t in sorted({0, T // 2, T - 1}):
        q2, tree2 = q * 8, np.full(T, (1 << T) - 1, np.uint64)
        q2[t], tree2[t] = q[t], tree[t]
        o2, lse2 = run(q2, tree2)
        assert_bits_equal(o2[t], o[t], f"o of token {t}")
        assert_bits_equal(lse2[t], lse[t], f"lse of token {t}")
        assert (o2 != o).any()


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("T,pos0", [(4, 1000), (12, 800)])
def test_a_token_alone_and_in_a_batch(G, T, pos0, q8):  # noqa: F811
    """The first token of a batch as the only one: the same value within the bounds (the rows are split another way)."""
    r = np.random.default_rng(43)
    nqh, nkvh, n_ctx = 24, 4, pos0 + T
    k, v = rows_of_cache(r, nkvh, n_ctx, q8, n_ctx, 12)
    q = queries(r, T, nqh)
    dk, dv, pos = G.up(k), G.up(v), G.i32(pos0)
    many = [G.down(x)[:1] for x in G.tree(G.up(q), dk, dv, pos, None, T, nqh, nkvh, n_ctx, q8)]
    one = [G.down(x) for x in G.tree(G.up(q[:1]), dk, dv, pos, None, 1, nqh, nkvh, n_ctx, q8)]
    _, _, bo, bl = attend(q[:1], R.values(k, nkvh, n_ctx, q8), R.values(v, nkvh, n_ctx, q8), R.visible(1, pos0, n_ctx, None), q8)
    near(many[0], one[0].astype(np.float64), 2 * bo, "o")
    near(many[1], one[1].astype(np.float64), 2 * bl, "lse")


# Of attn_weights: 1024 workgroups up to two row tiles, each of whose four waves walks tiles of its own, 512 of up to four,
# else 256. Over f16, 12 row tiles are one group, two to a wave; the last case is several groups.
@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("T,g,nkvh,pos0,n_ctx,rows", [
    (10, 1, 256, 1140, 1160, None), (20, 1, 256, 1157, 1180, 0xf3a5f), (64, 1, 64, 2395, 2459, 0xf0f0ffff1234f00f), (40, 2, 64, 1501, 1541, None),
    (64, 3, 16, 4700, 4764, None), (64, 3, 16, 4711, 4790, 0x00000000ffff0001), (64, 6, 16, 4700, 4764, None)])
def test_weights_over_many_tiles(G, T, g, nkvh, pos0, n_ctx, rows, q8):  # noqa: F811
    r = np.random.default_rng(T * g + pos0)
    nqh, end, row_tiles = nkvh * g, pos0 + T, -(-T * g // 16)
    groups = 1024 if row_tiles <= 2 else 512 if row_tiles <= 4 else 256
    assert -(-end // 32) // (groups // nkvh) >= 9
    k, _ = rows_of_cache(r, nkvh, n_ctx, q8, end, 0)
    q, tree = queries(r, T, nqh), R.random_tree(r, T)
    vis = R.visible(T, pos0, n_ctx, tree)
    k64 = np.nan_to_num(R.values(k, nkvh, n_ctx, q8))
    used = np.array([rows is None or bool(rows >> t & 1) for t in range(T)])
    lse = np.zeros((T, nkvh, g), np.float32)
    want, off = np.zeros((2, nkvh, n_ctx))
    q4 = q.astype(np.float64).reshape(T, nkvh, g, 256)
    for kh in range(nkvh):
        s = SCALE * (q4[:, kh] @ k64[kh].T)
        x = np.where(vis[:, None], s, -np.inf)
        m = x.max(-1)
        lse[:, kh] = m + np.log(np.exp(x - m[..., None]).sum(-1))
        ls = lse[:, kh].astype(np.float64)[..., None]
        p = np.where(used[:, None, None], np.exp(x - ls), 0)
        want[kh] = p.sum((0, 1))
        off[kh] = (p * (score_bound(q4[:, kh], k64[kh], s, SCALE) + (np.abs(s) + np.abs(ls)) * 2.0 ** -22 + 2.0 ** -22)).sum((0, 1))
    acc = r.uniform(0, 3, (nkvh, n_ctx)).astype(np.float32)
    want[:, :pos0] += acc[:, :pos0]
    want[:, end:] = acc[:, end:]
    d = G.up(acc)
    G.ops.attn_weights(G.up(q), G.up(lse.reshape(T, nqh)), G.up(k), G.i32(pos0), G.u64(tree), T, SCALE, nqh, nkvh, n_ctx, q8, d,
                       rows=None if rows is None else G.u64([rows]))
    # up to T g terms of one row are added in float32, 2^-24 of the running sum each, and the row's weight
    near(G.down(d), want, off + np.abs(want) * (np.sqrt(T * g) + 4) * 2.0 ** -23, "acc")
    assert_bits_equal(G.down(d)[:, end:], acc[:, end:], "rows behind the last")
