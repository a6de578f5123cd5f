"""Attention over the K/V cache on the GPU: a token's result does not depend on the others'."""
import numpy as np
import pytest

import attnref as R
from conftest import assert_bits_equal
from test_gpu_attn import G, SCALE, near  # noqa: F401
from test_gpu_attn_edges import attend

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
