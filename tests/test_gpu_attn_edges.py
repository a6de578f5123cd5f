"""Attention over the K/V cache on the GPU where it can go wrong and tests/test_gpu_attn.py does not look, against a plain
64-bit form: query values far below their row's largest."""
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


def attend(q, k, v, vis, scale=SCALE):
    """o, lse and the bounds of their errors, as R.attend's, but with each row's weight off by its own score's error.
    q [T][nqh][256]; k, v [nkvh][n_ctx][256]; vis [T][n_ctx]."""
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
        bo[:, kh] = off @ np.abs(v[kh]) + (off.sum(-1, keepdims=True) + common) * mean
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
    eo, el, bo, bl = attend(q, k, v, vis)
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
