"""A batch of sequences over a K/V cache in pages on the GPU: its rows written (bit for bit), read back (exactly), attended to
(within the bounds of tests/attnref.py), and drafted tokens verified (exactly); and the four together in a HIP graph. Memory
that no call may read holds NaN."""
import numpy as np
import pytest

import attnref as R
import cfgdata as cd
import pagedref as P
from conftest import assert_bits_equal
from test_gpu_attn import G, SCALE, near  # noqa: F401

pytestmark = pytest.mark.gpu
TYPES = [P.F16, P.Q8, P.Q8_Q4]


def handle(G, kp, vp, table, type):  # noqa: F811
    return G.ops.KvPages(G.up(kp.buf), G.up(vp.buf), G.up(table), kp.nkvh, kp.page, type)


def attn(G, q, kv, pos, cu, most, nqh, scale=SCALE):  # noqa: F811
    T = q.shape[0]
    o, lse = G.full((T, nqh, 256), 7.0), G.full((T, nqh), 7.0)
    G.ops.attn_paged(q, kv, pos, cu, T, most, scale, nqh, o, G.ws(G.ops.attn_paged_ws_bytes(kv, T, most, nqh)), lse=lse)
    return o, lse


def check(G, q, kp, vp, table, type, pos, new, most, nqh, got=None):  # noqa: F811
    """Runs attn_paged (unless `got`) and holds it to the plain form."""
    o, lse = got or attn(G, G.up(q), handle(G, kp, vp, table, type), G.i32(*pos), G.up(P.cu_of(new)), most, nqh)
    eo, el, bo, bl = P.attend(q, kp, vp, table, pos, new, SCALE)
    o, lse = G.down(o), G.down(lse)
    n = int(sum(new))
    near(o[:n], eo, bo, "o")
    seen = np.isfinite(el)
    assert np.array_equal(seen, lse[:n] != -np.inf)
    near(lse[:n][seen], el[seen], bl[seen], "lse")
    assert np.all(o[n:] == 7) and np.all(lse[n:] == 7)


# (rows before the batch, new tokens, rows of a page, query heads, kv heads)
BATCHES = [
    ([0], [1], 32, 24, 4),                          # a sequence's first token
    ([30], [1], 32, 24, 4),
    ([31], [1], 32, 24, 4),                         # a tile and a page, exactly
    ([32], [1], 64, 24, 4),
    ([0, 63, 64, 127, 5], [1, 1, 1, 1, 1], 64, 24, 4),
    ([700, 3, 129, 40], [1, 0, 1, 2], 64, 24, 4),   # no token, one, two
    ([0, 0, 0], [0, 3, 0], 32, 6, 2),
    ([1000, 33, 500], [4, 1, 4], 128, 24, 4),       # drafts: two row tiles
    ([95, 10], [5, 2], 32, 24, 4),                  # 30 query rows
    ([95, 10, 300], [6, 1, 3], 32, 24, 4),          # 36: two units a kv head
    ([40, 7], [64, 11], 64, 24, 4),                 # as many as there can be
    ([100, 200], [1, 1], 64, 7, 7),
    ([77, 12], [1, 1], 64, 16, 1),                  # a full row tile
    ([77, 12], [1, 1], 64, 24, 1),                  # one and a half
    ([77, 1], [3, 1], 256, 40, 1),                  # 120 query rows of one kv head
    ([5000, 17, 900], [1, 1, 1], 64, 24, 4),        # parts of a long one, joined
    ([9000], [2], 32, 6, 1),
]


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("pos,new,page,nqh,nkvh", BATCHES)
def test_attn(G, pos, new, page, nqh, nkvh, type):  # noqa: F811
    r = np.random.default_rng(sum(pos) + 7 * sum(new) + nqh)
    kp, vp, table = P.make_pages(r, pos, new, page, nkvh, type)
    q = (r.standard_normal((sum(new), nqh, 256)) * 1.5).astype(np.float32)
    check(G, q, kp, vp, table, type, pos, new, max(new), nqh)


@pytest.mark.parametrize("type", TYPES)
def test_attn_of_many_sequences(G, type):  # noqa: F811
    """More sequences than threads of a workgroup, short ones, some without tokens; and rows of tokens behind the last."""
    r = np.random.default_rng(3)
    pos = [int(x) for x in r.integers(0, 70, 600)]
    new = [int(x) for x in r.integers(0, 3, 600)]
    kp, vp, table = P.make_pages(r, pos, new, 32, 2, type)
    q = (r.standard_normal((sum(new) + 5, 4, 256)) * 1.5).astype(np.float32)
    check(G, q, kp, vp, table, type, pos, new, 2, 4)


@pytest.mark.parametrize("type", TYPES)
def test_attn_without_cu_is_one_token_each(G, type):  # noqa: F811
    r = np.random.default_rng(4)
    pos, new = [130, 0, 64], [1, 1, 1]
    kp, vp, table = P.make_pages(r, pos, new, 64, 4, type)
    q = r.standard_normal((3, 24, 256)).astype(np.float32)
    check(G, q, kp, vp, table, type, pos, new, 1, 24,
          attn(G, G.up(q), handle(G, kp, vp, table, type), G.i32(*pos), None, 1, 24))


@pytest.mark.parametrize("type", TYPES)
def test_attn_rows_that_do_not_exist(G, type):  # noqa: F811
    """Pages that are none (before, among and behind others), tokens past the table's end, before row 0, of no row at all."""
    r = np.random.default_rng(5)
    pos, new = [200, 150, 70, 638, 20, 639], [2, 1, 3, 2, 2, 1]
    kp, vp, table = P.make_pages(r, pos, new, 64, 4, type, holes=[(0, 0), (1, 1), (2, 1), (3, 2), (3, 3), (4, 0)], extra=0)
    pos = [200, 150, 70, 639, -1, 640]  # the table ends at row 640
    q = r.standard_normal((sum(new), 24, 256)).astype(np.float32)
    assert table.shape[1] == 10
    check(G, q, kp, vp, table, type, pos, new, 3, 24)


@pytest.mark.parametrize("type", TYPES)
def test_attn_leaves_out_tokens_behind_max_tokens(G, type):  # noqa: F811
    r = np.random.default_rng(6)
    pos, new = [50, 9], [5, 2]
    kp, vp, table = P.make_pages(r, pos, new, 32, 4, type)
    q = r.standard_normal((7, 24, 256)).astype(np.float32)
    kv = handle(G, kp, vp, table, type)
    o, lse = (G.down(x) for x in attn(G, G.up(q), kv, G.i32(*pos), G.up(P.cu_of(new)), 3, 24))
    eo, el, bo, bl = P.attend(q, kp, vp, table, pos, new, SCALE)
    on = [0, 1, 2, 5, 6]
    # the tokens taken are the same rows; those left out are no rows of the sequence then, but no token before sees them
    near(o[on], eo[on], bo[on], "o")
    near(lse[on], el[on], bl[on], "lse")
    assert np.all(o[3:5] == 7) and np.all(lse[3:5] == 7)


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("cu", [[0, 5, 3, 9], [-4, 2, 2, 100], [3, 3, 3, 3], [7, 1, 0, -1]])
def test_attn_with_bad_token_offsets_stays_inside(G, cu, type):  # noqa: F811
    """What cu holds is cut to 0 .. T and to rise; nothing else is promised, but that nothing outside is read or written."""
    r = np.random.default_rng(8)
    pos, T = [50, 9, 20], 8
    kp, vp, table = P.make_pages(r, pos, [8, 8, 8], 32, 4, type)
    q = G.up(r.standard_normal((T, 24, 256)).astype(np.float32))
    o, lse = attn(G, q, handle(G, kp, vp, table, type), G.i32(*pos), G.i32(*cu), 8, 24)
    assert np.isfinite(G.down(o)).all()


@pytest.mark.parametrize("type", TYPES)
def test_attn_gives_the_same_bits(G, type):  # noqa: F811
    r = np.random.default_rng(9)
    pos, new = [4000, 33, 900, 2], [2, 1, 3, 1]
    kp, vp, table = P.make_pages(r, pos, new, 64, 4, type)
    q, kv = G.up(r.standard_normal((7, 24, 256)).astype(np.float32)), handle(G, kp, vp, table, type)
    first = [G.down(x).copy() for x in attn(G, q, kv, G.i32(*pos), G.up(P.cu_of(new)), 3, 24)]
    for _ in range(3):
        for a, b in zip(first, attn(G, q, kv, G.i32(*pos), G.up(P.cu_of(new)), 3, 24)):
            assert_bits_equal(G.down(b), a, "again")


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("type", TYPES)
def test_attn_values_that_are_not_finite(G, type, bad):  # noqa: F811
    """V rows that hold one: it reaches the tokens that see the row, and no others."""
    r = np.random.default_rng(10)
    pos, new = [70, 40], [3, 2]
    kp, vp, table = P.make_pages(r, pos, new, 32, 2, type)
    for row in (3, 71):  # a row that all of sequence 0's tokens see; the row of its second token
        p, j = table[0, row // 32], row % 32
        if type == P.F16:
            vp.codes[p, 1, j].view(np.float16)[17] = bad
        else:
            vp.scales[p, 1, j].view(np.float16)[2] = bad
            vp.codes[p, 1, j] = 0x22 if type == P.Q8_Q4 else 5  # a code of -6, or 5
    q = r.standard_normal((5, 12, 256)).astype(np.float32)
    o = G.down(attn(G, G.up(q), handle(G, kp, vp, table, type), G.i32(*pos), G.up(P.cu_of(new)), 3, 12)[0])
    with np.errstate(invalid="ignore"):
        eo, _, bo, _ = P.attend(q, kp, vp, table, pos, new, SCALE)
    fine = np.isfinite(eo)
    assert np.array_equal(np.isfinite(o), fine)
    assert not fine[:3, 6:].all() and fine[3:].all() and fine[:, :6].all()
    near(o[fine], eo[fine], bo[fine], "o")


@pytest.mark.parametrize("type", TYPES)
def test_attn_pages_behind_2_31_bytes(G, type):  # noqa: F811
    """The last pages of a pool of more than 2^31 bytes, a page table in no order."""
    import torch

    r = np.random.default_rng(11)
    page, nkvh, pos, new = 1024, 4, [3000], [2]
    kp, vp, table = P.make_pages(r, pos, new, page, nkvh, type)
    kb, vb = kp.buf.shape[1], vp.buf.shape[1]
    n = (1 << 31) // vb + 10
    dk, dv = (torch.zeros(n, b, dtype=torch.uint8, device=G.i32(0).device) for b in (kb, vb))
    at = {int(p): n - 1 - 2 * i for i, p in enumerate(table[0][table[0] >= 0])}
    for p, i in at.items():
        dk[i], dv[i] = G.up(kp.buf[p]), G.up(vp.buf[p])
    moved = np.array([[at.get(int(p), -1) for p in table[0]]], np.int32)
    q = r.standard_normal((2, 24, 256)).astype(np.float32)
    kv = G.ops.KvPages(dk, dv, G.up(moved), nkvh, page, type)
    check(G, q, kp, vp, table, type, pos, new, 2, 24, attn(G, G.up(q), kv, G.i32(*pos), G.up(P.cu_of(new)), 2, 24))


# ---------------------------------------------------------------- rows written
def prep(G, kv, qg, kx, vx, qw, kw, pos, cu, nqh, rope3=None, rdelta=None):  # noqa: F811
    T = qg.shape[0]
    qn = G.full((T, nqh, 256), 7.0)
    G.ops.attn_prep_paged(G.up(qg), G.up(kx), G.up(vx), G.up(qw), G.up(kw), qn, kv, G.i32(*pos), None if cu is None else G.up(cu), T,
                          1e-6, cd.THETA_SCALE, nqh, rope3=None if rope3 is None else G.up(rope3),
                          rdelta=None if rdelta is None else G.i32(*rdelta))
    return G.down(qn)


def prep_inputs(r, T, nqh, nkvh):
    return [(s * r.standard_normal(x)).astype(np.float32) for s, x in ((2, (T, nqh, 512)), (1, (T, nkvh, 256)), (1, (T, nkvh, 256)))] + \
        [(1 + 0.1 * r.standard_normal(256)).astype(np.float32) for _ in range(2)]


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("pos,new,page,nqh,nkvh,extra", [
    ([0], [1], 32, 24, 4, "none"), ([31, 150000, 64], [1, 1, 1], 32, 24, 4, "none"), ([31, 0, 7, 90], [3, 0, 40, 1], 32, 24, 4, "rdelta"),
    ([5, 63], [2, 2], 64, 7, 1, "rope3"), ([10, 700], [70, 33], 64, 24, 4, "rdelta"),
    ([3] * 70, [1, 2] * 35, 32, 3, 3, "rdelta"), ([1], [60], 128, 90, 5, "none")])
def test_prep(G, oracle, pos, new, page, nqh, nkvh, extra, type):  # noqa: F811
    """Queries and f16 / q8_0 rows as attn_prep leaves them, bit for bit; 4-bit rows from their definition; no other byte."""
    r = np.random.default_rng(sum(pos) + sum(new))
    T, cu, B = sum(new), P.cu_of(new), len(pos)
    low = [p // page * page if p > 1000 else 0 for p in pos]  # a far position: the pages before it are none
    kp, vp, table = P.make_pages(r, [p - a for p, a in zip(pos, low)], new, page, nkvh, type)
    wide = np.full((B, max(a // page for a in low) + table.shape[1]), -1, np.int32)
    for b in range(B):
        wide[b, low[b] // page:low[b] // page + table.shape[1]] = table[b]
    qg, kx, vx, qw, kw = prep_inputs(r, T + 2, nqh, nkvh)  # two tokens of no sequence
    rope3 = r.integers(0, 5000, (T + 2, 3)).astype(np.int32) if extra == "rope3" else None
    rdelta = [int(x) for x in r.integers(-3, 50, B)] if extra == "rdelta" else None
    ek, ev = (P.Pool(len(p.buf), nkvh, page, p.bits, 0) for p in (kp, vp))
    ek.buf[:], ev.buf[:] = kp.buf, vp.buf
    kv = handle(G, kp, vp, wide, type)
    qn = prep(G, kv, qg, kx, vx, qw, kw, pos, cu, nqh, rope3, rdelta)
    for b in range(B):
        n = new[b]
        if not n:
            continue
        s = slice(cu[b], cu[b + 1])
        kc, vc = (np.zeros(nkvh * n * (512 if type == P.F16 else 272), np.uint8) for _ in range(2))
        # a contiguous cache of the new rows alone: the rotary position goes by rdelta
        e = oracle.attn_prep(qg[s].reshape(-1), kx[s].reshape(-1), vx[s].reshape(-1), qw, kw, kc, vc, 0, n, 1e-6, cd.THETA_SCALE,
                             nqh, nkvh, n, type != P.F16, rope3=None if rope3 is None else rope3[s],
                             rdelta=(rdelta[b] if rdelta else 0) - pos[b])
        assert_bits_equal(qn[s].reshape(-1), e, "qn")
        for pool, c in ((ek, kc), (ev, vc)):
            for t in range(n):
                j = pos[b] + t
                if pool.bits == 4:
                    codes, scales = P.row_parts(vx[cu[b] + t], 4)
                elif pool.bits == 16:
                    codes, scales = c.reshape(nkvh, n, 512)[:, t], None
                else:
                    codes, scales = c[:nkvh * n * 256].reshape(nkvh, n, 256)[:, t], c[nkvh * n * 256:].reshape(nkvh, n, 16)[:, t]
                pool.put(wide[b, j // page], j % page, codes, scales)
    assert np.array_equal(G.down(kv.k), ek.buf) and np.array_equal(G.down(kv.v), ev.buf)
    assert np.all(qn[T:] == 7)


@pytest.mark.parametrize("type", TYPES)
def test_prep_rows_that_do_not_exist(G, type):  # noqa: F811
    """Tokens past the table's end, before row 0, or whose page is none: queries, and no byte of the pages."""
    r = np.random.default_rng(12)
    kp, vp, table = P.make_pages(r, [60, 60, 60], [2, 2, 2], 64, 4, type, holes=[(1, 0), (2, 0)], extra=0)
    kv = handle(G, kp, vp, table, type)
    qg, kx, vx, qw, kw = prep_inputs(r, 6, 24, 4)
    qn = prep(G, kv, qg, kx, vx, qw, kw, [64, -2, 10], P.cu_of([2, 2, 2]), 24)
    assert np.array_equal(G.down(kv.k), kp.buf) and np.array_equal(G.down(kv.v), vp.buf) and not (qn == 7).any()


def test_prep_four_bits_of_odd_values(G):  # noqa: F811
    """Blocks of zeros, of one value, whose largest values are a and -a, of subnormal numbers, and with halves to round."""
    r = np.random.default_rng(13)
    T, nkvh = 12, 2
    qg, kx, vx, qw, kw = prep_inputs(r, T, 4, nkvh)
    vx[0] = 0
    vx[1] = 0.5
    vx[2, :, 5::32], vx[2, :, 9::32] = 4, -4
    vx[3, :, 5::32], vx[3, :, 9::32] = -4, 4
    vx[4] *= np.float32(1e-39)
    vx[5] *= np.float32(1e-44)
    vx[6] *= np.float32(60000)
    d = np.float32(0.375)
    vx[7] = (r.integers(-16, 16, vx[7].shape) / 2 * d).astype(np.float32)
    vx[7, :, ::32] = 8 * d
    vx[8], vx[8, :, ::32] = -0.0, -3e-38
    kp, vp, table = P.make_pages(r, [0], [T], 32, nkvh, P.Q8_Q4)
    kv = handle(G, kp, vp, table, P.Q8_Q4)
    prep(G, kv, qg, kx, vx, qw, kw, [0], P.cu_of([T]), 4)
    codes, scales = P.row_parts(vx, 4)
    for t in range(T):
        vp.put(table[0, 0], t, codes[t], scales[t])
    assert np.array_equal(G.down(kv.v), vp.buf)


# ---------------------------------------------------------------- rows read
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("kind", ["float32", "float16", "bfloat16"])
def test_read(G, kind, type):  # noqa: F811
    import torch

    r = np.random.default_rng(14)
    rows, page, nkvh, n_out = [1, 300, 64, 0, 129, 33], 32, 3, 131
    kp, vp, table = P.make_pages(r, rows, [0] * 6, page, nkvh, type, holes=[(4, 1), (4, 2)])
    start, count = [0, 7, 0, 0, 40, 30], [1, 200, 64, 5, 89, -2]  # 200: cut to n_out; sequence 3 has no pages
    kv = handle(G, kp, vp, table, type)
    dt = getattr(torch, kind)
    for with_start in (True, False):
        for which in (3, 1, 2):
            outs = [G.full((6, nkvh, n_out, 256), 7.0, dt) if which >> i & 1 else None for i in range(2)]
            G.ops.kv_pages_read(kv, G.i32(*start) if with_start else None, G.i32(*count), n_out, *outs)
            for out, pool in zip(outs, (kp, vp)):
                if out is None:
                    continue
                want = np.full((6, nkvh, n_out, 256), 7.0)
                for b in range(6):
                    n = max(0, min(count[b], n_out))
                    a = start[b] if with_start else 0
                    x, there = pool.values(table[b], a + n)
                    x[:, ~there] = 0
                    want[b, :, :n] = x[:, a:]
                torch.cuda.synchronize()
                want = torch.from_numpy(want).to(torch.float32).to(dt)  # a code times a scale is exact in float32
                got = out.cpu()
                assert torch.equal(torch.nan_to_num(got, 9.0), torch.nan_to_num(want, 9.0))


@pytest.mark.parametrize("type", TYPES)
def test_read_gives_a_cache_for_attn_tree(G, type):  # noqa: F811
    """A sequence taken out of the pages as f16: attn_tree over it agrees with the plain form over its values."""
    import torch

    r = np.random.default_rng(15)
    n, nkvh, nqh = 300, 4, 24
    kp, vp, table = P.make_pages(r, [n], [0], 64, nkvh, type)
    kc, vc = (G.full((1, nkvh, n, 256), 0.0, torch.float16) for _ in range(2))
    G.ops.kv_pages_read(handle(G, kp, vp, table, type), None, G.i32(n), n, kc, vc)
    q = r.standard_normal((1, nqh, 256)).astype(np.float32)
    o, _ = G.tree(G.up(q), kc, vc, G.i32(n - 1), None, 1, nqh, nkvh, n, False)
    k, v = (G.down(x)[0].astype(np.float64) for x in (kc, vc))
    eo, _, bo, _ = R.attend(q, k, v, R.visible(1, n - 1, n, None), SCALE)
    near(G.down(o), eo, bo, "o")


# ---------------------------------------------------------------- drafts verified
def probabilities(r, T, V, peak):
    x = r.standard_normal((T, V)).astype(np.float32) * 2
    for t in range(T):
        x[t, r.integers(0, V, 4)] += peak
    e = np.exp(x - x.max(1, keepdims=True), dtype=np.float32)
    return e / e.sum(1, keepdims=True, dtype=np.float32)


def verify(G, p, q, ids, parent, u, ul, cu, V, ld=0):  # noqa: F811
    import torch

    T, B = len(ids), len(cu) - 1
    out, path, n_path, pos = np.full(T, 55, np.int32), np.full(T, 66, np.int32), np.full(B, 77, np.int32), np.arange(B, dtype=np.int32)

    def rows(x):
        if x is None or not ld:
            return None if x is None else G.up(x)
        wide = G.full((T, ld), float("nan"))
        wide[:, :V] = G.up(x)
        return wide[:, :V]

    d = [G.up(x) for x in (out, path, n_path, pos)]
    G.ops.draft_verify(rows(p), rows(q), G.up(ids), None if parent is None else G.up(parent), G.up(u), G.up(ul), G.up(cu), B, V,
                       d[0], d[1], d[2], G.ws(G.ops.draft_verify_ws_bytes(B, V)), pos=d[3])
    got = [G.down(x) for x in d]
    want = P.verify(p, q, ids, parent, u, ul, cu, V, out, path, n_path, pos)
    for g, w, what in zip(got, want, ("out", "path", "n_path", "pos")):
        assert np.array_equal(g, w), (what, g[:20], w[:20])
    return got


def drafts(r, p, q, T, V):
    """Tokens drawn from q (p where there is none): likely to stand."""
    ids = np.zeros(T, np.int32)
    for t in range(1, T):
        row = (p[t - 1] if q is None else q[t]).astype(np.float64)
        ids[t] = r.choice(V, p=row / row.sum())
    return ids


@pytest.mark.parametrize("V,ld", [(1, 0), (2, 0), (63, 64), (4096, 0), (4097, 0), (4097, 4100), (32003, 0), (50000, 50003)])
@pytest.mark.parametrize("with_q", [True, False])
@pytest.mark.parametrize("new", [[4], [1], [1, 4, 0, 2, 7, 4, 3], [64, 65, 20]])
def test_verify_chain(G, new, with_q, V, ld):  # noqa: F811
    r = np.random.default_rng(V + sum(new) + with_q)
    cu = P.cu_of(new)
    T = sum(new)
    p = probabilities(r, T, V, 8)
    q = None
    if with_q:
        q = np.roll(p, 1, 0) * (1 + 0.3 * r.standard_normal((T, V))).clip(0.05).astype(np.float32)
        q = (q / q.sum(1, keepdims=True)).astype(np.float32)
    verify(G, p, q, drafts(r, p, q, T, V), None, r.random(T).astype(np.float32), r.random(len(new)).astype(np.float32), cu, V, ld)


@pytest.mark.parametrize("V", [5, 300, 20011])
@pytest.mark.parametrize("seed", range(4))
def test_verify_tree(G, seed, V):  # noqa: F811
    """Trees of likely drafts, among them the same token twice after one parent, parents that are none and ids outside."""
    r = np.random.default_rng(seed + V)
    new = [64, 1, 12, 0, 33]
    cu, T = P.cu_of(new), sum(new)
    p = probabilities(r, T, V, 9)
    ids, parent = np.zeros(T, np.int32), np.full(T, -1, np.int32)
    for b, n in enumerate(new):
        for t in range(1, n):
            a = parent[cu[b] + t] = int(r.integers(max(0, t - 6), t))
            ids[cu[b] + t] = np.argsort(-p[cu[b] + a])[r.integers(0, min(V, 4))]
    if seed == 3:
        parent[5], parent[7], parent[66], ids[3], ids[70] = -7, 40, 1000, V, -1
    for _ in range(5):
        verify(G, p, None, ids, parent, r.random(T).astype(np.float32), r.random(5).astype(np.float32), cu, V)


def test_verify_ends_of_the_random_numbers(G):  # noqa: F811
    """u of 0 and just below 1, outside [0, 1) and NaN; p equal to q, p below q everywhere, no weight at all, one token with
    all of it, NaN among the weights."""
    r = np.random.default_rng(16)
    V, ends = 9001, [0.0, 1 - 2.0 ** -24, 1.0, -1.0, np.nan, 0.5]
    B = 12 * len(ends)
    new = [2] * B
    cu, T = P.cu_of(new), 2 * B
    p = probabilities(r, T, V, 6)
    q = np.roll(p, 1, 0).copy()
    ids = np.zeros(T, np.int32)
    for b in range(B):
        i, k = 2 * b, b // len(ends)
        ids[i + 1] = int(p[i].argmax())
        if k == 1:
            p[i] *= np.float32(0.5)  # below q everywhere
            ids[i + 1] = int(p[i].argmin())
        elif k == 2:
            p[i:i + 2] = 0
        elif k == 3:
            p[i:i + 2] = 0
            p[i:i + 2, 8999] = 1
        elif k == 4:
            p[i:i + 2, 17] = p[i:i + 2, 8192] = np.nan
        elif k == 5:
            ids[i + 1] = [V, -1, 2 ** 31 - 1, -2 ** 31, V, -1][b % 6]
        elif k >= 6:
            q[i + 1] = r.permutation(q[i + 1])
            ids[i + 1] = r.integers(0, V)
    u = r.random(T).astype(np.float32)
    ul = np.array([ends[b % len(ends)] for b in range(B)], np.float32)
    u[1::2][:B // 2] = ul[:B // 2]
    verify(G, p, q, ids, None, u, ul, cu, V)
    verify(G, p, None, ids, None, u, ul, cu, V)


def test_verify_a_model_s_vocabulary(G):  # noqa: F811
    r = np.random.default_rng(17)
    V, new = 248320, [4, 3, 4]
    cu, T = P.cu_of(new), sum(new)
    p = probabilities(r, T, V, 11)
    q = np.roll(p, 1, 0) * (1 + 0.3 * r.standard_normal((T, V))).clip(0.05).astype(np.float32)
    q = (q / q.sum(1, keepdims=True)).astype(np.float32)
    ids = drafts(r, p, q, T, V)
    for _ in range(4):
        verify(G, p, q, ids, None, r.random(T).astype(np.float32), r.random(3).astype(np.float32), cu, V)


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("type", TYPES)
def test_a_step_of_a_batch(G, oracle, type):  # noqa: F811
    """Rows written, attended to, drafts verified and positions moved, then the next token of each sequence: in a HIP graph on a
    stream of its own, replayed with eager work between; and the rows of the accepted path read back."""
    import torch

    r = np.random.default_rng(18)
    o, dev = G.ops, G.i32(0).device
    B, nqh, nkvh, page, V, old = 3, 24, 4, 32, 1003, [200, 31, 64]
    new, room = [4, 3, 4], [8, 8, 8]
    cu, T = P.cu_of(new), sum(new)
    kp, vp, table = P.make_pages(r, old, room, page, nkvh, type)
    qg, kx, vx, qw, kw = prep_inputs(r, T, nqh, nkvh)
    p = probabilities(r, T, V, 8)
    q = np.roll(p, 1, 0)
    ids, u, ul = drafts(r, p, q, T, V), r.random(T).astype(np.float32), r.random(B).astype(np.float32)
    k0, v0 = G.up(kp.buf), G.up(vp.buf)
    kv = o.KvPages(k0.clone(), v0.clone(), G.up(table), nkvh, page, type)
    d = [G.up(x) for x in (qg, kx, vx, qw, kw, p, q, ids, u, ul)]
    pos, dcu = G.i32(*old), G.up(cu)
    qn, out, lse = G.full((T, nqh, 256), 0.0), G.full((T, nqh, 256), 0.0), G.full((T, nqh), 0.0)
    q1, o1 = G.full((B, nqh, 256), 0.0), G.full((B, nqh, 256), 0.0)
    tok, path, n_path = (torch.zeros(n, dtype=torch.int32, device=dev) for n in (T, T, B))
    back = [G.full((B, nkvh, 5, 256), 0.0) for _ in range(2)]
    start = G.i32(*old)
    ws = G.ws(max(o.attn_paged_ws_bytes(kv, T, 4, nqh), o.attn_paged_ws_bytes(kv, B, 1, nqh), o.draft_verify_ws_bytes(B, V)))

    def step():
        o.attn_prep_paged(*d[:5], qn, kv, pos, dcu, T, 1e-6, cd.THETA_SCALE, nqh)
        o.attn_paged(qn, kv, pos, dcu, T, 4, SCALE, nqh, out, ws, lse=lse)
        o.draft_verify(d[5], d[6], d[7], None, d[8], d[9], dcu, B, V, tok, path, n_path, ws, pos=pos)
        o.attn_prep_paged(*d[:5], q1, kv, pos, None, B, 1e-6, cd.THETA_SCALE, nqh)
        o.attn_paged(q1, kv, pos, None, B, 1, SCALE, nqh, o1, ws)
        o.kv_pages_read(kv, start, n_path, 5, *back)

    def reset():
        kv.k.copy_(k0), kv.v.copy_(v0), pos.copy_(start)
        for x in (qn, out, lse, q1, o1, tok, path, n_path, *back):
            x.zero_()

    def results():
        return {w: G.down(x).copy() for w, x in (("qn", qn), ("out", out), ("lse", lse), ("q1", q1), ("o1", o1), ("tok", tok), ("path", path),
                                                   ("n", n_path), ("pos", pos), ("k", kv.k), ("v", kv.v), ("bk", back[0]), ("bv", back[1]))}

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

    want = P.verify(p, q, ids, None, u, ul, cu, V, *(np.zeros(n, np.int32) for n in (T, T, B)), np.array(old, np.int32))
    for w, x in zip(("tok", "path", "n", "pos"), want):
        assert np.array_equal(eager[w], x), w
    at = eager["pos"]
    # the pages now hold the batch's rows, and behind the accepted ones the next token's
    kp.buf[:], vp.buf[:] = eager["k"], eager["v"]
    assert len(set(eager["n"])) > 1 or eager["n"][0] > 1
    eo, _, bo, _ = P.attend(eager["q1"], kp, vp, table, [int(x) for x in at], [1] * B, SCALE)
    near(eager["o1"], eo, bo, "the next token")
    for b in range(B):
        n = int(eager["n"][b])
        for x, pool in ((eager["bk"], kp), (eager["bv"], vp)):
            assert np.array_equal(x[b, :, :n], pool.values(table[b], old[b] + n)[0][:, old[b]:].astype(np.float32))
            assert np.all(x[b, :, n:] == 0)
    # the drafts' attention saw the rows before the next token took one's place: written again, they give it
    o.attn_prep_paged(*d[:5], qn, kv, start, dcu, T, 1e-6, cd.THETA_SCALE, nqh)
    kp.buf[:], vp.buf[:] = G.down(kv.k), G.down(kv.v)
    eo, el, bo, bl = P.attend(eager["qn"], kp, vp, table, old, new, SCALE)
    near(eager["out"], eo, bo, "the drafts")
    near(eager["lse"], el, bl, "the drafts' sums")


def test_a_tree_on_one_contiguous_cache(G):  # noqa: F811
    """draft_verify's path and count are kv_accept's: a tree's accepted rows move to their place."""
    r = np.random.default_rng(19)
    T, nkvh, n_ctx, pos0, V = 12, 2, 64, 20, 500
    parent = np.array([-1, 0, 0, 1, 1, 2, 3, 3, 4, 6, 6, 7], np.int32)
    p = probabilities(r, T, V, 9)
    ids = np.array([0] + [int(np.argsort(-p[a])[t % 2]) for t, a in enumerate(parent) if t], np.int32)
    u = np.full(T, 0.05, np.float32)
    cache = r.integers(0, 256, nkvh * n_ctx * 272).astype(np.uint8)
    dc, dpos, dpath, dn, dout = G.up(cache), G.i32(pos0), G.i32(*[0] * T), G.i32(0), G.i32(*[0] * T)
    G.ops.draft_verify(G.up(p), None, G.up(ids), G.up(parent), G.up(u), G.up(np.array([0.3], np.float32)), G.i32(0, T), 1, V, dout, dpath,
                       dn, G.ws(G.ops.draft_verify_ws_bytes(1, V)))
    G.ops.kv_accept([dc], [], dpos, dpath, dn, T, nkvh, n_ctx, True)
    path, n = G.down(dpath), int(G.down(dn)[0])
    assert n > 2 and list(path[:n]) != list(range(n))  # a branch was taken
    rows = lambda x: np.concatenate([x[:nkvh * n_ctx * 256].reshape(nkvh, n_ctx, 256), x[nkvh * n_ctx * 256:].reshape(nkvh, n_ctx, 16)], 2)  # noqa: E731
    want = rows(cache).copy()
    want[:, pos0:pos0 + n] = rows(cache)[:, pos0 + path[:n]]
    assert np.array_equal(rows(G.down(dc)), want)
