"""Attention over a K/V cache in pages on the GPU where it can go wrong and tests/test_gpu_paged.py does not look, against a plain
64-bit form with the bounds of tests/test_gpu_attn_edges.py: query values far below their row's largest, V rows of very
different size, scales of 0, more and fewer sequences than a wave has lanes, long sequences, calls at the same time, and what
lies behind a workspace."""
import numpy as np
import pytest

import attnref as R
import pagedref as P
from conftest import assert_bits_equal
from test_gpu_attn import G, SCALE, near  # noqa: F401
from test_gpu_attn_edges import attend
from test_gpu_paged import TYPES, attn, handle

pytestmark = pytest.mark.gpu


def pages_of(r, k, v, page, type):
    """Pools and table of one sequence with the values k, v [nkvh][n][256], as attn_prep_paged stores them."""
    nkvh, n, _ = k.shape
    need = -(-n // page)
    table = r.permutation(need + 1)[None, :need].astype(np.int32)
    pools = []
    for x, is_v in ((k, False), (v, True)):
        pool = P.Pool(need + 1, nkvh, page, P.bits_of(type, is_v), 0xFF)
        codes, scales = P.row_parts(x.astype(np.float32), pool.bits)
        for j in range(n):
            pool.put(table[0, j // page], j % page, codes[:, j], None if scales is None else scales[:, j])
        pools.append(pool)
    return pools[0], pools[1], table


def check(G, r, q, k, v, T, type, page=64):  # noqa: F811
    n = k.shape[1]
    kp, vp, table = pages_of(r, k, v, page, type)
    o, lse = attn(G, G.up(q), handle(G, kp, vp, table, type), G.i32(n - T), G.i32(0, T), T, q.shape[1])
    k64, v64 = kp.values(table[0], n)[0], vp.values(table[0], n)[0]
    eo, el, bo, bl = attend(q, k64, v64, R.visible(T, n - T, n, None), type != P.F16)
    near(G.down(o), eo, bo, "o")
    near(G.down(lse), el, bl, "lse")


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("T", [1, 4, 8])
def test_query_values_far_below_the_largest(G, T, type):  # noqa: F811
    """One value of q is 2^22 times the others, where K is small; the scores come from the others, where K is large."""
    r = np.random.default_rng(23)
    n, nqh, nkvh = 100 + T, 24, 4
    k, v = r.standard_normal((nkvh, n, 256)) * 1000, r.standard_normal((nkvh, n, 256))
    k[:, :, :32] *= 2.0 ** -20
    q = (r.standard_normal((T, nqh, 256)) * 2.0 ** -18).astype(np.float32)
    q[:, :, 0] = 16
    check(G, r, q, k, v, T, type)


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("where", ["first tile", "own rows"])
@pytest.mark.parametrize("T", [1, 3, 5, 9])
def test_a_large_row_of_little_weight(G, T, where, type):  # noqa: F811
    """A V row 2^26 (f16: 2^20) times as large as the others with 2^-69 of their weight gives next to nothing, and the others
    keep their precision."""
    r = np.random.default_rng(17)
    n, nqh, nkvh = 170 + T, 24, 4
    j = 3 if where == "first tile" else n - T
    k, v = r.standard_normal((nkvh, n, 256)), r.standard_normal((nkvh, n, 256)) * 2.0 ** -9
    k[:, :, :32] = 0
    k[:, j, 0] = -16  # times 48 and the scale: a score of -48
    v[:, j] *= 2.0 ** (20 if type == P.F16 else 24)
    q = r.standard_normal((T, nqh, 256)).astype(np.float32)
    q[:, :, 0] = 48
    check(G, r, q, k, v, T, type, 32)


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("T", [1, 4])
def test_a_large_row_whose_weight_shrinks(G, T, type):  # noqa: F811
    """The scores rise by 60 over the rows, and the first rows' values are the largest: whatever reference they were summed
    with, the last rows, which have all the weight, keep their precision."""
    r = np.random.default_rng(29)
    nkvh, n = 4, 1000 + T
    k, v = r.standard_normal((nkvh, n, 256)), r.standard_normal((nkvh, n, 256))
    k[:, :, :32] = 0
    at = np.arange(n) / n
    k[:, :, 0] = 16 * at
    v *= (2.0 ** np.where(at < 0.1, 8, -10))[:, None]
    q = r.standard_normal((T, 24, 256)).astype(np.float32)
    q[:, :, 0] = 60
    check(G, r, q, k, v, T, type)


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("T", [1, 4])
@pytest.mark.parametrize("zero", ["k", "v", "some v", "q", "all"])
def test_zeros(G, zero, T, type):  # noqa: F811
    """Rows, or blocks, whose scales are 0, and queries that are."""
    r = np.random.default_rng(31)
    nkvh, n = 2, 200 + T
    k, v = r.standard_normal((nkvh, n, 256)), r.standard_normal((nkvh, n, 256))
    q = r.standard_normal((T, 12, 256)).astype(np.float32)
    if zero in ("k", "all"):
        k[:] = 0
    if zero in ("v", "all"):
        v[:] = 0
    if zero == "some v":
        v[:, ::3] = 0
        v[:, :, 64:96] = 0
        v[:, 40:80] *= 2.0 ** -12
    if zero in ("q", "all"):
        q[:] = 0
    check(G, r, q, k, v, T, type)


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("T", [1, 4])
def test_very_unequal_scores(G, T, type):  # noqa: F811
    """Scores from -3000 to 3000: all the weight on one row, wherever it lies."""
    r = np.random.default_rng(33)
    nkvh, n = 4, 300 + T
    k, v = r.standard_normal((nkvh, n, 256)) * 50, r.standard_normal((nkvh, n, 256))
    q = (r.standard_normal((T, 24, 256)) * 60).astype(np.float32)
    check(G, r, q, k, v, T, type)


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("T", [1, 3])
def test_a_long_sequence(G, T, type):  # noqa: F811
    r = np.random.default_rng(35)
    pos, new = [20011, 5, 700], [T, 1, T]
    kp, vp, table = P.make_pages(r, pos, new, 512, 1, type)
    q = r.standard_normal((sum(new), 8, 256)).astype(np.float32)
    o, lse = attn(G, G.up(q), handle(G, kp, vp, table, type), G.i32(*pos), G.up(P.cu_of(new)), T, 8)
    eo, el, bo, bl = P.attend(q, kp, vp, table, pos, new, SCALE)
    near(G.down(o), eo, bo, "o")
    near(G.down(lse), el, bl, "lse")


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("n", [63, 64, 256])
def test_sequences_without_tokens_change_no_bit(G, n, type):  # noqa: F811
    """The plan of up to 64 sequences, of more, and of several to a thread: the same parts, and the same bits, where sequences
    without tokens make the difference."""
    r = np.random.default_rng(37)
    pos = [int(x) for x in np.exp(r.uniform(0, 7, n))]
    new = [int(x) for x in r.integers(0, 4, n)]
    new[5] = 3
    kp, vp, table = P.make_pages(r, pos, new, 64, 2, type)
    q = G.up(r.standard_normal((sum(new), 12, 256)).astype(np.float32))
    first = [G.down(x).copy() for x in attn(G, q, handle(G, kp, vp, table, type), G.i32(*pos), G.up(P.cu_of(new)), 3, 12)]
    for more in (1, 70, 700):
        at = np.sort(r.integers(0, n + 1, more))
        pos2, new2 = (np.insert(np.array(x), at, y) for x, y in ((pos, 9), (new, 0)))
        table2 = np.insert(table, at, -1, axis=0)
        got = attn(G, q, handle(G, kp, vp, table2, type), G.i32(*(int(x) for x in pos2)), G.up(P.cu_of(new2)), 3, 12)
        for a, b in zip(first, got):
            assert_bits_equal(G.down(b), a, f"{more} more")


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("T", [1, 4])
def test_calls_at_the_same_time(G, T, type):  # noqa: F811
    """Two streams, a workspace each."""
    import torch

    r = np.random.default_rng(39)
    pos, new = [3000, 77, 1200], [T] * 3
    kp, vp, table = P.make_pages(r, pos, new, 64, 4, type)
    kv, dpos, cu = handle(G, kp, vp, table, type), G.i32(*pos), G.up(P.cu_of(new))
    qs = [G.up(r.standard_normal((3 * T, 24, 256)).astype(np.float32)) for _ in range(2)]
    want = [[G.down(x).copy() for x in attn(G, q, kv, dpos, cu, T, 24)] for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [(G.full((3 * T, 24, 256), 0.0), G.full((3 * T, 24), 0.0), G.ws(G.ops.attn_paged_ws_bytes(kv, 3 * T, T, 24))) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, q, (o, lse, ws) in zip(streams, qs, outs):
            with torch.cuda.stream(s):
                G.ops.attn_paged(q, kv, dpos, cu, 3 * T, T, SCALE, 24, o, ws, lse=lse)
    torch.cuda.synchronize()
    for (o, lse, _), w in zip(outs, want):
        assert_bits_equal(G.down(o), w[0], "o")
        assert_bits_equal(G.down(lse), w[1], "lse")


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("n_seqs,T,nqh,nkvh", [(1, 1, 24, 4), (1, 5, 24, 4), (300, 1, 6, 1), (3, 64, 24, 4), (40, 4, 24, 4)])
def test_nothing_behind_the_workspace_is_written(G, n_seqs, T, nqh, nkvh, type):  # noqa: F811
    import torch

    r = np.random.default_rng(41)
    pos, new = [int(x) for x in np.exp(r.uniform(0, 8 if n_seqs < 10 else 6, n_seqs))], [T] * n_seqs
    kp, vp, table = P.make_pages(r, pos, new, 64, nkvh, type)
    kv, total = handle(G, kp, vp, table, type), n_seqs * T
    need = G.ops.attn_paged_ws_bytes(kv, total, T, nqh)
    ws = G.full((need + 4096,), 0x5A, torch.uint8)
    o = G.full((total, nqh, 256), 0.0)
    G.ops.attn_paged(G.up(r.standard_normal((total, nqh, 256)).astype(np.float32)), kv, G.i32(*pos), G.up(P.cu_of(new)), total, T, SCALE,
                     nqh, o, ws[:need])
    assert np.isfinite(G.down(o)).all() and np.all(G.down(ws[need:]) == 0x5A)
    V = 9000
    need = G.ops.draft_verify_ws_bytes(n_seqs, V)
    ws = G.full((need + 4096,), 0x5A, torch.uint8)
    p = torch.softmax(torch.randn(total, V, device=o.device), -1)
    ids, u = G.full((total,), 3, torch.int32), G.full((total,), 0.5)
    out, path, n_path = (G.full((x,), 0, torch.int32) for x in (total, total, n_seqs))
    G.ops.draft_verify(p, None, ids, None, u, G.full((n_seqs,), 0.25), G.up(P.cu_of(new)), n_seqs, V, out, path, n_path, ws[:need])
    assert np.all(G.down(ws[need:]) == 0x5A) and (G.down(n_path) >= 1).all()


@pytest.mark.parametrize("type", TYPES)
def test_attn_before_and_behind_all_positions(G, type):  # noqa: F811
    """Positions at the ends of 32 bits: nothing is read or written outside; a sequence far past its table sees all of it."""
    r = np.random.default_rng(43)
    n = 128
    kp, vp, table = P.make_pages(r, [n - 2, n - 2, n - 2], [2, 2, 2], 64, 4, type, extra=0)
    kv = handle(G, kp, vp, table, type)
    q = r.standard_normal((6, 24, 256)).astype(np.float32)
    o, lse = attn(G, G.up(q), kv, G.i32(2 ** 31 - 1, -2 ** 31, n), G.up(P.cu_of([2, 2, 2])), 2, 24)
    eo, el, bo, bl = P.attend(q, kp, vp, table, [n, n, n], [2, 2, 2], SCALE)
    near(G.down(o)[[0, 1, 4, 5]], eo[[0, 1, 4, 5]], bo[[0, 1, 4, 5]], "o")
    assert np.all(G.down(o)[2:4] == 0) and np.all(G.down(lse)[2:4] == -np.inf)
    G.ops.attn_prep_paged(G.up(r.standard_normal((6, 24, 512)).astype(np.float32)), *(G.full((6, 4, 256), 1.0) for _ in range(2)),
                          *(G.full((256,), 1.0) for _ in range(2)), G.full((6, 24, 256), 0.0), kv, G.i32(2 ** 31 - 1, -2 ** 31, n),
                          G.up(P.cu_of([2, 2, 2])), 6, 1e-6, 0.6, 24)
    assert np.array_equal(G.down(kv.k), kp.buf) and np.array_equal(G.down(kv.v), vp.buf)
    back = [G.full((3, 4, 40, 256), 7.0) for _ in range(2)]
    G.ops.kv_pages_read(kv, G.i32(2 ** 31 - 1, -2 ** 31, n - 20), G.i32(40, 40, 2 ** 31 - 1), 40, *back)
    for x, pool in zip(back, (kp, vp)):
        x = G.down(x)
        assert np.all(x[:2] == 0) and np.all(x[2, :, 20:] == 0)
        assert np.array_equal(x[2, :, :20], pool.values(table[2], n)[0][:, n - 20:].astype(np.float32))
