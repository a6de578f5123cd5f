"""attn_paged with many query rows a kv head on the GPU, where a unit's size changes, within the bounds of tests/attnref.py."""
import numpy as np
import pytest

import pagedref as P
from test_gpu_attn import G, SCALE, near  # noqa: F401
from test_gpu_paged import TYPES, attn, check, handle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("most", [5, 6, 8, 10, 11, 20, 22, 43])  # 30 to 258 query rows of 24 heads over 4
def test_sizes_of_units(G, most, type):  # noqa: F811
    r = np.random.default_rng(most)
    pos, new = [2500, 0, 63, 31, 300], [most, most, 1, 0, max(1, most - 3)]
    kp, vp, table = P.make_pages(r, pos, new, 32, 4, type)
    q = (r.standard_normal((sum(new), 24, 256)) * 1.5).astype(np.float32)
    check(G, q, kp, vp, table, type, pos, new, most, 24)


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("most", [7, 12, 40])
def test_more_sequences_than_a_wave_has_lanes(G, most, type):  # noqa: F811
    r = np.random.default_rng(most)
    n = 70
    pos = [int(x) for x in r.integers(0, 90, n - 1)] + [1500]
    new = [int(x) for x in r.integers(0, 4, n - 1)] + [most]
    kp, vp, table = P.make_pages(r, pos, new, 64, 2, type)
    q = (r.standard_normal((sum(new), 12, 256)) * 1.5).astype(np.float32)
    check(G, q, kp, vp, table, type, pos, new, most, 12)


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("most", [7, 12, 25])
def test_pages_that_are_none(G, most, type):  # noqa: F811
    """Before, among and behind others; a sequence of none at all; tokens past the table's end."""
    r = np.random.default_rng(most)
    pos, new = [900, 150, 70, 1021, 20], [most, 1, most, 3, most]
    holes = [(0, 0), (0, 7), (0, 8), (0, 9), (0, 28), (1, 1), (2, 2), (3, 3), (3, 30), (4, 0), (4, 1)]
    kp, vp, table = P.make_pages(r, pos, new, 32, 4, type, holes=holes, extra=0)
    assert table.shape[1] == 32
    pos[3] = 1022
    q = r.standard_normal((sum(new), 24, 256)).astype(np.float32)
    check(G, q, kp, vp, table, type, pos, new, most, 24)


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("most", [7, 12, 25])
def test_values_that_are_not_finite(G, most, type, bad):  # noqa: F811
    """V rows that hold one: a row that all tokens see, rows of the drafts' own; they reach the tokens that see them alone."""
    r = np.random.default_rng(10)
    pos, new = [170, 40], [most, 2]
    kp, vp, table = P.make_pages(r, pos, new, 32, 2, type)
    for row, dim in ((3, 17), (171, 66), (170 + most - 1, 200)):
        p, j = table[0, row // 32], row % 32
        if type == P.F16:
            vp.codes[p, 1, j].view(np.float16)[dim] = bad
        else:
            vp.scales[p, 1, j].view(np.float16)[dim // 32] = bad
            vp.codes[p, 1, j] = 0x22 if type == P.Q8_Q4 else 5
    q = r.standard_normal((sum(new), 12, 256)).astype(np.float32)
    o = G.down(attn(G, G.up(q), handle(G, kp, vp, table, type), G.i32(*pos), G.up(P.cu_of(new)), most, 12)[0])
    with np.errstate(invalid="ignore"):
        eo, _, bo, _ = P.attend(q, kp, vp, table, pos, new, SCALE)
    fine = np.isfinite(eo)
    assert np.array_equal(np.isfinite(o), fine)
    assert fine[0, 6:, 66].all() and not fine[1, 6:, 66].any() and fine[most - 2, 6:, 200].all() and not fine[most - 1, 6:, 200].any()
    assert fine[most:].all() and fine[:, :6].all()
    near(o[fine], eo[fine], bo[fine], "o")


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("most", [7, 12, 64])
def test_nothing_behind_the_workspace_is_written(G, most, type):  # noqa: F811
    """Many equal sequences, and one long one: as many parts as there can be."""
    import torch

    r = np.random.default_rng(most)
    for pos in ([40] * 90, [9000]):
        new = [most] * len(pos)
        kp, vp, table = P.make_pages(r, pos, new, 64, 1, type)
        kv, T = handle(G, kp, vp, table, type), sum(new)
        n = G.ops.attn_paged_ws_bytes(kv, T, most, 6)
        ws = torch.full((n + 4096,), 0xA5, dtype=torch.uint8, device=G.i32(0).device)
        q = r.standard_normal((T, 6, 256)).astype(np.float32)
        o, lse = G.full((T, 6, 256), 7.0), G.full((T, 6), 7.0)
        G.ops.attn_paged(G.up(q), kv, G.i32(*pos), G.up(P.cu_of(new)), T, most, SCALE, 6, o, ws[:n], lse=lse)
        assert (G.down(ws[n:]) == 0xA5).all()
        if len(pos) == 1 and most < 64:
            check(G, q, kp, vp, table, type, pos, new, most, 6, got=(o, lse))


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("most", [1, 4, 12])
def test_a_captured_call_follows_the_lengths(G, most, type):  # noqa: F811
    """Captured at short lengths, replayed as lengths, tokens and the table change: the eager call's bits each time."""
    import torch

    r = np.random.default_rng(most)
    nqh, nkvh, B = 24, 4, 5
    kp, vp, table = P.make_pages(r, [6000, 700, 64, 31, 3000], [most] * B, 64, nkvh, type)
    kv = handle(G, kp, vp, table, type)
    T = B * most
    q = G.up(r.standard_normal((T, nqh, 256)).astype(np.float32))
    pos, cu = G.i32(*[3] * B), G.up(P.cu_of([1] * B))
    ws = G.ws(G.ops.attn_paged_ws_bytes(kv, T, most, nqh))
    out = [G.full((T, nqh, 256), 7.0), G.full((T, nqh), 7.0)]

    def call():
        G.ops.attn_paged(q, kv, pos, cu, T, most, SCALE, nqh, out[0], ws, lse=out[1])

    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    steps = [([6000, 700, 64, 31, 3000], [most] * B, None), ([0, 699, 2, 30, 1000], [1, 0, most, most, 0], None),
             ([5000, 0, 0, 0, 0], [0, most, 1, 0, 0], None), ([700, 6000, 31, 64, 3000], [most] * B, [1, 0, 3, 2, 4])]
    for at, new, order in steps:
        pos.copy_(G.i32(*at)), cu.copy_(G.up(P.cu_of(new)))
        kv.table.copy_(G.up(table if order is None else table[order]))
        got = []
        for run in (call, g.replay):
            for x in out:
                x.fill_(7.0)
            run()
            got.append([G.down(x).copy() for x in out])
        for a, b in zip(*got):
            assert np.array_equal(a.view(np.uint8), b.view(np.uint8))
        assert np.isfinite(got[1][0]).all()
