"""attn_paged where the plan of its parts changes with the total of all rows: over codes, many units of more than 16 query rows have
parts of half their share (512 to the whole), but none under 32 tiles of 32 rows; shorter shares stay whole. Sequences of four
kinds share their kind's pages, which nothing writes, and its queries, so the plain 64-bit form is taken four times alone."""
import numpy as np
import pytest

import pagedref as P
from conftest import assert_bits_equal
from test_gpu_attn import G, SCALE, near  # noqa: F401
from test_gpu_paged import handle

pytestmark = pytest.mark.gpu
POS, NEW, NQH, NKVH = [12990, 8000, 700, 5001], [3, 2, 1, 3], 12, 2


@pytest.fixture(scope="module", params=[P.Q8, P.Q8_Q4])
def kinds(request):
    r = np.random.default_rng(51)
    kp, vp, table = P.make_pages(r, POS, NEW, 128, NKVH, request.param)
    q = (r.standard_normal((sum(NEW), NQH, 256)) * 1.5).astype(np.float32)
    return request.param, kp, vp, table, q, P.attend(q, kp, vp, table, POS, NEW, SCALE)


# sequences of each kind, and the share of a slot in tiles: halved; halved to the least; as it is (80 sequences and more are laid
# out by the workgroup's waves together)
@pytest.mark.parametrize("counts,share", [([28, 12, 12, 12], 66), ([10, 12, 20, 22], 44), ([2, 2, 55, 5], 14), ([30, 40, 40, 40], 116),
                                          ([8, 8, 34, 30], 43)])
def test_parts_of_half_a_share(G, kinds, counts, share):  # noqa: F811
    import torch

    type, kp, vp, table, q, (eo, el, bo, bl) = kinds
    tiles = [-(-(p + n) // 32) for p, n in zip(POS, NEW)]
    assert -(-sum(c * NKVH * (-(-t // 4) * 4) for c, t in zip(counts, tiles)) // 512) == share
    of = np.random.default_rng(sum(counts)).permutation(np.repeat(np.arange(4), counts))
    first = P.cu_of(NEW)
    at = np.concatenate([np.arange(first[k], first[k + 1]) for k in of])  # each token's row of q and of the plain form
    new = [NEW[k] for k in of]
    T, kv, guard = len(at), handle(G, kp, vp, table[of], type), 4096
    need = G.ops.attn_paged_ws_bytes(kv, T, 3, NQH)
    ws = G.full((need + guard,), 0xFF, torch.uint8)
    o, lse = G.full((T + 9, NQH, 256), 7.0), G.full((T + 9, NQH), 7.0)
    G.ops.attn_paged(G.up(q[at]), kv, G.i32(*(POS[k] for k in of)), G.up(P.cu_of(new)), T, 3, SCALE, NQH, o[:T], ws[:need], lse=lse[:T])
    o, lse = G.down(o), G.down(lse)
    assert np.all(G.down(ws[need:]) == 0xFF) and np.all(o[T:] == 7) and np.all(lse[T:] == 7)
    near(o[:T], eo[at], bo[at], "o")
    near(lse[:T], el[at], bl[at], "lse")
    for row in range(sum(NEW)):  # sequences of a kind are cut alike
        same = np.nonzero(at == row)[0]
        assert_bits_equal(o[same], np.repeat(o[same[:1]], len(same), 0), "o")
        assert_bits_equal(lse[same], np.repeat(lse[same[:1]], len(same), 0), "lse")
