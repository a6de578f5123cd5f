"""The plain forms of tests/pagedref.py against their definitions in other words (no GPU needed)."""
from fractions import Fraction

import numpy as np
import pytest

import pagedref as P


def test_four_bits():
    r = np.random.default_rng(1)
    x = r.standard_normal((5, 256)).astype(np.float32)
    x[1, :32] = 0
    x[2, 0], x[2, 1] = 9, -9
    c, s = P.row_parts(x, 4)
    y = P.row_values(c, s, 4)
    d = np.abs(s.view(np.float16).astype(np.float64)).repeat(32, -1)
    # codes 0 .. 15: half a step off, and a whole one at the end that 15 stands for
    assert np.all(np.abs(y - x) <= d * (1 + 2.0 ** -10) + 8 * d * 2.0 ** -11)
    assert np.all(np.abs(y - x)[np.abs(x) < 6.5 * d] <= (0.5 + 2.0 ** -6) * d[np.abs(x) < 6.5 * d])
    assert np.all(y[1, :32] == 0) and y[2, 1] == -9 and abs(y[2, 0] - 9 * 7 / 8) < 1e-2
    big = np.abs(x.reshape(5, 8, 32)).argmax(-1)  # the largest comes back but for its scale's rounding
    for i in (0, 3, 4):
        for b in range(8):
            k = 32 * b + big[i, b]
            assert abs(y[i, k] - x[i, k]) <= abs(x[i, k]) * 2.0 ** -11


def test_pick_is_the_inverse_of_the_sums():
    w = P.weights(np.array([0.25, 0.0, 0.5, 0.0, 0.25, 0.0]))
    for u, want in ((0, 0), (0.2499, 0), (0.25, 2), (0.74, 2), (0.75, 4), (1.0, 4), (2.0, 4), (np.nan, 0), (-1, 0)):
        assert P.pick(w, np.float32(u)) == want, u
    assert P.pick(w * 0, np.float32(0.5)) == -1
    x = np.random.default_rng(2).random(1000) * 1e-3
    assert all(int(a) == round(Fraction(float(b)) * 2 ** 40) for a, b in zip(P.weights(x), x))


def laws(q, tree):
    """(drawn tokens' frequencies, the target's) of the token behind the root, over many verifications."""
    r = np.random.default_rng(7)
    V, n = 5, 15000
    p = r.dirichlet(np.ones(V), 4).astype(np.float32)
    qq = r.dirichlet(np.ones(V), 4).astype(np.float32)
    seen = np.zeros(V)
    for _ in range(n):
        if tree:  # two different drafts after the root, one behind the first
            ids, parent = np.array([0, 1, 3, 2]), np.array([-1, 0, 0, 1])
        else:
            ids, parent = np.array([0] + [r.choice(V, p=qq[t] / qq[t].sum()) for t in (1, 2, 3)]), None
        u, ul = r.random(4).astype(np.float32), r.random(1).astype(np.float32)
        out, path, m, pos = P.verify(p, qq if q else None, ids, parent, u, ul, np.array([0, 4]), V, np.zeros(4, int), np.zeros(4, int),
                                     np.zeros(1, int), np.array([10]))
        assert pos[0] == 10 + m[0] and (path >= 0).sum() == m[0] and (out >= 0).sum() == m[0]
        seen[out[0]] += 1
    return seen / n, p[0].astype(np.float64)


@pytest.mark.parametrize("q,tree", [(True, False), (False, True)])
def test_verified_tokens_have_the_target_s_distribution(q, tree):
    got, want = laws(q, tree)
    # five standard deviations of a frequency of 15000 draws
    assert np.all(np.abs(got - want) < 5 * np.sqrt(want * (1 - want) / 15000))
