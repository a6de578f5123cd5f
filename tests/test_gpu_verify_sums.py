"""Draws of draft_verify whose weights sum far past 1 on the GPU, against whole numbers of any size (no rounding anywhere): where
the row is a pattern over and over and u a whole number of its parts, u times the sum lies on a border between two tokens."""
from fractions import Fraction

import numpy as np
import pytest

import pagedref as P
from test_gpu_attn import G  # noqa: F401

pytestmark = pytest.mark.gpu


def pick(w, u):
    """Least index whose sum of the whole numbers w up to it exceeds u times the sum of all; -1 where that is 0."""
    total = sum(int(x) for x in w)
    if total == 0:
        return -1
    want, at = Fraction(float(np.float32(u))) * total, 0
    for i, x in enumerate(w):
        at += int(x)
        if at > want:
            return i


def draw(G, p, u, q=None, ids=None):  # noqa: F811
    """out of draft_verify for sequences of one token (with q: two, the second of which u of 1 - 2^-24 refuses), p and q [..][V]."""
    B, V = len(u), p.shape[-1]
    each = 1 if ids is None else 2
    T = B * each
    cu = G.up(np.arange(0, T + 1, each, dtype=np.int32))
    out, path, n_path = G.i32(*[7] * T), G.i32(*[7] * T), G.i32(*[7] * B)
    G.ops.draft_verify(G.up(p), None if q is None else G.up(q), G.i32(*[0] * T) if ids is None else G.up(ids), None,
                       G.full((T,), 1 - 2.0 ** -24), G.up(np.asarray(u, np.float32)), cu, B, V, out, path, n_path,
                       G.ws(G.ops.draft_verify_ws_bytes(B, V)))
    assert np.all(G.down(n_path) == 1)
    return G.down(out)[::each]


@pytest.mark.parametrize("part,parts", [(4096, 8), (5001, 16), (12289, 4), (31040, 8), (124160, 2)])
@pytest.mark.parametrize("kind", ["uniform", "ones and little"])
def test_borders_of_large_sums(G, kind, part, parts):  # noqa: F811
    r = np.random.default_rng(part + parts)
    B = 24
    if kind == "uniform":
        one = r.random((B, part)).astype(np.float32)
    else:
        one = np.where(r.random((B, part)) < 0.9, 1, r.integers(1, 2 ** 20, (B, part)) * 2.0 ** -40).astype(np.float32)
    u = (1 + np.arange(B) % (parts - 1)).astype(np.float32) / parts
    got = draw(G, np.tile(one, (1, parts)), u)
    # the sum up to the end of part i is i / parts of the whole, and not above it: the token is the next part's first one
    assert np.all(one[:, 0] > 0)
    assert np.array_equal(got, (1 + np.arange(B) % (parts - 1)) * part), (got, part)


@pytest.mark.parametrize("V", [4096, 9001, 40000])
def test_any_random_numbers(G, V):  # noqa: F811
    r = np.random.default_rng(V)
    B = 6
    p = np.where(r.random((B, V)) < 0.5, r.random((B, V)) * 3, r.random((B, V)) * 2.0 ** -30).astype(np.float32)
    u = np.array([0, 2.0 ** -40, 2.0 ** -149, 0.3, 0.9999, 1 - 2.0 ** -24], np.float32)
    assert list(draw(G, p, u)) == [pick(P.weights(p[b].astype(np.float64)), u[b]) for b in range(B)]


def test_large_sums_of_differences(G):  # noqa: F811
    """A refused draft: weights of max(p - q, 0), a pattern of 5001 values eight times."""
    r = np.random.default_rng(5)
    B, part, parts = 14, 5001, 8
    one = r.random((B, part)).astype(np.float32)
    p = np.repeat(np.tile(one, (1, parts)), 2, 0)
    q = np.repeat(np.tile((one * r.random((B, part))).astype(np.float32), (1, parts)), 2, 0)
    p[:, 17], q[:, 17] = 0, 1  # the draft, which is refused
    ids = np.full(2 * B, 17, np.int32)
    u = (r.integers(1, parts, B) / parts).astype(np.float32)
    got = draw(G, p, u, q, ids)
    assert list(got) == [pick(P.weights(p[2 * b].astype(np.float64) - q[2 * b + 1]), u[b]) for b in range(B)]


@pytest.mark.parametrize("weight", [1.0, 0.75, 2.0 ** -40])
def test_the_largest_vocabulary(G, weight):  # noqa: F811
    """2^24 tokens of one weight: the token is the whole part of u 2^24, also where the sum is 2^64 times 2^-40."""
    V = 1 << 24
    for u in (0.0, 0.5, 1 - 2.0 ** -24, 2.0 ** -24, 0.3):
        assert draw(G, np.full((1, V), weight, np.float32), [u])[0] == int(float(np.float32(u)) * V), u
