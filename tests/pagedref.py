"""Plain 64-bit forms (numpy) of the operators over a K/V cache in pages and of the verification of drafts, from their
definitions; attention itself, with its error bounds, is tests/attnref.py's."""
import numpy as np

import attnref as R

HD = 256
F16, Q8, Q8_Q4 = 0, 1, 2


def bits_of(type, v):
    return 16 if type == F16 else 4 if v and type == Q8_Q4 else 8


def row_parts(x, bits):
    """Bytes of the codes and of the scales of rows x [.., 256] in float32, as they are stored."""
    x = np.asarray(x, np.float32)
    if bits == 16:
        return x.astype(np.float16).view(np.uint8), None
    b = x.reshape(*x.shape[:-1], 8, 32)
    with np.errstate(all="ignore"):
        if bits == 8:
            d = np.abs(b).max(-1, keepdims=True) / np.float32(127)
            inv = np.where(d != 0, np.float32(1) / d, np.float32(0))
            y = b * inv
            c = (np.sign(y) * np.floor(np.abs(y.astype(np.float64)) + 0.5)).astype(np.int8).reshape(x.shape).view(np.uint8)
        else:
            lo, hi = b.min(-1, keepdims=True), b.max(-1, keepdims=True)
            d = np.where(-lo >= hi, lo, hi) / np.float32(-8)
            inv = np.where(d != 0, np.float32(1) / d, np.float32(0))
            u = np.clip(np.trunc(b * inv + np.float32(8.5)), 0, 15).astype(np.uint8)
            c = (u[..., :16] | (u[..., 16:] << 4)).reshape(*x.shape[:-1], 128)
    return c, d[..., 0].astype(np.float16).view(np.uint8)


def row_values(codes, scales, bits):
    """Values [.., 256] in 64 bits of stored rows."""
    if bits == 16:
        return np.ascontiguousarray(codes).view(np.float16).astype(np.float64)
    d = np.ascontiguousarray(scales).view(np.float16).astype(np.float64)[..., None]
    if bits == 8:
        c = np.ascontiguousarray(codes).view(np.int8).astype(np.float64).reshape(*codes.shape[:-1], 8, 32)
    else:
        c = codes.reshape(*codes.shape[:-1], 8, 16)
        c = np.concatenate([c & 15, c >> 4], -1).astype(np.float64) - 8
    with np.errstate(invalid="ignore"):
        return (c * d).reshape(*codes.shape[:-1], 256)


class Pool:
    """Pages of K or V on the host: the bytes, and views of their codes and scales."""

    def __init__(self, n_pages, nkvh, page, bits, fill):
        self.bits, self.nkvh, self.page = bits, nkvh, page
        self.cb = HD * bits // 8
        self.buf = np.full((n_pages, nkvh * page * (self.cb + (0 if bits == 16 else 16))), fill, np.uint8)
        m = nkvh * page * self.cb
        self.codes = self.buf[:, :m].reshape(n_pages, nkvh, page, self.cb)
        self.scales = None if bits == 16 else self.buf[:, m:].reshape(n_pages, nkvh, page, 16)

    def put(self, page, row, codes, scales):  # codes [nkvh][..]
        self.codes[page, :, row] = codes
        if scales is not None:
            self.scales[page, :, row] = scales

    def values(self, table, n):
        """[nkvh][n][256] of a sequence's rows, and which exist."""
        out, there = np.zeros((self.nkvh, n, HD)), np.zeros(n, bool)
        for j in range(n):
            p = int(table[j // self.page]) if j // self.page < len(table) else -1
            if 0 <= p < len(self.buf):
                there[j] = True
                s = None if self.scales is None else self.scales[p, :, j % self.page]
                out[:, j] = row_values(self.codes[p, :, j % self.page], s, self.bits)
        return out, there


def make_pages(r, pos, new, page, nkvh, type, std=1.0, holes=(), extra=1):
    """K and V pools and the table of sequences with pos[b] + new[b] rows of random values, their pages in no order. What
    nobody may read is NaN: every page's other rows, and the pages of no sequence. holes: (sequence, page) without a page."""
    end = [max(0, p + n) for p, n in zip(pos, new)]
    need = [-(-n // page) for n in end]
    n_pages, most = sum(need) + 2, max(max(need), 1) + extra
    order = list(r.permutation(n_pages))
    table = np.full((len(pos), most), -1, np.int32)
    pools = []
    for v in (False, True):
        bits = bits_of(type, v)
        pools.append(Pool(n_pages, nkvh, page, bits, 0xFF))  # f16 0xFFFF: NaN
    for b, n in enumerate(need):
        for i in range(n):
            table[b, i] = order.pop()
            rows = min(page, end[b] - i * page)
            for pool in pools:
                if pool.bits == 16:
                    c, s = (r.standard_normal((nkvh, rows, HD)) * std).astype(np.float16).view(np.uint8), None
                else:
                    c = r.integers(0, 256, (nkvh, rows, pool.cb)).astype(np.uint8)
                    if pool.bits == 8:
                        c = np.where(c == 128, 0, c).astype(np.uint8)
                    s = (r.uniform(0.2, 1.8, (nkvh, rows, 8)) * std / (73 if pool.bits == 8 else 4.6)).astype(np.float16)
                    if pool.bits == 4:
                        s = np.where(r.random(s.shape) < 0.5, s, -s)
                    s = np.ascontiguousarray(s).view(np.uint8)
                pool.codes[table[b, i], :, :rows] = c
                if s is not None:
                    pool.scales[table[b, i], :, :rows] = s
    for b, i in holes:
        table[b, i] = -1 if (b + i) % 2 else n_pages
    return pools[0], pools[1], table


def cu_of(new):
    return np.concatenate([[0], np.cumsum(new)]).astype(np.int32)


def attend(q, kp, vp, table, pos, new, scale, tree=None):
    """o, lse and their bounds for all tokens of the batch (R.attend's for each sequence); tree: a mask for each token."""
    parts = []
    cu = cu_of(new)
    for b, n in enumerate(new):
        if not n:
            continue
        end = max(0, min(pos[b] + n, table.shape[1] * kp.page))
        k, there = kp.values(table[b], end)
        v, _ = vp.values(table[b], end)
        vis = R.visible(n, pos[b], end, None if tree is None else tree[cu[b]:cu[b + 1]]) & there
        k[:, ~there] = v[:, ~there] = 0
        if end == 0:
            k = v = np.zeros((kp.nkvh, 1, HD))
            vis = np.zeros((n, 1), bool)
        parts.append(R.attend(q[cu[b]:cu[b + 1]], k, v, vis, scale))
    return [np.concatenate([p[i] for p in parts]) for i in range(4)]


def weights(x):
    """Whole numbers of 2^-40 of the values x (float64), clamped to [0, 1], to the nearest, ties to even."""
    x = np.where(np.isnan(x), 0.0, np.clip(x, 0, 1))
    return np.rint(x * 2.0 ** 40).astype(np.int64)


def pick(w, u):
    """Least index whose sum of w up to it exceeds u times the whole (one rounding to float64); -1 where there is no weight."""
    total = int(w.sum())
    if total <= 0:
        return -1
    u = np.float32(0 if not u > 0 else min(u, np.float32(1 - 2.0 ** -24)))
    want = float(u) * (total / 2.0 ** 40)
    return int(np.argmax(np.cumsum(w) / 2.0 ** 40 > want))


def verify(p, q, ids, parent, u, u_last, cu, V, out, path, n_path, pos):
    """draft_verify in place on copies of out, path, n_path and pos."""
    out, path, n_path, pos = out.copy(), path.copy(), n_path.copy(), pos.copy()
    for b in range(len(cu) - 1):
        c0, nt = cu[b], min(64, cu[b + 1] - cu[b])
        if nt <= 0:
            n_path[b] = 0
            continue
        x, row = ids[c0:c0 + nt], p[c0:c0 + nt].astype(np.float64)
        prob = lambda t, i: row[t, i] if 0 <= i < V else 0.0  # noqa: E731
        stand, bad = [0], []
        if q is not None:
            t = 1
            while t < nt:
                qq = np.float64(q[c0 + t, x[t]]) if 0 <= x[t] < V else 0.0
                if not np.float64(u[c0 + t]) * qq < prob(t - 1, x[t]):
                    break
                stand.append(t)
                t += 1
            w = weights(row[t - 1] - q[c0 + t].astype(np.float64)) if t < nt else weights(row[t - 1])
            if w.sum() == 0:
                w = weights(row[t - 1])
        else:
            node, rest = 0, 1.0
            for t in range(1, nt):
                par = t - 1 if parent is None else parent[c0 + t]
                if par != node or not 0 <= par < t:
                    continue
                pr = 0.0 if x[t] in bad else prob(node, x[t])
                if np.float64(u[c0 + t]) * rest < pr:
                    node, rest, bad = t, 1.0, []
                    stand.append(t)
                else:
                    rest -= pr
                    bad.append(x[t])
            w = weights(row[node])
            w[[i for i in bad if 0 <= i < V]] = 0
        n = len(stand)
        out[c0:c0 + nt] = path[c0:c0 + nt] = -1
        out[c0:c0 + n - 1] = x[stand[1:]]
        out[c0 + n - 1] = pick(w, u_last[b])
        path[c0:c0 + n] = stand
        n_path[b] = n
        pos[b] += n
    return out, path, n_path, pos


def accept(pool, table, pos, cu, path, n_path):
    """kv_accept_paged in place on a pool's codes and scales; pos as draft_verify leaves it."""
    def place(b, j):
        i = j // pool.page
        p = int(table[b, i]) if 0 <= i < table.shape[1] else -1
        return (p, slice(None), j % pool.page) if 0 <= p < len(pool.buf) else None

    for b in range(len(cu) - 1):
        nt = min(64, cu[b + 1] - cu[b])
        moves = []
        for i in range(min(n_path[b], nt)):
            t = int(path[cu[b] + i])
            if not 0 <= t < nt:
                break
            a, z = (place(b, pos[b] - int(n_path[b]) + x) for x in (t, i))
            if a and z:
                moves.append((z, [x[a].copy() for x in (pool.codes, pool.scales) if x is not None]))
        for z, rows in moves:
            for x, row in zip((pool.codes, pool.scales), rows):
                x[z] = row
