"""Plain 64-bit forms of the operators over the K/V cache (numpy), written from their definitions, and the error bounds that
the GPU tests hold the float32 results to."""
import numpy as np

HD, BLOCK = 256, 64


def make_cache(r, nkvh, n_ctx, q8, std=1.0, garbage_from=None):
    """A cache's bytes. Rows from `garbage_from` on are what nobody may read: NaN (f16) or NaN scales (q8)."""
    if not q8:
        h = (r.standard_normal((nkvh, n_ctx, HD)) * std).astype(np.float16)
        if garbage_from is not None:
            h[:, garbage_from:] = np.nan
        return h.reshape(-1).view(np.uint8)
    codes = r.integers(-127, 128, (nkvh, n_ctx, HD)).astype(np.int8)
    scales = (r.uniform(0.2, 1.8, (nkvh, n_ctx, 8)) * std / 73).astype(np.float16)
    if garbage_from is not None:
        scales[:, garbage_from:] = np.nan
    return join_q8(codes, scales)


def join_q8(codes, scales):
    return np.concatenate([codes.reshape(-1).view(np.uint8), scales.reshape(-1).view(np.uint8)])


def split_q8(buf, nkvh, n_ctx):
    m = nkvh * n_ctx * HD
    return buf[:m].view(np.int8).reshape(nkvh, n_ctx, HD), buf[m:].view(np.float16).reshape(nkvh, n_ctx, 8)


def values(buf, nkvh, n_ctx, q8):
    """[nkvh][n_ctx][256] in 64 bits."""
    if not q8:
        return buf.view(np.float16).reshape(nkvh, n_ctx, HD).astype(np.float64)
    c, d = split_q8(buf, nkvh, n_ctx)
    return c.astype(np.float64) * np.repeat(d.astype(np.float64), 32, axis=2)


def random_tree(r, T, empty=()):
    """Ancestor masks; tokens in `empty` see no drafted row, not even their own."""
    masks = []
    for t in range(T):
        p = int(r.integers(max(-1, t - 5), t)) if t else -1
        masks.append((1 << t) | (masks[p] if p >= 0 else 0))
    return np.array([0 if t in empty else m for t, m in enumerate(masks)], np.uint64)


def visible(T, pos0, n_ctx, tree):
    """[T][n_ctx] truth values."""
    j = np.arange(n_ctx)
    out = np.zeros((T, n_ctx), bool)
    for t in range(T):
        out[t] = j < pos0
        m = (1 << (t + 1)) - 1 if tree is None else int(tree[t])
        for u in range(T):
            if (m >> u) & 1 and 0 <= pos0 + u < n_ctx:
                out[t, pos0 + u] = True
    return out


def block_visible(T, pos0, n_ctx, idx):
    """[T][nkvh][n_ctx]: how often token t sees a row through its list."""
    j = np.arange(n_ctx)
    out = np.zeros((T, idx.shape[1], n_ctx), np.int64)
    for t in range(T):
        for kh in range(idx.shape[1]):
            for b in idx[t, kh]:
                if b >= 0:
                    out[t, kh] += (j // BLOCK == b) & (j <= pos0 + t)
    return out


def attend(q, k, v, vis, scale):
    """o, lse and the bounds of their errors. q [T][nqh][256]; k, v [nkvh][n_ctx][256]; vis [T][n_ctx] or (counts)
    [T][nkvh][n_ctx].

    The bounds: a score is a float32 sum of 256 products whose query factor holds 2^-21 (two f16 terms, cut off); its
    rounding errors, at most 2^-23 of the running sum each, add up like 16 of them (their signs are independent), so
    |ds| <= (2^-21 + 16 * 2^-23) scale sum |q k|, with 2^-23 |s| more for the change of base. A weight is then off by |ds|
    plus 2^-22 (the exponential) plus 2^-21 (its two terms); numerator and denominator both, and the float32 sums over n
    rows add sqrt(n) 2^-23 each, over at most 600 parts joined 2^-22 more."""
    T, nqh, _ = q.shape
    nkvh, n_ctx, _ = k.shape
    g = nqh // nkvh
    o, bound = np.zeros((T, nqh, HD)), np.zeros((T, nqh, HD))
    lse, lse_bound = np.full((T, nqh), -np.inf), np.zeros((T, nqh))
    q = q.astype(np.float64)
    for h in range(nqh):
        kh = h // g
        for t in range(T):
            w = vis[t] if vis.ndim == 2 else vis[t, kh]
            at = np.nonzero(w)[0]
            if not len(at):
                continue
            s = scale * (k[kh, at] @ q[t, h])
            m = s.max()
            p = np.exp(s - m) * w[at]
            o[t, h] = (p / p.sum()) @ v[kh, at]
            lse[t, h] = m + np.log(p.sum())
            ds = scale * (np.abs(k[kh, at]) @ np.abs(q[t, h])) * (2.0 ** -21 + 16 * 2.0 ** -23) + np.abs(s) * 2.0 ** -23
            rel = 2 * (ds.max() + 2.0 ** -22 + 2.0 ** -21) + 2 * np.sqrt(len(at)) * 2.0 ** -23 + 2.0 ** -22
            bound[t, h] = rel * ((p / p.sum()) @ np.abs(v[kh, at]))
            lse_bound[t, h] = rel + np.abs(lse[t, h]) * 2.0 ** -22
    return o, lse, bound, lse_bound


def weights(q, lse, k, vis, scale, rows, acc, pos0, T):
    """acc after attn_weights, and the bound of its error."""
    nkvh, n_ctx, _ = k.shape
    g = q.shape[1] // nkvh
    out = acc.astype(np.float64).copy()
    add, off = np.zeros_like(out), np.zeros_like(out)
    for t in range(T):
        if not (rows >> t) & 1:
            continue
        for h in range(q.shape[1]):
            at = np.nonzero(vis[t])[0]
            if not len(at):
                continue
            s = scale * (k[h // g, at] @ q[t, h].astype(np.float64))
            p = np.exp(s - np.float64(lse[t, h]))
            ds = scale * (np.abs(k[h // g, at]) @ np.abs(q[t, h].astype(np.float64))) * (2.0 ** -21 + 16 * 2.0 ** -23)
            add[h // g, at] += p
            off[h // g, at] += p * (ds + (np.abs(s) + abs(lse[t, h])) * 2.0 ** -22 + 2.0 ** -22)
    new = (np.arange(n_ctx) >= pos0) & (np.arange(n_ctx) < pos0 + T)
    out[:, ~new] += add[:, ~new]
    out[:, new] = add[:, new]
    return out, off + np.abs(out) * 2.0 ** -22


def kept_rows(acc, n, keep, first, last):
    """[nkvh][keep], -1 behind the last."""
    out = np.full((acc.shape[0], keep), -1, np.int64)
    for kh in range(acc.shape[0]):
        if n <= keep:
            out[kh, :n] = np.arange(n)
            continue
        mid = list(range(first, n - last))
        key = [(-np.inf if np.isnan(acc[kh, j]) else float(acc[kh, j]), not np.isnan(acc[kh, j])) for j in mid]
        order = sorted(range(len(mid)), key=lambda i: (-key[i][0], not key[i][1], mid[i]))
        chosen = sorted(mid[i] for i in order[:keep - first - last])
        out[kh] = list(range(first)) + chosen + list(range(n - last, n))
    return out


def q8_pair(lo, hi):
    """Codes of lo and hi with one scale (float32 roundings), and the scale."""
    if not (np.isfinite(lo).all() and np.isfinite(hi).all()):
        return np.zeros(HD, np.int8), np.zeros(HD, np.int8), np.float32(np.inf)
    amax = np.float32(max(np.abs(lo).max(), np.abs(hi).max()))
    if amax < 2.0 ** -100:
        return np.zeros(HD, np.int8), np.zeros(HD, np.int8), np.float32(0)
    d = np.float32(np.float64(amax) / 127)
    inv = np.float32(1 / np.float64(d))
    code = lambda x: (lambda y: np.sign(y) * np.floor(np.abs(y) + 0.5))(  # noqa: E731
        (np.float32(x).astype(np.float64) * np.float64(inv)).astype(np.float32).astype(np.float64)).astype(np.int8)
    return code(lo), code(hi), d


def bounds(k, end):
    """lo, hi [nkvh][nblk][256], d [nkvh][nblk] of the blocks that hold rows before `end`."""
    nkvh, n_ctx, _ = k.shape
    nblk = -(-n_ctx // BLOCK)
    lo, hi, d = np.zeros((nkvh, nblk, HD), np.int8), np.zeros((nkvh, nblk, HD), np.int8), np.zeros((nkvh, nblk), np.float32)
    for kh in range(nkvh):
        for b in range(-(-end // BLOCK)):
            rows = k[kh, b * BLOCK:min(end, (b + 1) * BLOCK)]
            with np.errstate(invalid="ignore"):
                lo[kh, b], hi[kh, b], d[kh, b] = q8_pair(rows.min(0), rows.max(0))
    return lo, hi, d


def select(q, lo, hi, d, pos0, n_ctx, nsel, first, last):
    T, nqh, _ = q.shape
    nkvh, nblk, _ = lo.shape
    g = nqh // nkvh
    out = np.full((T, nkvh, nsel), -1, np.int64)
    for t in range(T):
        nb = 0 if pos0 + t < 0 else min(nblk, (pos0 + t) // BLOCK + 1)
        for kh in range(nkvh):
            best = np.full(nb, -np.inf, np.float32)
            for h in range(kh * g, (kh + 1) * g):
                c, _, dq = q8_pair(q[t, h], q[t, h])
                if np.isinf(dq):
                    dq = np.float32(0)
                c = c.astype(np.int64)
                dot = np.maximum(c, 0) @ hi[kh, :nb].astype(np.int64).T + np.minimum(c, 0) @ lo[kh, :nb].astype(np.int64).T
                best = np.maximum(best, dot.astype(np.float32) * dq)
            with np.errstate(invalid="ignore"):
                score = np.where(np.isinf(d[kh, :nb]), np.float32(np.inf), best * d[kh, :nb])
            b = np.arange(nb)
            must = (b < first) | (b >= nb - last)
            chosen = np.sort(np.lexsort((b, -score, ~must))[:nsel])  # the ends, then by score, then the lower one
            out[t, kh, :len(chosen)] = chosen
    return out
