"""Timed cases of the operators that read and keep the K/V cache which attn_prep writes, at the head layout of the model
this library serves (24 query heads, 4 K/V heads, head width 256) and at others: attention of a tree of drafted tokens
(one token is plain decoding), the accumulation of attention weights and the eviction of the lightest rows, attention
over blocks of 64 rows that a cheap score selects for each token, and the move of an accepted path's rows.

run() computes each operator in plain torch, in 32 bits, or calls the library where `own` is true; exact() restates each
from its definition in 64 bits. A cache is one byte buffer: f16 [nkvh][n_ctx][256], or int8 [nkvh][n_ctx][256] followed by
f16 scales [nkvh][n_ctx][8] (one per 32 values). Rows of a cache that are moved are returned as stored: codes and scales
are copied, not computed.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
HD = 256      # head width
BLOCK = 64    # rows of a block of the sparse attention
PKG = os.path.join(os.getcwd(), "qwen27-engine_amd")


def _ops():
    name = "qwen27_engine_amd"
    if name not in sys.modules:
        spec = importlib.util.spec_from_file_location(name, os.path.join(PKG, "__init__.py"), submodule_search_locations=[PKG])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name].ops


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # the first tokens of a chat: nothing but latency
        {"name": "tree_t1_37_q8", "kind": "tree", "T": 1, "n": 37, "n_ctx": 4096, "q8": True, "nqh": 24, "nkvh": 4},
        # plain decoding deep in a long document
        {"name": "tree_t1_150000_q8", "kind": "tree", "T": 1, "n": 150000, "n_ctx": 180224, "q8": True, "nqh": 24, "nkvh": 4},
        # verification of a small tree of drafts in an ordinary conversation, f16 cache
        {"name": "tree_t12_32771_f16", "kind": "tree", "T": 12, "n": 32771, "n_ctx": 40960, "q8": False, "nqh": 24, "nkvh": 4},
        # the widest tree (or the last 64 tokens of a prompt, whose attention scores an eviction) over a long context
        {"name": "tree_t64_131072_q8", "kind": "tree", "T": 64, "n": 131072, "n_ctx": 180224, "q8": True, "nqh": 24, "nkvh": 4},
        # the weights of one decoded token added up over a long cache
        {"name": "weights_t1_150000_q8", "kind": "weights", "T": 1, "n": 150000, "n_ctx": 180224, "q8": True, "nqh": 24,
         "nkvh": 4},
        # the weights of a prompt's last 32 tokens, f16 cache
        {"name": "weights_t32_20001_f16", "kind": "weights", "T": 32, "n": 20001, "n_ctx": 32768, "q8": False, "nqh": 24,
         "nkvh": 4},
        # a prompt's cache evicted into a smaller one for decoding
        {"name": "evict_20001_4096_f16", "kind": "evict", "n": 20001, "n_ctx": 32768, "keep": 4096, "first": 4, "last": 256,
         "in_place": False, "q8": False, "nkvh": 4},
        # a long cache evicted where it lies
        {"name": "evict_150000_16384_q8", "kind": "evict", "n": 150000, "n_ctx": 180224, "keep": 16384, "first": 4, "last": 1024,
         "in_place": True, "q8": True, "nkvh": 4},
        # sparse decoding of one token over a long cache: newest block's bounds, selection, attention
        {"name": "blocks_t1_150000_q8", "kind": "blocks", "T": 1, "n": 150000, "n_ctx": 180224, "nsel": 64, "first": 1, "last": 4,
         "q8": True, "nqh": 24, "nkvh": 4},
        # a ragged batch of a prompt, each token with blocks of its own
        {"name": "blocks_t1027_32768_f16", "kind": "blocks", "T": 1027, "n": 32768, "n_ctx": 40960, "nsel": 32, "first": 1,
         "last": 2, "q8": False, "nqh": 24, "nkvh": 4},
        # the accepted path of a verified tree, K, V and weights of the 16 attention layers at once
        {"name": "accept_t12_16layers_q8", "kind": "accept", "T": 12, "n": 1500, "n_ctx": 2048, "n_path": 4, "layers": 16,
         "q8": True, "nkvh": 4},
        # the same for the widest tree and a long path, f16 cache
        {"name": "accept_t64_16layers_f16", "kind": "accept", "T": 64, "n": 1500, "n_ctx": 2048, "n_path": 17, "layers": 16,
         "q8": False, "nkvh": 4},
    ]


def draw(rng):
    def size(lo, hi):
        return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    kind = rng.choice(["tree", "tree", "weights", "evict", "blocks", "accept"])
    q8 = rng.random() < 0.6
    nqh, nkvh = rng.choice([(24, 4), (24, 4), (12, 2), (16, 4), (16, 2), (7, 1)])
    case = {"kind": kind, "q8": q8, "nkvh": nkvh}
    if kind in ("tree", "weights"):
        T, n = size(1, 64), size(1, 131072)
        while T * n > 64 * 65536:
            T = (T + 1) // 2
        case.update(T=T, n=n, n_ctx=n + T + rng.randint(0, 4096), nqh=nqh)
    elif kind == "evict":
        n = size(100, 150000)
        keep = size(50, min(n, 16384))
        first = rng.randint(0, min(8, keep))
        case.update(n=n, n_ctx=n + rng.randint(0, 4096), keep=keep, first=first, last=rng.randint(0, (keep - first) // 2),
                    in_place=rng.random() < 0.5)
    elif kind == "blocks":
        T, n = size(1, 1027), size(1, 131072)
        while T * n > 1027 * 32768:
            T = (T + 1) // 2
        nsel = size(4, 64)
        case.update(T=T, n=n, n_ctx=n + T + rng.randint(0, 4096), nsel=nsel, first=rng.randint(0, 2), last=rng.randint(1, 2),
                    nqh=nqh)
    else:
        T = size(2, 64)
        case.update(T=T, n=size(1, 1900), n_ctx=2048, n_path=rng.randint(1, T), layers=rng.randint(1, 16))
    return case


# ---------------------------------------------------------------- inputs
class _Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(int(seed) * 2 + 1)

    def n(self, *shape):
        return torch.randn(shape, device=DEV, generator=self.g)

    def ints(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, device=DEV, generator=self.g)


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _cache(x, q8):
    """The byte buffer of f32 rows x [nkvh][n_ctx][256], quantized as attn_prep does."""
    if not q8:
        return x.to(torch.float16).reshape(-1).view(torch.uint8)
    b = x.view(-1, 8, 32)
    d = b.abs().amax(-1, keepdim=True) / 127
    codes = torch.where(d > 0, b / d, torch.zeros_like(b))
    codes = torch.trunc(codes + codes.sign() * 0.5)
    return torch.cat([codes.to(torch.int8).reshape(-1).view(torch.uint8), d.to(torch.float16).reshape(-1).view(torch.uint8)])


def _views(buf, nkvh, n_ctx, q8):
    """(codes [nkvh][n_ctx][256], scales [nkvh][n_ctx][8] or None) of a cache's buffer."""
    if not q8:
        return buf.view(torch.float16).view(nkvh, n_ctx, HD), None
    m = nkvh * n_ctx * HD
    return buf[:m].view(torch.int8).view(nkvh, n_ctx, HD), buf[m:].view(torch.float16).view(nkvh, n_ctx, 8)


def _rows(buf, nkvh, n_ctx, q8, n, dtype):
    """The values of rows 0 .. n - 1, [nkvh][n][256] in `dtype`."""
    c, d = _views(buf, nkvh, n_ctx, q8)
    c = c[:, :n].to(dtype)
    return c if d is None else (c.view(nkvh, n, 8, 32) * d[:, :n, :, None].to(dtype)).view(nkvh, n, HD)


def _tree(r, T):
    """Ancestor masks [T] of a random tree: each token follows the context or one of the eight before it."""
    parent = (torch.arange(T, device=DEV) - 1 - r.ints(0, 8, T)).clamp(min=-1).tolist()
    masks = []
    for t, p in enumerate(parent):
        masks.append((1 << t) | (masks[p] if p >= 0 else 0))
    return torch.tensor([m - (1 << 64) if m >= 1 << 63 else m for m in masks], dtype=torch.int64, device=DEV)


def prepare(case, seed):
    r, kind = _Rand(seed), case["kind"]
    nkvh, q8, n, n_ctx = case["nkvh"], case["q8"], case["n"], case["n_ctx"]
    st = {"case": case, "pos0": _i32(n)}
    if kind == "accept":
        T, L = case["T"], case["layers"]
        st["kv"] = torch.stack([_cache(r.n(nkvh, n_ctx, HD), q8) for _ in range(2 * L)])  # K and V of every layer
        st["accs"] = torch.exp(2 * r.n(L, nkvh, n_ctx))
        path = torch.randperm(T, device=DEV, generator=r.g)[:case["n_path"]].sort().values
        st["path"] = torch.cat([path, path.new_zeros(T - path.numel())]).to(torch.int32)
        st["n_path"] = _i32(case["n_path"])
        if own:  # a program's caches lie where they lie: their addresses are listed once
            st["caches"], st["weights"] = _ops().kv_pointers(list(st["kv"])), _ops().kv_pointers(list(st["accs"]))
        return st
    # keys with channels of unequal strength, a shared direction that many queries look for, and heavier rows
    chan = torch.exp(0.4 * r.n(nkvh, 1, HD))
    topic = r.n(nkvh, 1, HD)
    k = r.n(nkvh, n_ctx, HD) * chan + topic * (torch.rand(nkvh, n_ctx, 1, device=DEV, generator=r.g) < 0.02) * 0.7
    st["k"] = _cache(k, q8)
    del k
    st["v"] = _cache(r.n(nkvh, n_ctx, HD), q8)
    if kind == "evict":
        st["acc"] = torch.exp(2 * r.n(nkvh, n_ctx))
        st["n_out"] = n_ctx if case["in_place"] else case["keep"] + 512
        if case["in_place"]:
            st["ko"], st["vo"], st["acc_o"] = st["k"], st["v"], st["acc"]
        else:
            row = (HD + 16) if q8 else 2 * HD
            st["ko"], st["vo"] = (torch.zeros(nkvh * st["n_out"] * row, dtype=torch.uint8, device=DEV) for _ in range(2))
            st["acc_o"] = torch.zeros(nkvh, st["n_out"], device=DEV)
        if own:
            st["kept"] = torch.empty(nkvh, case["keep"], dtype=torch.int32, device=DEV)
            st["ws"] = torch.empty(_ops().kv_evict_ws_bytes(nkvh, n_ctx, case["keep"], q8, case["in_place"]),
                                   dtype=torch.uint8, device=DEV)
        return st
    T, nqh = case["T"], case["nqh"]
    st["q"] = (r.n(T, nkvh, nqh // nkvh, HD) * 1.5 + topic[None] * 0.8).reshape(T, nqh, HD).contiguous()
    st["scale"] = HD ** -0.5
    if kind == "weights":
        st["acc"] = torch.exp(r.n(nkvh, n_ctx))
    if kind in ("tree", "weights"):
        st["tree"] = _tree(r, T)
    if kind == "weights":
        # the log sums that attn_tree gave for these queries
        kf = _rows(st["k"], nkvh, n_ctx, q8, min(n + T, n_ctx), torch.float32)
        st["lse"] = _plain_scores(st, kf).logsumexp(-1).permute(1, 0, 2).reshape(T, nqh).contiguous()
    if kind == "blocks":
        # the bounds of the rows before this batch, as earlier calls left them
        nblk = -(-n_ctx // BLOCK)
        st["lo"], st["hi"] = (torch.zeros(nkvh, nblk, HD, dtype=torch.int8, device=DEV) for _ in range(2))
        st["kd"] = torch.zeros(nkvh, nblk, device=DEV)
        kf = _rows(st["k"], nkvh, n_ctx, q8, n, torch.float32)
        _put_bounds(st, kf, 0, -(-n // BLOCK), n)
        if own:
            kb = torch.empty(_ops().kv_block_bytes(nkvh, n_ctx), dtype=torch.uint8, device=DEV)
            m = nkvh * nblk * HD
            kb[:m], kb[m:2 * m] = st["lo"].view(torch.uint8).view(-1), st["hi"].view(torch.uint8).view(-1)
            kb[2 * m:] = st["kd"].view(-1).view(torch.uint8)
            st["kb"] = kb
            st["lo"], st["hi"] = (kb[i * m:(i + 1) * m].view(torch.int8).view(nkvh, nblk, HD) for i in range(2))
            st["kd"] = kb[2 * m:].view(torch.float32).view(nkvh, nblk)
    if own:
        o = _ops()
        st["o"] = torch.empty(T, nqh, HD, device=DEV)
        if kind == "tree":
            st["lse"] = torch.empty(T, nqh, device=DEV)
            nbytes = o.attn_tree_ws_bytes(T, nqh, nkvh, n_ctx)
        elif kind == "blocks":
            st["idx"] = torch.empty(T, nkvh, case["nsel"], dtype=torch.int32, device=DEV)
            nbytes = max(o.attn_select_ws_bytes(T, nkvh, n_ctx), o.attn_blocks_ws_bytes(T, nqh, nkvh, case["nsel"]))
        else:
            nbytes = 0
        st["ws"] = torch.empty(nbytes, dtype=torch.uint8, device=DEV)
    return st


# ---------------------------------------------------------------- the plain forms
def _plain_visible(st, T, n, total):
    """[T][total]: token t sees every row before n and the drafted rows of its mask."""
    j = torch.arange(total, device=DEV)
    bit = (st["tree"][:, None] >> (j - n).clamp(min=0, max=63)[None]) & 1
    return (j < n)[None] | (bit == 1)


def _plain_scores(st, kf):
    """scale * q . k of the rows kf [nkvh][total][256] as [nkvh][T][group][total], -inf where hidden."""
    case, nkvh, total = st["case"], kf.shape[0], kf.shape[1]
    T, g = case["T"], case["nqh"] // nkvh
    q = st["q"].to(kf.dtype).view(T, nkvh, g, HD).permute(1, 0, 2, 3).reshape(nkvh, T * g, HD)
    s = torch.bmm(q * st["scale"], kf.transpose(1, 2).contiguous()).view(nkvh, T, g, total)
    return s.masked_fill_(~_plain_visible(st, T, case["n"], total)[None, :, None], float("-inf"))


def _plain_attend(s, vf):
    """softmax(s) v and the log of the sum of exponentials; a row with nothing visible gives zeros and -inf."""
    m = s.amax(-1, keepdim=True).clamp(min=torch.finfo(s.dtype).min)
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    nkvh, T, g = s.shape[:3]
    o = torch.bmm(p.view(nkvh, T * g, -1), vf).view(nkvh, T, g, HD) / total.clamp(min=torch.finfo(s.dtype).tiny)
    lse = (m + total.log()).squeeze(-1)
    return (o.permute(1, 0, 2, 3).reshape(T, nkvh * g, HD).contiguous(),
            lse.permute(1, 0, 2).reshape(T, nkvh * g).contiguous())


def _run_tree(st):
    c = st["case"]
    total = min(c["n"] + c["T"], c["n_ctx"])
    kf, vf = (_rows(st[w], c["nkvh"], c["n_ctx"], c["q8"], total, torch.float32) for w in ("k", "v"))
    return _plain_attend(_plain_scores(st, kf), vf)


def _run_weights(st):
    c = st["case"]
    n, total, nkvh, T = c["n"], min(c["n"] + c["T"], c["n_ctx"]), c["nkvh"], c["T"]
    s = _plain_scores(st, _rows(st["k"], nkvh, c["n_ctx"], c["q8"], total, torch.float32))
    lse = st["lse"].view(T, nkvh, -1).permute(1, 0, 2)[..., None]
    w = (s - lse).exp_().sum((1, 2))
    st["acc"][:, :n] += w[:, :n]
    st["acc"][:, n:total] = w[:, n:]  # the weights of new rows begin here
    return st["acc"]


def _plain_kept(acc, n, keep, first, last):
    """[nkvh][min(n, keep)]: the kept rows in order; among equal weights the lowest rows stay."""
    nkvh = acc.shape[0]
    if n <= keep:
        return torch.arange(n, device=DEV).expand(nkvh, n)
    heavy = acc[:, first:n - last].sort(dim=1, descending=True, stable=True).indices[:, :keep - first - last] + first
    ends = torch.cat([torch.arange(first, device=DEV), torch.arange(n - last, n, device=DEV)]).expand(nkvh, first + last)
    return torch.cat([heavy, ends], 1).sort(dim=1).values


def _run_evict(st):
    c = st["case"]
    nkvh, q8, keep = c["nkvh"], c["q8"], c["keep"]
    idx = _plain_kept(st["acc"], c["n"], keep, c["first"], c["last"])
    m = idx.shape[1]
    for a, b in (("k", "ko"), ("v", "vo")):
        for x, y in zip(_views(st[a], nkvh, c["n_ctx"], q8), _views(st[b], nkvh, st["n_out"], q8)):
            if x is not None:
                y[:, :m] = x.gather(1, idx[..., None].expand(-1, -1, x.shape[2]))
    st["acc_o"][:, :m] = st["acc"].gather(1, idx)
    kept = torch.full((nkvh, keep), -1, dtype=torch.int32, device=DEV)
    kept[:, :m] = idx
    return kept


def _q8_rows(lo, hi):
    """int8 codes of lo and hi [.., 256] with one scale d = max|.| / 127 for both, and d."""
    amax = torch.maximum(lo.abs().amax(-1), hi.abs().amax(-1))
    # 64 bits and one rounding each: the float32 quotient, reciprocal and products, correctly rounded
    d = torch.where(amax >= 2.0 ** -100, amax.double() / 127, torch.zeros_like(amax, dtype=torch.float64)).float()
    inv = torch.where(d > 0, 1 / d.double(), torch.zeros_like(d, dtype=torch.float64)).float()[..., None]
    out = []
    for x in (lo, hi):
        y = (x.double() * inv.double()).float()
        out.append(torch.trunc(y.double() + y.sign() * 0.5).to(torch.int8))
    return out[0], out[1], d


def _put_bounds(st, kf, b0, b1, n):
    """Bounds of blocks b0 .. b1 - 1 from the rows kf [nkvh][n][256] of the cache, into st's lo, hi and kd."""
    nkvh = kf.shape[0]
    pad = b1 * BLOCK - n
    rows = torch.cat([kf[:, b0 * BLOCK:], kf[:, -1:].expand(-1, pad, -1)], 1) if pad else kf[:, b0 * BLOCK:]
    rows = rows.view(nkvh, b1 - b0, BLOCK, HD)
    st["lo"][:, b0:b1], st["hi"][:, b0:b1], st["kd"][:, b0:b1] = _q8_rows(rows.amin(2), rows.amax(2))


def _plain_select(st, total):
    """[T][nkvh][nsel] selected blocks in order, -1 behind the last."""
    c = st["case"]
    T, n, nkvh, nsel = c["T"], c["n"], c["nkvh"], c["nsel"]
    g, nb = c["nqh"] // nkvh, -(-total // BLOCK)
    qc, _, qd = _q8_rows(st["q"].view(T, nkvh, g, HD), st["q"].view(T, nkvh, g, HD))
    q = qc.float().permute(1, 0, 2, 3).reshape(nkvh, T * g, HD)
    lo, hi = (st[w][:, :nb].float().transpose(1, 2).contiguous() for w in ("lo", "hi"))
    dot = torch.bmm(q.clamp(min=0), hi) + torch.bmm(q.clamp(max=0), lo)  # whole numbers below 2^24: exact
    s = (dot.view(nkvh, T, g, nb) * qd.permute(1, 0, 2)[..., None]).amax(2) * st["kd"][:, None, :nb]
    b = torch.arange(nb, device=DEV)[None]
    mine = ((n + torch.arange(T, device=DEV)) // BLOCK)[:, None]  # the block of the token itself
    s = torch.where((b < c["first"]) | (b > mine - c["last"]), torch.full_like(s, float("inf")), s)
    s = torch.where(b <= mine, s, torch.full_like(s, float("-inf")))
    top = s.sort(dim=-1, descending=True, stable=True).indices[..., :nsel]
    top = torch.where(top <= mine[None], top, torch.full_like(top, nb)).sort(dim=-1).values
    idx = torch.full((T, nkvh, nsel), -1, dtype=torch.int32, device=DEV)
    idx[..., :top.shape[-1]] = torch.where(top < nb, top, torch.full_like(top, -1)).permute(1, 0, 2)
    return idx


def _block_scores(st, kf, idx, nb):
    """Scores of the rows kf [nkvh][total][256] as [nkvh][T][group][total], -inf outside the selected blocks."""
    c, nkvh, total = st["case"], kf.shape[0], kf.shape[1]
    T, g = c["T"], c["nqh"] // nkvh
    seen = torch.zeros(nkvh, T, nb + 1, dtype=torch.bool, device=DEV)
    at = idx.permute(1, 0, 2).long()
    seen.scatter_(2, torch.where(at < 0, torch.full_like(at, nb), at), True)
    j = torch.arange(total, device=DEV)
    vis = seen[..., j // BLOCK] & (j[None] <= c["n"] + torch.arange(T, device=DEV)[:, None])[None]
    q = st["q"].to(kf.dtype).view(T, nkvh, g, HD).permute(1, 0, 2, 3).reshape(nkvh, T * g, HD)
    s = torch.bmm(q * st["scale"], kf.transpose(1, 2).contiguous()).view(nkvh, T, g, total)
    return s.masked_fill_(~vis[:, :, None], float("-inf"))


def _run_blocks(st):
    c = st["case"]
    total = min(c["n"] + c["T"], c["n_ctx"])
    nb = -(-total // BLOCK)
    kf, vf = (_rows(st[w], c["nkvh"], c["n_ctx"], c["q8"], total, torch.float32) for w in ("k", "v"))
    _put_bounds(st, kf, c["n"] // BLOCK, nb, total)
    idx = _plain_select(st, total)
    return idx, _plain_attend(_block_scores(st, kf, idx, nb), vf)[0]


def _kv_views(st):
    """(codes [2 layers][nkvh][n_ctx][256], scales or None) of the caches of every layer."""
    c, kv = st["case"], st["kv"]
    shape = (kv.shape[0], c["nkvh"], c["n_ctx"])
    if not c["q8"]:
        return kv.view(torch.float16).view(*shape, HD), None
    m = c["nkvh"] * c["n_ctx"] * HD
    return kv[:, :m].view(torch.int8).unflatten(1, (*shape[1:], HD)), kv[:, m:].view(torch.float16).unflatten(1, (*shape[1:], 8))


def _run_accept(st):
    codes, d = _kv_views(st)
    i = torch.arange(st["case"]["T"], device=DEV)
    dst = st["pos0"] + i
    src = st["pos0"] + torch.where(i < st["n_path"], st["path"], i)  # rows behind the path stay as they are
    codes[:, :, dst] = codes[:, :, src]
    if d is not None:
        d[:, :, dst] = d[:, :, src]
    st["accs"][:, :, dst] = st["accs"][:, :, src]


# ---------------------------------------------------------------- one pass
def run(st):
    c = st["case"]
    kind, nkvh, n_ctx, q8 = c["kind"], c["nkvh"], c["n_ctx"], c["q8"]
    if kind == "tree":
        if own:
            _ops().attn_tree(st["q"], st["k"], st["v"], st["pos0"], st["tree"], c["T"], st["scale"], c["nqh"], nkvh, n_ctx, q8,
                             st["o"], st["ws"], lse=st["lse"])
            return {"o": st["o"], "lse": st["lse"]}
        o, lse = _run_tree(st)
        return {"o": o, "lse": lse}
    if kind == "weights":
        if own:
            _ops().attn_weights(st["q"], st["lse"], st["k"], st["pos0"], st["tree"], c["T"], st["scale"], c["nqh"], nkvh, n_ctx,
                                q8, st["acc"])
            return {"acc": st["acc"]}
        return {"acc": _run_weights(st)}
    if kind == "evict":
        if own:
            _ops().kv_evict(st["k"], st["v"], st["acc"], st["pos0"], c["keep"], c["first"], c["last"], st["ko"], st["vo"],
                            st["acc_o"], st["n_out"], st["kept"], nkvh, n_ctx, q8, st["ws"])
            kept = st["kept"]
        else:
            kept = _run_evict(st)
        return {"kept": kept, "acc": st["acc_o"], "k": _views(st["ko"], nkvh, st["n_out"], q8),
                "v": _views(st["vo"], nkvh, st["n_out"], q8)}
    if kind == "blocks":
        if own:
            m, o = _ops(), st["o"]
            m.kv_block_bounds(st["k"], st["pos0"], c["T"], nkvh, n_ctx, q8, st["kb"])
            m.attn_select(st["q"], st["kb"], st["pos0"], c["T"], c["nqh"], nkvh, n_ctx, c["nsel"], c["first"], c["last"],
                          st["idx"], st["ws"])
            m.attn_blocks(st["q"], st["k"], st["v"], st["pos0"], st["idx"], c["T"], c["nsel"], st["scale"], c["nqh"], nkvh, n_ctx,
                          q8, o, st["ws"])
            idx = st["idx"]
        else:
            idx, o = _run_blocks(st)
        return {"idx": idx, "o": o, "lo": st["lo"], "hi": st["hi"], "kd": st["kd"]}
    if own:
        _ops().kv_accept(st["caches"], st["weights"], st["pos0"], st["path"], st["n_path"], c["T"], nkvh, n_ctx, q8)
    else:
        _run_accept(st)
    return {"kv": _kv_views(st), "acc": st["accs"]}


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    nkvh, n, kind = case["nkvh"], case["n"], case["kind"]
    row = HD + 16 if case["q8"] else 2 * HD
    if kind == "accept":
        return {"bytes": 2.0 * case["n_path"] * nkvh * case["layers"] * (2 * row + 4), "flops": 0.0}
    if kind == "evict":
        m = min(n, case["keep"])
        return {"bytes": nkvh * (4.0 * n + 2 * m * (2 * row + 4) + 4 * case["keep"]), "flops": 0.0}
    T, nqh = case["T"], case["nqh"]
    total = min(n + T, case["n_ctx"])
    qo = 4.0 * T * nqh * HD
    if kind == "tree":
        return {"bytes": 2.0 * nkvh * total * row + 2 * qo + 4 * T * nqh, "flops": 4.0 * HD * nqh * T * total}
    if kind == "weights":
        return {"bytes": nkvh * total * (row + 8.0) + qo + 4 * T * nqh, "flops": 2.0 * HD * nqh * T * total}
    nb = -(-total // BLOCK)
    read = min(total, T * case["nsel"] * BLOCK)
    mine = min(total, case["nsel"] * BLOCK)
    return {"bytes": nkvh * (nb * (2.0 * HD + 4) + 2.0 * read * row) + 2 * qo + 4 * T * nkvh * case["nsel"],
            "flops": 4.0 * HD * nqh * T * mine + 4.0 * HD * nqh * T * nb}


# ---------------------------------------------------------------- from the definitions, in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    kind, nkvh, n, n_ctx, q8 = case["kind"], case["nkvh"], case["n"], case["n_ctx"], case["q8"]
    if kind in ("evict", "accept"):
        return None  # rows are chosen and copied: nothing is computed
    T, nqh = case["T"], case["nqh"]
    g, total = nqh // nkvh, min(n + T, n_ctx)
    q = st["q"].double() * st["scale"]
    heads, idx, acc = [], None, []
    if kind == "blocks":
        idx = _exact_idx(case, st, total)
    for kh in range(nkvh):
        k, v = (_exact_rows(st[w], kh, nkvh, n_ctx, q8, total) for w in ("k", "v"))
        s = (q[:, kh * g:(kh + 1) * g].reshape(T * g, HD) @ k.t()).view(T, g, total)
        hidden = torch.zeros(T, total, dtype=torch.bool, device=DEV)
        if kind == "blocks":
            listed_ = torch.zeros(T, -(-total // BLOCK), device=DEV)
            listed_.scatter_add_(1, idx[:, kh].clamp(min=0).long(), (idx[:, kh] >= 0).float())
            hidden |= listed_.repeat_interleave(BLOCK, 1)[:, :total] == 0
            hidden |= torch.arange(total, device=DEV)[None] > n + torch.arange(T, device=DEV)[:, None]
        else:
            masks = st["tree"].tolist()
            for t in range(T):
                for j in range(n, total):
                    hidden[t, j] = not (masks[t] >> (j - n)) & 1
        s.masked_fill_(hidden[:, None], float("-inf"))
        if kind == "weights":
            w = torch.exp(s - st["lse"].double()[:, kh * g:(kh + 1) * g, None]).sum((0, 1))
            a = st["acc"][kh].double()
            a[:n] += w[:n]
            a[n:total] = w[n:]
            acc.append(a)
        else:
            lse = torch.logsumexp(s, -1)
            heads.append((torch.exp(s - lse[..., None]).view(T * g, total) @ v, lse))
    if kind == "weights":
        return {"acc": torch.stack(acc)}
    o = torch.cat([h[0].view(T, g, HD) for h in heads], 1)
    if kind == "blocks":
        return {"idx": None, "o": o, "lo": None, "hi": None, "kd": None}
    return {"o": o, "lse": torch.cat([h[1] for h in heads], 1)}


def _exact_rows(buf, kh, nkvh, n_ctx, q8, total):
    """Rows 0 .. total - 1 of K/V head kh in 64 bits, from the bytes of the cache."""
    if not q8:
        at = kh * n_ctx * HD * 2
        return buf[at:at + total * HD * 2].view(torch.float16).view(total, HD).double()
    at, sc = kh * n_ctx * HD, nkvh * n_ctx * HD + kh * n_ctx * 16
    x = buf[at:at + total * HD].view(torch.int8).view(total, HD).double()
    return x * buf[sc:sc + total * 16].view(torch.float16).view(total, 8).double().repeat_interleave(32, 1)


def _exact_idx(case, st, total):
    """The selected blocks [T][nkvh][nsel], from the definition: scores of the whole-number bounds, rounded where it rounds."""
    T, n, nkvh, nsel = case["T"], case["n"], case["nkvh"], case["nsel"]
    g, nb, b0 = case["nqh"] // case["nkvh"], -(-total // BLOCK), case["n"] // BLOCK

    def scale(x):
        d = (x / 127).float().double()
        return d, (1 / d).float().double()

    def code(x, inv):
        y = (x * inv).float().double()
        return torch.sign(y) * torch.floor(y.abs() + 0.5)

    lo, hi, kd = st["lo"].double(), st["hi"].double(), st["kd"].double()
    for kh in range(nkvh):
        k = _exact_rows(st["k"], kh, nkvh, case["n_ctx"], case["q8"], total)
        for b in range(b0, nb):
            rows = k[b * BLOCK:(b + 1) * BLOCK]
            a, z = rows.min(0).values, rows.max(0).values
            d, inv = scale(torch.maximum(a.abs().max(), z.abs().max()))
            lo[kh, b], hi[kh, b], kd[kh, b] = code(a, inv), code(z, inv), d
    q = st["q"].double().view(T, nkvh, g, HD)
    qd, qi = scale(q.abs().amax(-1, keepdim=True))
    qc = code(q, qi)
    best = torch.full((T, nkvh, nb), float("-inf"), dtype=torch.float64, device=DEV)
    for kh in range(nkvh):
        for h in range(g):
            x = qc[:, kh, h]
            dot = torch.where(x > 0, x, torch.zeros_like(x)) @ hi[kh, :nb].t() + torch.where(x < 0, x, torch.zeros_like(x)) @ lo[kh, :nb].t()
            best[:, kh] = torch.maximum(best[:, kh], (dot * qd[:, kh, h]).float().double())
        best[:, kh] = (best[:, kh] * kd[kh, :nb]).float().double()
    block = torch.arange(nb, device=DEV)
    mine = (n + torch.arange(T, device=DEV)) // BLOCK
    must = (block[None] < case["first"]) | (block[None] > mine[:, None] - case["last"])
    best.masked_fill_(must[:, None], float("inf"))
    best.masked_fill_((block[None] > mine[:, None])[:, None], float("-inf"))
    # the rank of a block: those of a higher score, and those of the same one before it
    order = torch.argsort(best, dim=-1, descending=True, stable=True)
    rank = torch.empty_like(order)
    rank.scatter_(2, order, block.expand_as(order).contiguous())
    chosen = (rank < nsel) & (block[None] <= mine[:, None])[:, None]
    idx = torch.full((T, nkvh, nsel + 1), -1, dtype=torch.int64, device=DEV)
    place = torch.where(chosen, chosen.cumsum(-1) - 1, torch.full_like(order, nsel))
    idx.scatter_(2, place, block.expand_as(order).contiguous())
    return idx[..., :nsel]
