"""Timed cases of the operators that serve a batch of sequences from a K/V cache in pages, at the head layout of the model
this library serves (24 query heads, 4 K/V heads, head width 256, vocabulary 248320) and at others: attention of each
sequence's new tokens over its pages, the norms, rotation and quantising write that fill them, the rows read back as
values, and the verification of drafted tokens against the target's probabilities.

run() computes each operator in plain torch, or calls the library where `own` is true; exact() restates each from its
definition in 64 bits.

A page of K or V is a cache of `page` rows as attn_prep lays it out: f16 [nkvh][page][256], or codes [nkvh][page][256]
followed by f16 scales [nkvh][page][8] (one per 32 values); a code has 8 bits, or 4: byte j < 16 of a block's 16 holds
value j in its low and value j + 16 in its high half, each the code, 0 .. 15, of (code - 8) * scale.
Types of a cache: 0 f16; 1 K and V in 8 bits; 2 K in 8 bits, V in 4.
table [sequences][max_pages] gives the pages of a sequence, pos its rows before this batch, and tokens cu[b] .. cu[b + 1] - 1
are its new ones.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
HD = 256  # head width
F16, Q8, Q8_Q4 = 0, 1, 2
PKG = os.path.join(os.getcwd(), "qwen27-engine_amd")
EPS = 1e-6
# the model's: 1e7^(-2/64) in float32
THETA = float(torch.tensor(1e7, dtype=torch.float32) ** torch.tensor(-2.0 / 64, dtype=torch.float32))
OUT = [torch.float32, torch.float16, torch.bfloat16]


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
    model = {"nqh": 24, "nkvh": 4}
    return [
        # the first tokens of the only chat: nothing but latency
        {"name": "attn_b1_37_q8", "kind": "attn", "B": 1, "new": 1, "short": 37, "long": 37, "page": 64, "type": Q8, **model},
        # plain decoding of an ordinary batch, prompts of every length
        {"name": "attn_b32_16k_q8", "kind": "attn", "B": 32, "new": 1, "short": 101, "long": 16384, "page": 64, "type": Q8, **model},
        # verification of three drafts beside each sequence's last token, V in 4 bits to hold more sequences
        {"name": "attn_b48_t4_32k_q4", "kind": "attn", "B": 48, "new": 4, "short": 500, "long": 32768, "page": 64, "type": Q8_Q4,
         **model},
        # one long document among short chats, f16 cache
        {"name": "attn_b8_one_131072_f16", "kind": "attn", "B": 8, "new": 1, "short": 333, "long": 131072, "one": True, "page": 128,
         "type": F16, **model},
        # the new rows of one decoded token written and read back: latency
        {"name": "prep_b1_q8", "kind": "prep", "B": 1, "new": 1, "short": 700, "long": 700, "page": 64, "type": Q8, "out": 1, **model},
        # a batch's step with drafts
        {"name": "prep_b64_t4_q4", "kind": "prep", "B": 64, "new": 4, "short": 10, "long": 150000, "page": 32, "type": Q8_Q4, "out": 1,
         **model},
        # the prompts of four sequences, one after another in a ragged batch of some 4000 tokens
        {"name": "prep_b4_prompts_f16", "kind": "prep", "B": 4, "new": 1999, "short": 1, "long": 30000, "page": 128, "type": F16,
         "out": 1, **model},
        # a short sequence's rows as float32
        {"name": "read_b1_500_q8_f32", "kind": "read", "B": 1, "new": 0, "short": 500, "long": 500, "page": 64, "type": Q8, "out": 0,
         **model},
        # sequences taken out of the pages as f16 caches
        {"name": "read_b8_32k_q4_f16", "kind": "read", "B": 8, "new": 0, "short": 1001, "long": 32768, "page": 64, "type": Q8_Q4,
         "out": 1, **model},
        # one sequence's three drafts, each drawn from a distribution of its own
        {"name": "verify_b1_t4", "kind": "verify", "B": 1, "new": 4, "vocab": 248320, "tree": False},
        # the same for a batch
        {"name": "verify_b64_t4", "kind": "verify", "B": 64, "new": 4, "vocab": 248320, "tree": False},
        # trees of drafts without probabilities, such as attn_tree attends to
        {"name": "verify_b4_tree64", "kind": "verify", "B": 4, "new": 64, "vocab": 248320, "tree": True},
    ]


def draw(rng):
    def size(lo, hi):
        return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    kind = rng.choice(["attn", "attn", "attn", "prep", "prep", "read", "verify", "verify"])
    if kind == "verify":
        tree = rng.random() < 0.4
        return {"kind": kind, "B": size(1, 16 if tree else 64), "new": rng.randint(2, 16 if tree else 4), "vocab": size(1000, 248320),
                "tree": tree}
    nqh, nkvh = rng.choice([(24, 4), (24, 4), (12, 2), (16, 2), (8, 8), (7, 1), (32, 4)])
    case = {"kind": kind, "nqh": nqh, "nkvh": nkvh, "type": rng.choice([F16, Q8, Q8, Q8_Q4]), "page": rng.choice([32, 64, 64, 128])}
    B, short = size(1, 64), size(1, 20000)
    if kind == "attn":
        case.update(new=rng.choice([1, 1, rng.randint(1, 8)]), short=short, long=size(short, 131072))
    elif kind == "prep":
        case.update(new=size(1, 2048), short=short, long=size(short, 150000), out=rng.choice([1, 2]))
    else:
        case.update(new=0, short=short, long=size(short, 65536), out=rng.randint(0, 2))
    case["B"] = B
    # no more than the largest listed case of its kind, of which the rows of the longest sequence are B times in all
    most, rows = {"attn": (550e6, 2_000_000), "prep": (280e6, 3_000_000), "read": (420e6, 400_000)}[kind]
    while case["B"] > 1 and (work(case)["bytes"] > most or case["B"] * case["long"] * nkvh > 4 * rows):
        case["B"] = (case["B"] + 1) // 2
    while case["long"] > case["short"] and (work(case)["bytes"] > most or case["B"] * case["long"] * nkvh > 4 * rows):
        case["long"] = max(case["short"], case["long"] * 3 // 4)
    return case


def _shares(n):
    """n numbers in [0, 1], spread evenly, in no order."""
    return [(0.5 + i * 0.6180339887498949) % 1.0 for i in range(n)]


def _lengths(case):
    """Rows of each sequence, those of the new tokens among them."""
    lo, hi, B = case["short"], case["long"], case["B"]
    if case.get("one"):
        return [hi if b == B // 2 else lo + 17 * b for b in range(B)]
    if B == 1:
        return [hi]
    return [round(math.exp(math.log(lo) + (math.log(hi) - math.log(lo)) * x)) for x in _shares(B)]


def _counts(case):
    """New tokens of each sequence: 1 to `new`, all of them in the first."""
    n = case["new"]
    return [n if b == 0 or n < 2 else 1 + int((n - 0.01) * x) for b, x in enumerate(_shares(case["B"]))]


def _rows(case):
    """(rows before the batch, new tokens) of each sequence."""
    new = _counts(case)
    if case["kind"] == "prep":
        return _lengths(case), new
    return [max(0, n - t) for n, t in zip(_lengths(case), new)], new


# ---------------------------------------------------------------- inputs
class _Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(int(seed) * 2 + 1)

    def n(self, *shape):
        return torch.randn(shape, device=DEV, generator=self.g)

    def u(self, *shape):
        return torch.rand(shape, device=DEV, generator=self.g)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _cu(new):
    at = [0]
    for n in new:
        at.append(at[-1] + n)
    return at


def _codes8(x):
    """int8 codes [.., 256] and f16 scales [.., 8] of f32 rows: d = amax / 127, code = round(x (1 / d)), halves away from 0."""
    b = x.unflatten(-1, (8, 32))
    d = (b.abs().amax(-1, keepdim=True).double() / 127).float()
    inv = torch.where(d > 0, (1 / d.double()).float(), torch.zeros_like(d))
    y = b * inv
    return torch.trunc(y.double() + y.sign() * 0.5).to(torch.int8).flatten(-2), d.squeeze(-1).to(torch.float16)


def _codes4(x):
    """uint8 [.., 128] of two codes each and f16 scales [.., 8]: d = e / -8 for the value e of largest magnitude (the
    negative one of two), code = min(15, trunc(x (1 / d) + 8.5))."""
    b = x.unflatten(-1, (8, 32))
    lo, hi = b.amin(-1, keepdim=True), b.amax(-1, keepdim=True)
    d = torch.where(-lo >= hi, lo, hi) / -8
    inv = torch.where(d != 0, (1 / d.double()).float(), torch.zeros_like(d))
    y = b * inv
    c = torch.trunc(y + 8.5).clamp(max=15).to(torch.uint8)
    return (c[..., :16] | (c[..., 16:] << 4)).flatten(-2), d.squeeze(-1).to(torch.float16)


def _bits(case, v):
    return 16 if case["type"] == F16 else 4 if v and case["type"] == Q8_Q4 else 8


def _row_bytes(case):
    """Bytes of a K and a V row of one head."""
    return sum(2 * HD if _bits(case, v) == 16 else HD * _bits(case, v) // 8 + 16 for v in (False, True))


def _pack(x, bits):
    """Pages' bytes [pages][..] from f32 rows x [pages][nkvh][page][256]."""
    if bits == 16:
        return x.to(torch.float16).flatten(1).view(torch.uint8)
    codes, scales = _codes8(x) if bits == 8 else _codes4(x)
    return torch.cat([codes.flatten(1).view(torch.uint8), scales.flatten(1).view(torch.uint8)], 1)


def _parts(buf, case, v):
    """Views of a buffer of pages: f16 [pages][nkvh][page][256], or codes [..][256 or 128] and scales [..][8]."""
    nkvh, page, bits = case["nkvh"], case["page"], _bits(case, v)
    if bits == 16:
        return buf.view(torch.float16).view(-1, nkvh, page, HD), None
    m = nkvh * page * HD * bits // 8
    codes, scales = buf[:, :m], buf[:, m:].view(torch.float16)
    return ((codes.view(torch.int8) if bits == 8 else codes).unflatten(1, (nkvh, page, HD * bits // 8)),
            scales.unflatten(1, (nkvh, page, 8)))


def prepare(case, seed):
    r, kind, B = _Rand(seed), case["kind"], case["B"]
    st = {"case": case}
    if kind == "verify":
        return _prepare_verify(st, r)
    nkvh, page = case["nkvh"], case["page"]
    pos, new = _rows(case)
    cu = _cu(new)
    T, end = cu[-1], [p + n for p, n in zip(pos, new)]
    st["max_pages"] = max(-(-n // page) for n in end) + 1
    # the pages lie in no order; those of a sequence behind its last row are none
    need = [-(-n // page) for n in end]
    n_pages = sum(need) + 3
    where = torch.randperm(n_pages, device=DEV, generator=r.g).to(torch.int32)
    at = _i32(_cu(need))[:-1, None] + torch.arange(st["max_pages"], device=DEV)
    used = torch.arange(st["max_pages"], device=DEV) < _i32(need)[:, None]
    st["table"] = torch.where(used, where[at.clamp(max=n_pages - 1).long()], torch.full_like(at, -1).int())
    st["pos"], st["cu"] = _i32(pos), _i32(cu)
    if kind == "prep":
        row = lambda v: nkvh * page * (2 * HD if _bits(case, v) == 16 else HD * _bits(case, v) // 8 + 16)  # noqa: E731
        st["k"], st["v"] = (torch.zeros(n_pages, row(v), dtype=torch.uint8, device=DEV) for v in (False, True))
        nqh = case["nqh"]
        st["qg"] = r.n(T, nqh, 2 * HD) * 2  # queries beside their gates
        st["kin"] = r.n(T, nkvh, HD) * torch.exp(0.5 * r.n(nkvh, HD))
        st["vin"] = r.n(T, nkvh, HD)
        st["qw"], st["kw"] = 1 + 0.1 * r.n(HD), 1 + 0.1 * r.n(HD)
        st["rdelta"] = torch.zeros(B, dtype=torch.int32, device=DEV)
        st["qn"] = torch.zeros(T, nqh, HD, device=DEV)
        st["count"], st["n_out"] = _i32(new), max(new)
    else:
        # keys with channels of unequal strength and a shared direction that many queries look for
        chan, topic = torch.exp(0.4 * r.n(nkvh, 1, HD)), r.n(nkvh, 1, HD)
        k = r.n(n_pages, nkvh, page, HD) * chan
        st["k"] = _pack(k.add_(topic * (r.u(n_pages, nkvh, page, 1) < 0.02) * 0.7), _bits(case, False))
        del k
        st["v"] = _pack(r.n(n_pages, nkvh, page, HD), _bits(case, True))
    if kind == "read":
        st["count"], st["n_out"] = _i32(end), max(end)
    if kind in ("prep", "read"):
        st["ko"], st["vo"] = (torch.zeros(B, nkvh, st["n_out"], HD, dtype=OUT[case["out"]], device=DEV) for _ in range(2))
    if kind == "attn":
        nqh, g = case["nqh"], case["nqh"] // nkvh
        st["q"] = (r.n(T, nkvh, g, HD) * 1.5 + topic[None] * 0.8).reshape(T, nqh, HD).contiguous()
        st["scale"] = HD ** -0.5
        st["o"], st["lse"] = torch.empty(T, nqh, HD, device=DEV), torch.empty(T, nqh, device=DEV)
    return st


def _prepare_verify(st, r):
    c = st["case"]
    B, V, new = c["B"], c["vocab"], c["new"]
    counts = [new] * B if c["tree"] else _counts(c)
    cu = _cu(counts)
    T = cu[-1]
    st["cu"], st["pos"] = _i32(cu), _i32([100 + 7 * b for b in range(B)])
    # a few likely tokens before a long tail, as a language model's next-token probabilities have
    logits = r.n(T, V).mul_(2.0)
    logits.scatter_add_(1, (r.u(T, 8) * V).long(), 9 + 2 * r.n(T, 8))
    st["p"] = torch.softmax(logits, -1)
    st["u"], st["u_last"] = r.u(T), r.u(B)
    if c["tree"]:
        # each token follows one of the eight before it; the drafts are likely tokens of their parent's distribution
        back = 1 + (r.u(B, new) * 8).int()
        parent = (torch.arange(new, device=DEV, dtype=torch.int32) - back).clamp(min=0)
        parent[:, 0] = -1
        st["parent"] = parent.view(-1).contiguous()
        row = (torch.arange(B, device=DEV)[:, None] * new + parent.clamp(min=0)).view(-1)
        top = st["p"].topk(4, dim=1).indices
        st["ids"] = top[row, (r.u(T) * 4).long()].to(torch.int32)
        return st
    # the drafts' probabilities: those of a smaller model, near the target's; row t belongs to token t
    q = torch.softmax(logits.add_(r.n(T, V).mul_(0.7)), -1)
    st["q"] = torch.roll(q, 1, 0)
    st["ids"] = torch.multinomial(st["q"], 1, generator=r.g).view(-1).to(torch.int32)
    return st


# ---------------------------------------------------------------- the plain forms
def _gather(buf, st, v, n):
    """Values [B][nkvh][n][256], f32, of rows 0 .. n - 1 of every sequence (rows that it does not have: anything)."""
    c = st["case"]
    pages = -(-n // c["page"])
    t = st["table"][:, :pages].clamp(min=0).long()
    codes, scales = _parts(buf, c, v)
    x = codes[t].transpose(1, 2).flatten(2, 3)[:, :, :n]  # [B][nkvh][n][..]
    if scales is None:
        return x.float()
    d = scales[t].transpose(1, 2).flatten(2, 3)[:, :, :n].float()
    x = x.unflatten(-1, (8, -1))
    if _bits(c, v) == 4:
        x = torch.cat([x & 15, x >> 4], -1).float() - 8
    return (x.float() * d[..., None]).flatten(-2)


def _spread(x, st, fill):
    """Rows x [T][..] of the tokens as [B][new][..], `fill` where a sequence has fewer."""
    c = st["case"]
    cu = st["cu"].long()
    t = torch.arange(c["new"], device=DEV)
    has = t < (cu[1:] - cu[:-1])[:, None]
    at = torch.where(has, cu[:-1, None] + t, torch.zeros_like(t))
    y = x[at]
    return torch.where(has.view(has.shape + (1,) * (y.dim() - 2)), y, torch.full_like(y, fill)), has


def _run_attn(st):
    c = st["case"]
    nkvh, g, B, new = c["nkvh"], c["nqh"] // c["nkvh"], c["B"], c["new"]
    n = (st["max_pages"] - 1) * c["page"]
    q, has = _spread(st["q"], st, 0.0)
    q = q.view(B, new, nkvh, g, HD).permute(0, 2, 1, 3, 4).reshape(B * nkvh, new * g, HD) * st["scale"]
    k = _gather(st["k"], st, False, n).view(B * nkvh, n, HD)
    s = torch.bmm(q, k.transpose(1, 2).contiguous()).view(B, nkvh, new, g, n)
    del k
    seen = torch.arange(n, device=DEV) <= (st["pos"][:, None] + torch.arange(new, device=DEV))[..., None]
    s.masked_fill_(~seen[:, None, :, None], float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    v = _gather(st["v"], st, True, n).view(B * nkvh, n, HD)
    o = torch.bmm(p.view(B * nkvh, new * g, n), v).view(B, nkvh, new, g, HD) / total
    lse = (m + total.log()).squeeze(-1)
    return (o.permute(0, 2, 1, 3, 4).reshape(B, new, nkvh * g, HD)[has], lse.permute(0, 2, 1, 3).reshape(B, new, nkvh * g)[has])


def _angles(st):
    """cos and sin [T][32] of the rotation: the angle is the float32 product of the position and theta^j in float32."""
    T = st["qn"].shape[0]
    t = torch.arange(T, device=DEV)
    b = torch.searchsorted(st["cu"][1:].long(), t, right=True)
    where = (st["pos"][b] - st["rdelta"][b] + t - st["cu"][b]).float()
    freq = torch.tensor([THETA ** j for j in range(32)], dtype=torch.float32, device=DEV)
    a = (where[:, None] * freq).double()
    return a.cos().float(), a.sin().float()


def _norm_rope(x, w, cos, sin):
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
    a, b, rest = y[..., :32], y[..., 32:64], y[..., 64:]
    cos, sin = cos[:, None], sin[:, None]
    return torch.cat([a * cos - b * sin, a * sin + b * cos, rest], -1)


def _put(buf, st, v, x):
    """Writes the new rows x [T][nkvh][256] to their places in the pages."""
    c = st["case"]
    t = torch.arange(x.shape[0], device=DEV)
    b = torch.searchsorted(st["cu"][1:].long(), t, right=True)
    row = st["pos"][b].long() + t - st["cu"][b]
    page, slot = st["table"][b, row // c["page"]].long(), row % c["page"]
    parts = _parts(buf, c, v)
    values = {16: lambda: (x.to(torch.float16), None), 8: lambda: _codes8(x), 4: lambda: _codes4(x)}[_bits(c, v)]()
    parts[0][page, :, slot] = values[0]
    if values[1] is not None:
        parts[1][page, :, slot] = values[1]


def _read_back(st, first, count, n):
    """Rows first[b] .. first[b] + count[b] - 1 of each sequence into st's ko and vo, from their first row on."""
    c = st["case"]
    i = torch.arange(n, device=DEV)
    row = (first[:, None] + i).long()
    page = st["table"].gather(1, (row // c["page"]).clamp(max=st["max_pages"] - 1)).clamp(min=0).long()
    has = (i < count[:, None])[:, None, :, None]
    for buf, out, v in ((st["k"], st["ko"], False), (st["v"], st["vo"], True)):
        codes, scales = _parts(buf, c, v)
        x = codes[page, :, row % c["page"]].transpose(1, 2)  # [B][nkvh][n][..]
        if scales is None:
            x = x.float()
        else:
            x = x.unflatten(-1, (8, -1))
            if _bits(c, v) == 4:
                x = torch.cat([x & 15, x >> 4], -1).float() - 8
            x = (x.float() * scales[page, :, row % c["page"]].transpose(1, 2).float()[..., None]).flatten(-2)
        torch.where(has, x.to(out.dtype), out, out=out)


def _run_prep(st):
    cos, sin = _angles(st)
    st["qn"].copy_(_norm_rope(st["qg"][..., :HD], st["qw"], cos, sin))
    _put(st["k"], st, False, _norm_rope(st["kin"], st["kw"], cos, sin))
    _put(st["v"], st, True, st["vin"])
    _read_back(st, st["pos"], st["count"], st["n_out"])


def _weights(x):
    """Multiples of 2^-40 in [0, 1], whose float64 sums are exact in any order."""
    return (x.clamp(0, 1) + 6144.0) - 6144.0


def _pick(w, u):
    """Smallest index whose sum up to it exceeds u times the whole sum."""
    c = w.cumsum(-1)
    return torch.searchsorted(c, u.double()[:, None] * c[:, -1:], right=True).squeeze(1)


def _run_chain(st):
    c = st["case"]
    ids, has = _spread(st["ids"].long(), st, 0)
    u, _ = _spread(st["u"], st, 0.0)
    B, new = ids.shape
    row = st["cu"][:-1, None].long() + torch.arange(new, device=DEV)
    last = row.clamp(max=st["p"].shape[0] - 1)
    ok = u[:, 1:].double() * st["q"][last[:, 1:], ids[:, 1:]].double() < st["p"][last[:, :-1], ids[:, 1:]].double()
    n = (ok & has[:, 1:]).long().cumprod(1).sum(1)  # accepted drafts
    stop = n + 1 < has.sum(1)  # one was refused
    at = row.gather(1, n[:, None]).squeeze(1)
    p = st["p"][at].double()
    q = st["q"][(at + 1).clamp(max=st["q"].shape[0] - 1)].double() * stop[:, None]
    w = _weights(p - q)
    w = torch.where(w.sum(1, keepdim=True) > 0, w, _weights(p))
    token = _pick(w, st["u_last"])
    i = torch.arange(new, device=DEV)
    nxt = torch.cat([ids[:, 1:], ids[:, :1]], 1)
    out = torch.where(i < n[:, None], nxt, torch.where(i == n[:, None], token[:, None], torch.full_like(nxt, -1)))
    path = torch.where(i <= n[:, None], i, torch.full_like(nxt, -1))
    return out[has].int(), path[has].int(), (n + 1).int()


def _run_tree(st):
    c = st["case"]
    B, new, V = c["B"], c["new"], c["vocab"]
    ids, parent, u = st["ids"].view(B, new).long(), st["parent"].view(B, new), st["u"].view(B, new).double()
    p = st["p"].view(B, new, V)
    b = torch.arange(B, device=DEV)
    w = p[b[:, None], parent.clamp(min=0).long(), ids].double()  # the drafts' probabilities after their parents
    node = torch.zeros(B, dtype=torch.int32, device=DEV)
    rest = torch.ones(B, dtype=torch.float64, device=DEV)
    tried = torch.zeros(B, new, dtype=torch.bool, device=DEV)
    path = torch.zeros(B, new, dtype=torch.bool, device=DEV)
    path[:, 0] = True
    for t in range(1, new):  # a walk: each step needs the one before
        here = parent[:, t] == node
        again = (tried & (ids == ids[:, t:t + 1])).any(1)
        x = torch.where(again, torch.zeros_like(rest), w[:, t])
        yes = here & (u[:, t] * rest < x)
        no = here & ~yes
        node = torch.where(yes, torch.full_like(node, t), node)
        rest = torch.where(yes, torch.ones_like(rest), torch.where(no, rest - x, rest))
        tried &= ~yes[:, None]
        tried[:, t] = no
        path[:, t] = yes
    left = p[b, node.long()].double()
    left = left.scatter(1, torch.where(tried, ids, ids[:, :1] * 0), torch.where(tried, torch.zeros_like(w), left[:, :1]))
    # index 0 stands for the drafts that were not tried; where it was, it is zero
    left[:, 0] = torch.where((tried & (ids == 0)).any(1), torch.zeros_like(rest), p[b, node.long(), 0].double())
    token = _pick(_weights(left), st["u_last"])
    n = path.sum(1)
    i = torch.arange(new, device=DEV)
    order = torch.where(path, i, i + new).sort(1).values  # the accepted tokens first
    order = torch.where(i < n[:, None], order, torch.full_like(order, -1))
    nxt = torch.cat([order[:, 1:], torch.full_like(order[:, :1], -1)], 1)
    out = torch.where(nxt >= 0, ids.gather(1, nxt.clamp(min=0)), torch.where(i == n[:, None] - 1, token[:, None], torch.full_like(nxt, -1)))
    return out.view(-1).int(), order.view(-1).int(), n.int()


# ---------------------------------------------------------------- one pass
def _kv(st):
    """The handle and the workspace that a program keeps beside its pages."""
    o, c = _ops(), st["case"]
    if "kv" not in st:
        st["kv"] = o.KvPages(st["k"], st["v"], st["table"], c["nkvh"], c["page"], c["type"])
        if c["kind"] == "attn":
            st["ws"] = torch.empty(o.attn_paged_ws_bytes(st["kv"], st["q"].shape[0], c["new"], c["nqh"]), dtype=torch.uint8, device=DEV)
    return o, st["kv"]


def run(st):
    c = st["case"]
    kind = c["kind"]
    if kind == "verify":
        if own:
            o = _ops()
            if "ws" not in st:
                st["ws"] = torch.empty(o.draft_verify_ws_bytes(c["B"], c["vocab"]), dtype=torch.uint8, device=DEV)
                st["out"], st["path"] = torch.empty_like(st["ids"]), torch.empty_like(st["ids"])
                st["n_path"] = torch.empty(c["B"], dtype=torch.int32, device=DEV)
            o.draft_verify(st["p"], st.get("q"), st["ids"], st.get("parent"), st["u"], st["u_last"], st["cu"], c["B"], c["vocab"],
                           st["out"], st["path"], st["n_path"], st["ws"], pos=st["pos"])
            out, path, n = st["out"], st["path"], st["n_path"]
        else:
            out, path, n = _run_tree(st) if c["tree"] else _run_chain(st)
            st["pos"] += n
        return {"out": out, "path": path, "n_path": n, "pos": st["pos"]}
    if kind == "attn":
        if own:
            o, kv = _kv(st)
            o.attn_paged(st["q"], kv, st["pos"], st["cu"], st["q"].shape[0], c["new"], st["scale"], c["nqh"], st["o"], st["ws"],
                         lse=st["lse"])
            return {"o": st["o"], "lse": st["lse"]}
        o, lse = _run_attn(st)
        return {"o": o, "lse": lse}
    if kind == "prep":
        if own:
            o, kv = _kv(st)
            o.attn_prep_paged(st["qg"], st["kin"], st["vin"], st["qw"], st["kw"], st["qn"], kv, st["pos"], st["cu"], st["qn"].shape[0],
                              EPS, THETA, c["nqh"], rdelta=st["rdelta"])
            o.kv_pages_read(kv, st["pos"], st["count"], st["n_out"], st["ko"], st["vo"])
        else:
            _run_prep(st)
        return {"qn": st["qn"], "k": st["ko"], "v": st["vo"]}
    if own:
        o, kv = _kv(st)
        o.kv_pages_read(kv, None, st["count"], st["n_out"], st["ko"], st["vo"])
    else:
        _read_back(st, torch.zeros_like(st["pos"]), st["count"], st["n_out"])
    return {"k": st["ko"], "v": st["vo"]}


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind, B = case["kind"], case["B"]
    if kind == "verify":
        # the row of p that the next token is drawn from; where a draft was refused, as in about half of the chains, one of q
        return {"bytes": B * case["vocab"] * (4.0 if case["tree"] else 6.0), "flops": 0.0}
    pos, new = _rows(case)
    nqh, nkvh, T = case["nqh"], case["nkvh"], sum(new)
    rows = sum(p + n for p, n in zip(pos, new))
    row = _row_bytes(case)
    if kind == "attn":
        return {"bytes": float(nkvh * rows * row + 4 * T * nqh * (2 * HD + 1)),
                "flops": 4.0 * HD * nqh * sum(n * (p + n) for p, n in zip(pos, new))}
    back = 2 * HD * (4 if case["out"] == 0 else 2)  # a row of K and of V read back
    if kind == "read":
        return {"bytes": float(nkvh * rows * (row + back)), "flops": 0.0}
    return {"bytes": float(T * (nqh * HD * 8 + nkvh * (HD * 8 + 2 * row + back))), "flops": 0.0}


# ---------------------------------------------------------------- from the definitions, in 64 bits
def _exact_rows(buf, case, v, pages, n):
    """Rows 0 .. n - 1, [nkvh][n][256], of the sequence whose pages are listed."""
    nkvh, page, bits = case["nkvh"], case["page"], _bits(case, v)
    x = buf[pages[:-(-n // page)].long()]
    if bits == 16:
        return x.view(torch.float16).view(-1, nkvh, page, HD).permute(1, 0, 2, 3).reshape(nkvh, -1, HD)[:, :n].double()
    m = nkvh * page * HD * bits // 8
    d = x[:, m:].contiguous().view(torch.float16).view(-1, nkvh, page, 8).double().repeat_interleave(32, -1)
    y = x[:, :m].contiguous()
    if bits == 8:
        y = y.view(torch.int8).view(-1, nkvh, page, HD).double()
    else:
        y = y.view(-1, nkvh, page, 8, 16).int()
        y = torch.stack([y % 16, y // 16], -2).view(-1, nkvh, page, HD).double() - 8
    return (y * d).permute(1, 0, 2, 3).reshape(nkvh, -1, HD)[:, :n]


def exact(case, seed):
    kind = case["kind"]
    if kind == "verify":
        return None  # whole numbers: which tokens are accepted and drawn
    st = prepare(case, seed)
    pos, new = _rows(case)
    cu, nkvh, nqh = _cu(new), case["nkvh"], case["nqh"]
    if kind == "read":
        out = [torch.zeros(case["B"], nkvh, st["n_out"], HD, dtype=torch.float64, device=DEV) for _ in range(2)]
        for b, n in enumerate(p + t for p, t in zip(pos, new)):
            for buf, y, v in ((st["k"], out[0], False), (st["v"], out[1], True)):
                y[b, :, :n] = _exact_rows(buf, case, v, st["table"][b], n)
        return {"k": out[0], "v": out[1]}
    if kind == "attn":
        os, ls, g = [], [], nqh // nkvh
        for b in range(case["B"]):
            n, t = pos[b] + new[b], new[b]
            k, v = (_exact_rows(st[w], case, w == "v", st["table"][b], n) for w in ("k", "v"))
            q = st["q"][cu[b]:cu[b + 1]].double().view(t, nkvh, g, HD).permute(1, 0, 2, 3).reshape(nkvh, t * g, HD)
            s = torch.bmm(q, k.transpose(1, 2).contiguous()).mul_(st["scale"]).view(nkvh, t, g, n)
            hidden = torch.arange(n, device=DEV)[None] > pos[b] + torch.arange(t, device=DEV)[:, None]
            s.masked_fill_(hidden[:, None], float("-inf"))
            l = torch.logsumexp(s, -1)
            o = torch.bmm(torch.exp(s - l[..., None]).view(nkvh, t * g, n), v).view(nkvh, t, g, HD)
            os.append(o.permute(1, 0, 2, 3).reshape(t, nqh, HD))
            ls.append(l.permute(1, 0, 2).reshape(t, nqh))
        return {"o": torch.cat(os), "lse": torch.cat(ls)}
    # prep: queries, and the new rows before they were quantised are no output; V's values follow from its inputs alone
    freq = (torch.tensor(THETA, dtype=torch.float64) ** torch.arange(32)).float()
    where = torch.tensor([p + t for p, n in zip(pos, new) for t in range(n)], dtype=torch.float32)
    a = (where[:, None] * freq).double().to(DEV)[:, None]  # the angle is a float32 product by definition

    def turned(x, w):
        x = x.double()
        y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / HD + EPS) * w.double()
        z = y.clone()
        z[..., :32] = y[..., :32] * torch.cos(a) - y[..., 32:64] * torch.sin(a)
        z[..., 32:64] = y[..., :32] * torch.sin(a) + y[..., 32:64] * torch.cos(a)
        return z

    return {"qn": turned(st["qg"][..., :HD], st["qw"]), "k": None, "v": None}
