"""Operators over paged session caches: what is measured, in plain torch and through the library.

A pool holds K/V pages of every layer, `[layers][pages][2 * kv_heads][page][128]` in bf16 or as INT8 /
INT4 codes with f16 scales per 32 dims; a session is a row of page ids and a token count.

Kinds:
  attend   s2pk_paged_attention: ragged rows of many sessions over their pages, causal or
           with a draft tree's visibility words; one decode row a session up to prompt chunks.
  append   s2pk_paged_append: fused qkv rows to normed, rotated queries and appended K/V.
  share    s2pk_pages_fork + s2pk_pages_reserve: continuations of one prompt share its pages,
           then every session gets room for its next tokens (a shared last page is copied).
  reclaim  s2pk_pages_free + s2pk_pages_compact: finished sessions give their pages back and the
           pages still in use move to the front of the pool.
"""
import ctypes
import math
import os
import sys

import torch

own = False

DEV = "cuda"
HD = 128
EPS = 1e-6
BASE = 1e6
TREE16 = [-1, 0, 0, 1, 1, 2, 2, 3, 3, 4, 5, 6, 6, 7, 8, 10, 11]


# ------------------------------------------------------------------ the cases

def _attend(name, bits, sessions, shortest, longest, rows, page, tree=False, qh=32, kvh=8):
    return {"name": name, "kind": "attend", "bits": bits, "sessions": sessions,
            "shortest": shortest, "longest": longest, "rows": rows, "page": page, "tree": tree,
            "qh": qh, "kvh": kvh}


def _append(name, bits, sessions, shortest, longest, rows, page, qh=32, kvh=8):
    return {"name": name, "kind": "append", "bits": bits, "sessions": sessions,
            "shortest": shortest, "longest": longest, "rows": rows, "page": page, "qh": qh,
            "kvh": kvh}


def listed():
    return [
        # the first decode row of one short session: latency alone
        _attend("attend_one_row_100", 16, 1, 100, 100, 1, 16),
        # a lockstep decode tick of 32 ragged sessions over 4-bit pages
        _attend("attend_decode_int4_32", 4, 32, 511, 4095, 1, 32),
        # decode of 16 long sessions over bf16 pages
        _attend("attend_decode_bf16_16x8192", 16, 16, 8191, 8191, 1, 64),
        # eight K = 4 chains to verify over INT8 pages of the smallest size, ragged
        _attend("attend_verify_int8_8x5", 8, 8, 256, 4096, 5, 16),
        # four 16-node draft trees at 8,192 tokens
        _attend("attend_tree_bf16_4x17", 16, 4, 8192, 8192, 17, 64, True),
        # prompt chunks of two sessions behind their earlier chunks
        _attend("attend_prefill_bf16_2x2048", 16, 2, 1500, 2048, 2048, 64),
        # the rows of a lockstep tick of 64 sessions into bf16 pages
        _append("append_tick_bf16_64", 16, 64, 17, 4001, 1, 32),
        # prompt chunks of four sessions into INT8 pages
        _append("append_prefill_int8_4x2048", 8, 4, 0, 1000, 2048, 64),
        # one 1,000-token prompt forked into four continuations
        {"name": "share_4_of_1000", "kind": "share", "sessions": 8, "forks": 4, "tokens": 1000,
         "page": 16, "layers": 4, "pages": 700, "want": 1},
        # a long prompt forked into 32 continuations of drafts, whole backbone, page bookkeeping
        # of a large pool
        {"name": "share_32_of_4090", "kind": "share", "sessions": 64, "forks": 32, "tokens": 4090,
         "page": 16, "layers": 36, "pages": 1500, "want": 17},
        # a few pages to move
        {"name": "reclaim_12_pages", "kind": "reclaim", "sessions": 16, "live": 100, "moved": 12,
         "page": 16, "layers": 4, "pages": 333},
        # a pool that half of the sessions left, whole backbone
        {"name": "reclaim_200_pages", "kind": "reclaim", "sessions": 64, "live": 600, "moved": 200,
         "page": 16, "layers": 36, "pages": 1500},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "append", "append", "share", "reclaim"])
    page = rng.choice([16, 32, 64, 128])
    kvh, group = rng.choice([(8, 4), (8, 4), (8, 4), (4, 8), (2, 4), (8, 1), (1, 16), (4, 2)])
    if kind == "attend":
        bits = rng.choice([16, 16, 8, 4])
        shape = rng.choice(["decode", "decode", "verify", "tree", "prefill"])
        sessions = _log_int(rng, 1, 48) if shape != "prefill" else rng.randint(1, 4)
        longest = _log_int(rng, 1, 8000 if shape != "prefill" else 2000)
        rows = {"decode": 1, "verify": rng.randint(2, 8), "tree": 17,
                "prefill": _log_int(rng, 20, 1500)}[shape]
        while sessions * longest > 131072 or sessions * rows > 2048:
            sessions = max(1, sessions // 2)
        c = _attend("", bits, sessions, max(0, longest // rng.randint(1, 8)), longest, rows, page,
                    shape == "tree", kvh * group, kvh)
    elif kind == "append":
        rows = _log_int(rng, 1, 1500)
        sessions = max(1, min(_log_int(rng, 1, 64), 6000 // rows))
        longest = _log_int(rng, 1, 4000)
        c = _append("", rng.choice([16, 16, 8, 4]), sessions, longest // 2, longest, rows, page,
                    kvh * group, kvh)
    elif kind == "share":
        forks = _log_int(rng, 1, 24)
        tokens = _log_int(rng, 3, 4000)
        page = rng.choice([16, 32])
        want = rng.choice([1, 5, 17, rng.randint(2, 100)])
        c = {"kind": "share", "sessions": 3 + forks + rng.randint(0, 9), "forks": forks,
             "tokens": tokens, "page": page, "layers": rng.randint(1, 18), "want": want}
        c["pages"] = 3 * (tokens // page + 1) + (forks + 6) * (want // page + 3) + rng.randint(0, 200)
    else:
        live = _log_int(rng, 9, 500)
        c = {"kind": "reclaim", "sessions": rng.randint(4, 40), "live": live,
             "moved": rng.randint(1, max(1, live // 3)), "page": rng.choice([16, 32]),
             "layers": rng.randint(1, 18)}
        c["pages"] = 2 * live + rng.randint(50, 300)
    c.pop("name", None)
    return c


# -------------------------------------------------------------- shapes of a case

def _spread(lo, hi, n):
    """n lengths between lo and hi, the last one hi"""
    return [lo + int((hi - lo) * ((0.381966 * (n - 1 - i)) % 1.0)) if i < n - 1 else hi
            for i in range(n)]


def _lens(c):
    return _spread(c["shortest"], c["longest"], c["sessions"])


def _rows(c):
    """rows of every session: alike for drafts and ticks, ragged for prompt chunks"""
    r = c["rows"]
    if r < 18:
        return [r] * c["sessions"]
    return _spread(r * 2 // 3, r, c["sessions"])


def _el(bits):
    return {16: 128, 8: 128, 4: 64}[bits]


def _slot_bytes(bits):
    return {16: 256, 8: 136, 4: 72}[bits]


def _vis(c):
    """slots a row sees, summed over the rows (and the tree's depth of each node)"""
    if not c.get("tree"):
        return sum(sum(n + i + 1 for i in range(r)) for n, r in zip(_lens(c), _rows(c)))
    return sum(sum(n + _depth(i) + 1 for i in range(r)) for n, r in zip(_lens(c), _rows(c)))


def _depth(i):
    d = 0
    while TREE16[i] >= 0:
        d, i = d + 1, TREE16[i]
    return d


def _words():
    """visibility words of the draft tree: a node sees its ancestors and itself"""
    out = []
    for i in range(len(TREE16)):
        w, j = 0, i
        while j >= 0:
            w |= 1 << j
            j = TREE16[j]
        out.append(w)
    return out


def work(c):
    k = c["kind"]
    if k == "attend":
        rows, spans = sum(_rows(c)), sum(n + r for n, r in zip(_lens(c), _rows(c)))
        return {"bytes": spans * 2 * c["kvh"] * _slot_bytes(c["bits"]) + 2 * rows * c["qh"] * 256,
                "flops": 4 * 128 * c["qh"] * _vis(c)}
    if k == "append":
        rows = sum(_rows(c))
        return {"bytes": rows * ((2 * c["qh"] + 2 * c["kvh"]) * 256
                                 + 2 * c["kvh"] * _slot_bytes(c["bits"]) + 256),
                "flops": rows * 128 * (6 * c["qh"] + 10 * c["kvh"])}
    page = 16 * c["page"] * 256 * c["layers"]
    state = 8 * c["pages"]
    if k == "share":
        # the parent and its forks all go on writing behind a partly filled page: each but
        # the last of them needs a copy of it
        copied = c["forks"] if c["tokens"] % c["page"] else 0
        return {"bytes": 2 * copied * page + state + 8 * c["forks"] * (c["tokens"] // c["page"] + 1),
                "flops": 0}
    return {"bytes": 2 * c["moved"] * page + state, "flops": 0}


# ------------------------------------------------------------------ the inputs

def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1000003 + salt) & 0x7FFFFFFFFFFFFFFF)
    return g


def _randn(g, *shape, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32) * scale).to(dtype)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _pool(g, bits, layers, pages, kvh, page):
    """a pool whose every slot holds values (codes and scales of values of unit variance)"""
    shape = (layers, pages, 2 * kvh, page)
    if bits == 16:
        kv = torch.empty(*shape, HD, dtype=torch.bfloat16, device=DEV)
        kv.normal_(generator=g)
        return kv, None
    if bits == 8:
        kv = torch.randint(-127, 128, (*shape, HD), generator=g, device=DEV, dtype=torch.int8)
        top = 127 * 0.577
    else:
        kv = torch.randint(-128, 128, (*shape, HD // 2), generator=g, device=DEV, dtype=torch.int8)
        top = 8 * 0.577
    scales = torch.rand(*shape, 4, generator=g, device=DEV) * 0.6 + 0.7
    return kv, (scales / top).to(torch.float16)


def _rope_table(n_pos):
    """[n_pos][64] (cos, sin) of the rotation, in bf16"""
    i = torch.arange(64, dtype=torch.float64, device=DEV)
    inv = (1.0 / torch.pow(torch.tensor(BASE, dtype=torch.float64, device=DEV), 2 * i / HD)).float()
    ang = torch.arange(n_pos, dtype=torch.float32, device=DEV)[:, None] * inv[None, :]
    return torch.stack([ang.double().cos(), ang.double().sin()], -1).float().to(torch.bfloat16)


def prepare(case, seed):
    c, g = dict(case), _gen(seed, 77)
    k = c["kind"]
    if k in ("attend", "append"):
        lens, rows = _lens(c), _rows(c)
        need = [-(-(n + r) // c["page"]) for n, r in zip(lens, rows)]
        layers = 2
        pages = sum(need) + 3
        st = {"case": c, "layer": 1, "max_rows": max(rows),
              "max_len": max(n + r for n, r in zip(lens, rows)), "rows": sum(rows)}
        st["kv"], st["scales"] = _pool(g, c["bits"], layers, pages, c["kvh"], c["page"])
        perm = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
        table = torch.full((c["sessions"], max(need)), -1, dtype=torch.int32, device=DEV)
        at = 0
        for s, n in enumerate(need):
            table[s, :n] = perm[at:at + n]
            at += n
        st["table"] = table
        st["len"] = _i32(lens)
        row0 = [0]
        for r in rows:
            row0.append(row0[-1] + r)
        st["row0"] = _i32(row0)
        if k == "attend":
            # a few dims carry more of the scores, as after trained norms
            w = _randn(g, HD, scale=0.4, dtype=torch.float32).exp()
            st["q"] = (_randn(g, st["rows"], c["qh"], HD, dtype=torch.float32) * w).to(torch.bfloat16)
            st["vis"] = None
            if c["tree"]:
                st["vis"] = torch.tensor(_words() * c["sessions"], dtype=torch.int64, device=DEV)
        else:
            st["qkv"] = _randn(g, st["rows"], (c["qh"] + 2 * c["kvh"]) * HD, scale=2.0)
            st["qn"] = _randn(g, HD, scale=0.1, dtype=torch.float32).add_(1).to(torch.bfloat16)
            st["kn"] = _randn(g, HD, scale=0.1, dtype=torch.float32).add_(1).to(torch.bfloat16)
            st["rope"] = _rope_table(st["max_len"] + 1)
        return st
    st = {"case": c}
    st["kv"], _ = _pool(g, 16, c["layers"], c["pages"], 8, c["page"])
    n, pages = c["sessions"], c["pages"]
    perm = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    if k == "share":
        held = -(-c["tokens"] // c["page"])
        # the parent, two bystanders of half its length, the rest empty
        owned = [held, held // 2, held // 2] + [0] * (n - 3)
        toks = [c["tokens"], (held // 2) * c["page"], (held // 2) * c["page"]] + [0] * (n - 3)
        width = held + c["want"] // c["page"] + 2
        order = perm
        st["src"] = _i32([0] * c["forks"])
        st["dst"] = _i32(list(range(3, 3 + c["forks"])))
        st["want"] = _i32([c["want"] if s == 0 or 3 <= s < 3 + c["forks"] else 0 for s in range(n)])
    else:
        # even sessions stay, odd ones are freed; `moved` of the pages that stay lie behind
        # the first `live` of the pool
        live, moved = c["live"], min(c["moved"], c["live"], pages - c["live"])
        low = torch.randperm(live, generator=g, device=DEV)
        high = torch.randperm(pages - live, generator=g, device=DEV) + live
        stay = torch.cat([low[:live - moved], high[:moved]])
        stay = stay[torch.randperm(live, generator=g, device=DEV)]
        gone = torch.cat([low[live - moved:], high[moved:]])
        gone = gone[torch.randperm(gone.numel(), generator=g, device=DEV)]
        n_even, n_odd = (n + 1) // 2, n // 2
        leave = min(gone.numel() - 3, live)
        e = [live // n_even + (i < live % n_even) for i in range(n_even)]
        o = [leave // n_odd + (i < leave % n_odd) for i in range(n_odd)]
        owned = [e[s // 2] if s % 2 == 0 else o[s // 2] for s in range(n)]
        toks = [max(0, p * c["page"] - (s % 5)) for s, p in enumerate(owned)]
        width = max(owned) + 2
        parts, ie, io = [], 0, 0
        for s, p in enumerate(owned):
            if s % 2 == 0:
                parts.append(stay[ie:ie + p])
                ie += p
            else:
                parts.append(gone[io:io + p])
                io += p
        order = torch.cat(parts).to(torch.int32)
        st["keep"] = _i32([-1 if s % 2 == 0 else 0 for s in range(n)])
    # one buffer: ref [pages], table [n][width], held [n], len [n]
    ref = torch.zeros(pages, dtype=torch.int32, device=DEV)
    ref[order[:sum(owned)].long()] = 1
    table = torch.full((n, width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for s, p in enumerate(owned):
        table[s, :p] = order[at:at + p]
        at += p
    st["width"] = width
    st["start"] = torch.cat([ref, table.reshape(-1), _i32(owned), _i32(toks)])
    st["state"] = st["start"].clone()
    return st


def _views(st):
    c = st["case"]
    n, w, pages, s = c["sessions"], st["width"], c["pages"], st["state"]
    a = pages + n * w
    return s[:pages], s[pages:a].view(n, w), s[a:a + n], s[a + n:a + 2 * n]


# -------------------------------------------------------------- the plain forms

def _values(kv, scales, bits):
    """what codes stand for, in float32"""
    if bits == 16:
        return kv.float()
    if bits == 4:
        lo, hi = ((kv & 15) ^ 8) - 8, kv >> 4
        kv = torch.stack([lo, hi], -1).flatten(-2)
    return (kv.float().unflatten(-1, (4, 32)) * scales.float()[..., None]).flatten(-2)


def _session_kv(st):
    """every session's pages as [sessions, slots, 2 kvh, 128] in float32"""
    at = st["table"].clamp_min(0).long()
    kv = st["kv"][st["layer"]][at]
    sc = None if st["scales"] is None else st["scales"][st["layer"]][at]
    v = _values(kv, sc, st["case"]["bits"])  # [S, P, 2 kvh, page, 128]
    return v.permute(0, 2, 1, 3, 4).flatten(2, 3)  # [S, 2 kvh, P * page, 128]


def _plain_attend(st):
    c = st["case"]
    S, R, KVH, G = c["sessions"], st["max_rows"], c["kvh"], c["qh"] // c["kvh"]
    kv = _session_kv(st)
    T = kv.shape[2]
    row0, n = st["row0"].long(), st["len"].long()
    i = torch.arange(R, device=DEV)
    at = row0[:-1, None] + i  # [S, R] the row of the batch, those past a session's last unused
    real = at < row0[1:, None]
    at = at.clamp_max(st["rows"] - 1)
    q = st["q"][at].float().view(S, R, KVH, G, HD).permute(0, 2, 1, 3, 4).reshape(S, KVH, R * G, HD)
    scores = torch.matmul(q, kv[:, :KVH].transpose(2, 3).contiguous()) / math.sqrt(HD)
    slot = torch.arange(T, device=DEV)
    if st["vis"] is None:
        seen = slot <= (n[:, None] + i)[..., None]
    else:
        node = slot - n[:, None, None]
        word = st["vis"][at][..., None]
        seen = (node < 0) | ((node < R) & ((word >> node.clamp(0, 63)) & 1).bool())
    scores.view(S, KVH, R, G, T).masked_fill_(~seen[:, None, :, None, :], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    o = torch.matmul(p, kv[:, KVH:]) / p.sum(-1, keepdim=True)
    o = o.view(S, KVH, R, G, HD).permute(0, 2, 1, 3, 4).reshape(S, R, c["qh"] * HD)
    return o[real].to(torch.bfloat16)


def _slots(st):
    """page and place of every row's own slot"""
    c = st["case"]
    row0 = st["row0"].long()
    r = torch.arange(st["rows"], device=DEV)
    s = torch.searchsorted(row0[1:].contiguous(), r, right=True)
    slot = st["len"].long()[s] + r - row0[s]
    return st["table"].long()[s, slot // c["page"]], slot % c["page"], slot


def _plain_norm_rope(x, w, cs):
    """x [rows, heads, 128] float32: RMS norm a head (a bf16 tensor between the two, as the
    separate launchers leave it), then the rotation of neighbouring pairs"""
    q = x * x
    for h in (64, 32, 16, 8, 4, 2, 1):  # pairwise, halves first
        q = q[..., :h] + q[..., h:]
    inv = 1.0 / torch.sqrt(q / HD + EPS)
    y = (x * inv * w.float()).to(torch.bfloat16).float().unflatten(-1, (64, 2))
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    return torch.stack([y[..., 0] * c - y[..., 1] * s, y[..., 1] * c + y[..., 0] * s],
                       -1).flatten(-2).to(torch.bfloat16)


def _codes(x, bits):
    """x [..., 128] bf16: codes and f16 scales of its groups of 32"""
    top = 127.0 if bits == 8 else 7.0
    x = x.float().unflatten(-1, (4, 32))
    s = (x.abs().amax(-1) / torch.full((), top, device=DEV)).to(torch.float16)
    f = s.float()[..., None]
    q = torch.where(f > 0, torch.round(x / f), 0.0).clamp(-top, top).flatten(-2).to(torch.int8)
    if bits == 4:
        q = (q[..., 0::2] & 15) | (q[..., 1::2] << 4)
    return q, s


def _written(st):
    """the layer's pages after the append: bf16, or what the codes stand for in f16"""
    kv, bits = st["kv"][st["layer"]], st["case"]["bits"]
    if bits == 16:
        return kv
    if bits == 4:
        kv = torch.stack([((kv & 15) ^ 8) - 8, kv >> 4], -1).flatten(-2)
    return kv.unflatten(-1, (4, 32)) * st["scales"][st["layer"]][..., None]


def _plain_append(st):
    c = st["case"]
    qh, kvh = c["qh"], c["kvh"]
    x = st["qkv"].float().view(st["rows"], qh + 2 * kvh, HD)
    page, at, slot = _slots(st)
    cs = st["rope"][slot].float()
    q = _plain_norm_rope(x[:, :qh], st["qn"], cs)
    new = torch.cat([_plain_norm_rope(x[:, qh:qh + kvh], st["kn"], cs),
                     st["qkv"].view(st["rows"], -1, HD)[:, qh + kvh:]], 1)
    if c["bits"] == 16:
        st["kv"][st["layer"]][page, :, at] = new
    else:
        codes, scales = _codes(new, c["bits"])
        st["kv"][st["layer"]][page, :, at] = codes
        st["scales"][st["layer"]][page, :, at] = scales
    return {"q": q, "kv": _written(st)}


def _plain_share(st):
    c, page = st["case"], st["case"]["page"]
    st["state"].copy_(st["start"])
    ref, table, held, length = _views(st)
    src, dst = st["src"].long(), st["dst"].long()
    # fork: the pages of the source's tokens, one more reference each
    n = (length[src] + page - 1) // page
    j = torch.arange(st["width"], device=DEV)
    shared = j < n[:, None]
    table[dst] = torch.where(shared, table[src], -1)
    ref.index_add_(0, table[src][shared].long(), torch.ones((), dtype=torch.int32, device=DEV)
                   .expand(int(shared.sum())))
    held[dst], length[dst] = n.int(), length[src]
    # reserve: pages that are missing, and a copy of a last page that others hold too
    want = st["want"]
    room = (length + want + page - 1) // page
    fits = (want > 0) & (room <= st["width"])
    more = torch.where(fits, (room - held).clamp_min(0), 0)
    last = length // page
    partly = fits & (length % page > 0)
    mine = torch.where(partly, table.gather(1, last.long().clamp_max(st["width"] - 1)[:, None])[:, 0], -1)
    same = (mine[:, None] == mine[None, :]) & partly[:, None] & partly[None, :]
    before = torch.tril(same, -1).sum(1)
    copy = partly & (before < ref[mine.clamp_min(0).long()] - 1)
    need = more + copy
    free = (ref == 0).nonzero()[:, 0]
    upto = need.cumsum(0)
    ok = fits & (upto <= free.numel())
    first = upto - need
    copy &= ok
    # the copy takes the session's first new page, the missing ones the rest in order
    s = copy.nonzero()[:, 0]
    old, new = mine[s].long(), free[first[s]]
    st["kv"][:, new] = st["kv"][:, old]
    ref.index_add_(0, old, torch.full_like(s, -1, dtype=torch.int32))
    table[s, last[s].long()] = new.int()
    ref[new] = 1
    k = j - held[:, None]
    fill = ok[:, None] & (k >= 0) & (k < more[:, None])
    ids = free[((first + copy)[:, None] + k).clamp(0, free.numel() - 1)]
    table[fill] = ids[fill].int()
    ref[ids[fill]] = 1
    held += torch.where(ok, more, 0).int()
    return {"state": st["state"], "granted": ok.int(), "kv": st["kv"]}


def _plain_reclaim(st):
    c, page = st["case"], st["case"]["page"]
    st["state"].copy_(st["start"])
    ref, table, held, length = _views(st)
    keep = st["keep"]
    n = torch.where(keep >= 0, torch.minimum(held, (torch.minimum(keep, length) + page - 1) // page), held)
    j = torch.arange(st["width"], device=DEV)
    drop = (j >= n[:, None]) & (j < held[:, None])
    ref.index_add_(0, table[drop].long(), torch.full((int(drop.sum()),), -1, dtype=torch.int32,
                                                     device=DEV))
    table[drop] = -1
    length.copy_(torch.where(keep >= 0, torch.minimum(keep, length), length))
    held.copy_(n)
    # compact: the pages in use behind the first `live` move into the free ones before them
    used = ref > 0
    live = int(used.sum())
    holes = (~used[:live]).nonzero()[:, 0]
    movers = used[live:].nonzero()[:, 0] + live
    st["kv"][:, holes] = st["kv"][:, movers]
    to = torch.arange(c["pages"], dtype=torch.int32, device=DEV)
    to[movers] = holes.int()
    ref[holes] = ref[movers]
    ref[movers] = 0
    inside = j < held[:, None]
    table[inside] = to[table[inside].long()]
    return {"state": st["state"], "live": live, "kv": st["kv"]}


# ------------------------------------------------------------ the library's calls

def _lib():
    pkg = os.path.join(os.getcwd(), "s2pro-native_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import s2pamd
    return s2pamd, s2pamd.load()


def _bind(st):
    """the descriptors and workspaces that a program keeps beside its caches"""
    m, lib = _lib()
    c, b = st["case"], {"m": m, "lib": lib}
    kvh = c.get("kvh", 8)
    b["pool"] = m.PagePool(kv=st["kv"].data_ptr(),
                           scales=None if st.get("scales") is None else st["scales"].data_ptr(),
                           layers=st["kv"].shape[0], pages=st["kv"].shape[1], kv_heads=kvh,
                           page=c["page"], bits=c.get("bits", 16))
    if c["kind"] in ("attend", "append"):
        b["batch"] = m.PageBatch(table=st["table"].data_ptr(), len=st["len"].data_ptr(),
                                 row0=st["row0"].data_ptr(), sessions=c["sessions"],
                                 max_pages=st["table"].shape[1], rows=st["rows"],
                                 max_rows=st["max_rows"], max_len=st["max_len"])
        if c["kind"] == "attend":
            n = lib.s2pk_paged_attention_work_floats(ctypes.byref(b["batch"]), c["qh"], kvh)
            b["work"] = torch.empty(max(1, n), dtype=torch.float32, device=DEV)
    else:
        ref, table, held, length = _views(st)
        b["tab"] = m.PageTables(ref=ref.data_ptr(), table=table.data_ptr(), held=held.data_ptr(),
                                len=length.data_ptr(), sessions=c["sessions"],
                                max_pages=st["width"])
        n = lib.s2pk_pages_work_ints(ctypes.byref(b["pool"]), ctypes.byref(b["tab"]))
        b["work"] = torch.empty(n, dtype=torch.int32, device=DEV)
        b["live"] = torch.zeros((), dtype=torch.int64, device=DEV)  # the call writes its low word
    b["pool_p"] = ctypes.byref(b["pool"])
    b["batch_p"] = ctypes.byref(b["batch"]) if "batch" in b else None
    b["tab_p"] = ctypes.byref(b["tab"]) if "tab" in b else None
    st["bound"] = b
    return b


def _own_run(st):
    b = st.get("bound") or _bind(st)
    m, lib, c = b["m"], b["lib"], st["case"]
    s = torch.cuda.current_stream().cuda_stream
    k = c["kind"]
    if k == "attend":
        out = torch.empty(st["rows"], c["qh"] * HD, dtype=torch.bfloat16, device=DEV)
        m.hip_check(lib.s2pk_paged_attention(
            b["pool_p"], b["batch_p"], st["layer"], st["q"].data_ptr(), c["qh"],
            None if st["vis"] is None else st["vis"].data_ptr(), out.data_ptr(),
            b["work"].data_ptr(), s), "paged attention")
        return out
    if k == "append":
        q = torch.empty(st["rows"], c["qh"], HD, dtype=torch.bfloat16, device=DEV)
        m.hip_check(lib.s2pk_paged_append(
            b["pool_p"], b["batch_p"], st["layer"], st["qkv"].data_ptr(), c["qh"],
            st["qn"].data_ptr(), st["kn"].data_ptr(), EPS, st["rope"].data_ptr(),
            st["rope"].shape[0], None, q.data_ptr(), s), "paged append")
        return {"q": q, "kv": _written(st)}
    st["state"].copy_(st["start"])
    if k == "share":
        granted = torch.empty(c["sessions"], dtype=torch.int32, device=DEV)
        m.hip_check(lib.s2pk_pages_fork(b["pool_p"], b["tab_p"], st["src"].data_ptr(),
                                        st["dst"].data_ptr(), c["forks"], None, s), "fork")
        m.hip_check(lib.s2pk_pages_reserve(b["pool_p"], b["tab_p"], st["want"].data_ptr(),
                                           granted.data_ptr(), b["work"].data_ptr(), s), "reserve")
        return {"state": st["state"], "granted": granted, "kv": st["kv"]}
    live = b["live"]
    m.hip_check(lib.s2pk_pages_free(b["pool_p"], b["tab_p"], st["keep"].data_ptr(), s), "free")
    m.hip_check(lib.s2pk_pages_compact(b["pool_p"], b["tab_p"], live.data_ptr(),
                                       b["work"].data_ptr(), s), "compact")
    return {"state": st["state"], "live": live, "kv": st["kv"]}


def run(state):
    if own:
        return _own_run(state)
    return {"attend": _plain_attend, "append": _plain_append, "share": _plain_share,
            "reclaim": _plain_reclaim}[state["case"]["kind"]](state)


# -------------------------------------------------------------------- 64 bits

def exact(case, seed):
    """Attention and the appended rows in binary64, session by session; nothing is computed
    by the page calls."""
    if case["kind"] not in ("attend", "append"):
        return None
    st = prepare(case, seed)
    c = st["case"]
    lens, rows, kvh, qh, page = _lens(c), _rows(c), c["kvh"], c["qh"], c["page"]
    layer = st["layer"]

    def f64(kv, sc):
        if c["bits"] == 16:
            return kv.double()
        if c["bits"] == 4:
            u = kv.to(torch.int16) & 255
            kv = torch.stack([u % 16, u // 16], -1).reshape(*u.shape[:-1], HD)
            kv = torch.where(kv > 7, kv - 16, kv)
        return kv.double() * sc.double().repeat_interleave(32, -1)

    if c["kind"] == "attend":
        out, r0 = [], 0
        for s, (n, r) in enumerate(zip(lens, rows)):
            ids = st["table"][s, :-(-(n + r) // page)].long()
            kv = f64(st["kv"][layer, ids], None if st["scales"] is None else st["scales"][layer, ids])
            kv = kv.transpose(0, 1).reshape(2 * kvh, -1, HD)[:, :n + r]
            own_rows = torch.zeros(r, n + r, dtype=torch.bool, device=DEV)
            for i in range(r):
                own_rows[i, :n] = True
                j = i
                while j >= 0:
                    own_rows[i, n + j] = True
                    if not c["tree"]:
                        own_rows[i, n:n + j] = True
                        break
                    j = TREE16[j]
            q = st["q"][r0:r0 + r].double().view(r, kvh, qh // kvh, HD)
            o = torch.empty(r, kvh, qh // kvh, HD, dtype=torch.float64, device=DEV)
            for h in range(kvh):
                z = (q[:, h].reshape(-1, HD) @ kv[h].t().contiguous()) * HD ** -0.5
                z = z.view(r, -1, n + r).masked_fill(~own_rows[:, None], -math.inf)
                o[:, h] = torch.softmax(z, -1).view(-1, n + r).matmul(kv[kvh + h]).view(r, -1, HD)
            out.append(o.reshape(r, qh * HD))
            r0 += r
        return torch.cat(out)
    x = st["qkv"].double().view(st["rows"], -1, HD)
    pos = torch.cat([torch.arange(n, n + r, device=DEV) for n, r in zip(lens, rows)])
    turn = torch.complex(st["rope"][pos, :, 0].double(), st["rope"][pos, :, 1].double())[:, None]

    def turned(a, w):
        a = a / (a.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()
        a = a.to(torch.bfloat16).double().view(*a.shape[:-1], 64, 2)
        return torch.view_as_real(torch.view_as_complex(a.contiguous()) * turn).flatten(-2)

    q, k, v = turned(x[:, :qh], st["qn"]), turned(x[:, qh:qh + kvh], st["kn"]), x[:, qh + kvh:]
    new = torch.cat([k, v], 1)
    kv = f64(st["kv"][layer], None if st["scales"] is None else st["scales"][layer])
    if c["bits"] != 16:
        top = 127 if c["bits"] == 8 else 7
        x = new.to(torch.bfloat16).double().view(*new.shape[:-1], 4, 32)
        s = (x.abs().amax(-1, keepdim=True) / top).half().double()
        new = torch.where(s > 0, (x / s).round().clamp(-top, top) * s, 0.0).flatten(-2)
    r0 = 0
    for s, (n, r) in enumerate(zip(lens, rows)):
        at = torch.arange(n, n + r, device=DEV)
        kv[st["table"][s].long()[at // page], :, at % page] = new[r0:r0 + r]
        r0 += r
    return {"q": q, "kv": kv if c["bits"] == 16 else kv.unflatten(-1, (4, 32))}
