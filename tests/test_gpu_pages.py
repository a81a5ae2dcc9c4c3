"""The pages' bookkeeping against a model in plain Python, and the calls of a paged
session together: reserve, append, attend, fork, commit, free, compact."""
import ctypes

import numpy as np
import pytest
import torch

import s2pamd
from gpu_util import DEV, P, S
from paged_util import (HD, Batch, Pool, attend, check, dev_i32, keep, rand_q, reference, tree_words)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    return s2pamd.load()


class Model:
    """counts and tables as the header states them"""

    def __init__(self, pages, sessions, max_pages, page):
        self.ref, self.page, self.max_pages = [0] * pages, page, max_pages
        self.tab = [[] for _ in range(sessions)]
        self.len = [0] * sessions

    def cover(self, n):
        return -(-n // self.page)

    def reserve(self, want):
        granted, copies = [0] * len(want), []
        holders = {}
        free = [i for i, r in enumerate(self.ref) if r == 0]
        dead, at, plan = False, 0, []
        for s, w in enumerate(want):
            if w <= 0:
                continue
            room = self.cover(self.len[s] + w)
            if room > self.max_pages:
                continue
            more = max(0, room - len(self.tab[s]))
            mine = self.tab[s][self.len[s] // self.page] if self.len[s] % self.page else None
            copy = mine is not None and holders.get(mine, 0) < self.ref[mine] - 1
            if mine is not None:
                holders[mine] = holders.get(mine, 0) + 1
            if dead or at + more + copy > len(free):
                dead = True
                continue
            plan.append((s, free[at:at + more + copy], copy, mine))
            at += more + copy
        for s, ids, copy, mine in plan:
            granted[s] = 1
            if copy:
                self.tab[s][self.len[s] // self.page] = ids[0]
                self.ref[mine] -= 1
                copies.append((mine, ids[0]))
            self.tab[s] += ids[int(copy):]
            for i in ids:
                self.ref[i] = 1
        return granted, copies

    def fork(self, src, dst):
        done = []
        state = [(list(t), n) for t, n in zip(self.tab, self.len)]
        for i, (a, b) in enumerate(zip(src, dst)):
            n = len(self.tab)
            ok = 0 <= a < n and 0 <= b < n and a not in dst and b not in src and b not in dst[:i]
            ok = ok and not state[b][0] and state[a][1] > 0
            if ok:
                ids = state[a][0][:self.cover(state[a][1])]
                self.tab[b], self.len[b] = list(ids), state[a][1]
                for p in ids:
                    self.ref[p] += 1
            done.append(int(ok))
        return done

    def free(self, keep_):
        for s, k in enumerate(keep_):
            if k < 0:
                continue
            n = min(k, self.len[s])
            c = self.cover(n)
            for p in self.tab[s][c:]:
                self.ref[p] -= 1
            self.tab[s], self.len[s] = self.tab[s][:c], n

    def compact(self):
        live = sum(r > 0 for r in self.ref)
        holes = [i for i in range(live) if self.ref[i] == 0]
        movers = [i for i in range(live, len(self.ref)) if self.ref[i]]
        to = dict(zip(movers, holes))
        for a, b in to.items():
            self.ref[b], self.ref[a] = self.ref[a], 0
        self.tab = [[to.get(p, p) for p in t] for t in self.tab]
        return live, list(to.items())


class Dev:
    def __init__(self, lib, pool, sessions, max_pages):
        self.lib, self.pool, self.n, self.w = lib, pool, sessions, max_pages
        self.ref = dev_i32(np.zeros(pool.pages))
        self.table = dev_i32(np.full((sessions, max_pages), -1))
        self.held, self.len = dev_i32(np.zeros(sessions)), dev_i32(np.zeros(sessions))
        self.t = s2pamd.PageTables(ref=self.ref.data_ptr(), table=self.table.data_ptr(),
                                   held=self.held.data_ptr(), len=self.len.data_ptr(),
                                   sessions=sessions, max_pages=max_pages)
        self.p = pool.desc()
        n = lib.s2pk_pages_work_ints(ctypes.byref(self.p), ctypes.byref(self.t))
        self.work = keep(torch.full((n + 64,), -77, dtype=torch.int32, device=DEV))

    def call(self, f, *a):
        s2pamd.hip_check(f(ctypes.byref(self.p), ctypes.byref(self.t), *a, S()), f.__name__)
        assert (self.work[-64:] == -77).all()  # the workspace's end

    def reserve(self, want):
        g = keep(torch.full((self.n,), -5, dtype=torch.int32, device=DEV))
        self.call(self.lib.s2pk_pages_reserve, P(dev_i32(want)), P(g), P(self.work))
        return g.tolist()

    def fork(self, src, dst):
        d = keep(torch.full((len(src),), -5, dtype=torch.int32, device=DEV))
        self.call(self.lib.s2pk_pages_fork, P(dev_i32(src)), P(dev_i32(dst)), len(src), P(d))
        return d.tolist()

    def free(self, k):
        self.call(self.lib.s2pk_pages_free, P(dev_i32(k)))

    def compact(self):
        n = dev_i32([-5])
        self.call(self.lib.s2pk_pages_compact, P(n), P(self.work))
        return int(n)

    def same(self, m, what):
        assert self.ref.tolist() == m.ref, what
        assert self.len.tolist() == m.len, what
        assert self.held.tolist() == [len(t) for t in m.tab], what
        tab = self.table.tolist()
        for s, t in enumerate(m.tab):
            assert tab[s][:len(t)] == t, (what, s)


@pytest.mark.parametrize("bits,page,kvh,layers", [(16, 16, 8, 3), (8, 32, 1, 2), (4, 16, 2, 1),
                                                  (4, 256, 8, 1)])
@pytest.mark.parametrize("pages,sessions", [(40, 12), (9000, 70)])
def test_random_calls(lib, bits, page, kvh, layers, pages, sessions):
    if pages > 1000:
        kvh, layers, page = 1, 1, 16
    r = np.random.default_rng(bits + pages)
    max_pages = 9 if pages < 100 else 300
    pool = Pool(1, bits, pages, kvh, page, layers)
    d, m = Dev(lib, pool, sessions, max_pages), Model(pages, sessions, max_pages, page)
    body = [t.clone() for t in (pool.kv, pool.scales) if t is not None]
    seen = set()
    for step in range(30):
        op = r.choice(["reserve", "reserve", "fork", "free", "compact"])
        moves = []
        if op == "reserve":
            top = max_pages * page // 3
            want = [int(x) for x in r.integers(-2, 3, sessions) * r.integers(0, top, sessions)]
            got, moves = m.reserve(want)
            assert d.reserve(want) == got, step
            seen.update(got)
            # the granted tokens are written: lengths grow, not always as far as the room
            for s, g in enumerate(got):
                if g:
                    m.len[s] += int(r.integers(0, want[s] + 1))
            d.len.copy_(torch.tensor(m.len, dtype=torch.int32))
        elif op == "fork":
            n = int(r.integers(1, 2 * sessions))
            src, dst = (r.integers(-1, sessions + 1, n).tolist() for _ in range(2))
            assert d.fork(src, dst) == m.fork(src, dst), step
        elif op == "free":
            k = [int(x) for x in np.where(r.random(sessions) < 0.4,
                                          r.integers(0, max_pages * page, sessions) // 2, -1)]
            k = [0 if x > 0 and r.random() < 0.4 else x for x in k]
            d.free(k)
            m.free(k)
        else:
            live, moves = m.compact()
            assert d.compact() == live, step
        d.same(m, (step, op))
        for a, b in moves:
            for t in body:
                t[:, b] = t[:, a]
        for t, w in zip((pool.kv, pool.scales), body):
            assert torch.equal(t.view(torch.int16), w.view(torch.int16)), (step, op)
    assert seen == {0, 1}


def test_a_full_table_of_sessions_and_a_captured_call(lib):
    """1,024 sessions that all share one prompt's last page, in one graph"""
    pages, n = 3000, 1024
    pool = Pool(1, 16, pages, 1, 16)
    d, m = Dev(lib, pool, n, 4), Model(pages, n, 4, 16)
    want = [20] + [0] * (n - 1)
    d.reserve(want), m.reserve(want)
    m.len[0] = 20
    d.len[0] = 20
    src, dst, one = dev_i32([0] * (n - 1)), dev_i32(list(range(1, n))), dev_i32([1] * n)
    first = [t.clone() for t in (d.ref, d.table, d.held, d.len)]
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    granted = dev_i32(np.zeros(n))
    with torch.cuda.graph(graph, stream=side):
        st = s2pamd.stream_ptr(side)
        a = ctypes.byref(d.p), ctypes.byref(d.t)
        s2pamd.hip_check(lib.s2pk_pages_fork(*a, P(src), P(dst), n - 1, None, st))
        s2pamd.hip_check(lib.s2pk_pages_reserve(*a, P(one), P(granted), P(d.work), st))
    m.fork([0] * (n - 1), list(range(1, n)))
    got, copies = m.reserve([1] * n)
    assert len(copies) == n - 1
    for step in range(3):
        for t, f in zip((d.ref, d.table, d.held, d.len), first):
            t.copy_(f)
        granted.zero_()
        for _, b in copies:
            pool.kv[:, b] = 0
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        d.same(m, step)
        assert granted.tolist() == got
        for a_, b in copies[::97]:
            assert torch.equal(pool.kv[:, b], pool.kv[:, a_])


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_a_serving_loop(lib, bits):
    """Two sessions prefill a prompt in chunks, one is forked into two continuations, all
    decode and verify trees, one ends, the pool is compacted and the rest go on: the
    attention's outputs are those of each session's own tokens at every step."""
    kvh, g, page, layers, pages, n, width = 2, 4, 16, 2, 60, 6, 12
    qh = kvh * g
    pool = Pool(1, bits, pages, kvh, page, layers)
    d, m = Dev(lib, pool, n, width), Model(pages, n, width, page)
    rope = keep(torch.empty(512, 64, 2, dtype=torch.bfloat16, device=DEV))
    s2pamd.hip_check(lib.s2pk_rope_table(P(rope), 512, HD, 1e6, S()))
    wn = keep(torch.ones(HD, dtype=torch.bfloat16, device=DEV))
    # per session and layer, the K/V values of its tokens: [tokens][2 kvh][128]
    hist = [[np.zeros((0, 2 * kvh, HD)) for _ in range(layers)] for _ in range(n)]
    state = {"seed": 10}

    def step(rows, parent=None, path=None):
        """rows[s] new rows of session s; a tree keeps path[s] of them behind the root"""
        want = [r for r in rows]
        assert d.reserve(want) == [int(r > 0) for r in rows]
        m.reserve(want)
        d.same(m, "reserve")
        b = Batch(d.table.cpu().numpy(), m.len, rows, page)
        b.d_table, b.d_len = d.table, d.len
        vis = pos = None
        if parent:
            words = [w for r in rows if r for w in tree_words(parent)]
            vis = keep(torch.tensor(words, dtype=torch.int64, device=DEV))
            deep = [bin(w).count("1") - 1 for w in tree_words(parent)]
            pos = dev_i32([m.len[s] + x for s, r in enumerate(rows) if r for x in deep])
        desc, new = b.desc(), []
        for layer in range(layers):
            state["seed"] += 1
            qkv = rand_q(state["seed"], b.rows, qh + 2 * kvh, 1.5)
            q = keep(torch.empty(b.rows, qh * HD, dtype=torch.bfloat16, device=DEV))
            s2pamd.hip_check(lib.s2pk_paged_append(
                ctypes.byref(d.p), ctypes.byref(desc), layer, P(qkv), qh, P(wn), P(wn), 1e-6,
                P(rope), 512, P(pos), P(q), S()))
            pool.layer = layer
            out = attend(lib, pool, b, q, qh, vis)
            want_o, tol = reference(pool, b, q, qh, words if parent else None)
            check(out, want_o, tol, f"layer {layer}")
            # the pages hold the session's own history and the new rows behind it
            for s, r in enumerate(rows):
                if not r:
                    continue
                t = m.len[s] + r
                vals = pool.values(m.tab[s][:-(-t // page)], layer)
                vals = vals.transpose(0, 2, 1, 3).reshape(-1, 2 * kvh, HD)
                assert np.array_equal(vals[:m.len[s]], hist[s][layer]), (s, layer)
                new.append((s, layer, vals[m.len[s]:t]))
        if parent:
            arr = np.zeros(b.rows, np.int32)
            acc = np.zeros(n, np.int32)
            for s, r in enumerate(rows):
                if r:
                    arr[b.row0[s]:b.row0[s] + len(path[s])] = path[s]
                    acc[s] = len(path[s])
            s2pamd.hip_check(lib.s2pk_paged_commit(ctypes.byref(d.p), ctypes.byref(desc),
                                                   P(dev_i32(arr)), P(dev_i32(acc)), P(d.len), S()))
            stay = {s: [0] + list(path[s]) for s, r in enumerate(rows) if r}
        else:
            stay = {s: list(range(r)) for s, r in enumerate(rows) if r}
            d.len.add_(dev_i32(rows))
        for s, layer, v in new:
            hist[s][layer] = np.concatenate([hist[s][layer], v[stay[s]]])
        for s in stay:
            m.len[s] += len(stay[s])
        assert d.len.tolist() == m.len

    step([40, 25, 0, 0, 0, 0])
    step([33, 4, 0, 0, 0, 0])
    assert d.fork([0, 0], [3, 4]) == m.fork([0, 0], [3, 4]) == [1, 1]
    for s in (3, 4):
        hist[s] = list(hist[0])
    step([1, 1, 0, 1, 1, 0])
    tree = [-1, 0, 0, 1, 2, 2, 4]
    step([7, 7, 0, 7, 7, 0], tree, {0: [2, 4, 6], 1: [1], 3: [], 4: [2, 5]})
    k = [-1, 0, -1, 50, -1, -1]
    d.free(k), m.free(k)
    hist[1] = [np.zeros((0, 2 * kvh, HD))] * layers
    hist[3] = [h[:50] for h in hist[3]]
    step([1, 0, 0, 1, 1, 30])
    assert d.compact() == m.compact()[0]
    d.same(m, "compact")
    assert max(p for t in m.tab for p in t) == sum(x > 0 for x in m.ref) - 1
    step([5, 0, 20, 1, 1, 3])
    step([1, 0, 1, 1, 1, 1])


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("rows", [1, 5])
def test_a_captured_tick(lib, bits, rows):
    """room, append, attention and commit of every layer in one graph: its replays are the eager
    ticks bit for bit while the sessions grow past pages and share a prompt"""
    kvh, g, page, layers, pages, n, width, ticks = 2, 4, 16, 2, 64, 3, 20, 12
    qh, total = kvh * g, n * rows
    rope = keep(torch.empty(512, 64, 2, dtype=torch.bfloat16, device=DEV))
    s2pamd.hip_check(lib.s2pk_rope_table(P(rope), 512, HD, 1e6, S()))
    want, row0 = dev_i32([rows] * n), dev_i32(np.arange(n + 1) * rows)
    acc = [[(3 * t + s) % rows for s in range(n)] for t in range(ticks)]
    path = dev_i32(np.tile(np.arange(1, rows + 1), n))
    sides = []
    for _ in range(2):
        pool = Pool(5, bits, pages, kvh, page, layers)
        d = Dev(lib, pool, n, width)
        assert d.reserve([21, 0, 0]) == [1, 0, 0]
        d.len.copy_(dev_i32([21, 0, 0]))
        assert d.fork([0, 0], [1, 2]) == [1, 1]
        b = s2pamd.PageBatch(table=d.table.data_ptr(), len=d.len.data_ptr(),
                             row0=row0.data_ptr(), sessions=n, max_pages=width, rows=total,
                             max_rows=rows, max_len=width * page)
        floats = lib.s2pk_paged_attention_work_floats(ctypes.byref(b), qh, kvh)
        sides.append(dict(
            pool=pool, d=d, b=b, granted=dev_i32([0] * n), acc=dev_i32([0] * n),
            qkv=keep(torch.empty(layers, total, (qh + 2 * kvh) * HD, dtype=torch.bfloat16,
                                 device=DEV)),
            q=keep(torch.empty(total, qh * HD, dtype=torch.bfloat16, device=DEV)),
            out=keep(torch.empty(layers, total, qh * HD, dtype=torch.bfloat16, device=DEV)),
            work=keep(torch.empty(floats, dtype=torch.float32, device=DEV))))

    def tick(x, st):
        d, b = x["d"], ctypes.byref(x["b"])
        p = ctypes.byref(d.p)
        ok = s2pamd.hip_check
        ok(lib.s2pk_pages_reserve(p, ctypes.byref(d.t), P(want), P(x["granted"]), P(d.work), st))
        for i in range(layers):
            ok(lib.s2pk_paged_append(p, b, i, P(x["qkv"][i]), qh, None, None, 1e-6, P(rope), 512,
                                     None, P(x["q"]), st))
            ok(lib.s2pk_paged_attention(p, b, i, P(x["q"]), qh, None, P(x["out"][i]), P(x["work"]),
                                        st))
        ok(lib.s2pk_paged_commit(p, b, P(path), P(x["acc"]), P(d.len), st))

    eager, graphed = sides
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        tick(graphed, s2pamd.stream_ptr(side))
    for t in range(ticks):
        new = rand_q(100 + t, layers * total, qh + 2 * kvh, 1.5)
        for x in sides:
            x["qkv"].copy_(new.view_as(x["qkv"]))
            x["acc"].copy_(torch.tensor(acc[t], dtype=torch.int32))
        torch.cuda.synchronize()
        tick(eager, S())
        graph.replay()
        torch.cuda.synchronize()
        assert eager["granted"].tolist() == [1] * n
        for a, b in zip((eager["d"].ref, eager["d"].table, eager["d"].len, eager["out"],
                         eager["pool"].kv),
                        (graphed["d"].ref, graphed["d"].table, graphed["d"].len, graphed["out"],
                         graphed["pool"].kv)):
            assert torch.equal(a, b), t
    assert eager["d"].len.tolist() == [21 + sum(a[s] + 1 for a in acc) for s in range(n)]
