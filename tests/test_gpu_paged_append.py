"""s2pk_paged_append against the separate launchers, bit for bit, and against
binary64; the RoPE table; the commit of accepted nodes."""
import ctypes

import numpy as np
import pytest
import torch

import pyoracle as po
import s2pamd
from gpu_util import DEV, P, S, bf16_vals, to_dev, to_host
from paged_util import (HD, Batch, Pool, attend, check, dev_i32, keep, new_batch, pages_for, rand_q,
                        reference, tree_words)

pytestmark = pytest.mark.gpu
BASE, EPS = 1e6, 1e-6


@pytest.fixture(scope="module")
def lib():
    return s2pamd.load()


@pytest.fixture(scope="module")
def table(lib):
    t = torch.empty(3000, 64, 2, dtype=torch.bfloat16, device=DEV)
    s2pamd.hip_check(lib.s2pk_rope_table(P(t), 3000, 128, BASE, S()))
    torch.cuda.synchronize()
    return t


def test_table_against_binary64(lib, table):
    """the angle is the product of the position and 1 / base^(2i/128), both in f32, so its
    cos and sin are off by at most the angle's rounding (2^-23 of it with the inverse's) and
    the bf16 step"""
    p = np.arange(3000, dtype=np.float64)[:, None]
    a = p * (1.0 / np.power(BASE, 2 * np.arange(64) / 128.0))[None]
    got = bf16_vals(to_host(table.view(torch.int16), np.uint16)).reshape(3000, 64, 2)
    for i, f in enumerate((np.cos, np.sin)):
        assert (np.abs(got[..., i] - f(a)) <= 2.0 ** -8 * np.abs(f(a)) + a * 2.0 ** -22 + 1e-30).all()
    far = keep(torch.empty(300000, 64, 2, dtype=torch.bfloat16, device=DEV))
    s2pamd.hip_check(lib.s2pk_rope_table(P(far), 300000, 128, BASE, S()))
    assert torch.equal(far[:3000], table)


def weights(seed, norm):
    if not norm:
        return None, None
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return [keep((torch.randn(HD, generator=g, device=DEV) * 0.2 + 1).to(torch.bfloat16))
            for _ in range(2)]


def append(lib, pool, b, qkv, qh, qn, kn, rope, pos=None, q=None, layer=None):
    if q is None:
        q = keep(torch.empty(b.rows, qh * HD, dtype=torch.bfloat16, device=DEV))
    p, d = pool.desc(), b.desc()
    s2pamd.hip_check(lib.s2pk_paged_append(
        ctypes.byref(p), ctypes.byref(d), pool.layer if layer is None else layer, P(qkv), qh,
        P(qn), P(kn), EPS, P(rope), rope.shape[0], P(pos), P(q), S()), "paged append")
    return q


def separate(lib, pool, b, qkv, qh, qn, kn, pos, max_seq=4096):
    """q and one contiguous cache a row from the launchers that do one thing each"""
    n, kvh, bits = b.rows, pool.kvh, pool.bits
    q, k, v = (keep(torch.empty(n, w * HD, dtype=torch.bfloat16, device=DEV))
               for w in (qh, kvh, kvh))
    ok = s2pamd.hip_check
    ok(lib.s2pk_qkv_split(P(qkv), P(q), P(k), P(v), n, qh * HD, kvh * HD, S()))
    ok(lib.s2pk_qk_norm(P(q), P(qn), n, qh, HD, EPS, S()))
    ok(lib.s2pk_qk_norm(P(k), P(kn), n, kvh, HD, EPS, S()))
    ok(lib.s2pk_rope_pos(P(q), P(k), n, qh, kvh, HD, P(pos), BASE, S()))
    # one slot a row: a cache of max_seq 1
    at = dev_i32(np.zeros(n))
    el = {16: 256, 8: 128, 4: 64}[bits]
    kc, vc = (keep(torch.zeros(n, kvh, el, dtype=torch.uint8, device=DEV)) for _ in range(2))
    ks, vs = (keep(torch.zeros(n, kvh, 4, dtype=torch.float16, device=DEV)) for _ in range(2))

    def ptrs(t):
        return keep(torch.tensor([t[i].data_ptr() for i in range(n)], dtype=torch.int64, device=DEV))

    if bits == 16:
        ok(lib.s2pk_kv_append_ptrs(P(k), P(v), P(ptrs(kc)), P(ptrs(vc)), n, kvh, HD, P(at), 1, S()))
    else:
        ok(lib.s2pk_kv_append8_ptrs(P(k), P(v), P(ptrs(kc)), P(ptrs(vc)), P(ptrs(ks)), P(ptrs(vs)),
                                    n, kvh, HD, P(at), 1, bits, S()))
    torch.cuda.synchronize()
    return q, torch.cat([kc, vc], 1), torch.cat([ks, vs], 1)


def places(b):
    """(row, page id, place) of every row that belongs to a session"""
    out = []
    for s, (n, r) in enumerate(zip(b.lens, b.nrows)):
        for i in range(r):
            out.append((int(b.row0[s]) + i, int(b.table[s, (n + i) // b.page]), (n + i) % b.page))
    return out


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("page,kvh,g,lens,rows,norm", [
    (16, 8, 4, [0, 15, 16, 100, 2000], [1, 1, 1, 1, 1], True),
    (32, 8, 4, [0, 31, 300], [5, 5, 5], True),
    (16, 2, 4, [7, 0, 64], [70, 0, 33], True),
    (256, 1, 16, [250], [40], False),
    (64, 3, 3, [5, 9], [3, 130], True)])
def test_bits_of_the_separate_launchers(lib, table, bits, page, kvh, g, lens, rows, norm):
    qh = kvh * g
    pool = Pool(1, bits, pages_for(page, lens, rows), kvh, page, layers=2, layer=1)
    b = new_batch(2, pool.pages, page, lens, rows)
    qkv = rand_q(3, b.rows, qh + 2 * kvh, 3.0)
    qkv[0, qh * HD:qh * HD + 32] = 0  # a group of zeros
    qn, kn = weights(4, norm)
    before = pool.kv.clone(), None if pool.scales is None else pool.scales.clone()
    q = append(lib, pool, b, qkv, qh, qn, kn, table)
    pos = dev_i32(np.concatenate([np.arange(n, n + r) for n, r in zip(lens, rows)]))
    wq, wkv, wsc = separate(lib, pool, b, qkv, qh, qn, kn, pos)
    assert torch.equal(q, wq)
    at = places(b)
    r, ids, pl = (torch.tensor([a[i] for a in at], device=DEV) for i in range(3))
    assert torch.equal(pool.kv[1][ids, :, pl].view(torch.uint8), wkv[r])
    if bits != 16:
        assert torch.equal(pool.scales[1][ids, :, pl], wsc[r])
    # nothing else moved
    for t, o in zip((pool.kv, pool.scales), before):
        if t is not None:
            assert torch.equal(t[0], o[0])
            o[1][ids, :, pl] = t[1][ids, :, pl]
            assert torch.equal(t[1], o[1])


@pytest.mark.parametrize("bits", [16, 8])
def test_against_binary64(lib, table, bits):
    """q = turn(bf16(x inv w)): the normed value is rounded to bf16 (2^-8 of it; the f32 norm
    may carry it over a border, hence twice), the product with cos, sin and the result (2^-8)"""
    kvh, g, page, lens, rows = 2, 4, 16, [40, 1000], [20, 9]
    qh = kvh * g
    pool = Pool(1, bits, pages_for(page, lens, rows), kvh, page)
    b = new_batch(2, pool.pages, page, lens, rows)
    qkv = rand_q(3, b.rows, qh + 2 * kvh, 2.0)
    qn, kn = weights(4, True)
    q = append(lib, pool, b, qkv, qh, qn, kn, table)
    x = qkv.double().view(b.rows, -1, HD).cpu().numpy()
    pos = np.concatenate([np.arange(n, n + r) for n, r in zip(lens, rows)])
    cs = table.double().cpu().numpy()[pos]
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS)
    for part, w, got in ((y[:, :qh], qn, q.double().view(b.rows, qh, HD).cpu().numpy()),
                         (y[:, qh:qh + kvh], kn, None)):
        z = (part * w.double().cpu().numpy()).reshape(b.rows, -1, 64, 2)
        c, s = cs[:, None, :, 0], cs[:, None, :, 1]
        o = np.stack([z[..., 0] * c - z[..., 1] * s, z[..., 1] * c + z[..., 0] * s], -1)
        mag = (np.abs(z[..., 0]) + np.abs(z[..., 1]))[..., None] * 2.0 ** -7
        if got is None:
            vals = np.stack([pool.values([i])[0][:kvh, p] for _, i, p in places(b)])
            got = vals
            # a code is off by half a step of its group's scale
            if bits == 8:
                top = np.abs(o).reshape(b.rows, kvh, 4, 32).max(-1, keepdims=True)
                mag = mag + (top * (0.51 / 127 + 2.0 ** -10) * np.ones((1, 1, 1, 32))).reshape(
                    b.rows, kvh, 64, 2)
        got = got.reshape(o.shape)
        assert (np.abs(got - o) <= mag + 2.0 ** -8 * np.abs(o)).all()


@pytest.mark.parametrize("bits", [16, 4])
def test_positions_of_a_tree_and_rows_left_out(lib, table, bits):
    page, kvh, g = 16, 2, 4
    lens, rows = [30, 40, -3, 9], [4, 3, 1, 2]
    qh = kvh * g
    pool = Pool(1, bits, 20, kvh, page)
    ok = new_batch(2, pool.pages, page, [30, 40, 0, 9], rows)
    tab = ok.table.copy()
    tab[1, :] = pool.pages + 3  # pages that are not there
    b = Batch(tab, lens, rows, page, total=sum(rows) + 5)
    qkv = rand_q(3, b.rows, qh + 2 * kvh, 2.0)
    qn, kn = weights(4, True)
    depth = [30, 31, 31, 32, 40, 41, 42, 0, -1, 3000, 0, 0, 0, 0, 0]
    pos = dev_i32(depth)
    kv0 = pool.kv.clone()
    q = keep(torch.full((b.rows, qh * HD), 7.0, dtype=torch.bfloat16, device=DEV))
    append(lib, pool, b, qkv, qh, qn, kn, table, pos, q)
    clip = dev_i32(np.clip(depth, 0, 2999))
    wq, wkv, _ = separate(lib, pool, b, qkv, qh, qn, kn, clip)
    assert torch.equal(q[:7], wq[:7])   # session 1's queries too, though its pages are missing
    assert (q[7:] == 7.0).all()         # a negative length, two positions outside, padding
    moved = (pool.kv != kv0).flatten(4).any(-1).sum() if bits != 16 else None
    for i in range(4):
        s = 30 + i
        got = pool.kv[0, int(tab[0, s // page]), :, s % page].contiguous().view(torch.uint8)
        assert torch.equal(got, wkv[i])
        pool.kv[0, int(tab[0, s // page]), :, s % page] = kv0[0, int(tab[0, s // page]), :, s % page]
    assert torch.equal(pool.kv, kv0), moved


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_commit(lib, bits):
    page, kvh, layers = 16, 2, 3
    lens, rows = [10, 30, 0, 45, 7], [17, 17, 17, 17, 17]
    pool = Pool(1, bits, pages_for(page, lens, rows), kvh, page, layers)
    b = new_batch(2, pool.pages, page, lens, rows)
    paths = [[2, 5, 11], [], [1, 2, 3], [16], [3]]
    n_acc = [3, 0, 3, 1, -1]
    path = np.full(b.rows, 99, np.int32)
    for s, p in enumerate(paths):
        path[17 * s:17 * s + len(p)] = p
    want = [t.clone() for t in (pool.kv, pool.scales) if t is not None]
    for s, p in enumerate(paths):
        if n_acc[s] < 0:
            continue
        for d, node in enumerate(p, 1):
            f, t = lens[s] + node, lens[s] + d
            for w in want:
                w[:, int(b.table[s, t // page]), :, t % page] = \
                    w[:, int(b.table[s, f // page]), :, f % page]
    p, d = pool.desc(), b.desc()
    s2pamd.hip_check(lib.s2pk_paged_commit(ctypes.byref(p), ctypes.byref(d), P(dev_i32(path)),
                                           P(dev_i32(n_acc)), P(b.d_len), S()))
    for t, w in zip((pool.kv, pool.scales), want):
        assert torch.equal(t, w)
    assert b.d_len.tolist() == [14, 31, 4, 47, 7]
    # nodes that are none move nothing; counts past the rows are the rows
    path[:] = [-4, 2 ** 31 - 1, 17, 0, 1] * 17
    s2pamd.hip_check(lib.s2pk_paged_commit(ctypes.byref(p), ctypes.byref(d), P(dev_i32(path)),
                                           P(dev_i32([1000] * 5)), None, S()))
    for t, w in zip((pool.kv, pool.scales), want):
        assert torch.equal(t, w)


@pytest.mark.parametrize("bits", [8, 4])
def test_codes_of_values_next_to_a_half(lib, table, bits):
    """c = rint(x / s) with the f32 quotient, for values on a half step and next to it, scales that are
    powers of two and others, down to f16's smallest"""
    kvh, page, n, most = 4, 64, 512, 127 if bits == 8 else 7
    rng = np.random.default_rng(bits)
    pool = Pool(1, bits, n // page + 1, kvh, page)
    b = new_batch(2, pool.pages, page, [0], [n])
    top = np.exp2(rng.uniform(-26, 12, (n, kvh, 4, 1))).astype(np.float32)
    top[::3] = most * np.exp2(rng.integers(-20, 8, (len(top[::3]), kvh, 4, 1)))
    half = (rng.integers(-most, most, (n, kvh, 4, 32)) + 0.5) / most
    x = np.where(rng.random(half.shape) < 0.7, half, rng.uniform(-1, 1, half.shape)) * top
    x[..., :1] = top
    v = torch.tensor(x.reshape(n, kvh, HD), dtype=torch.float32).to(torch.bfloat16)
    x = v.float().numpy().reshape(n, kvh, 4, 32)
    qkv = keep(torch.zeros(n, 3 * kvh, HD, dtype=torch.bfloat16, device=DEV))
    qkv[:, 2 * kvh:] = v.to(DEV)
    append(lib, pool, b, qkv.view(n, -1), kvh, None, None, table)
    s = (np.abs(x).max(-1, keepdims=True) / np.float32(most)).astype(np.float16).astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where(s > 0, np.clip(np.rint(x / s), -most, most), 0)
    got = np.stack([pool.values([i])[0][kvh:, p] for _, i, p in places(b)])
    assert np.array_equal(got.reshape(x.shape), c * s.astype(np.float64))
