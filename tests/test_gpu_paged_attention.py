"""s2pk_paged_attention against binary64 with tolerances counted from its
roundings (paged_util.reference)."""
import ctypes

import numpy as np
import pytest
import torch

import s2pamd
from gpu_util import DEV, P, to_host
from paged_util import (HD, Batch, Pool, attend, check, dev_i32, keep, new_batch, pages_for, rand_q,
                        reference, tree_words)

pytestmark = pytest.mark.gpu
TREE16 = [-1, 0, 0, 1, 1, 2, 2, 3, 3, 4, 5, 6, 6, 7, 8, 10, 11]


@pytest.fixture(scope="module")
def lib():
    return s2pamd.load()


def run(lib, seed, bits, page, kvh, g, lens, rows, vis=None, scale=1.0, layers=1, layer=0):
    pool = Pool(seed, bits, pages_for(page, lens, rows), kvh, page, layers, layer)
    b = new_batch(seed, pool.pages, page, lens, rows)
    q = rand_q(seed + 1, b.rows, kvh * g, scale)
    dv = None if vis is None else keep(torch.tensor(np.array(vis, np.uint64).view(np.int64),
                                                    device=DEV))
    out = attend(lib, pool, b, q, kvh * g, dv)
    check(out, *reference(pool, b, q, kvh * g, vis), f"bits {bits} page {page}")
    return pool, b, q, out


DECODE = [0, 1, 14, 15, 16, 31, 32, 63, 64, 100, 127, 128, 129, 511, 1000]


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_decode_lengths(lib, bits, page):
    run(lib, 100 + page + bits, bits, page, 2, 4, DECODE, [1] * len(DECODE))


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("kvh,g", [(1, 1), (3, 2), (2, 3), (1, 8), (1, 16), (2, 5)])
def test_head_groups(lib, bits, kvh, g):
    run(lib, 7 * g + bits, bits, 32, kvh, g, [70, 0, 33, 200], [1, 2, 5, 3])


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_chains_of_ragged_rows(lib, bits):
    run(lib, 300 + bits, bits, 16, 8, 4, [0, 5, 300, 64, 1, 700], [5, 1, 0, 8, 7, 3], layers=3,
        layer=2)


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("n", [0, 50, 300])
def test_draft_trees(lib, bits, n):
    lens, rows = [n, n + 13], [17, 17]
    run(lib, 400 + bits + n, bits, 32, 2, 4, lens, rows, vis=tree_words(TREE16) * 2)


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_words_of_64_rows_and_empty_rows(lib, bits):
    r = np.random.default_rng(5)
    words = [int(w) for w in r.integers(0, 1 << 63, 64, dtype=np.uint64) * 2 + 1]
    words[0] = words[40] = 0  # with no prefix these rows see nothing: zeros
    words[63] = (1 << 64) - 1
    _, b, _, out = run(lib, 500 + bits, bits, 16, 1, 4, [0], [64], vis=words)
    got = out.view(64, -1).float()
    assert not got[0].any() and not got[40].any() and got[1].any()
    run(lib, 510 + bits, bits, 16, 1, 4, [45], [64], vis=words)


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("lens,rows", [([0], [70]), ([37, 0], [33, 129]), ([300], [257]),
                                       ([5, 90, 1], [9, 12, 100])])
def test_prompt_chunks(lib, bits, lens, rows):
    run(lib, 600 + sum(rows) + bits, bits, 64, 2, 4, lens, rows)
    run(lib, 601 + sum(rows) + bits, bits, 16, 1, 3, lens, rows)


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_peaked_and_flat_scores(lib, bits):
    """scores far apart (one slot takes nearly everything) and all alike"""
    run(lib, 700 + bits, bits, 32, 2, 4, [400, 900], [1, 4], scale=12.0)
    run(lib, 701 + bits, bits, 32, 2, 4, [400, 900], [1, 40], scale=0.0)


def test_one_slot_returns_v(lib):
    pool, b, q, out = run(lib, 9, 16, 16, 2, 4, [0, 0], [1, 1])
    for s in range(2):
        v = pool.kv[0, int(b.table[s, 0]), 2:, 0]  # [kvh][128]
        assert torch.equal(out[s].view(2, 4, 128), v[:, None].expand(2, 4, 128))


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("lens,rows,tree", [([30, 100], [1, 1], False), ([30, 100], [5, 3], False),
                                            ([40], [17], True), ([20, 3], [60, 33], False)])
def test_values_that_no_row_sees(lib, bits, lens, rows, tree):
    """NaN and infinities in every slot behind a session and in whole foreign pages change
    nothing; in a node's slot they reach the rows that see it and no others."""
    seed, page, kvh, g = 800 + bits + sum(rows), 32, 2, 4
    pool = Pool(seed, bits, pages_for(page, lens, rows) + 2, kvh, page)
    b = new_batch(seed, pool.pages, page, lens, rows)
    vis = tree_words(TREE16) if tree else None
    dv = None if vis is None else keep(torch.tensor(vis, dtype=torch.int64, device=DEV))
    q = rand_q(seed + 1, b.rows, kvh * g)
    want, tol = reference(pool, b, q, kvh * g, vis)
    clean = attend(lib, pool, b, q, kvh * g, dv).clone()
    used = torch.zeros(pool.pages, page, dtype=torch.bool, device=DEV)
    for s, (n, r) in enumerate(zip(lens, rows)):
        for j in range(n + r):
            used[int(b.table[s, j // page]), j % page] = True
    t = pool.kv[0] if bits == 16 else pool.scales[0]
    junk = torch.where(torch.rand(t.shape, device=DEV) < 0.5, float("nan"), float("inf")).to(t.dtype)
    t.copy_(torch.where(used[:, None, :, None], t, junk))
    assert torch.equal(attend(lib, pool, b, q, kvh * g, dv), clean)
    check(clean, want, tol)
    # the second node of session 0: rows that see it turn NaN, the others keep their bits
    if rows[0] < 2:
        return
    slot = lens[0] + 1
    t[int(b.table[0, slot // page]), kvh:, slot % page] = float("nan")
    t[int(b.table[0, slot // page]), :kvh, slot % page] = float("inf")
    out = attend(lib, pool, b, q, kvh * g, dv)
    for i in range(b.rows):
        sees = i < rows[0] and (bool(vis[i] & 2) if tree else i >= 1)
        if sees:
            assert torch.isnan(out[i].float()).all(), i
        else:
            assert torch.equal(out[i], clean[i]), i


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("rows", [[1, 2, 1], [40, 17, 1]])
def test_pages_that_are_not_there(lib, bits, rows):
    """ids outside the pool: their slots are seen by nobody; a session with no page at all
    gets zeros"""
    page, kvh, g, lens = 16, 2, 4, [70, 40, 20]
    pool = Pool(900 + bits, bits, pages_for(page, lens, rows), kvh, page)
    b = new_batch(1, pool.pages, page, lens, rows)
    table = b.table.copy()
    table[0, 1] = pool.pages
    table[0, 3] = -7
    table[1, 0] = 2 ** 31 - 1
    table[2, :] = -1
    b = Batch(table, lens, rows, page)
    q = rand_q(2, b.rows, kvh * g)
    out = attend(lib, pool, b, q, kvh * g)
    check(out, *reference(pool, b, q, kvh * g))
    assert not out[-1].float().any()


@pytest.mark.parametrize("most", [1, 5, 100])
def test_sessions_left_out_and_padding(lib, most):
    """rows of sessions that do not fit, and rows of none, stay as they were"""
    page, kvh, g = 16, 2, 4
    lens, rows = [20, 30, -1, 60, 5], [min(most, 3), most + 1, 1, most, 1]
    safe = [20, 30, 0, 60, 5]
    pool = Pool(31, 16, pages_for(page, safe, rows), kvh, page)
    ok = new_batch(3, pool.pages, page, safe, rows)
    # session 1 has too many rows, 2 a negative length, 3 is too long
    b = Batch(ok.table, lens, rows, page, total=sum(rows) + 7, max_rows=most, max_len=59 + most)
    q = rand_q(4, b.rows, kvh * g)
    out = keep(torch.full((b.rows, kvh * g * 128), 3.5, dtype=torch.bfloat16, device=DEV))
    attend(lib, pool, b, q, kvh * g, out=out)
    want, tol = reference(pool, b, q, kvh * g)
    untouched = np.isnan(want).all((1, 2))
    assert untouched.sum() == most + 1 + 1 + most + 7
    check(out, want, tol)
    assert (out[torch.tensor(untouched, device=DEV)] == 3.5).all()
    # row counts that make no sense leave everything
    for row0 in ([0, -5, 3, 2, 9, 4], [5, 5, 5, 5, 5, 5], [7, 3, 2 ** 31 - 1, 2, 1, 0]):
        b.d_row0 = dev_i32(row0)
        out.fill_(3.5)
        attend(lib, pool, b, q, kvh * g, out=out)
        assert torch.isfinite(out.float()).all()


@pytest.mark.parametrize("rows", [1, 33])
def test_offsets_past_32_bits(lib, rows):
    """the second layer of a pool of 10 GiB, pages behind 4 GiB"""
    page, kvh, pages = 256, 8, 2601
    kv = keep(torch.empty(2, pages, 2 * kvh, page, 128, dtype=torch.bfloat16, device=DEV))
    pool = Pool(1, 16, 2, kvh, page)
    pool.kv, pool.pages, pool.layers, pool.layer = kv, pages, 2, 1
    ids = [pages - 1, 2500, 0]
    for i in ids:
        kv[1, i].normal_()
    b = Batch([ids], [2 * page + 100], [rows], page)
    q = rand_q(5, rows, 32)
    check(attend(lib, pool, b, q, 32), *reference(pool, b, q, 32))


@pytest.mark.parametrize("bits,rows", [(16, 1), (4, 5), (8, 40)])
def test_captured_replayed_and_on_another_stream(lib, bits, rows):
    """one graph replayed while the sessions grow; two workspaces on two streams at once"""
    page, kvh, g, n = 16, 2, 4, 3
    lens = [100, 3, 250]
    pool = Pool(41, bits, 80, kvh, page)
    b = new_batch(6, pool.pages, page, [x + 64 for x in lens], [rows] * n)
    b.lens = lens
    b.d_len.copy_(torch.tensor(lens, dtype=torch.int32))
    q = rand_q(7, b.rows, kvh * g)
    out = keep(torch.zeros(b.rows, kvh * g * 128, dtype=torch.bfloat16, device=DEV))
    desc = b.desc()
    work = [keep(torch.empty(lib.s2pk_paged_attention_work_floats(ctypes.byref(desc), kvh * g, kvh),
                             dtype=torch.float32, device=DEV)) for _ in range(2)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        attend(lib, pool, b, q, kvh * g, out=out, stream=side, work=work[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        attend(lib, pool, b, q, kvh * g, out=out, stream=side, work=work[0])
    for step in range(3):
        b.lens = [x + 17 * step for x in lens]
        b.d_len.copy_(torch.tensor(b.lens, dtype=torch.int32))
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check(out, *reference(pool, b, q, kvh * g), f"replay {step}")
    other = keep(torch.zeros_like(out))
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(4):
        attend(lib, pool, b, q, kvh * g, out=out, stream=first, work=work[0])
        attend(lib, pool, b, q, kvh * g, out=other, stream=second, work=work[1])
    torch.cuda.synchronize()
    assert torch.equal(out, other)
    check(out, *reference(pool, b, q, kvh * g))


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_same_bits_every_time_and_many_sessions(lib, bits):
    lens = [(37 * i) % 300 for i in range(200)]
    pool, b, q, out = run(lib, 51 + bits, bits, 16, 1, 4, lens, [1] * 200)
    for _ in range(3):
        assert torch.equal(attend(lib, pool, b, q, 4), out)


def test_a_long_session(lib):
    """33,000 slots; every split of it counts"""
    run(lib, 61, 4, 256, 1, 4, [33000, 10], [1, 1])
    run(lib, 62, 16, 128, 1, 4, [20000], [6])


@pytest.mark.parametrize("bits,rows", [(16, 1), (8, 5), (4, 2), (16, 40), (8, 40), (4, 33)])
def test_as_many_sessions_as_there_can_be(lib, bits, rows):
    lens = [(31 * i) % 50 for i in range(1024)]
    nrows = [rows if i % 97 == 5 else (i % 3 if rows > 1 else 1) for i in range(1024)]
    run(lib, 71 + bits + rows, bits, 16, 1, 2, lens, nrows)


@pytest.mark.parametrize("bits,rows", [(8, 1), (4, 1), (8, 40), (4, 40)])
@pytest.mark.parametrize("kscale,qscale", [(2.0 ** 16, 2.0 ** -16), (2.0 ** 14, 2.0 ** -14), (2.0 ** 9, 2.0 ** -8),
                                           (2.0 ** -4, 2.0 ** 6), (1.0, 2.0 ** 17)])
def test_far_off_magnitudes_of_codes(lib, bits, rows, kscale, qscale):
    """K scales of hundreds (values past 65,504), queries past f16's range: powers of two change
    no rounding where the cache's scales stay normal"""
    lens, nrows, page, kvh, g = [150, 20], [rows, 3], 32, 2, 4
    pool = Pool(81 + bits, bits, pages_for(page, lens, nrows), kvh, page)
    f = kscale if bits == 8 else kscale / 16
    pool.scales[:, :, :kvh] = (pool.scales[:, :, :kvh].float() * f).to(torch.float16)
    b = new_batch(8, pool.pages, page, lens, nrows)
    q = rand_q(9, b.rows, kvh * g, qscale * (1 if qscale < 1e4 else 2.0 ** -17))
    if qscale > 1e4:  # one vector of huge queries, orthogonal to all but a few dims
        q = q.clone()
        q.view(b.rows, kvh * g, 128)[0, 0, 3:] = 0
        q.view(b.rows, kvh * g, 128)[0, 0, :3] = 2.0 ** 17
        keep(q)
    check(attend(lib, pool, b, q, kvh * g), *reference(pool, b, q, kvh * g))


@pytest.mark.parametrize("bits,rows", [(16, 1), (8, 1), (4, 5), (16, 40), (8, 40), (4, 40)])
def test_a_nan_query_stays_in_its_row_and_head(lib, bits, rows):
    lens, nrows, page, kvh, g = [90, 30], [rows, rows], 16, 2, 4
    pool = Pool(91 + bits, bits, pages_for(page, lens, nrows), kvh, page)
    b = new_batch(10, pool.pages, page, lens, nrows)
    q = rand_q(11, b.rows, kvh * g)
    clean = attend(lib, pool, b, q, kvh * g).clone()
    q.view(b.rows, kvh * g, 128)[rows - 1, 3, 17] = float("nan")
    out = attend(lib, pool, b, q, kvh * g).view(b.rows, kvh * g, 128)
    assert torch.isnan(out[rows - 1, 3].float()).all()
    out[rows - 1, 3] = clean.view_as(out)[rows - 1, 3]
    assert torch.equal(out.view_as(clean), clean)


@pytest.mark.parametrize("rows", [1, 40])
def test_scores_that_are_all_minus_infinity(lib, rows):
    """the softmax of nothing but -inf is NaN by its formula, unlike that of no slot"""
    pool = Pool(95, 16, 4, 1, 16)
    pool.kv[:, :, 0] = float("-inf")
    b = Batch([[2, 1, 0]], [3], [rows], 16)
    q = keep(torch.ones(rows, 2 * 128, dtype=torch.bfloat16, device=DEV))
    assert torch.isnan(attend(lib, pool, b, q, 2).float()).all()


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("rows", [1, 5, 40, 100])
def test_bits_do_not_depend_on_what_lies_behind_the_end(lib, bits, rows):
    page, kvh, g = 64, 2, 4
    lens, n = [70, 300, 1], [rows, 1, rows]
    pool = Pool(51, bits, pages_for(page, lens, n), kvh, page)
    b = new_batch(52, pool.pages, page, lens, n)
    q = rand_q(53, b.rows, kvh * g)
    outs = []
    for fill in (0.0, 60000.0, float("nan")):
        for s in range(len(lens)):
            end = lens[s] + n[s]
            if end % page:
                t = pool.kv if bits == 16 else pool.scales
                t[0, int(b.table[s, end // page]), :, end % page:] = fill
        outs.append(attend(lib, pool, b, q, kvh * g))
    for o in outs[1:]:
        assert torch.equal(o, outs[0])


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("rows", [1, 5, 8, 20, 100])
def test_bounds_far_above_the_lengths(lib, bits, rows):
    """host bounds for 100,000 slots and 200 rows more than there are; 5 and 8 rows over INT8 then
    go through two vector tiles a wave"""
    page, kvh, g = 256, 2, 4
    lens, n = [0, 700, 31, 255, 1000, 256, 3, 90], [rows, 1, rows, rows, 2, rows, rows, 1]
    n = [min(x, rows) for x in n]
    pool = Pool(61, bits, pages_for(page, lens, n), kvh, page)
    b = new_batch(62, pool.pages, page, lens, n)
    b.table = np.pad(b.table, ((0, 0), (0, 400 - b.table.shape[1])), constant_values=-1)
    b.d_table = dev_i32(b.table)
    q = rand_q(63, b.rows, kvh * g)
    for most in (rows, rows + 200):
        b.max_len, b.max_rows = 100_000, most
        check(attend(lib, pool, b, q, kvh * g), *reference(pool, b, q, kvh * g), f"{most}")


@pytest.mark.parametrize("rows", [5, 8])
def test_two_vector_tiles_with_trees_and_unseen_values(lib, rows):
    """INT8, 17 to 32 query vectors, enough rounds for two vector tiles a wave"""
    page, kvh, g = 64, 4, 4
    lens, n = [4000, 4100, 3999, 64, 0, 2500], [rows] * 6
    pool = Pool(64, 8, pages_for(page, lens, n), kvh, page)
    b = new_batch(65, pool.pages, page, lens, n, max_len=50_000)
    b.table = np.pad(b.table, ((0, 0), (0, 800 - b.table.shape[1])), constant_values=-1)
    b.table[1, 3] = pool.pages  # a page that is not there
    b.d_table = dev_i32(b.table)
    words = tree_words(TREE16[:rows]) * 6
    words[2 * rows + 1] = 0  # sees the prefix alone
    words[4 * rows + 2] = 0  # sees nothing
    unseen = lens[3] + rows - 1
    for i in range(rows):
        words[3 * rows + i] &= ~(1 << (rows - 1))
    pool.scales[0, int(b.table[3, unseen // page]), :, unseen % page] = float("nan")
    q = rand_q(66, b.rows, kvh * g)
    vis = keep(torch.tensor(np.array(words, np.uint64).view(np.int64), device=DEV))
    want = reference(pool, b, q, kvh * g, words)
    check(attend(lib, pool, b, q, kvh * g, vis), *want)


@pytest.mark.parametrize("bits,rows", [(8, 1), (4, 5), (8, 40), (4, 40), (8, 100), (4, 100)])
@pytest.mark.parametrize("vscale", [2.0 ** 14, 2.0 ** 9, 2.0 ** -12])
def test_far_off_values_of_codes(lib, bits, rows, vscale):
    """V scales of hundreds in the prefix, among the nodes and alone in a tile, and tiny ones; some
    groups only, so that a tile holds both; a NaN and an infinite scale that one row's view leaves out"""
    page, kvh, g = 32, 2, 4
    lens, n = [150, 20], [rows, min(rows, 3)]
    pool = Pool(71, bits, pages_for(page, lens, n), kvh, page)
    b = new_batch(72, pool.pages, page, lens, n)
    v = pool.scales[0, :, kvh:]
    v[:, :, ::3, 1:3] = (v[:, :, ::3, 1:3].float() * vscale).to(torch.float16)
    last = lens[0] + rows - 1
    bad = pool.scales[0, int(b.table[0, last // page]), kvh:, last % page]
    bad[0, 2], bad[1, 0] = float("nan"), float("inf")
    q = rand_q(73, b.rows, kvh * g)
    out = attend(lib, pool, b, q, kvh * g)
    with np.errstate(invalid="ignore"):
        want, tol = reference(pool, b, q, kvh * g)
    seen = rows - 1  # the one row that sees the bad scales
    got = out.float().view(b.rows, kvh, g, HD).cpu()
    assert torch.isnan(got[seen, 0, :, 64:96]).all()
    assert not torch.isfinite(got[seen, 1, :, :32]).any()
    keep_rows = [i for i in range(b.rows) if i != seen]
    flat = torch.tensor(keep_rows, device=DEV)
    check(out[flat], want[keep_rows], tol[keep_rows], f"{vscale}")
