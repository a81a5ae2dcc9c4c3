"""The refusals of the paged-cache calls (no GPU): bad arguments are errors before
anything is launched, no rows is success, sizes are pure functions."""
import ctypes
import subprocess
from pathlib import Path

import pytest

import s2pamd
from s2pamd import PageBatch, PagePool, PageTables

ROOT = Path(__file__).resolve().parent.parent
A = 1 << 20  # an aligned address, never read
MIRRORS = [("s2p_page_pool", PagePool), ("s2p_page_batch", PageBatch),
           ("s2p_page_tables", PageTables)]


@pytest.fixture(scope="module")
def lib():
    return s2pamd.load()


def pool(**kw):
    d = dict(kv=A, scales=None, layers=2, pages=8, kv_heads=8, page=16, bits=16)
    return ctypes.byref(PagePool(**{**d, **kw}))


def batch(**kw):
    d = dict(table=A, len=A, row0=A, sessions=2, max_pages=4, rows=2, max_rows=1, max_len=64)
    return ctypes.byref(PageBatch(**{**d, **kw}))


def tables(**kw):
    d = dict(ref=A, table=A, held=A, len=A, sessions=4, max_pages=4)
    return ctypes.byref(PageTables(**{**d, **kw}))


BAD_POOL = [dict(kv=None), dict(kv=A + 8), dict(bits=5), dict(bits=8), dict(bits=4, scales=A + 8),
            dict(page=8), dict(page=48), dict(page=512), dict(page=0), dict(layers=0),
            dict(pages=0), dict(pages=-1), dict(pages=(1 << 21) + 1), dict(kv_heads=0),
            dict(kv_heads=2000)]
BAD_BATCH = [dict(table=None), dict(len=None), dict(row0=None), dict(sessions=0),
             dict(sessions=1025), dict(max_pages=0), dict(max_rows=0), dict(max_len=0),
             dict(max_len=65), dict(max_rows=65, max_len=64)]
BAD_TABLES = [dict(ref=None), dict(table=None), dict(held=None), dict(len=None), dict(sessions=0),
              dict(sessions=1025), dict(max_pages=0)]


def attention(lib, p, b, layer=0, q=A, qh=32, vis=None, out=2 * A, work=A):
    return lib.s2pk_paged_attention(p, b, layer, q, qh, vis, out, work, None)


def append(lib, p, b, layer=0, qkv=A, qh=32, qn=A, kn=A, rope=A, n_pos=64, q=2 * A):
    return lib.s2pk_paged_append(p, b, layer, qkv, qh, qn, kn, 1e-6, rope, n_pos, None, q, None)


@pytest.mark.parametrize("kw", BAD_POOL, ids=str)
def test_bad_pools(lib, kw):
    p = pool(**kw)
    assert attention(lib, p, batch()) != 0
    assert append(lib, p, batch()) != 0
    assert lib.s2pk_paged_commit(p, batch(), A, A, None, None) != 0
    assert lib.s2pk_pages_reserve(p, tables(), A, A, A, None) != 0
    assert lib.s2pk_pages_fork(p, tables(), A, A, 1, None, None) != 0
    assert lib.s2pk_pages_free(p, tables(), A, None) != 0
    assert lib.s2pk_pages_compact(p, tables(), None, A, None) != 0


@pytest.mark.parametrize("kw", BAD_BATCH, ids=str)
def test_bad_batches(lib, kw):
    assert attention(lib, pool(), batch(**kw)) != 0
    assert append(lib, pool(), batch(**kw)) != 0
    assert lib.s2pk_paged_commit(pool(), batch(**kw), A, A, None, None) != 0


@pytest.mark.parametrize("kw", BAD_TABLES, ids=str)
def test_bad_tables(lib, kw):
    t = tables(**kw)
    assert lib.s2pk_pages_reserve(pool(), t, A, A, A, None) != 0
    assert lib.s2pk_pages_fork(pool(), t, A, A, 1, None, None) != 0
    assert lib.s2pk_pages_free(pool(), t, A, None) != 0
    assert lib.s2pk_pages_compact(pool(), t, None, A, None) != 0


def test_other_arguments(lib):
    p, b, t = pool(), batch(), tables()
    for kw in (dict(layer=-1), dict(layer=2), dict(q=None), dict(q=A + 2), dict(out=None),
               dict(out=2 * A + 8), dict(work=None), dict(work=A + 4), dict(qh=0), dict(qh=-32),
               dict(qh=12), dict(qh=17 * 8), dict(vis=A + 4)):
        assert attention(lib, p, b, **kw) != 0, kw
    # visibility words have 64 bits
    assert attention(lib, p, batch(max_rows=65, max_len=64 + 1, max_pages=5), vis=A) != 0
    for kw in (dict(layer=2), dict(qkv=None), dict(qkv=A + 2), dict(q=None), dict(rope=None),
               dict(rope=A + 4), dict(n_pos=0), dict(qn=None), dict(kn=None), dict(kn=A + 2),
               dict(qh=12)):
        assert append(lib, p, b, **kw) != 0, kw
    assert lib.s2pk_paged_commit(p, b, None, A, None, None) != 0
    assert lib.s2pk_paged_commit(p, b, A, None, None, None) != 0
    assert lib.s2pk_paged_commit(p, batch(max_rows=65, max_len=70, max_pages=5), A, A, None,
                                 None) != 0
    assert lib.s2pk_pages_reserve(p, t, None, A, A, None) != 0
    assert lib.s2pk_pages_reserve(p, t, A, A, None, None) != 0
    assert lib.s2pk_pages_fork(p, t, None, A, 1, None, None) != 0
    assert lib.s2pk_pages_fork(p, t, A, None, 1, None, None) != 0
    assert lib.s2pk_pages_free(p, t, None, None) != 0
    assert lib.s2pk_pages_compact(p, t, None, None, None) != 0
    assert lib.s2pk_rope_table(A, 4, 64, 1e6, None) != 0
    assert lib.s2pk_rope_table(A, 4, 128, -1.0, None) != 0
    assert lib.s2pk_rope_table(None, 4, 128, 1e6, None) != 0
    for f in (lib.s2pk_pages_reserve, ):
        assert f(None, t, A, A, A, None) != 0
        assert f(p, None, A, A, A, None) != 0


def test_outputs_in_place_of_inputs(lib):
    """other blocks still read the rows that one writes"""
    assert attention(lib, pool(), batch(), q=A, out=A) != 0
    assert append(lib, pool(), batch(), qkv=A, q=A) != 0


def test_more_rounds_than_are_counted(lib):
    big = dict(sessions=1024, max_pages=1 << 22, max_len=1 << 30)
    assert attention(lib, pool(page=256), batch(**big)) != 0
    assert lib.s2pk_paged_attention_work_floats(batch(**big), 32, 8) > 0


def test_no_rows_is_success(lib):
    b = batch(rows=0)
    assert attention(lib, None, b) == 0
    assert append(lib, None, b) == 0
    assert lib.s2pk_paged_commit(None, b, None, None, None, None) == 0
    assert lib.s2pk_pages_fork(None, None, None, None, 0, None, None) == 0
    assert lib.s2pk_rope_table(None, 0, 128, 1e6, None) == 0


def test_struct_mirrors(tmp_path):
    """the ctypes mirrors lie as the header says"""
    lines = [f'P("{c}.{f}", offsetof({c}, {f}));' for c, m in MIRRORS for f, _ in m._fields_]
    lines += [f'P("{c}", sizeof({c}));' for c, _ in MIRRORS]
    src = tmp_path / "layout.cpp"
    src.write_text("#define __HIP_PLATFORM_AMD__ 1\n#include <cstdio>\n#include <s2pro/paged.h>\n"
                   '#define P(n, v) std::printf("%s %zu\\n", n, (size_t)(v))\n'
                   "int main() { " + "\n".join(lines) + " }\n")
    exe = tmp_path / "layout"
    subprocess.run(["g++", "-std=c++17", "-w", f"-I{ROOT}/include", "-I/opt/rocm/include", str(src),
                    "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    got = {a: int(b) for a, b in (x.split() for x in out.splitlines())}
    for c, m in MIRRORS:
        assert got[c] == ctypes.sizeof(m)
        for f, _ in m._fields_:
            assert got[f"{c}.{f}"] == getattr(m, f).offset, f


def test_sizes(lib):
    assert lib.s2p_page_pool_bytes(pool()) == 2 * 8 * 16 * 16 * 256
    assert lib.s2p_page_pool_scale_bytes(pool()) == 0
    q = pool(bits=4, scales=A)
    assert lib.s2p_page_pool_bytes(q) == 2 * 8 * 16 * 16 * 64
    assert lib.s2p_page_pool_scale_bytes(q) == 2 * 8 * 16 * 16 * 8
    # past 32 bits
    assert lib.s2p_page_pool_bytes(pool(pages=100000, layers=36)) == 36 * 100000 * 16 * 16 * 256
    assert lib.s2pk_paged_attention_work_floats(batch(), 32, 8) > 0
    assert lib.s2pk_paged_attention_work_floats(batch(), 33, 8) == 0
    assert lib.s2pk_paged_attention_work_floats(None, 32, 8) == 0
    assert lib.s2pk_pages_work_ints(pool(), tables()) >= 8 + 4
