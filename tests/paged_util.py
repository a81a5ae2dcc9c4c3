"""Pools, batches and a binary64 reference for the paged-cache tests."""
import ctypes

import numpy as np
import torch

import s2pamd
from gpu_util import DEV, LIVE, bf16_bits, bf16_vals, to_host

HD = 128


def keep(t):
    LIVE.append(t)
    return t


def dev_i32(v):
    return keep(torch.tensor(np.asarray(v, np.int32), device=DEV))


class Pool:
    """A pool of random values on the GPU and what it stands for on the host."""

    def __init__(self, seed, bits, pages, kvh, page, layers=1, layer=0):
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        self.bits, self.pages, self.kvh, self.page = bits, pages, kvh, page
        self.layers, self.layer = layers, layer
        shape = (layers, pages, 2 * kvh, page)
        self.scales = None
        if bits == 16:
            self.kv = torch.randn(*shape, HD, generator=g, device=DEV).to(torch.bfloat16)
        else:
            n = HD if bits == 8 else HD // 2
            self.kv = torch.randint(-127, 128, (*shape, n), generator=g, device=DEV,
                                    dtype=torch.int8)
            s = torch.rand(*shape, 4, generator=g, device=DEV) + 0.5
            self.scales = (s / (73 if bits == 8 else 4.6)).to(torch.float16)
        for t in (self.kv, self.scales):
            if t is not None:
                keep(t)

    def desc(self):
        return s2pamd.PagePool(kv=self.kv.data_ptr(),
                               scales=None if self.scales is None else self.scales.data_ptr(),
                               layers=self.layers, pages=self.pages, kv_heads=self.kvh,
                               page=self.page, bits=self.bits)

    def values(self, ids, layer=None):
        """[len(ids)][2 kvh][page][128] in binary64"""
        layer = self.layer if layer is None else layer
        ids = torch.as_tensor(np.asarray(ids, np.int64), device=DEV)
        kv = self.kv[layer][ids].cpu()
        if self.bits == 16:
            return kv.double().numpy()
        kv = kv.numpy()
        if self.bits == 4:
            u = kv.view(np.uint8)
            kv = np.stack([u & 15, u >> 4], -1).reshape(*u.shape[:-1], HD).astype(np.int32)
            kv = np.where(kv > 7, kv - 16, kv)
        sc = self.scales[layer][ids].cpu().numpy().astype(np.float64)
        return kv * np.repeat(sc, 32, -1)


class Batch:
    def __init__(self, table, lens, rows, page, total=None, max_rows=None, max_len=None):
        self.table = np.asarray(table, np.int32)
        self.lens, self.nrows, self.page = list(lens), list(rows), page
        self.row0 = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.rows = int(self.row0[-1]) if total is None else total
        self.max_rows = max_rows or max(1, max(rows))
        self.max_len = max_len or max(1, max(n + r for n, r in zip(lens, rows)))
        self.d_table, self.d_len, self.d_row0 = map(dev_i32, (self.table, lens, self.row0))

    def desc(self):
        return s2pamd.PageBatch(table=self.d_table.data_ptr(), len=self.d_len.data_ptr(),
                                row0=self.d_row0.data_ptr(), sessions=len(self.lens),
                                max_pages=self.table.shape[1], rows=self.rows,
                                max_rows=self.max_rows, max_len=self.max_len)


def new_batch(seed, pool_pages, page, lens, rows, **kw):
    """every session on random pages of its own"""
    need = [-(-(n + r) // page) for n, r in zip(lens, rows)]
    ids = np.random.default_rng(seed).permutation(pool_pages)[:sum(need)]
    table = np.full((len(lens), max(1, max(need))), -1, np.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = ids[at:at + n]
        at += n
    return Batch(table, lens, rows, page, **kw)


def pages_for(page, lens, rows):
    return sum(-(-(n + r) // page) for n, r in zip(lens, rows)) + 2


def attend(lib, pool, batch, q, qh, vis=None, out=None, stream=None, work=None):
    if out is None:
        out = keep(torch.empty(batch.rows, qh * HD, dtype=torch.bfloat16, device=DEV))
    b, p = batch.desc(), pool.desc()
    if work is None:
        n = lib.s2pk_paged_attention_work_floats(ctypes.byref(b), qh, pool.kvh)
        assert n > 0
        work = keep(torch.empty(n, dtype=torch.float32, device=DEV))
    s2pamd.hip_check(lib.s2pk_paged_attention(
        ctypes.byref(p), ctypes.byref(b), pool.layer, s2pamd.dptr(q), qh, s2pamd.dptr(vis),
        s2pamd.dptr(out), s2pamd.dptr(work), s2pamd.stream_ptr(stream)), "paged attention")
    return out


def reference(pool, batch, q, qh, vis=None):
    """(output, tolerance) [rows][qh][128] in binary64; rows of no session are NaN.

    The tolerance counts a kernel's roundings: the output to bf16 (2^-8 of it), p to
    bf16 and, over codes, v to bf16 (2^-8 of sum p |v| / l each), over codes also k to
    bf16, which moves a score by at most 2^-8 sum |q k| / sqrt(128) and with it p's share
    of the output; 2^-10 more on p covers the f32 sums and exponentials."""
    rows, kvh, page = batch.rows, pool.kvh, pool.page
    g = qh // kvh
    qv = bf16_vals(q.cpu().view(torch.int16).numpy().view(np.uint16)).astype(np.float64).reshape(
        rows, kvh, g, HD)
    out = np.full((rows, kvh, g, HD), np.nan)
    tol = np.zeros_like(out)
    h8 = 2.0 ** -8
    for s, (n, r) in enumerate(zip(batch.lens, batch.nrows)):
        r0 = int(batch.row0[s])
        if r <= 0 or n < 0 or r > batch.max_rows or n + r > batch.max_len:
            continue
        ids = batch.table[s, :-(-(n + r) // page)]
        there = np.repeat((ids >= 0) & (ids < pool.pages), page)[:n + r]
        kv = pool.values(np.where((ids >= 0) & (ids < pool.pages), ids, 0))
        kv = kv.transpose(1, 0, 2, 3).reshape(2 * kvh, -1, HD)[:, :n + r]
        for i in range(r):
            seen = there.copy()
            if vis is None:
                seen[n + i + 1:] = False
            else:
                for b in range(r):
                    seen[n + b] &= bool((int(vis[r0 + i]) >> b) & 1)
            j = np.nonzero(seen)[0]
            if not len(j):
                out[r0 + i] = 0
                continue
            for h in range(kvh):
                k, v, x = kv[h, j], kv[kvh + h, j], qv[r0 + i, h]
                z = x @ k.T / np.sqrt(HD)
                p = np.exp(z - z.max(1, keepdims=True))
                p /= p.sum(1, keepdims=True)
                o = p @ v
                e = (h8 * (1 if pool.bits == 16 else 2) + 2.0 ** -10) * (p @ np.abs(v))
                if pool.bits != 16:
                    dz = h8 * (np.abs(x) @ np.abs(k).T) / np.sqrt(HD)
                    e += (p * np.expm1(dz)) @ np.abs(v) + (p * np.expm1(dz)).sum(1)[:, None] * np.abs(o)
                out[r0 + i, h], tol[r0 + i, h] = o, e + h8 * np.abs(o)
    return out.reshape(rows, qh, HD), tol.reshape(rows, qh, HD)


def check(got, want, tol, what=""):
    got = bf16_vals(to_host(got.view(torch.int16), np.uint16)).astype(np.float64).reshape(want.shape)
    rows = ~np.isnan(want).all((1, 2))
    bad = ~(np.abs(got - want) <= tol + 1e-30) & rows[:, None, None]
    assert not bad.any(), (
        f"{what}: {int(bad.sum())} of {bad.size} off; first {np.argwhere(bad)[0]}, got "
        f"{got[bad][:4]}, want {want[bad][:4]}, tolerance {tol[bad][:4]}")
    # on average a rounding is far below its bound
    err = np.linalg.norm((got - want)[rows]) / max(1e-30, np.linalg.norm(want[rows]))
    assert err < 8e-3, (what, err)


def rand_q(seed, rows, qh, scale=1.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return keep((torch.randn(rows, qh * HD, generator=g, device=DEV) * scale).to(torch.bfloat16))


def tree_words(parent):
    out = []
    for i in range(len(parent)):
        w, j = 0, i
        while j >= 0:
            w |= 1 << j
            j = parent[j]
        out.append(w)
    return out


__all__ = [n for n in dir() if not n.startswith("_")] + ["bf16_bits"]
