"""Plain models of the operators for a batch of sequences, for the tests: a
paged cache as Python lists, attention and 4-bit products in 64 bits."""
import ctypes

import numpy as np
import torch

import motoria_amd as M

TORCH = {M.MHIP_F32: torch.float32, M.MHIP_F16: torch.float16, M.MHIP_BF16: torch.bfloat16}
TYPES = [M.MHIP_F32, M.MHIP_F16, M.MHIP_BF16]


def esize(t):
    return 4 if t == M.MHIP_F32 else 2


def rounded(a, t):
    """float64 values of a rounded to type t, and its bytes as integers."""
    x = torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(TORCH[t])
    raw = x.view(torch.int32 if t == M.MHIP_F32 else torch.int16).numpy()
    return x.double().numpy(), raw


def values(raw, t):
    """float64 values of integers that hold elements of type t."""
    x = torch.from_numpy(np.ascontiguousarray(raw))
    return x.view(TORCH[t]).double().numpy()


class Cache:
    """A cache on the GPU and its model: every call goes to both."""

    def __init__(self, g, **kw):
        kw = dict(dict(type=M.MHIP_F32, n_layers=2, n_kv_heads=2, head_dim=32, page=16, n_pages=40,
                       max_seqs=8, max_blocks=9), **kw)
        self.g, self.d = g, M.PageDims(**kw)
        self.gpu = M.Pages(g, self.d)
        d = self.d
        self.int = np.int32 if d.type == M.MHIP_F32 else np.int16
        shape = (d.n_layers, d.n_pages, d.n_kv_heads, d.page, d.head_dim)
        rng = np.random.default_rng(1)
        self.k = rounded(rng.standard_normal(shape), d.type)[1].reshape(shape)
        self.v = rounded(rng.standard_normal(shape), d.type)[1].reshape(shape)
        self.load()
        self.table = [[] for _ in range(d.max_seqs)]
        self.len = [0] * d.max_seqs
        self.refs = [0] * d.n_pages
        self.held = []

    def load(self):
        for p, a in ((self.gpu.arrays.k, self.k), (self.gpu.arrays.v, self.v)):
            a = np.ascontiguousarray(a)
            self.g.check(M.lib().mhip_h2d(self.g.h, p, a.ctypes.data, a.nbytes), "h2d")

    def up(self, a, dtype=np.int32):
        p = self.g.upload(np.ascontiguousarray(a, dtype))
        self.held.append(p)
        return p

    def close(self):
        for p in self.held:
            self.g.free(p)
        self.held = []
        self.gpu.close()

    # -- the model's own steps
    def take(self):
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def copy_rows(self, a, b, rows):
        self.k[:, b, :, :rows] = self.k[:, a, :, :rows]
        self.v[:, b, :, :rows] = self.v[:, a, :, :rows]

    # -- calls
    def extend(self, seqs, counts, model=True):
        self.gpu.extend(self.up(seqs), None if counts is None else self.up(counts), len(seqs))
        if model:
            for s, n in zip(seqs, counts if counts is not None else [1] * len(seqs)):
                self.len[s] += n
                while len(self.table[s]) * self.d.page < self.len[s]:
                    self.table[s].append(self.take())

    def write(self, layer, seqs, counts, k, v, top, pad=0):
        """k, v: integers [n][top][heads * hd] (rows pad values further apart)."""
        d = self.d
        w = d.n_kv_heads * d.head_dim

        def rows(a):
            r = np.zeros((len(seqs) * top, w + pad), self.int)
            r[:, :w] = a.reshape(-1, w)
            return r
        self.gpu.write(layer, self.up(seqs), None if counts is None else self.up(counts), len(seqs),
                       top, self.up(rows(k), self.int), self.up(rows(v), self.int), w + pad)
        for i, s in enumerate(seqs):
            n = top if counts is None else counts[i]
            for j in range(n):
                b, r = divmod(self.len[s] - n + j, d.page)
                for mine, new in ((self.k, k), (self.v, v)):
                    mine[layer, self.table[s][b], :, r] = new[i, j].reshape(d.n_kv_heads, -1)

    def fork(self, src, dst, deep=False, model=True):
        self.gpu.fork(self.up(src), self.up(dst), len(src), M.MHIP_PAGES_DEEP if deep else 0)
        if not model:
            return
        page = self.d.page
        for a, b in zip(src, dst):
            full = 0 if deep else self.len[a] // page
            self.table[b] = self.table[a][:full]
            for p in self.table[b]:
                self.refs[p] += 1
            self.len[b] = self.len[a]
            for x in range(full, len(self.table[a])):
                self.table[b].append(self.take())
                self.copy_rows(self.table[a][x], self.table[b][x], min(page, self.len[a] - x * page))

    def free(self, seqs):
        self.gpu.free(self.up(seqs), len(seqs))
        for s in seqs:
            for p in self.table[s]:
                self.refs[p] -= 1
            self.table[s], self.len[s] = [], 0

    def compact(self):
        self.gpu.compact()
        n = sum(r > 0 for r in self.refs)
        movers = [p for p in range(n, self.d.n_pages) if self.refs[p] > 0]
        for hole, p in zip([h for h in range(n) if self.refs[h] == 0], movers):
            self.copy_rows(p, hole, self.d.page)
            self.refs[hole], self.refs[p] = self.refs[p], 0
            self.table = [[hole if x == p else x for x in r] for r in self.table]

    # -- comparison
    def books(self):
        d, a, g = self.d, self.gpu.arrays, self.g
        return (g.download(a.table, (d.max_seqs, d.max_blocks), np.int32),
                g.download(a.len, (d.max_seqs,), np.int32),
                g.download(a.refs, (d.n_pages,), np.int32))

    def check(self, bits=0):
        table, lens, refs = self.books()
        want = np.full(table.shape, -1)
        for s, r in enumerate(self.table):
            want[s, :len(r)] = r
        assert np.array_equal(table, want), (table, want)
        assert lens.tolist() == self.len and refs.tolist() == self.refs
        for p, mine in ((self.gpu.arrays.k, self.k), (self.gpu.arrays.v, self.v)):
            assert np.array_equal(self.g.download(p, mine.shape, self.int), mine)
        assert self.gpu.status() == (bits, sum(r == 0 for r in self.refs))

    def rows(self, which, layer, slot, n):
        """float64 [n][heads][hd] of a slot's first n tokens."""
        a = values(self.k if which == "k" else self.v, self.d.type)[layer]
        if n <= 0:
            return np.zeros((0, self.d.n_kv_heads, self.d.head_dim))
        return np.concatenate([a[p].transpose(1, 0, 2) for p in self.table[slot]])[:n]


def attention(q, k, v, scale):
    """One token's heads in 64 bits: q [heads][hd], k and v [tokens][kv][hd]."""
    n, kv, hd = k.shape
    out = np.zeros(q.shape)
    if n == 0:
        return out
    g = q.shape[0] // kv
    with np.errstate(all="ignore"):
        for h in range(q.shape[0]):
            s = scale * (k[:, h // g] @ q[h])
            e = np.exp(s - s.max())
            out[h] = (e / e.sum()) @ v[:, h // g]
    return out


def attention_tolerance(q, k, v, o, scale, t, parts=64):
    """How far a computed row may be off, element by element. u = 2^-24:
    a score is a sum of hd products in fp32, off by at most (hd + 4) u times the sum
    of the products' sizes; a weight's relative error is that of its score and the
    maximum's, and of two exponentials (2^-21); the two sums add a rounding per
    token and part. With 16-bit caches a weight is rounded (half a step), and l
    is the sum of the rounded ones: two half steps at most. The output is rounded
    once."""
    u, eps = 2.0 ** -24, torch.finfo(TORCH[t]).eps
    n, kv, hd = k.shape
    tol = np.zeros(q.shape)
    if n == 0:
        return tol
    g = q.shape[0] // kv
    for h in range(q.shape[0]):
        with np.errstate(all="ignore"):  # (rows that are not finite are not compared by it)
            size = scale * (np.abs(k[:, h // g]) @ np.abs(q[h])).max()
        e = 2 * (hd + 4) * u * size + 2.0 ** -21 + (n + 2 * parts + 16) * u
        weight = 0.0 if t == M.MHIP_F32 else 2 * eps / 2
        tol[h] = (2 * e + weight) * np.abs(v[:, h // g]).max(0) + eps / 2 * np.abs(o[h])
    return tol


def q4_weights(codes, scales, group):
    """float64 weights of codes [rows][cols/2] and fp16 scales [rows][cols/group]."""
    n = np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1).astype(np.int64)
    n = np.where(n > 7, n - 16, n).astype(np.float64)
    return n * np.repeat(scales.astype(np.float64), group, axis=1)


def q4_tolerance(w, x, o, t):
    """How far a product may be off: fp32 x enters within 2^-23 of each value; the
    sum of cols products rounds at most once a product in fp32 (2^-23 each, were it to
    cut rather than round); the output is rounded once."""
    size = np.abs(x) @ np.abs(w).T
    eps = torch.finfo(TORCH[t]).eps
    return size * ((w.shape[1] + 64) * 2.0 ** -23 + 2.0 ** -23) + eps / 2 * np.abs(o)
