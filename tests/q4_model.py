"""A plain model of a key/value cache in 4 bits, for the tests: its bytes by
their addresses, the codes by their definition, attention, accumulated weights and
eviction in 64 bits. Pages, slots and calls that every cache has are
shared_model's."""
import numpy as np
import torch

import motoria_amd as M
from shared_model import TORCH, Cache


def addresses(page, hd, keys):
    """For token t and element d of a page: the byte and the half of its code, and the
    first byte of its s and m."""
    t, d = np.arange(page)[:, None], np.arange(hd)[None]
    g = hd // 32
    if keys:
        word = (t * 4 + d % 32 // 8) * g + d // 32
        nibble = d % 8 // 2 + 4 * (d % 2)
        byte, high = word * 4 + nibble // 2, nibble % 2 + 0 * t
        low = page * hd // 2 + page * hd // 16 + 2 * (t * g + d // 32)
    else:
        byte = ((t // 4 * 16 + d % 32 // 2) * g + d // 32) * 4 + np.array([0, 2, 1, 3])[t % 4]
        high = d % 2 + 0 * t
        low = page * hd // 2 + page * hd // 16 + 2 * ((t // 4 * g + d // 32) * 4 + t % 4)
    scale = page * hd // 2 + 2 * ((t // 4 * g + d // 32) * 4 + t % 4)
    return byte, high, scale, low


def codes_of(x):
    """Codes, s and m (float16) of float32 x [..., 32] by the definition; what is not
    finite or too large is put in range first."""
    x = np.where(np.isnan(x), np.float32(0), np.clip(x, np.float32(-32768), np.float32(32768)))
    m = x.min(-1).astype(np.float16) + np.float16(0)  # (-0 as 0)
    diff = np.maximum(x.max(-1) - m.astype(np.float32), np.float32(0)) + np.float32(0)
    s = (diff / np.float32(15)).astype(np.float16)
    above = x.astype(np.float64) - m.astype(np.float64)[..., None]
    step = s.astype(np.float64)[..., None]
    c = sum((above >= (k + 0.5) * step).astype(np.int64) for k in range(15))
    return np.where(step > 0, c, 0), s, m


class CacheQ4(Cache):
    """A cache in 4 bits on the GPU and its model."""

    def __init__(self, g, **kw):
        kw = dict(dict(type=M.MHIP_Q4, n_layers=2, n_kv_heads=2, head_dim=64, page=16, n_pages=40,
                       max_seqs=8, max_blocks=9), **kw)
        self.g, self.d = g, M.PageDims(**kw)
        self.gpu = M.Pages(g, self.d)
        d = self.d
        self.int = np.uint8
        shape = (d.n_layers, d.n_pages, d.n_kv_heads, d.page * d.head_dim * 5 // 8)
        rng = np.random.default_rng(1)
        # pages that hold nothing are full of NaN and other bytes
        self.k, self.v = (rng.integers(0, 256, shape, dtype=np.uint8) for _ in (0, 1))
        for a in (self.k, self.v):
            tail = a[..., d.page * d.head_dim // 2:].reshape(*shape[:3], -1, 2)
            tail[..., 1] |= 0x7c
        self.load()
        self.table = [[] for _ in range(d.max_seqs)]
        self.len = [0] * d.max_seqs
        self.refs = [0] * d.n_pages
        self.held = []
        self.T = d.max_blocks * d.page
        self.w = rng.random((d.n_layers, d.max_seqs, d.n_kv_heads, self.T), dtype=np.float32)
        assert self.gpu.weights_bytes() == self.w.nbytes
        self.d_w = self.up(self.w, np.float32)
        self.at = [addresses(d.page, d.head_dim, keys) for keys in (True, False)]

    def copy_rows(self, a, b, rows):  # a page goes whole
        self.k[:, b], self.v[:, b] = self.k[:, a], self.v[:, a]

    def set_weights(self, w):
        self.w = np.ascontiguousarray(w, np.float32)
        self.g.check(M.lib().mhip_h2d(self.g.h, self.d_w, self.w.ctypes.data, self.w.nbytes), "h2d")

    # -- one token's bytes
    def put(self, which, layer, page, h, t, x):
        byte, high, scale, low = (a[t] for a in self.at[which])
        raw = (self.k, self.v)[which][layer, page, h]
        c, s, m = codes_of(x.reshape(-1, 32))
        c = c.reshape(-1)
        for d in range(len(byte)):
            raw[byte[d]] = (raw[byte[d]] & (0x0f if high[d] else 0xf0)) | c[d] << (4 * high[d])
        for j in range(len(byte) // 32):
            raw[scale[32 * j]:scale[32 * j] + 2] = s[j:j + 1].view(np.uint8)
            raw[low[32 * j]:low[32 * j] + 2] = m[j:j + 1].view(np.uint8)

    def get(self, which, layer, page, h):
        """float64 s c [page][hd] and m [page][hd] of a page."""
        byte, high, scale, low = self.at[which]
        raw = (self.k, self.v)[which][layer, page, h]
        c = (raw[byte] >> (4 * high)) & 15

        def half(at):
            two = np.stack([raw[at], raw[at + 1]], -1)
            return np.ascontiguousarray(two).view(np.float16)[..., 0].astype(np.float64)
        return half(scale) * c, half(low)

    def parts(self, which, layer, slot, n=None):
        """float64 s c and m, [n][heads][hd] each, of a slot's first n tokens."""
        n = self.len[slot] if n is None else n
        d = self.d
        out = np.zeros((2, len(self.table[slot]) * d.page, d.n_kv_heads, d.head_dim))
        with np.errstate(invalid="ignore"):
            for i, p in enumerate(self.table[slot]):
                for h in range(d.n_kv_heads):
                    out[:, i * d.page:(i + 1) * d.page, h] = self.get(which, layer, p, h)
        return out[0, :n], out[1, :n]

    # -- calls
    def rows_of(self, a, pad, t):
        """Rows of values (float32) as bytes of type t, pad values further apart; and rounded."""
        x = torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(TORCH[t])
        n, w = x.shape
        r = torch.zeros(n, w + pad, dtype=TORCH[t])
        r[:, :w] = x
        return r.view(torch.uint8).numpy(), x.float().numpy()

    def write_q4(self, layer, t, seqs, counts, k, v, top, pad=0, weights=True):
        """k, v: float32 [n * top][heads * hd]."""
        d = self.d
        raw = [self.rows_of(a, pad, t) for a in (k, v)]
        self.gpu.write_q4(layer, t, self.up(seqs), None if counts is None else self.up(counts), len(seqs), top,
                          self.up(raw[0][0], np.uint8), self.up(raw[1][0], np.uint8),
                          d.n_kv_heads * d.head_dim + pad, self.d_w if weights else None)
        for i, s in enumerate(seqs):
            n = top if counts is None else counts[i]
            for j in range(n):
                pos = self.len[s] - n + j
                b, r = divmod(pos, d.page)
                for which in (0, 1):
                    x = raw[which][1][i * top + j].reshape(d.n_kv_heads, -1)
                    for h in range(d.n_kv_heads):
                        self.put(which, layer, self.table[s][b], h, r, x[h])
                if weights:
                    self.w[layer, s, :, pos] = 0

    def fill(self, seqs, lens, rng, t=M.MHIP_F32, spread=1.0):
        """Slots of given lengths, every layer's rows at random (with some larger channels)."""
        self.extend(seqs, lens)
        d, top = self.d, max(max(lens), 1)
        for layer in range(d.n_layers):
            shape = (len(seqs) * top, d.n_kv_heads * d.head_dim)
            big = np.exp(0.5 * rng.standard_normal(shape[1])) * spread
            k, v = (rng.standard_normal(shape) * big + 0.3 * spread * rng.standard_normal(shape[1]) for _ in (0, 1))
            self.write_q4(layer, t, seqs, lens, k, v, top)

    def fork_weights(self, src, dst, deep=False, model=True):
        flags = M.MHIP_PAGES_DEEP if deep else 0
        real, self.gpu.fork = self.gpu.fork, lambda a, b, n, f: self.gpu.fork_weights(self.d_w, a, b, n, flags)
        try:
            self.fork(src, dst, deep, model)
        finally:
            self.gpu.fork = real
        if model:
            for a, b in zip(src, dst):
                self.w[:, b, :, :self.len[a]] = self.w[:, a, :, :self.len[a]]

    def evict(self, seqs, keep, recent, max_len=None, model=True):
        max_len = max([self.len[s] for s in seqs if 0 <= s < len(self.len)] + [0]) if max_len is None else max_len
        nbytes = self.gpu.evict_ws_bytes(len(seqs), keep, max_len)
        assert nbytes
        self.gpu.evict(self.d_w, self.up(seqs), len(seqs), keep, recent, max_len, self.up(np.full(nbytes, 0x7b), np.uint8))
        if not model:
            return
        d = self.d
        shared = {s: [self.refs[p] > 1 for p in self.table[s]] for s in seqs}
        old = {s: list(self.table[s]) for s in seqs}
        before = self.k.copy(), self.v.copy()
        nb, active = -(-keep // d.page), [s for s in seqs if self.len[s] > keep]
        for s in active:  # pages first, in the list's order, none of those given back
            self.table[s] = [self.take() if shared[s][b] else old[s][b] for b in range(nb)]
        for s in active:
            for b, p in enumerate(old[s]):
                if b >= nb or shared[s][b]:
                    self.refs[p] -= 1
        for s in active:
            n = self.len[s]
            for layer in range(d.n_layers):
                for h in range(d.n_kv_heads):
                    w = self.w[layer, s, h]
                    key = np.where(np.isnan(w), -np.inf, w)[:n - recent]
                    nan = np.isnan(w[:n - recent])
                    order = np.lexsort((np.arange(n - recent), nan, -key))[:keep - recent]
                    stay = np.concatenate([np.sort(order), np.arange(n - recent, n)]).astype(int)
                    for r, a in enumerate(stay):
                        self.move(before, layer, h, old[s][a // d.page], a % d.page, self.table[s][r // d.page], r % d.page)
                    w[:keep] = w[stay].copy()
            self.len[s] = keep

    def move(self, before, layer, h, pa, a, pb, b):
        for which, now in enumerate((self.k, self.v)):
            byte, _, scale, low = self.at[which]
            x, y = before[which][layer, pa, h], now[layer, pb, h]
            y[byte[b]] = x[byte[a]]
            for at in (scale, low):
                y[at[b]], y[at[b] + 1] = x[at[a]], x[at[a] + 1]

    def check(self, bits=0):
        super().check(bits)
        got = self.g.download(self.d_w, self.w.shape, np.float32)
        assert np.array_equal(got.view(np.uint32), self.w.view(np.uint32))


def attend(q, k, v, scale):
    """A token's heads in 64 bits: q [heads][hd]; k, v as parts() gives them, cut to what it
    sees. Output, weights [tokens][kv], the sums of the weights with the sizes of v, of s c and of s c and m
    apart, and how large the sums are that give the scores."""
    (ks, km), (vs, vm) = k, v
    n, kv, hd = ks.shape
    g = q.shape[0] // kv
    out, w, sizes = np.zeros(q.shape), np.zeros((n, kv)), np.zeros((3,) + q.shape)
    err = 0.0
    if n == 0:
        return out, w, sizes, err
    for h in range(q.shape[0]):
        kk, sc, mm = (ks + km)[:, h // g], vs[:, h // g], vm[:, h // g]
        s = scale * (kk @ q[h])
        e = np.exp(s - s.max())
        e /= e.sum()
        out[h] = e @ (sc + mm)
        for x, a in zip(sizes, (np.abs(sc + mm), sc, sc + np.abs(mm))):
            x[h] = e @ a
        w[:, h // g] += e
        err = max(err, scale * ((np.abs(ks) + np.abs(km))[:, h // g] @ np.abs(q[h])).max())
    return out, w, sizes, err


def tolerances(t, n, hd, sizes, err):
    """How far an output (before its own rounding) may be off, and a weight as a factor of
    itself. u = 2^-24. A score is a sum of hd products and G of
    the m, each of them cut or rounded in fp32 (2^-23, and sixteen times that where codes of 16-bit rows are
    lined up as larger than they are), G products with s; fp32 queries enter within
    2^-22. A weight's relative error is that of its score and of the row's reference, two exponentials'
    (2^-21) and the sums'. A weight enters within half a step of fp16 (2^-11, bf16 rows) or 2^-22 (two
    pieces) and is the same one for s c and m, so that is an error of it times v; its product with s is rounded by
    as much again, which is an error of s c alone; and the sums of s c and of m are apart in fp32, a
    rounding a product (sixteen times that for s c, as above), of their own sizes. fp16's least
    step adds 2^-30 a weight."""
    u = 2.0 ** -24
    v, sc, both = sizes
    cut = 1 if t == M.MHIP_F32 else 16
    e = err * ((hd * cut + 16) * 2 * u + (4 * u if t == M.MHIP_F32 else 0))
    weight = 2 * e + 2.0 ** -21 + (n + 80) * u
    once = 2.0 ** -11 if t == M.MHIP_BF16 else 2.0 ** -21
    return (weight + once) * v + once * sc + (n + 80) * u * both + (n / 32 + 8) * cut * 2 * u * sc + n * 2.0 ** -30 * sc, weight
