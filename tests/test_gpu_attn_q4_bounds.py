"""What attention over a cache in 4 bits promises of its roundings (include/mia_hip.h), against 64 bits, on
inputs whose scores are known so well that the roundings of weights and values are what is left."""
import numpy as np
import pytest

import motoria_amd as M
from q4_model import CacheQ4, codes_of
from shared_model import TYPES
from test_gpu_attn_q4 import call

pytestmark = pytest.mark.gpu
HALF = {  # of a value in [1, 2), and the least exponent
    M.MHIP_F32: (2.0 ** -24, -126), M.MHIP_F16: (2.0 ** -11, -14), M.MHIP_BF16: (2.0 ** -8, -126),
}


@pytest.fixture(scope="module")
def g():
    gpu = M.Gpu()
    yield gpu
    gpu.close()


def half_step(t, x):
    """Half a step of type t at x, and not more (relative to a value it is up to twice smaller)."""
    half, least = HALF[t]
    return np.exp2(np.maximum(np.floor(np.log2(np.abs(x) + 1e-300)), least)) * half


def rows_of(q, k, v, scale):
    """A token's heads in 64 bits, as q4_model.attend: output, weights [heads][tokens] and how large the sums
    are that give the scores."""
    (ks, km), (vs, vm) = k, v
    g = q.shape[0] // ks.shape[1]
    at = np.arange(q.shape[0]) // g
    s = scale * np.einsum("hd,thd->ht", q, (ks + km)[:, at])
    w = np.exp(s - s.max(1, keepdims=True))
    w /= w.sum(1, keepdims=True)
    err = scale * np.einsum("hd,thd->ht", np.abs(q), (np.abs(ks) + np.abs(km))[:, at]).max()
    return np.einsum("ht,thd->hd", w, (vs + vm)[:, at]), w, err


def bound(t, w, v, err, tiles, products=32):
    """How far an output may be off before its own rounding, and a weight as a factor of itself.
    A score: `products` of queries and codes that are not 0, each cut at 2^-23 of the largest by the matrix cores, a
    product with s and a sum (2^-23 each), and the m in one more; fp32 queries enter within 2^-22. Its
    weight is off by twice that (its own and the reference's), two exponentials' 2^-21 and the sums'. Weights enter
    within 2^-23 of their size or 2^-34 of the row's largest (or as nothing), their products with s within 3 2^-23 or, all
    of them, within 2^-18 (16-bit rows 2^-15) of the group's largest sum of weight x s x code, which is no more than that
    of weight x 15 s: n products are off by 2^-24 (1 + s / 2) each, times a code of 15, and their sum is
    (1 + s / 2) n / 4 (n / 32) at least, or they are not taken, so by 15 2^-22 = 2^-18.1 (15 2^-19 = 2^-15.1) of it. Sums over the tokens: a wavefront adds 32 at a time (2^-22 of the sum so far each),
    then wavefronts and parts are joined (2^-20)."""
    (vs, vm), g = v, w.shape[0] // v[0].shape[1]
    at = np.arange(w.shape[0]) // g
    e = err * ((products + 2) * 2.0 ** -23 + (2.0 ** -22 if t == M.MHIP_F32 else 0))
    weight = 2 * e + 2.0 ** -21 + 2.0 ** -22 + tiles * 2.0 ** -22 + 2.0 ** -20
    few = 2.0 ** -18 if t == M.MHIP_F32 else 2.0 ** -15
    n = vs.shape[0]
    most = vs.reshape(n, vs.shape[1], -1, 32).max(-1) * (15 / 14)  # (of 32 codes the greatest is 14 or 15)
    group = np.repeat(np.einsum("ht,thg->hg", w, most[:, at]), 32, -1)
    both = np.einsum("ht,thd->hd", w, (vs + np.abs(vm))[:, at])
    off = weight * both + few * group
    lost = np.einsum("ht,thd->hd", np.minimum(w, 2.0 ** -34 * w.max(1, keepdims=True)), (vs + np.abs(vm))[:, at])
    return off + 2.0 ** -22 * both + lost, weight


def check(c, t, heads, q, seqs, counts, top, max_len, scale, tiles, products=32, weights=False):
    """Rows held to the bound and one rounding, and the weights added up to theirs; prints how far they are off in
    units of that."""
    d = c.d
    if weights:
        c.set_weights(np.zeros_like(c.w))
    got = call(c, 0, t, heads, q, seqs, counts, top, max_len, scale, weights=weights)
    x = c.rows_of(q, 0, t)[1].astype(np.float64).reshape(len(seqs) * top, heads, d.head_dim)
    want, tol_w = np.zeros(c.w.shape), np.zeros(c.w.shape)
    for i, s in enumerate(seqs):
        n = top if counts is None else counts[i]
        k, v = c.parts(0, 0, s), c.parts(1, 0, s)
        for j in range(n):
            see = c.len[s] - n + j + 1
            seen = [a[:see] for a in v]
            o, w, err = rows_of(x[i * top + j], [a[:see] for a in k], seen, scale)
            off, fw = bound(t, w, seen, err, tiles, products)
            row = got[i * top + j]
            tol = off + half_step(t, np.abs(o) + off)
            over = np.abs(row - o) / (tol + 1e-300)
            print("row", s, j, "of", see, "worst", over.max(), "of the tolerance", flush=True)
            assert (over <= 1).all(), (s, j, np.abs(row - o).max(), over.max(), (over > 1).mean())
            sums = w.reshape(d.n_kv_heads, -1, see).sum(1)
            want[0, s, :, :see] += sums
            # (a weight of less than fp32's least is nothing)
            tol_w[0, s, :, :see] += (fw + see * 2.0 ** -34) * sums + 2.0 ** -120
    if weights:
        got_w = c.g.download(c.d_w, c.w.shape, np.float32).astype(np.float64)
        tol_w += (heads * top + 8) * 2.0 ** -24 * want
        assert (np.abs(got_w - want) <= tol_w).all(), (np.abs(got_w - want) / (tol_w + 1e-300)).max()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("heads,kv,hd,length,count", [(4, 1, 32, 100, 2), (16, 2, 64, 200, 1), (20, 1, 32, 130, 3), (4, 1, 160, 77, 1)])
def test_one_rounding(g, t, heads, kv, hd, length, count):
    """A row's output is its formula's, rounded once: scores of a few units, from one element of each query, so
    that what scores are off by is far below the output's step."""
    print("test_one_rounding", t, heads, kv, hd, length, count, flush=True)
    c = CacheQ4(g, n_layers=1, n_kv_heads=kv, head_dim=hd, page=16, n_pages=40, max_blocks=16, max_seqs=2)
    rng = np.random.default_rng(heads + hd)
    try:
        c.extend([0], [length])
        k, v = (rng.standard_normal((length, kv * hd)) for _ in (0, 1))
        c.write_q4(0, t, [0], [length], k, v, length)
        q = np.zeros((count, heads, hd))
        q[:, np.arange(heads), rng.integers(0, hd, heads)] = 1.5
        check(c, t, heads, q.reshape(count, -1), [0], [count], count, length, 1.0, length // 128 + 1)
    finally:
        c.close()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [32, 128])
def test_scores_of_queries_of_far_apart_sizes(g, t, hd):
    """A query with one element of 512 at a code of 1, one at a code of 0 and the others of about 2^-14 at codes
    of 15: all that is small has to reach the score. Seen by the weights, which are fp32. A score is off by 33 cuts
    of 2^-23 of its largest product (34 with the product with s); what is small is 2^-14 of it in all."""
    print("test_scores_of_queries_of_far_apart_sizes", t, hd, flush=True)
    n = 60
    c = CacheQ4(g, n_layers=1, n_kv_heads=1, head_dim=hd, page=16, max_seqs=2)
    try:
        step = np.linspace(2.0 ** -10, 1, n).astype(np.float16).astype(np.float32)  # a token's s, 15 of which are fp16's too
        code = np.full(hd, 15.0, np.float32)
        code[0], code[1] = 1, 0
        code[32::32] = 0  # (a least value of 0 in every group)
        c.extend([0], [n])
        k = step[:, None] * code
        c.write_q4(0, t, [0], [n], k, np.zeros_like(k), n)
        q = np.full((1, hd), 2.0 ** -14 * 1.5, np.float32)
        q[0, 0], q[0, 1], q[0, 32::32] = 512, 0, 0
        scale = 2.0 ** -6
        x = c.rows_of(q, 0, t)[1].astype(np.float64).reshape(1, hd)
        ks, km = c.parts(0, 0, 0)
        assert (km == 0).all() and (ks[:, 0, 0] > 0).all()
        start = np.zeros_like(c.w)
        c.set_weights(start)
        call(c, 0, t, 1, q, [0], None, 1, 144, scale)
        got = g.download(c.d_w, c.w.shape, np.float32)[0, 0, 0, :n].astype(np.float64)
        _, w, err = rows_of(x, (ks, km), c.parts(1, 0, 0), scale)
        less = np.abs(ks[:, 0, 2:] @ x[0, 2:] * scale).max()
        e = err * (34 * 2.0 ** -23 + (2.0 ** -22 if t == M.MHIP_F32 else 0))
        tol = 2 * e + 2.0 ** -21 + 2.0 ** -20
        assert less > 3 * tol  # (a score without them is seen)
        assert (np.abs(got / w[0] - 1) <= tol).all(), np.abs(got / w[0] - 1).max() / tol
    finally:
        c.close()


def one_far_ahead(c, t, n, heads, gap, values, seq=0):
    """A slot of n tokens of which the first gets a score that is `gap` powers of two above the others', which are
    all 0; its own values are 0. Returns the query: one element, so that scores are one product."""
    d = c.d
    c.extend([seq], [n])
    k = np.zeros((n, d.n_kv_heads, d.head_dim), np.float32)
    k[0, :, 0] = 15
    c.write_q4(0, t, [seq], [n], k.reshape(n, -1), values, n)
    q = np.zeros((1, heads, d.head_dim))
    q[:, :, 0] = gap * np.log(2) / 15
    return q.reshape(1, -1)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [32, 160])
@pytest.mark.parametrize("size,gap", [(1.0, 20.6), (750.0, 23.2), (7500.0, 22.2), (32000.0, 20.6), (7500.0, 30.0), (0.01, 25.0)])
def test_small_weights_of_large_values(g, t, hd, size, gap):
    """One weight of 1, at values of 0, and all others 2^-20 and less, at values of one size: what is small is all
    that there is. In one launch, in parts, and with weights added up in both ways."""
    print("test_small_weights_of_large_values", t, hd, size, gap, flush=True)
    rng = np.random.default_rng(int(gap * 10) + hd)
    for n, heads, top_len in ((500, 2, 500), (1500, 2, 1600), (500, 40, 500)):
        c = CacheQ4(g, n_layers=1, n_kv_heads=2, head_dim=hd, page=64, n_pages=30, max_blocks=25, max_seqs=2)
        try:
            v = size * (0.5 + 0.5 * rng.random((n, 2 * hd))) * np.where(np.arange(2 * hd) % 3 == 0, -1, 1)
            v[0] = 0
            q = one_far_ahead(c, t, n, heads, gap, v)
            check(c, t, heads, q, [0], None, 1, top_len, 1.0, n // 128 + 1, 1, weights=True)
        finally:
            c.close()


@pytest.mark.parametrize("t", TYPES)
def test_values_that_a_row_does_not_see(g, t):
    """Tokens of 2^15 within the first tile that the first rows do not see: they change nothing of those."""
    c = CacheQ4(g, n_layers=1, n_kv_heads=1, head_dim=64, page=16, n_pages=30, max_blocks=5, max_seqs=2)
    rng = np.random.default_rng(3)
    try:
        for seq, (n, count) in enumerate(((30, 20), (70, 50))):
            c.extend([seq], [n])
            k, v = (rng.standard_normal((n, 64)) for _ in (0, 1))
            v *= np.where(np.arange(n) < n - count + 3, 0.01, 30000)[:, None]
            c.write_q4(0, t, [seq], [n], k, np.clip(v, -32768, 32768), n)
            q = np.zeros((count, 4, 64))
            q[:, np.arange(4), rng.integers(0, 64, 4)] = 1.5
            check(c, t, 4, q.reshape(count, -1), [seq], [count], count, n, 1.0, 1, 1)
    finally:
        c.close()


@pytest.mark.parametrize("t", TYPES)
def test_large_values_of_no_weight(g, t):
    """Tokens of 2^15, the first of a slot or some of each tile, whose weights are 2^-60: what they add is far
    below what the others', of 0.01 and less, come to."""
    rng = np.random.default_rng(4)
    for n, top_len, which in ((300, 300, "first"), (300, 300, "some"), (1200, 1300, "some")):
        c = CacheQ4(g, n_layers=1, n_kv_heads=1, head_dim=64, page=16, n_pages=90, max_blocks=85, max_seqs=1)
        try:
            large = np.arange(n) < 20 if which == "first" else np.arange(n) % 31 == 7
            c.extend([0], [n])
            k = np.zeros((n, 64), np.float32)
            k[large, 0] = -15
            v = rng.standard_normal((n, 64)) * np.where(large, 1e5, 0.01 if which == "first" else 0.0005)[:, None]
            c.write_q4(0, t, [0], [n], k, np.clip(v, -32768, 32768), n)
            q = np.zeros((1, 4, 64))
            q[:, :, 0] = 60 * np.log(2) / 15
            check(c, t, 4, q.reshape(1, -1), [0], None, 1, top_len, 1.0, n // 128 + 1, 1)
        finally:
            c.close()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("heads,hd", [(4, 96), (20, 256)])
def test_groups_of_far_apart_sizes(g, t, heads, hd):
    """Groups of 32 channels from 2^15 down to 2^-13, one of zeros, in every token."""
    c = CacheQ4(g, n_layers=1, n_kv_heads=1, head_dim=hd, page=16, n_pages=20, max_blocks=13, max_seqs=1)
    rng = np.random.default_rng(5)
    n = 200
    try:
        c.extend([0], [n])
        k, v = (rng.standard_normal((n, hd)) for _ in (0, 1))
        size = np.exp2(np.linspace(13, -13, hd // 32))
        size[1] = 0
        c.write_q4(0, t, [0], [n], k, np.clip(v * np.repeat(size, 32), -32768, 32768), n)
        q = np.zeros((1, heads, hd))
        q[:, np.arange(heads), rng.integers(0, hd, heads)] = 1.5
        got = call(c, 0, t, heads, q.reshape(1, -1), [0], None, 1, n, 1.0, weights=False)
        assert (got[0, :, 32:64] == 0).all()
        check(c, t, heads, q.reshape(1, -1), [0], None, 1, n, 1.0, 2, 1)
    finally:
        c.close()


@pytest.mark.parametrize("t", [M.MHIP_F32, M.MHIP_BF16])
def test_the_largest_s(g, t):
    """Pages that a program fills by itself: any s and m that are finite."""
    c = CacheQ4(g, n_layers=1, n_kv_heads=1, head_dim=64, page=16, n_pages=8, max_blocks=5, max_seqs=1)
    rng = np.random.default_rng(6)
    try:
        c.fill([0], [77], rng, t)
        _, _, scale, low = c.at[1]
        for i, p in enumerate(c.table[0]):
            for r in range(16):
                for j in range(0, 64, 32):
                    s, m = np.float16(65504 if r % 3 else 9000), np.float16((-1) ** r * 65504)
                    c.v[0, p, 0, scale[r, j]:scale[r, j] + 2] = np.array([s]).view(np.uint8)
                    c.v[0, p, 0, low[r, j]:low[r, j] + 2] = np.array([m]).view(np.uint8)
        g.check(M.lib().mhip_h2d(g.h, c.gpu.arrays.v, c.v.ctypes.data, c.v.nbytes), "h2d")
        q = np.zeros((1, 3, 64))
        q[:, np.arange(3), [5, 40, 63]] = 2.0
        check(c, t, 3, q.reshape(1, -1), [0], None, 1, 77, 1.0, 1, 1)
    finally:
        c.close()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("heads,lens", [(4, (100, 40)), (4, (1500, 700)), (40, (100, 40))])
def test_weights_of_queries_that_are_not_finite(g, t, heads, lens):
    """A row whose query is not finite makes NaN of the weights of the positions that it sees, in its key/value
    head and slot, and of no others: scores kept and formed again, in one launch and in parts."""
    print("test_weights_of_queries_that_are_not_finite", t, heads, lens, flush=True)
    c = CacheQ4(g, n_layers=1, n_kv_heads=2, head_dim=64, page=64, n_pages=50, max_blocks=25, max_seqs=3)
    rng = np.random.default_rng(heads)
    try:
        c.fill([0, 2], list(lens), rng, t)
        q = rng.standard_normal((6, heads * 64))
        start = np.zeros_like(c.w)
        c.set_weights(start)
        good = call(c, 0, t, heads, q, [0, 2], [3, 3], 3, lens[0], 0.125)
        well = g.download(c.d_w, c.w.shape, np.float32)
        q[1, 5] = np.nan              # slot 0, its second new token, head 0 of the first key/value head
        q[3, 64 * heads - 7] = -np.inf  # slot 2, the first one, the last head
        c.set_weights(start)
        got = call(c, 0, t, heads, q, [0, 2], [3, 3], 3, lens[0], 0.125)
        w = g.download(c.d_w, c.w.shape, np.float32)
        bad = np.zeros((6, heads), bool)
        bad[1, 0] = bad[3, heads - 1] = True
        assert np.isnan(got[bad]).all() and np.array_equal(got[~bad], good[~bad])
        spoiled = np.zeros(w.shape, bool)
        spoiled[0, 0, 0, :lens[0] - 1] = spoiled[0, 2, 1, :lens[1] - 2] = True
        assert np.isnan(w[spoiled]).all()
        assert np.array_equal(w[~spoiled], well[~spoiled])
        assert c.gpu.status()[0] == 0
    finally:
        c.close()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("order", ["up", "down", "mixed"])
@pytest.mark.parametrize("heads,top", [(4, 3), (40, 3)])
def test_scores_of_thousands(g, t, order, heads, top):
    """Scores up to 20000, at least 30 apart: a row is the values of the greatest it sees, rounded, with a weight
    of 1 (of the two pieces of a weight 2^-21, of its product with s 2^-18 or 2^-15, of the reference that
    is the score itself nothing), and the others add less than 2^-40."""
    print("test_scores_of_thousands", t, order, heads, top, flush=True)
    n = 290
    c = CacheQ4(g, n_layers=1, n_kv_heads=2, head_dim=64, page=16, n_pages=40, max_blocks=20, max_seqs=2)
    rng = np.random.default_rng(8)
    try:
        size = {"up": np.arange(1, n + 1), "down": np.arange(n, 0, -1), "mixed": rng.permutation(n) + 1}[order] * 1.5
        k = np.zeros((n, 2, 64))
        k[:, :, 7] = size[:, None]
        v = rng.standard_normal((n, 128))
        c.extend([1], [n])
        c.write_q4(0, M.MHIP_F32, [1], [n], k.reshape(n, -1), v, n)
        q = np.zeros((top, heads, 64))
        q[:, :, 7] = 400
        (ks, km), (vs, vm) = c.parts(0, 0, 1), c.parts(1, 0, 1)
        score = (ks + km)[:, 0, 7] * 400 / 8
        assert np.diff(np.sort(score)).min() > 30 and score.max() > 20000
        c.set_weights(np.zeros_like(c.w))
        got = call(c, 0, t, heads, q.reshape(top, -1), [1], [top], top, n, 0.125)
        w = g.download(c.d_w, c.w.shape, np.float32)[0, 1, :, :n]
        want = np.zeros(n)
        few = 2.0 ** -18 if t == M.MHIP_F32 else 2.0 ** -15
        for j in range(top):
            see = n - top + j + 1
            at = int(score[:see].argmax())
            want[at] += heads // 2
            o = np.repeat((vs + vm)[at], heads // 2, 0)
            size15 = np.repeat(np.repeat(vs[at].reshape(2, 2, 32).max(-1), 32, -1) * 15 / 14, heads // 2, 0)
            off = 2.0 ** -20 * np.repeat((vs + np.abs(vm))[at], heads // 2, 0) + few * size15 + 2.0 ** -34
            tol = off + half_step(t, np.abs(o) + off)
            assert (np.abs(got[j] - o) <= tol).all(), (j, (np.abs(got[j] - o) / tol).max())
        assert (np.abs(w - want) <= 2.0 ** -20 * want + 2.0 ** -40).all()
    finally:
        c.close()


def test_pages_behind_32_bits_hold_what_is_attended_to(g):
    """Pages beyond 2^32 bytes of both arrays, by the s c and m that were written there: the bound is so small that
    zeros, or the tokens in another order of pages, would not pass."""
    d = M.PageDims(M.MHIP_Q4, 9, 8, 256, 128, 4 * 1024, 2, 4)
    p = M.Pages(g, d)
    rng = np.random.default_rng(10)
    held = []

    def up(x, dt=np.int32):
        held.append(g.upload(np.ascontiguousarray(x, dt)))
        return held[-1]
    L = M.lib()
    try:
        table = np.full((2, 4), -1, np.int32)
        table[1, :3] = [d.n_pages - 1, 0, d.n_pages - 2]
        lens = np.array([0, 300], np.int32)
        for at, x in ((p.arrays.table, table), (p.arrays.len, lens)):
            g.check(L.mhip_h2d(g.h, at, x.ctypes.data, x.nbytes), "h2d")
        width = 8 * 256
        rows = [rng.standard_normal((300, width)).astype(np.float32) for _ in (0, 1)]
        p.write_q4(8, M.MHIP_F32, up([1]), up([300]), 1, 300, *(up(x, np.float32) for x in rows), width)
        k, v = ([x.astype(np.float64) for x in (s[..., None] * code.astype(np.float64), m[..., None] + 0.0 * code)]
                for code, s, m in (codes_of(x.reshape(300, 8, -1, 32)) for x in rows))
        k, v = ([x.reshape(300, 8, 256) for x in y] for y in (k, v))
        q = rng.standard_normal((1, width)).astype(np.float32) * 2
        out = up(np.zeros((1, width)), np.float32)
        ws = up(np.zeros(p.attention_q4_ws_bytes(M.MHIP_F32, 8, 1, 1, 300, True)), np.uint8)
        sums = np.zeros(p.weights_bytes() // 4, np.float32)
        dw = up(sums, np.float32)
        p.attention_q4(8, M.MHIP_F32, 8, up(q, np.float32), width, out, width, up([1]), None, 1, 1, 300, 1 / 16, dw, ws)
        got = g.download(out, (8, 256), np.float32)
        x = q.astype(np.float64).reshape(8, 256)
        o, w, err = rows_of(x, k, v, 1 / 16)
        off, fw = bound(M.MHIP_F32, w, v, err, 3)
        tol = off + half_step(M.MHIP_F32, np.abs(o) + off)
        assert tol.max() < 0.02 and np.abs(o).max() > 0.5
        other = np.r_[128:256, 0:128, 256:300]
        for wrong in (0 * o, rows_of(x, k, [a[other] for a in v], 1 / 16)[0], rows_of(x, [a[other] for a in k], v, 1 / 16)[0]):
            assert (np.abs(wrong - o) > tol).mean() > 0.5
        assert (np.abs(got - o) <= tol).all(), (np.abs(got - o) / tol).max()
        got_w = g.download(dw, sums.shape, np.float32).reshape(9, 2, 8, -1)
        assert (np.abs(got_w[8, 1, :, :300] - w) <= (fw + 2.0 ** -20) * w).all()
        got_w[8, 1, :, :300] = 0
        assert (got_w == 0).all() and p.status()[0] == 0
    finally:
        for h in held:
            g.free(h)
        p.close()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("heads,count,n,parts", [(4, 1, 500, False), (40, 30, 480, False), (8, 2, 4500, False), (4, 1, 3000, True)])
def test_a_wavefront_on_its_own_goes_twice(g, t, heads, count, n, parts):
    """Positions of one wavefront (of a workgroup's four, 32 at a time) with values of 2^15 and no weight beside
    some of 2^-9: it does its part again, and the others do not; where a workgroup has more than 4096
    positions all do. Scores are kept, or formed again, for the weights, either way."""
    print("test_a_wavefront_on_its_own_goes_twice", t, heads, count, n, parts, flush=True)
    slots = 1 if parts or n < 512 else 600  # (so many that none is cut)
    c = CacheQ4(g, n_layers=1, n_kv_heads=1, head_dim=64, page=64, n_pages=n // 64 + 2 + slots, max_blocks=n // 64 + 2, max_seqs=slots)
    rng = np.random.default_rng(14)
    try:
        mine = np.arange(n) // 32 % 4 == 2
        large = mine & (np.arange(n) % 5 == 0)
        k = np.zeros((n, 64), np.float32)
        k[large, 0] = -15
        v = rng.standard_normal((n, 64)) * np.where(large, 1e5, np.where(mine, 2.0 ** -9, 1.0))[:, None]
        c.extend([0], [n])
        c.write_q4(0, t, [0], [n], k, np.clip(v, -32768, 32768), n)
        seqs, counts, lens = [0], [count], n
        if slots > 1:
            c.extend(list(range(1, slots)), [1] * (slots - 1))
            for s in range(1, slots):
                c.write_q4(0, t, [s], [1], np.ones((1, 64)), np.ones((1, 64)), 1)
            seqs, counts = list(range(slots)), [count] + [1] * (slots - 1)
        q = np.zeros((len(seqs) * count, heads, 64))
        q[:, :, 0] = 60 * np.log(2) / 15
        sizes = c.gpu.attention_q4_ws_bytes(t, heads, len(seqs), count, n)
        assert (sizes > 256) == parts
        check(c, t, heads, q.reshape(len(q), -1), seqs, counts, count, n, 1.0, n // 128 + 1, 1, weights=True)
    finally:
        c.close()


@pytest.mark.parametrize("t", [M.MHIP_F32, M.MHIP_BF16])
@pytest.mark.parametrize("size", [2.0 ** -13, 2.0 ** -17, 2.0 ** -21])
def test_the_smallest_values(g, t, size):
    """Keys and values whose m (and s) are below fp16's normal range: products with such an m are cut at 2^-37 of the
    largest weight, or of the largest of the query's sums over a group (three pieces of it for each group)."""
    print("test_the_smallest_values", t, size, flush=True)
    n, heads, hd = 200, 4, 64
    c = CacheQ4(g, n_layers=1, n_kv_heads=1, head_dim=hd, page=16, n_pages=20, max_blocks=13, max_seqs=1)
    rng = np.random.default_rng(15)
    scale = 0.25 / size
    try:
        c.extend([0], [n])
        k, v = (rng.standard_normal((n, hd)) * size for _ in (0, 1))
        c.write_q4(0, M.MHIP_F32, [0], [n], k, v, n)
        q = rng.standard_normal((1, heads, hd)) * 0.5
        got = call(c, 0, t, heads, q.reshape(1, -1), [0], None, 1, n, scale, weights=False)
        x = c.rows_of(q.reshape(1, -1), 0, t)[1].astype(np.float64).reshape(heads, hd)
        k, v = c.parts(0, 0, 0), c.parts(1, 0, 0)
        o, w, err = rows_of(x, k, v, scale)
        off, _ = bound(t, w, v, err, 2)
        cut = scale * 6 * 2.0 ** -37 * np.abs(x.reshape(heads, 2, 32).sum(-1)).max(-1)
        off = off + 2 * cut[:, None] * np.einsum("ht,thd->hd", w, np.repeat((v[0] + np.abs(v[1])), heads, 1))
        off = off + n * 2.0 ** -37 * w.max(1)[:, None]
        assert off.max() < size / 16
        tol = off + half_step(t, np.abs(o) + off)
        assert (np.abs(got[0] - o) <= tol).all(), (np.abs(got[0] - o) / tol).max()
    finally:
        c.close()
