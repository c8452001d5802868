"""Attention over a cache in 4 bits and the weights it adds up, against 64 bits on the
values that the cache holds: types, head layouts, lengths, masks, limits and replays."""
import ctypes

import numpy as np
import pytest
import torch

import motoria_amd as M
from q4_model import CacheQ4, attend, tolerances
from shared_model import TORCH, TYPES

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def g():
    gpu = M.Gpu()
    yield gpu
    gpu.close()


def call(c, layer, t, n_heads, q, seqs, counts, top, max_len, scale, weights=True, pad=0, ws=None):
    """Rows out (float64 [n * top][heads][hd]); q float32 [n * top][heads * hd], rounded to t."""
    d, g = c.d, c.g
    width, n = n_heads * d.head_dim, len(seqs)
    raw, _ = c.rows_of(q, pad, t)
    nbytes = c.gpu.attention_q4_ws_bytes(t, n_heads, n, top, max_len, weights)
    assert nbytes
    ws = c.up(np.full(nbytes, 0x7f), np.uint8) if ws is None else ws
    blank = np.full((n * top, raw.shape[1] + 0), 0x5a, np.uint8)
    out = c.up(blank, np.uint8)
    c.gpu.attention_q4(layer, t, n_heads, c.up(raw, np.uint8), width + pad, out, width + pad, c.up(seqs),
                       None if counts is None else c.up(counts), n, top, max_len, scale, c.d_w if weights else None, ws)
    got = g.download(out, blank.shape, np.uint8)
    rows = torch.from_numpy(got).view(TORCH[t])
    e = 4 if t == M.MHIP_F32 else 2
    assert (got[:, width * e:] == 0x5a).all()  # what is between the rows
    return rows[:, :width].double().numpy().reshape(n * top, n_heads, d.head_dim)


def check(c, layer, t, n_heads, q, seqs, counts, top, max_len, scale, weights=True, pad=0):
    d = c.d
    got = call(c, layer, t, n_heads, q, seqs, counts, top, max_len, scale, weights, pad)
    _, x = c.rows_of(q, 0, t)
    x = x.astype(np.float64).reshape(len(seqs) * top, n_heads, d.head_dim)
    want_w, tol_w = c.w.astype(np.float64), np.zeros(c.w.shape)
    eps = torch.finfo(TORCH[t]).eps
    for i, s in enumerate(seqs):
        n = top if counts is None else counts[i]
        k, v = c.parts(0, layer, s), c.parts(1, layer, s)
        for j in range(top):
            see = max(0, c.len[s] - n + j + 1) if j < n else 0
            o, w, sizes, err = attend(x[i * top + j], [a[:see] for a in k], [a[:see] for a in v], scale)
            off, fw = tolerances(t, see, d.head_dim, sizes, err)
            row = got[i * top + j]
            if see == 0:
                assert (row == 0).all(), (s, j)
                continue
            tol = off + eps / 2 * (np.abs(o) + off) + 2.0 ** -25
            assert (np.abs(row - o) <= tol).all(), (s, j, np.abs(row - o).max(), (np.abs(row - o) / tol).max())
            want_w[layer, s, :, :see] += w.T
            tol_w[layer, s, :, :see] += fw * w.T
    if weights:
        got_w = c.g.download(c.d_w, c.w.shape, np.float32)
        rows = n_heads // d.n_kv_heads * top
        tol_w = tol_w * (1 + 2.0 ** -20) + (rows + 8) * 2.0 ** -24 * want_w * (tol_w > 0)
        assert (np.abs(got_w - want_w) <= tol_w).all(), (np.abs(got_w - want_w) - tol_w).max()
        c.w = got_w
    c.check()
    return got


def queries(rng, n, heads, hd, scale):
    return rng.standard_normal((n, heads * hd)) * np.exp(0.5 * rng.standard_normal(heads * hd)) / (scale * np.sqrt(hd)) * 1.5


LAYOUTS = [  # heads, cache
    (16, dict(n_kv_heads=2, head_dim=128, n_layers=2)),                                   # 8 rows a head
    (4, dict(n_kv_heads=4, head_dim=64, n_layers=1, page=32, max_blocks=5)),              # as many heads as key/value heads
    (5, dict(n_kv_heads=1, head_dim=256, n_layers=1, page=64, max_blocks=3)),             # one head for all
    (20, dict(n_kv_heads=1, head_dim=32, n_layers=1, page=16)),                           # more than a tile of rows
    (6, dict(n_kv_heads=2, head_dim=96, n_layers=1, page=128, max_blocks=2)),
    (40, dict(n_kv_heads=2, head_dim=160, n_layers=1, page=32, max_blocks=5)),
    (3, dict(n_kv_heads=3, head_dim=224, n_layers=1, page=256, max_blocks=1)),
    (9, dict(n_kv_heads=1, head_dim=192, n_layers=1, page=16)),
]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("layout", range(len(LAYOUTS)))
def test_layouts(g, layout, t):
    """Every type, head size and ratio: one token, some, and chunks; lengths from none up."""
    print("test_layouts", LAYOUTS[layout], t, flush=True)
    heads, kw = LAYOUTS[layout]
    c = CacheQ4(g, **kw)
    d = c.d
    rng = np.random.default_rng(100 * layout + t)
    full = d.max_blocks * d.page
    scale = d.head_dim ** -0.5
    try:
        lens = [min(full, x) for x in (1, 33, 100, full - 2, 0, 17)]
        c.fill([0, 1, 2, 3, 4, 5], lens, rng, t)
        layer = d.n_layers - 1
        seqs = [3, 0, 4, 2, 1, 5]
        check(c, layer, t, heads, queries(rng, 6, heads, d.head_dim, scale), seqs, None, 1, max(lens), scale, pad=[0, 16][layout % 2])
        counts = [3, 1, 0, 5, 2, 4]
        check(c, layer, t, heads, queries(rng, 30, heads, d.head_dim, scale), seqs, counts, 5, full, scale, weights=layout % 2 == 0)
        check(c, layer, t, heads, queries(rng, 2 * 70, heads, d.head_dim, scale), [3, 1], [70, 33], 70, max(lens), scale)
    finally:
        c.close()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 63, 127, 128, 129, 160, 255, 257, 383, 500, 511, 513])
def test_lengths(g, t, length):
    """A slot's end anywhere in a tile, a wavefront's turn, a page."""
    c = CacheQ4(g, n_layers=1, n_kv_heads=1, head_dim=64, page=16, n_pages=40, max_blocks=33, max_seqs=2)
    rng = np.random.default_rng(length)
    try:
        c.fill([1], [length], rng, t)
        check(c, 0, t, 8, queries(rng, 1, 8, 64, 0.125), [1], None, 1, length, 0.125)
        n = min(length, 3)
        check(c, 0, t, 8, queries(rng, n, 8, 64, 0.125), [1], [n], n, 528, 0.125)
    finally:
        c.close()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("count", [12, 30, 70])
@pytest.mark.parametrize("max_len", [3000, 8000])
def test_weights_of_many_rows(g, t, count, max_len):
    """Rows of one, two and more turns, and wavefronts with one to four tiles of positions (as many as
    max_len gives them), of which slots fill some."""
    print("test_weights_of_many_rows", t, count, max_len, flush=True)
    c = CacheQ4(g, n_layers=1, n_kv_heads=8, head_dim=32, page=256, n_pages=8, max_blocks=32, max_seqs=2)
    rng = np.random.default_rng(count + max_len + t)
    scale = 32 ** -0.5
    try:
        c.fill([0, 1], [645, 75], rng, t)
        check(c, 0, t, 16, queries(rng, 2 * count, 16, 32, scale), [1, 0], [count - 3, count], count, max_len, scale)
    finally:
        c.close()


@pytest.mark.parametrize("t", TYPES)
def test_long_slots_in_parts(g, t):
    """Slots of several parts, of very different lengths; parts that a slot or a row does not reach."""
    c = CacheQ4(g, n_layers=1, n_kv_heads=2, head_dim=32, page=64, n_pages=330, max_blocks=150, max_seqs=4)
    rng = np.random.default_rng(t)
    scale = 32 ** -0.5
    try:
        c.fill([0, 1, 2, 3], [9001, 4097, 700, 5], rng, t)
        check(c, 0, t, 6, queries(rng, 4, 6, 32, scale), [2, 0, 3, 1], None, 1, 9600, scale)
        check(c, 0, t, 6, queries(rng, 8, 6, 32, scale), [1, 3], [4, 2], 4, 4097, scale)
    finally:
        c.close()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("heads,kv,hd", [(12, 4, 64), (5, 1, 96), (16, 2, 160), (8, 2, 256), (20, 1, 256), (40, 8, 128)])
def test_parts_of_every_layout(g, t, heads, kv, hd):
    print("test_parts_of_every_layout", t, heads, kv, hd, flush=True)
    c = CacheQ4(g, n_layers=1, n_kv_heads=kv, head_dim=hd, page=64, n_pages=60, max_blocks=25, max_seqs=3)
    rng = np.random.default_rng(heads + hd + t)
    scale = hd ** -0.5
    try:
        c.fill([0, 1, 2], [1500, 650, 1101], rng, t)
        check(c, 0, t, heads, queries(rng, 3, heads, hd, scale), [1, 0, 2], None, 1, 1600, scale)
        check(c, 0, t, heads, queries(rng, 9, heads, hd, scale), [2, 1, 0], [3, 0, 2], 3, 1500, scale)
    finally:
        c.close()


@pytest.mark.parametrize("t", TYPES)
def test_slots_longer_than_a_window_of_pages(g, t):
    """Where there are many items a workgroup goes through a long slot by itself, 4096 positions' pages at a
    time: tiles of many rows, and one token of many slots, whose scores are kept for the weights. As the values
    grow it goes through it twice."""
    print("test_slots_longer_than_a_window_of_pages", t, flush=True)
    scale = 32 ** -0.5
    for n, kv, heads, top, seqs in ((8, 1, 32, 65, [5, 0, 1, 2, 3, 4, 6, 7]), (230, 8, 16, 1, list(range(230)))):
        c = CacheQ4(g, n_layers=1, n_kv_heads=kv, head_dim=32, page=64, n_pages=n + 80, max_blocks=75, max_seqs=n)
        rng = np.random.default_rng(n + t)
        try:
            lens = [4700 if s == 5 else 1 + s % 60 for s in range(n)]
            others = [s for s in range(n) if s != 5]
            c.fill(others, [lens[s] for s in others], rng, t)
            c.extend([5], [4700])
            k, v = (rng.standard_normal((4700, kv * 32)) for _ in (0, 1))
            v *= np.exp2(np.linspace(-8, 12, 4700))[:, None]
            c.write_q4(0, t, [5], [4700], k, v, 4700)
            sizes = M.lib().mhip_attention_q4_ws_bytes(ctypes.byref(c.d), t, heads, n, top, 4800, 0)
            assert sizes == 256  # not cut into parts
            counts = None if top == 1 else [min(top, lens[s]) for s in seqs]
            check(c, 0, t, heads, queries(rng, n * top, heads, 32, scale), seqs, counts, top, 4800, scale)
        finally:
            c.close()


def test_two_contexts_at_once(g):
    """Two contexts (streams), each with a cache, weights and a workspace of its own and calls queued in turn
    without a wait, give what each gives alone."""
    rng = np.random.default_rng(17)
    other = M.Gpu()
    caches = []
    try:
        for gpu in (g, other):
            c = CacheQ4(gpu, n_layers=1, n_kv_heads=2, head_dim=128, page=32, max_blocks=40, max_seqs=6, n_pages=220)
            caches.append(c)
            c.fill(list(range(6)), [900 + 30 * i for i in range(6)], rng, M.MHIP_F16)
            c.dq = c.up(c.rows_of(rng.standard_normal((6, 8 * 128)), 0, M.MHIP_F16)[0], np.uint8)
            c.out = c.up(np.zeros((6, 2048)), np.uint8)
            c.ws = c.up(np.zeros(c.gpu.attention_q4_ws_bytes(M.MHIP_F16, 8, 6, 1, 1200, True)), np.uint8)
            c.seqs = c.up(np.arange(6))

        def step(c):
            c.gpu.attention_q4(0, M.MHIP_F16, 8, c.dq, 1024, c.out, 1024, c.seqs, None, 6, 1, 1200, 0.09, c.d_w, c.ws)
        alone = []
        for c in caches:
            c.set_weights(np.zeros_like(c.w))
            for _ in range(20):
                step(c)
            alone.append((c.g.download(c.out, (6, 2048), np.uint8), c.g.download(c.d_w, c.w.shape, np.float32)))
            c.set_weights(np.zeros_like(c.w))
        for _ in range(20):
            for c in caches:
                step(c)
        for c, (out, w) in zip(caches, alone):
            assert np.array_equal(c.g.download(c.out, (6, 2048), np.uint8), out) and out.any()
            assert np.array_equal(c.g.download(c.d_w, c.w.shape, np.float32).view(np.uint32), w.view(np.uint32))
    finally:
        for c in caches:
            c.close()
        other.close()


def test_parts_are_as_planned():
    """The long slots of the test above are cut: their workspace holds parts."""
    d = M.PageDims(M.MHIP_Q4, 1, 2, 32, 64, 330, 4, 150)
    L = M.lib()
    one = L.mhip_attention_q4_ws_bytes(ctypes.byref(d), M.MHIP_F32, 6, 4, 1, 100, 0)
    many = L.mhip_attention_q4_ws_bytes(ctypes.byref(d), M.MHIP_F32, 6, 4, 1, 9600, 0)
    assert many >= one + 2 * 4 * 6 * 32 * 4


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("spread", ["peaked", "large", "small", "one", "far"])
def test_scores_of_every_size(g, t, spread):
    """Softmaxes from flat to a single weight, queries and keys of far apart sizes, references that move."""
    c = CacheQ4(g, n_layers=1, n_kv_heads=1, head_dim=64, page=16, n_pages=40, max_blocks=33, max_seqs=2)
    rng = np.random.default_rng(5)
    q = rng.standard_normal((3, 4 * 64))
    scale = 0.125
    try:
        if spread == "peaked":
            q, size = q * 30, 1.0
        elif spread == "large":
            q, size = q * 300, 500.0
        elif spread == "small":
            q, size, scale = q * 2.0 ** -10, 2.0 ** -9, 2.0 ** 16
        elif spread == "one":
            q, size = q * 0, 1.0
        else:
            q, size = q * np.exp(2.5 * rng.standard_normal(q.shape)), 1.0
        c.extend([0], [500])
        k, v = (rng.standard_normal((500, 64)) * size for _ in (0, 1))
        k *= np.linspace(0.2, 1, 500)[:, None]  # later keys score higher
        c.write_q4(0, t, [0], [500], k, v, 500)
        check(c, 0, t, 4, q, [0], [3], 3, 528, scale)
    finally:
        c.close()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("order", ["up", "down", "spikes"])
def test_values_of_every_size(g, t, order):
    """Values that grow or shrink by 2^20 along a slot, so that what a wavefront sees first says nothing about
    the rest, and single tokens that are far larger than all others; more rows than a tile too."""
    c = CacheQ4(g, n_layers=1, n_kv_heads=1, head_dim=64, page=16, n_pages=60, max_blocks=50, max_seqs=2)
    rng = np.random.default_rng(11)
    n = 780
    try:
        size = np.exp2(np.linspace(-8, 12, n))
        if order == "down":
            size = size[::-1]
        elif order == "spikes":
            size = np.where(np.arange(n) % 97 == 60, 3000.0, 0.01)
        c.extend([0], [n])
        k, v = (rng.standard_normal((n, 64)) for _ in (0, 1))
        c.write_q4(0, t, [0], [n], k, v * size[:, None], n)
        check(c, 0, t, 4, queries(rng, 3, 4, 64, 0.125), [0], [3], 3, 800, 0.125)
        check(c, 0, t, 4, queries(rng, 20, 4, 64, 0.125), [0], [20], 20, 800, 0.125)
    finally:
        c.close()


@pytest.mark.parametrize("scale", [2.0 ** -64, 2.0 ** -20, 2.0 ** 64])
@pytest.mark.parametrize("t", [M.MHIP_F32, M.MHIP_BF16])
def test_scales(g, t, scale):
    """The limits of the scale, against queries that make up for it, or do not."""
    c = CacheQ4(g, n_layers=1, n_kv_heads=1, head_dim=32, page=16, max_seqs=2)
    rng = np.random.default_rng(8)
    try:
        c.fill([0], [77], rng, t)
        q = rng.standard_normal((2, 3 * 32))
        check(c, 0, t, 3, q / scale / 8, [0], [2], 2, 80, scale)
        if scale < 1:
            check(c, 0, t, 3, q, [0], [2], 2, 80, scale)          # every weight the same
    finally:
        c.close()


@pytest.mark.parametrize("t", TYPES)
def test_limits(g, t):
    """Slots out of range or longer than max_len are NaN rows with an error bit, others are right, and
    no weights are added for them."""
    c = CacheQ4(g, n_layers=1, n_kv_heads=2, head_dim=64)
    rng = np.random.default_rng(1)
    try:
        c.fill([0, 1, 2], [50, 90, 20], rng, t)
        q = queries(rng, 5, 4, 64, 0.125)
        got = call(c, 0, t, 4, q, [0, 8, 1, -5, 2], None, 1, 60, 0.125)
        assert c.gpu.status()[0] == M.MHIP_PAGES_BAD
        assert np.isnan(got[[1, 2, 3]]).all()
        w = c.g.download(c.d_w, c.w.shape, np.float32)
        assert np.array_equal(w[:, [1, 3, 4, 5, 6, 7]], c.w[:, [1, 3, 4, 5, 6, 7]])
        c.set_weights(c.w)
        good = check(c, 0, t, 4, q[[0, 4]], [0, 2], None, 1, 60, 0.125)
        assert np.array_equal(good, got[[0, 4]])
    finally:
        c.close()


@pytest.mark.parametrize("t", TYPES)
def test_a_page_out_of_range_counts_as_zeros(g, t):
    c = CacheQ4(g, n_layers=1, n_kv_heads=2, head_dim=64, page=16)
    rng = np.random.default_rng(2)
    try:
        c.fill([0], [70], rng, t)
        real = list(c.table[0])
        for bad in (-1, c.d.n_pages, 1 << 30):
            table = np.full((c.d.max_seqs, c.d.max_blocks), -1, np.int32)
            table[0, :5] = real
            table[0, 2] = bad
            g.check(M.lib().mhip_h2d(g.h, c.gpu.arrays.table, table.ctypes.data, table.nbytes), "h2d")
            q = queries(rng, 1, 4, 64, 0.125)
            got = call(c, 0, t, 4, q, [0], None, 1, 70, 0.125, weights=False)
            assert c.gpu.status()[0] == M.MHIP_PAGES_BAD
            x = c.rows_of(q, 0, t)[1].astype(np.float64).reshape(4, 64)
            k, v = c.parts(0, 0, 0), c.parts(1, 0, 0)
            for a in (*k, *v):
                a[32:48] = 0
            o, _, sizes, err = attend(x, k, v, 0.125)
            off = tolerances(t, 70, 64, sizes, err)[0]
            tol = off + torch.finfo(TORCH[t]).eps / 2 * (np.abs(o) + off) + 2.0 ** -25
            assert (np.abs(got[0] - o) <= tol).all()
    finally:
        c.close()


@pytest.mark.parametrize("t", TYPES)
def test_queries_that_are_not_finite(g, t):
    """They spoil their own row and no other."""
    c = CacheQ4(g, n_layers=1, n_kv_heads=1, head_dim=64)
    rng = np.random.default_rng(3)
    try:
        c.fill([0, 1], [100, 40], rng, t)
        q = queries(rng, 4, 4, 64, 0.125)
        good = call(c, 0, t, 4, q, [0, 1], [2, 2], 2, 100, 0.125, weights=False)
        q[0, 64 * 1 + 5] = np.nan
        q[3, 64 * 2 + 9] = np.inf
        got = call(c, 0, t, 4, q, [0, 1], [2, 2], 2, 100, 0.125, weights=False)
        bad = np.zeros((4, 4), bool)
        bad[0, 1] = bad[3, 2] = True
        assert np.isnan(got[bad]).all() and np.array_equal(got[~bad], good[~bad])
    finally:
        c.close()


def test_weights_are_the_same_every_time(g):
    """Sums do not depend on what else runs: twelve calls from the same start, bit for bit."""
    c = CacheQ4(g, n_layers=1, n_kv_heads=2, head_dim=64, page=16, n_pages=150, max_blocks=70, max_seqs=4)
    rng = np.random.default_rng(4)
    try:
        c.fill([0, 1, 2], [1000, 700, 30], rng)
        q = queries(rng, 3 * 9, 16, 64, 0.125)
        first = None
        start = c.w.copy()
        for _ in range(12):
            c.set_weights(start)
            out = call(c, 0, M.MHIP_F32, 16, q, [0, 1, 2], [9, 4, 9], 9, 1000, 0.125)
            w = g.download(c.d_w, c.w.shape, np.float32)
            if first is None:
                first = out, w
            assert np.array_equal(out, first[0]) and np.array_equal(w.view(np.uint32), first[1].view(np.uint32))
    finally:
        c.close()


@pytest.mark.parametrize("t", TYPES)
def test_a_budget_kept(g, t):
    """As a program uses them together: a prompt, forks of it, steps of a token each with weights added up, an
    eviction whenever a slot is past its budget, then a chunk of a next turn."""
    heads, layers = 8, 2
    c = CacheQ4(g, n_layers=layers, n_kv_heads=2, head_dim=64, page=16, n_pages=60, max_blocks=9, max_seqs=5)
    d = c.d
    rng = np.random.default_rng(6)
    width = d.n_kv_heads * d.head_dim
    try:
        c.fill([0], [75], rng, t)
        for layer in range(layers):
            check(c, layer, t, heads, queries(rng, 75, heads, 64, 0.125), [0], [75], 75, 75, 0.125)
        c.fork_weights([0, 0], [1, 2])
        seqs = [2, 0, 1]
        for step in range(7):
            c.extend(seqs, None)
            for layer in range(layers):
                k, v = (rng.standard_normal((3, width)) for _ in (0, 1))
                c.write_q4(layer, t, seqs, None, k, v, 1)
                check(c, layer, t, heads, queries(rng, 3, heads, 64, 0.125), seqs, None, 1, 144, 0.125)
            if c.len[2] > 78:
                c.evict(seqs, 64, 16)
                c.check()
        c.extend([1], [40])
        for layer in range(layers):
            k, v = (rng.standard_normal((40, width)) for _ in (0, 1))
            c.write_q4(layer, t, [1], [40], k, v, 40)
            check(c, layer, t, heads, queries(rng, 40, heads, 64, 0.125), [1], [40], 40, 144, 0.125)
        c.free(seqs)
        c.check()
    finally:
        c.close()


def test_graph_of_a_step(g):
    """A captured step of a batch (pages, rows, attention with weights in every layer, eviction), replayed: each
    replay gives what the same calls give eagerly on a second cache."""
    heads, layers, t = 8, 2, M.MHIP_BF16
    rng = np.random.default_rng(9)
    kw = dict(n_layers=layers, n_kv_heads=2, head_dim=64, page=16, n_pages=60, max_blocks=9, max_seqs=5)
    a, b = CacheQ4(g, **kw), CacheQ4(g, **kw)
    L = M.lib()
    try:
        for c in (a, b):
            c.fill([0, 1, 2], [70, 63, 10], np.random.default_rng(1), t)
            c.fork_weights([0], [4])
        seqs = [4, 2, 1, 0]
        q = queries(rng, 4 * layers, heads, 64, 0.125)
        kv = rng.standard_normal((2, 4, 128))
        step = []
        for c in (a, b):
            out = c.up(np.zeros((layers * 4, heads * 64)), np.uint16)
            ws = c.up(np.zeros(c.gpu.attention_q4_ws_bytes(t, heads, 4, 1, 144, True)), np.uint8)
            ews = c.up(np.zeros(c.gpu.evict_ws_bytes(4, 72, 144)), np.uint8)
            dq = c.up(c.rows_of(q, 0, t)[0], np.uint8)
            dk, dv = (c.up(c.rows_of(x, 0, t)[0], np.uint8) for x in kv)
            ds = c.up(seqs)

            def run(c=c, out=out, ws=ws, ews=ews, dq=dq, dk=dk, dv=dv, ds=ds):
                c.gpu.extend(ds, None, 4)
                for layer in range(layers):
                    at = layer * 4 * heads * 64 * 2
                    c.gpu.write_q4(layer, t, ds, None, 4, 1, dk, dv, 128, c.d_w)
                    c.gpu.attention_q4(layer, t, heads, dq + at, heads * 64, out + at, heads * 64, ds, None, 4, 1, 144,
                                       0.125, c.d_w, ws)
                c.gpu.evict(c.d_w, ds, 4, 72, 9, 144, ews)
            step.append((run, out))
        g.check(L.mhip_sync(g.h), "sync")
        g.check(L.mhip_graph_begin(g.h), "begin")
        step[0][0]()
        graph = ctypes.c_void_p()
        g.check(L.mhip_graph_end(g.h, ctypes.byref(graph)), "end")
        for replay in range(6):
            g.check(L.mhip_graph_launch(g.h, graph), "launch")
            step[1][0]()
            got, want = (g.download(out, (layers * 4, heads * 64), np.uint16) for _, out in step)
            assert np.array_equal(got, want), replay
            assert all(np.array_equal(x, y) for x, y in zip(a.books(), b.books()))
            assert np.array_equal(*(g.download(c.d_w, c.w.shape, np.float32).view(np.uint32) for c in (a, b)))
            assert np.array_equal(*(g.download(c.gpu.arrays.k, c.k.shape, np.uint8) for c in (a, b)))
            assert a.gpu.status() == b.gpu.status()
        L.mhip_graph_destroy(graph)
    finally:
        a.close()
        b.close()


def test_a_pool_behind_32_bits(g):
    """Pages beyond 2^32 bytes of both arrays are read where they are."""
    d = M.PageDims(M.MHIP_Q4, 9, 8, 256, 128, 4 * 1024, 2, 4)
    p = M.Pages(g, d)
    rng = np.random.default_rng(0)
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
        k, v = (rng.standard_normal((300, width)).astype(np.float32) for _ in (0, 1))
        p.write_q4(8, M.MHIP_F32, up([1]), up([300]), 1, 300, up(k, np.float32), up(v, np.float32), width)
        back = up(np.zeros((300, width)), np.float32), up(np.zeros((300, width)), np.float32)
        p.read_q4(8, M.MHIP_F32, up([1]), up([300]), 1, 300, *back, width)
        k, v = (g.download(x, (300, 8, 256), np.float32).astype(np.float64) for x in back)
        q = rng.standard_normal((1, width)).astype(np.float32) * 2
        out = up(np.zeros((1, width)), np.float32)
        ws = up(np.zeros(p.attention_q4_ws_bytes(M.MHIP_F32, 8, 1, 1, 300)), np.uint8)
        p.attention_q4(8, M.MHIP_F32, 8, up(q, np.float32), width, out, width, up([1]), None, 1, 1, 300, 1 / 16, None, ws)
        got = g.download(out, (8, 256), np.float32)
        o, _, sizes, err = attend(q.astype(np.float64).reshape(8, 256), (k, 0 * k), (v, 0 * v), 1 / 16)
        # (s c and m are not apart here: neither is larger than 16, as no value is beyond +-8)
        assert np.abs(v).max() < 8 and np.abs(k).max() < 8
        err += 16 * np.abs(q).sum() / 16
        tol = tolerances(M.MHIP_F32, 300, 256, np.abs(sizes) + 16, err)[0] + 2.0 ** -24 * np.abs(o)
        assert (np.abs(got - o) <= tol).all()
        assert p.status()[0] == 0
    finally:
        for h in held:
            g.free(h)
        p.close()
