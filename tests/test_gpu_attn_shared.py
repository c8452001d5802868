"""Attention over a paged cache (mhip_attention_shared) against 64 bits: types,
head layouts, lengths from zero to long, prefixes and pages that end inside
tiles, padded batches, several tokens a slot, values that are not finite in
masked places, repeats and graphs, and a whole layer of a batch together with the
4-bit products."""
import ctypes

import numpy as np
import pytest

import motoria_amd as M
from shared_model import (TYPES, Cache, attention, attention_tolerance, esize, q4_tolerance,
                          q4_weights, rounded, values)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def g():
    gpu = M.Gpu()
    yield gpu
    gpu.close()


def fill(c, lens, prefix, rng):
    """Slots of the given lengths, those behind slot 0 forks of its first
    `prefix` tokens; slot 0 itself is at least that long. All values random
    from the cache's own start."""
    c.extend([0], [prefix]) if prefix else None
    if prefix and len(lens) > 1:
        behind = [s for s in range(1, len(lens)) if lens[s] >= prefix]
        if behind:
            c.fork([0] * len(behind), behind)
    for s, n in enumerate(lens):
        if n > c.len[s]:
            c.extend([s], [n - c.len[s]])


def run(c, q, heads, seqs, counts, top, prefix, max_len, scale, prefix_seq=0, layer=0, pad=0, ws=None):
    """(rows, error bits): q float64 [n * top][heads * hd]."""
    t, g, w = c.d.type, c.g, heads * c.d.head_dim
    raw = np.zeros((len(q), w + pad), c.int)
    raw[:, :w] = rounded(q, t)[1].reshape(len(q), w)
    dq, n = c.up(raw, c.int), len(seqs)
    guard = np.full((len(q) + 1, w + pad), 0x5a5a if t else 0x5a5a5a5a, c.int)
    out = c.up(guard, c.int)
    need = c.gpu.attention_ws_bytes(heads, n, top, prefix, max_len)
    assert need > 0
    ws = ws or c.up(np.zeros(need, np.uint8), np.uint8)
    c.gpu.attention(layer, heads, dq, w + pad, out, w + pad, c.up(seqs),
                    None if counts is None else c.up(counts), n, top, prefix_seq, prefix, max_len, scale, ws)
    got = g.download(out, guard.shape, c.int)
    assert np.array_equal(got[len(q):], guard[len(q):]), "a row behind the last was written"
    assert np.array_equal(got[:, w:], guard[:, w:]), "a row's padding was written"
    return values(got[:len(q), :w], t).reshape(len(q), heads, -1), c.gpu.status()[0]


def want(c, q, heads, seqs, counts, top, scale, layer=0):
    """Each row in 64 bits, and how far it may be off."""
    rows, tol = [], []
    qv = rounded(q, c.d.type)[0].reshape(len(q), heads, -1)
    for i, s in enumerate(seqs):
        n = top if counts is None else counts[i]
        for j in range(top):
            lim = max(0, c.len[s] - n + j + 1) if j < n else 0
            k, v = c.rows("k", layer, s, lim), c.rows("v", layer, s, lim)
            o = attention(qv[i * top + j], k, v, scale)
            rows.append(o)
            tol.append(attention_tolerance(qv[i * top + j], k, v, o, scale, c.d.type))
    return np.array(rows), np.array(tol)


def close(got, rows, tol):
    assert np.array_equal(np.isnan(got), np.isnan(rows))
    ok = np.isfinite(rows)
    assert np.array_equal(got[~ok & ~np.isnan(rows)], rows[~ok & ~np.isnan(rows)])
    off = np.abs(got[ok] - rows[ok]) - tol[ok]
    assert off.max(initial=-1) <= 0, off.max()


# heads, kv heads, head size, page, lengths (slot 0 first), prefix, tokens a slot
LAYOUTS = [
    (1, 1, 16, 16, [1], 0, 1),
    (4, 2, 32, 16, [5, 16, 17, 64, 65], 0, 1),
    (8, 2, 64, 32, [40, 41, 97, 33], 33, 1),
    (32, 4, 128, 16, [300, 300, 412, 555, 301], 300, 1),
    (10, 2, 80, 64, [130, 200, 131], 128, 3),
    (6, 6, 48, 16, [70, 71, 100], 64, 1),
    (5, 1, 256, 128, [260, 300, 257, 514], 256, 1),
    (32, 4, 128, 16, [900] * 7, 850, 2),
    (16, 1, 96, 256, [300, 310, 1000], 299, 5),
    (8, 4, 112, 32, [64] * 20, 64, 1),
    (24, 8, 64, 16, [5000, 4999], 4097, 1),
]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("x", range(len(LAYOUTS)))
def test_against_64_bits(g, x, t):
    heads, kv, hd, page, lens, prefix, top = LAYOUTS[x]
    print("test_against_64_bits", LAYOUTS[x], t, flush=True)
    rng = np.random.default_rng(100 + x)
    blocks = -(-max(lens) // page) + 1
    c = Cache(g, type=t, n_layers=2, n_kv_heads=kv, head_dim=hd, page=page, max_blocks=blocks,
              max_seqs=len(lens) + 1, n_pages=blocks * len(lens) + 2)
    try:
        fill(c, lens, prefix, rng)
        seqs = rng.permutation(len(lens)).tolist()
        counts = [int(n) for n in rng.integers(1, top + 1, len(seqs))]
        q = rng.standard_normal((len(seqs) * top, heads * hd)) * 2
        scale = 1 / np.sqrt(hd)
        rows, tol = want(c, q, heads, seqs, counts, top, scale, layer=1)
        for p in (prefix, 0):  # with the prefix read once, and without
            got, bits = run(c, q, heads, seqs, counts, top, p, max(lens), scale, layer=1, pad=16)
            assert bits == 0
            close(got, rows, tol)
    finally:
        c.close()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n", [1, 2, 3, 5, 9, 17, 33])
def test_batches_of_any_size(g, n, t):
    """Every shape of the prefix's row tiles (8 rows a slot: 8 to 264)."""
    rng = np.random.default_rng(n)
    c = Cache(g, type=t, n_layers=1, n_kv_heads=2, head_dim=128, max_blocks=20, max_seqs=n,
              n_pages=20 + 12 * n)
    try:
        prefix = 210
        lens = [prefix + int(x) for x in rng.integers(0, 90, n)]
        fill(c, lens, prefix, rng)
        seqs = rng.permutation(n).tolist()
        q = rng.standard_normal((n, 16 * 128)) * 2
        rows, tol = want(c, q, 16, seqs, None, 1, 0.1)
        got, bits = run(c, q, 16, seqs, None, 1, prefix, 320, 0.1)
        assert bits == 0
        close(got, rows, tol)
    finally:
        c.close()


@pytest.mark.parametrize("t", TYPES)
def test_rows_that_see_little(g, t):
    """Empty slots, a slot twice, slots shorter than the prefix, counts of zero
    and beyond the slot's length, padding rows: zeros where nothing is seen."""
    rng = np.random.default_rng(8)
    c = Cache(g, type=t, n_layers=1, n_kv_heads=2, head_dim=64, max_blocks=20, max_seqs=8, n_pages=99)
    try:
        fill(c, [150, 150, 151, 170], 150, rng)
        c.fork([0], [5])
        # slot 4 holds the prefix's first 32 tokens and no more
        c.extend([4], [32])
        for mine in (c.k, c.v):
            for b in (0, 1):
                mine[:, c.table[4][b]] = mine[:, c.table[0][b]]
        c.load()
        seqs = [3, 6, 4, 3, 0, 2, 5, 4]
        counts = [3, 3, 3, 1, 0, 2, 3, 2]
        q = rng.standard_normal((24, 4 * 64)) * 2
        rows, tol = want(c, q, 4, seqs, counts, 3, 0.125)
        for prefix in (150, 100, 0):
            got, bits = run(c, q, 4, seqs, counts, 3, prefix, 200, 0.125)
            assert bits == 0
            close(got, rows, tol)
            assert (got[3:6] == 0).all() and (got[12:15] == 0).all() and (got[10:12] == 0).all()
        # more tokens than a slot has: its first rows are before its start
        c.extend([7], [2])
        seqs, counts = [7, 7], [3, 4]
        q = q[:8]
        rows, tol = want(c, q, 4, seqs, counts, 4, 0.125)
        got, bits = run(c, q, 4, seqs, counts, 4, 0, 16, 0.125)
        assert bits == 0 and (got[0] == 0).all()
        close(got, rows, tol)
    finally:
        c.close()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_values_that_are_not_finite(g, bad, t):
    """Infinities and NaN: behind a slot's end (the rest of its last page), in
    tokens that only later rows of the slot or longer slots see, and where they
    are seen. Rows that do not see them are as without."""
    rng = np.random.default_rng(9)
    c = Cache(g, type=t, n_layers=1, n_kv_heads=1, head_dim=64, page=32, max_blocks=8, max_seqs=4, n_pages=40)
    try:
        fill(c, [96, 120, 100, 130], 96, rng)
        c.extend([0], [9])
        worst = rounded(np.array([bad]), t)[1][0]
        for mine in (c.k, c.v):
            for s in range(4):
                b, r = divmod(c.len[s], 32)
                if r:
                    mine[:, c.table[s][b], :, r:] = worst           # behind the end
                b, r = divmod(c.len[s] - 2, 32)
                mine[0, c.table[s][b], 0, r, 5:9] = worst             # the last token but one
        free = [p for p in range(40) if c.refs[p] == 0]
        c.k[:, free] = worst
        c.v[:, free] = worst
        c.load()
        seqs, counts, q = [1, 0, 3, 2], [4, 4, 4, 2], rng.standard_normal((16, 4 * 64))
        q[:, 70] = 0.0
        rows, tol = want(c, q, 4, seqs, counts, 4, 0.125)
        assert np.isfinite(rows[[0, 1, 4, 5, 8, 9]]).all() and not np.isfinite(rows[[2, 3]]).all()
        for prefix in (96, 0):
            got, bits = run(c, q, 4, seqs, counts, 4, prefix, 130, 0.125)
            assert bits == 0
            close(got, rows, tol)
        # only values: weights of the rows that see them stay finite
        c.k = np.where(np.isfinite(values(c.k, t)), c.k, rounded(np.array([0.25]), t)[1][0]).astype(c.int)
        c.load()
        rows, tol = want(c, q, 4, seqs, counts, 4, 0.125)
        got, bits = run(c, q, 4, seqs, counts, 4, 96, 130, 0.125)
        close(got, rows, tol)
        # in the prefix itself, before and behind where a short slot ends
        c.free([2])
        c.extend([2], [40])
        for mine in (c.k, c.v):
            for b in (0, 1):
                mine[:, c.table[2][b]] = mine[:, c.table[0][b]]
        c.v[0, c.table[0][1], 0, 20, 3] = worst
        c.load()
        seqs, counts, q = [2, 0, 1], [1, 1, 1], q[:3]
        rows, tol = want(c, q, 4, seqs, counts, 1, 0.125)
        assert np.isfinite(rows[0]).all() and not np.isfinite(rows[1]).all()
        got, bits = run(c, q, 4, seqs, counts, 1, 96, 130, 0.125)
        assert bits == 0
        close(got, rows, tol)
    finally:
        c.close()


@pytest.mark.parametrize("t", TYPES)
def test_scores_far_apart(g, t):
    """Scores from the type's own range: one token far above all others, scores
    that fall with every token, and keys of the type's lowest value."""
    rng = np.random.default_rng(10)
    c = Cache(g, type=t, n_layers=1, n_kv_heads=1, head_dim=32, max_blocks=20, max_seqs=2, n_pages=40)
    try:
        fill(c, [200, 300], 0, rng)
        k = values(c.k, t)
        k[0, c.table[1][7], 0, 3] *= 60.0
        for i in range(200):
            k[0, c.table[0][i // 16], 0, i % 16, 0] = 100.0 - i
        c.k = rounded(k, t)[1].reshape(c.k.shape)
        c.load()
        q = rng.standard_normal((2, 2 * 32)) * 3
        q[0, 0] = q[0, 32] = 2.0
        rows, tol = want(c, q, 2, [0, 1], None, 1, 1.0)
        got, bits = run(c, q, 2, [0, 1], None, 1, 0, 320, 1.0)
        close(got, rows, tol)
        low = rounded(np.array([-3e38 if t != M.MHIP_F16 else -65504.0]), t)[1][0]
        c.k[0, c.table[0][3]] = low  # a page of the lowest value: weights 0, or the row is NaN
        c.load()
        q = np.abs(q)
        with np.errstate(all="ignore"):
            rows, tol = want(c, q, 2, [0, 1], None, 1, 1.0)
        got, bits = run(c, q, 2, [0, 1], None, 1, 0, 320, 1.0)
        ok = np.isfinite(rows)
        assert ok.all()
        off = np.abs(got[1] - rows[1]) - tol[1]
        assert off.max() <= 0 and np.isfinite(got).all()
        assert np.abs(got[0] - rows[0]).max() <= 0.02  # (its tolerance goes by the lowest value's size)
    finally:
        c.close()


def test_long_weights_of_fp16_count(g):
    """One token 2^20 above 4000 others, which together are 2^-8 of the sum."""
    c = Cache(g, type=M.MHIP_F16, n_layers=1, n_kv_heads=1, head_dim=16, max_blocks=300, max_seqs=1, n_pages=300)
    try:
        n = 4096
        c.extend([0], [n])
        k, v = np.zeros(c.k.shape), np.zeros(c.k.shape)
        k[0, c.table[0][0], 0, 0, 0] = 20 * np.log(2.0)
        v[0, :, 0, :, 1] = 1.0
        v[0, c.table[0][0], 0, 0, 1] = 0.0
        c.k, c.v = (rounded(a, c.d.type)[1].reshape(c.k.shape) for a in (k, v))
        c.load()
        q = np.zeros((1, 16))
        q[0, 0] = 1.0
        rows, tol = want(c, q, 1, [0], None, 1, 1.0)
        got, _ = run(c, q, 1, [0], None, 1, 0, n, 1.0)
        # half a step of the output, and half a step of each weight
        assert abs(got[0, 0, 1] / rows[0, 0, 1] - 1) <= 2.0 ** -10 + 2.0 ** -11
    finally:
        c.close()


def test_bad_pages_and_slots(g):
    """Indexes that only the device sees: pages out of range count as zeros, slots
    that cannot be are NaN, each with the error bit; other rows are right."""
    rng = np.random.default_rng(11)
    c = Cache(g, type=M.MHIP_BF16, n_layers=1, n_kv_heads=2, head_dim=64, max_blocks=10, max_seqs=4, n_pages=40)
    try:
        fill(c, [100, 90, 80], 0, rng)
        q = rng.standard_normal((3, 4 * 64))
        got, bits = run(c, q, 4, [0, 77, 2], None, 1, 0, 160, 0.125)
        rows, tol = want(c, q, 4, [0, 1, 2], None, 1, 0.125)
        assert bits == M.MHIP_PAGES_BAD and np.isnan(got[1]).all()
        close(got[[0, 2]], rows[[0, 2]], tol[[0, 2]])
        got, bits = run(c, q, 4, [0, 1, 2], None, 1, 0, 90, 0.125)  # slot 0 is longer
        assert bits == M.MHIP_PAGES_BAD and np.isnan(got[0]).all()
        close(got[1:], rows[1:], tol[1:])
        for page in (-1, 40, 2 ** 31 - 1):
            table, _, _ = c.books()
            table[1, 2] = page
            a = np.ascontiguousarray(table)
            g.check(M.lib().mhip_h2d(g.h, c.gpu.arrays.table, a.ctypes.data, a.nbytes), "h2d")
            got, bits = run(c, q, 4, [0, 1, 2], None, 1, 0, 160, 0.125)
            assert bits == M.MHIP_PAGES_BAD
            close(got[[0, 2]], rows[[0, 2]], tol[[0, 2]])
            k, v = c.rows("k", 0, 1, 90), c.rows("v", 0, 1, 90)
            k[32:48] = v[32:48] = 0
            qv = rounded(q, c.d.type)[0].reshape(3, 4, 64)[1]
            o = attention(qv, k, v, 0.125)
            close(got[1], o, attention_tolerance(qv, k, v, o, 0.125, c.d.type))
    finally:
        c.close()


def test_a_prefix_longer_than_its_slot(g):
    rng = np.random.default_rng(14)
    c = Cache(g, n_layers=1, n_kv_heads=1, head_dim=64, max_blocks=10, max_seqs=3, n_pages=40)
    try:
        fill(c, [40, 90], 0, rng)
        q = rng.standard_normal((1, 64))
        got, bits = run(c, q, 1, [1], None, 1, 64, 100, 0.125)
        assert bits == M.MHIP_PAGES_BAD
        got, bits = run(c, q, 1, [1], None, 1, 64, 100, 0.125, prefix_seq=1)
        assert bits == 0
        rows, tol = want(c, q, 1, [1], None, 1, 0.125)
        close(got, rows, tol)
    finally:
        c.close()


@pytest.mark.parametrize("scale", [2.0 ** -64, 2.0 ** -20, 4.0, 2.0 ** 64])
def test_scales(g, scale):
    """From one that makes all tokens equal to one that leaves the largest score
    alone (scores of small whole numbers, exact in fp32)."""
    rng = np.random.default_rng(15)
    c = Cache(g, n_layers=1, n_kv_heads=1, head_dim=16, max_blocks=20, max_seqs=2, n_pages=40)
    try:
        fill(c, [300, 130], 100, rng)
        c.k = rounded(rng.integers(-3, 4, c.k.shape), c.d.type)[1].reshape(c.k.shape)
        c.load()
        q = rng.integers(-2, 3, (2, 32)).astype(float)
        rows, _ = want(c, q, 2, [0, 1], None, 1, scale)
        got, bits = run(c, q, 2, [0, 1], None, 1, 100, 300, scale)
        assert bits == 0
        # weights of 2^-21 each, sums of 300 tokens
        assert np.abs(got - rows).max() <= np.abs(values(c.v, c.d.type)).max() * (2.0 ** -20 + 400 * 2.0 ** -24)
    finally:
        c.close()


@pytest.mark.parametrize("t", [M.MHIP_F32, M.MHIP_BF16])
def test_offsets_beyond_32_bits(g, t):
    """The last pages of a cache of over 2^32 bytes (and elements' bytes past
    2^31): written, forked, moved by compaction to the front, and read."""
    d = M.PageDims(t, 1, 1, 256, 256, 36000 if t else 18000, 4, 3)
    size, page = esize(t), 256 * 256 * esize(t)
    assert d.n_pages * page > 1 << 32
    c, L = M.Pages(g, d), M.lib()
    rng = np.random.default_rng(16)
    dt = np.int32 if t == M.MHIP_F32 else np.int16
    mem = []

    def up(a, dtype=np.int32):
        mem.append(g.upload(np.ascontiguousarray(a, dtype)))
        return mem[-1]
    try:
        # all pages but the last four are some other program's
        refs = np.ones(d.n_pages, np.int32)
        refs[-4:] = 0
        g.check(L.mhip_h2d(g.h, c.arrays.refs, refs.ctypes.data, refs.nbytes), "h2d")
        n = 300
        k, kr = rounded(rng.standard_normal((n, 256)), t)
        v, vr = rounded(rng.standard_normal((n, 256)), t)
        q, qr = rounded(rng.standard_normal((1, 256)) * 2, t)
        c.extend(up([2]), up([n]), 1)
        c.write(0, up([2]), up([n]), 1, n, up(kr, dt), up(vr, dt), 256)
        c.fork(up([2]), up([0]), 1)
        out = up(np.zeros(256), dt)
        ws = up(np.zeros(c.attention_ws_bytes(1, 1, 1, 256, 400)), np.uint8)
        want_row = attention(q.reshape(1, 256), k[:, None], v[:, None], 0.06)
        tol = attention_tolerance(q.reshape(1, 256), k[:, None], v[:, None], want_row, 0.06, t)

        def check(slot, prefix_seq):
            c.attention(0, 1, up(qr.reshape(1, 256), dt), 256, out, 256, up([slot]), None, 1, 1, prefix_seq, 256, 400,
                        0.06, ws)
            got = values(g.download(out, (256,), dt), t).reshape(1, 256)
            assert (np.abs(got - want_row) <= tol).all()
        check(2, 2)
        check(0, 2)
        assert c.status() == (0, 1)
        table = g.download(c.arrays.table, (4, 3), np.int32)
        assert table[2].tolist() == [d.n_pages - 4, d.n_pages - 3, -1]
        assert table[0].tolist() == [d.n_pages - 4, d.n_pages - 2, -1]
        refs = g.download(c.arrays.refs, (d.n_pages,), np.int32)
        refs[:-4] = 0  # the other program is gone
        g.check(L.mhip_h2d(g.h, c.arrays.refs, refs.ctypes.data, refs.nbytes), "h2d")
        c.compact()
        assert g.download(c.arrays.table, (4, 3), np.int32)[[0, 2]].tolist() == [[0, 2, -1], [0, 1, -1]]
        check(2, 0)
        check(0, 2)
        assert c.status() == (0, d.n_pages - 3)
    finally:
        for p in mem:
            g.free(p)
        c.close()


def test_two_contexts_at_once(g):
    """Two contexts (streams), each with a cache of its own and calls queued in
    turn without a wait, give what each gives alone."""
    rng = np.random.default_rng(17)
    other = M.Gpu()
    caches = []
    try:
        for gpu in (g, other):
            c = Cache(gpu, type=M.MHIP_F16, n_layers=1, n_kv_heads=2, head_dim=128, max_blocks=40, max_seqs=6,
                      n_pages=120)
            caches.append(c)
            fill(c, [400 + 30 * i for i in range(6)], 350, rng)
            c.q = rng.standard_normal((6, 8 * 128)) * 2
            c.dq = c.up(rounded(c.q, c.d.type)[1], c.int)
            c.out = c.up(np.zeros((6, 1024)), c.int)
            c.ws = c.up(np.zeros(c.gpu.attention_ws_bytes(8, 6, 1, 350, 600), np.uint8), np.uint8)
            c.seqs = c.up(np.arange(6))
        for _ in range(20):
            for c in caches:
                c.gpu.attention(0, 8, c.dq, 1024, c.out, 1024, c.seqs, None, 6, 1, 0, 350, 600, 0.09, c.ws)
        for c in caches:
            rows, tol = want(c, c.q, 8, range(6), None, 1, 0.09)
            close(values(c.g.download(c.out, (6, 1024), c.int), c.d.type).reshape(6, 8, 128), rows, tol)
    finally:
        for c in caches:
            c.close()
        other.close()


def test_repeats_and_replays_give_the_same_bits(g):
    """Two calls, and replays of a graph that shares its workspace with a second
    one, agree to the bit."""
    rng = np.random.default_rng(12)
    L = M.lib()
    c = Cache(g, type=M.MHIP_BF16, n_layers=1, n_kv_heads=4, head_dim=128, max_blocks=80, max_seqs=12,
              n_pages=300)
    try:
        lens = [1000 + 17 * i for i in range(12)]
        fill(c, lens, 1000, rng)
        need = c.gpu.attention_ws_bytes(32, 12, 1, 1000, 1280)
        ws = c.up(np.zeros(need, np.uint8), np.uint8)
        qs = [c.up(rounded(rng.standard_normal((12, 4096)), c.d.type)[1], c.int) for _ in (0, 1)]
        outs = [c.up(np.zeros((12, 4096)), c.int) for _ in (0, 1)]
        seqs = c.up(np.arange(12))

        def call(x):
            c.gpu.attention(0, 32, qs[x], 4096, outs[x], 4096, seqs, None, 12, 1, 0, 1000, 1280, 0.09, ws)

        def result(x):
            return g.download(outs[x], (12, 4096), c.int)
        call(0), call(1)
        first = result(0), result(1)
        graphs = []
        for x in (0, 1):
            g.check(L.mhip_graph_begin(g.h), "begin")
            call(x)
            p = ctypes.c_void_p()
            g.check(L.mhip_graph_end(g.h, ctypes.byref(p)), "end")
            graphs.append(p)
        for _ in range(3):
            for x in (0, 1):
                g.check(L.mhip_zero(g.h, outs[x], 12 * 4096 * 2), "zero")
                g.check(L.mhip_graph_launch(g.h, graphs[x]), "launch")
            assert np.array_equal(result(0), first[0]) and np.array_equal(result(1), first[1])
            call(1), call(0)
            assert np.array_equal(result(0), first[0]) and np.array_equal(result(1), first[1])
        for p in graphs:
            L.mhip_graph_destroy(p)
    finally:
        c.close()


@pytest.mark.parametrize("t", TYPES)
def test_a_layer_of_a_batch(g, t):
    """The operators as a decode step uses them, captured into one graph and
    replayed: rows of q, k and v by 4-bit products, the new tokens' pages and
    rows, attention behind a shared prompt, the output rows. Each step against
    64 bits on the step's own inputs."""
    rng = np.random.default_rng(13)
    heads, kv, hd, dim, n, prefix, group = 8, 2, 64, 256, 6, 70, 32
    width, kw = heads * hd, kv * hd
    L = M.lib()
    c = Cache(g, type=t, n_layers=1, n_kv_heads=kv, head_dim=hd, max_blocks=8, max_seqs=n, n_pages=60)
    try:
        fill(c, [prefix] * n, prefix, rng)
        weights = {}
        for name, (r, k) in dict(q=(width, dim), k=(kw, dim), v=(kw, dim), o=(dim, width)).items():
            codes = rng.integers(0, 256, (r, k // 2)).astype(np.uint8)
            scales = (0.02 * (0.5 + rng.random((r, k // group)))).astype(np.float16)
            weights[name] = (c.up(codes, np.uint8), c.up(scales, np.float16), r, k,
                             q4_weights(codes, scales, group))
        new = lambda w: c.up(np.zeros((n, w)), c.int)  # noqa: E731
        x, q, k, v, att, y = new(dim), new(width), new(kw), new(kw), new(width), new(dim)
        seqs = rng.permutation(n)
        dseqs, max_len = c.up(seqs), prefix + 20
        ws = c.up(np.zeros(c.gpu.attention_ws_bytes(heads, n, 1, prefix, max_len), np.uint8), np.uint8)
        qws = c.up(np.zeros(max(M.matvec_q4_ws_bytes(t, w, n) for w in (dim, width)), np.uint8), np.uint8)

        def product(name, out, src):
            codes, scales, r, cols, _ = weights[name]
            M.matvec_q4(g, t, out, r, codes, scales, group, src, cols, r, cols, n, qws)
        g.check(L.mhip_graph_begin(g.h), "begin")
        for name, out in (("q", q), ("k", k), ("v", v)):
            product(name, out, x)
        c.gpu.extend(dseqs, None, n)
        c.gpu.write(0, dseqs, None, n, 1, k, v, kw)
        c.gpu.attention(0, heads, q, width, att, width, dseqs, None, n, 1, 0, prefix, max_len, 0.125, ws)
        product("o", y, att)
        graph = ctypes.c_void_p()
        g.check(L.mhip_graph_end(g.h, ctypes.byref(graph)), "end")
        for step in range(18):
            xs, raw = rounded(rng.standard_normal((n, dim)), t)
            g.check(L.mhip_h2d(g.h, x, np.ascontiguousarray(raw).ctypes.data, raw.nbytes), "h2d")
            g.check(L.mhip_graph_launch(g.h, graph), "launch")
            got = {name: g.download(p, (n, w), c.int) for name, p, w in
                   (("q", q, width), ("k", k, kw), ("v", v, kw), ("att", att, width), ("y", y, dim))}
            val = {name: values(a, t) for name, a in got.items()}
            for name, src in (("q", xs), ("k", xs), ("v", xs)):
                w = weights[name][4]
                assert (np.abs(val[name] - src @ w.T) <= q4_tolerance(w, src, src @ w.T, t)).all(), name
            for i, s in enumerate(seqs):
                c.len[s] += 1
                if len(c.table[s]) * 16 < c.len[s]:
                    c.table[s].append(c.take())
                b, r = divmod(c.len[s] - 1, 16)
                c.k[0, c.table[s][b], :, r] = got["k"][i].reshape(kv, hd)
                c.v[0, c.table[s][b], :, r] = got["v"][i].reshape(kv, hd)
            if step in (0, 9, 17):
                c.check()
            rows, tol = want(c, val["q"], heads, seqs, None, 1, 0.125)
            close(val["att"].reshape(n, heads, hd), rows, tol)
            w = weights["o"][4]
            y64 = val["att"] @ w.T
            assert (np.abs(val["y"] - y64) <= q4_tolerance(w, val["att"], y64, t)).all()
        L.mhip_graph_destroy(graph)
    finally:
        c.close()
