"""Rows into and out of a cache in 4 bits, its pages' forks and moves, and eviction by
accumulated weight, against a model that knows every byte."""
import ctypes

import numpy as np
import pytest
import torch

import motoria_amd as M
from q4_model import CacheQ4, codes_of
from shared_model import TORCH, TYPES

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def g():
    gpu = M.Gpu()
    yield gpu
    gpu.close()


SHAPES = [dict(), dict(n_layers=1, n_kv_heads=1, head_dim=32), dict(n_kv_heads=5, head_dim=96, page=32, max_blocks=5),
          dict(n_layers=1, n_kv_heads=4, head_dim=256, page=64, max_blocks=3, n_pages=17),
          dict(n_layers=3, head_dim=128, page=256, max_blocks=2, n_pages=9),
          dict(n_layers=1, n_kv_heads=1, head_dim=224, page=128, max_blocks=2, n_pages=9),
          dict(n_layers=1, n_kv_heads=13, head_dim=160, max_blocks=4)]


def rows(rng, n, width):
    return [rng.standard_normal((n, width)) * np.exp(rng.standard_normal(width)) for _ in (0, 1)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_write_and_read(g, shape, t):
    print("test_write_and_read", SHAPES[shape], t, flush=True)
    c = CacheQ4(g, **SHAPES[shape])
    rng = np.random.default_rng(10 * shape + t)
    d = c.d
    width = d.n_kv_heads * d.head_dim
    try:
        for step, counts in enumerate(([3, 1, 0], [19, 0, 14], None, [1, 4, 7])):
            seqs = rng.permutation(d.max_seqs)[:3].tolist()
            c.extend(seqs, counts)
            top = 1 if counts is None else max(counts) + step % 2
            for layer in range(d.n_layers):
                k, v = rows(rng, 3 * top, width)
                pad = [0, 16][step % 2]
                c.write_q4(layer, t, seqs, counts, k, v, top, pad=pad, weights=step != 1)
            c.check()
            # and back: rows past the counts stay as they were
            n = [1] * 3 if counts is None else counts
            for layer in range(d.n_layers):
                blank = np.full((3 * top, (width + pad) * (4 if t == M.MHIP_F32 else 2)), 0x5a, np.uint8)
                dk, dv = c.up(blank, np.uint8), c.up(blank, np.uint8)
                c.gpu.read_q4(layer, t, c.up(seqs), None if counts is None else c.up(counts), 3, top, dk, dv, width + pad)
                for which, at in ((0, dk), (1, dv)):
                    want = torch.from_numpy(blank.copy()).view(TORCH[t])
                    for i, s in enumerate(seqs):
                        if n[i]:
                            a, b = c.parts(which, layer, s)
                            # s c is exact in fp32, the sum rounds once
                            x = torch.from_numpy((a + b)[-n[i]:].reshape(n[i], -1)).float().to(TORCH[t])
                            want[i * top:i * top + n[i], :width] = x
                    got = g.download(at, blank.shape, np.uint8)
                    assert np.array_equal(got, want.view(torch.uint8).numpy()), (step, layer, which)
    finally:
        c.close()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("count", [4, 5, 6, 7, 8, 9, 17])
def test_tokens_in_fours(g, count, t):
    """Calls that begin and end anywhere in a four of tokens, and what was there beside them."""
    print("test_tokens_in_fours", count, t, flush=True)
    c = CacheQ4(g, n_layers=2, n_kv_heads=2, head_dim=96, page=16, max_seqs=4, max_blocks=4, n_pages=16)
    rng = np.random.default_rng(10 * count + t)
    width = 2 * 96
    try:
        seqs = [2, 0, 3, 1]
        for counts in ([0, 1, 2, 3], [count, 3, count - 1, count], [1] * 4, [2, count, count, 1]):
            c.extend(seqs, counts)
            k, v = rows(rng, 4 * count, width)
            for layer in (0, 1):
                c.write_q4(layer, t, seqs, counts, k, v, count, weights=layer == 0)
            c.check()
            blank = np.zeros((4 * count, width * (4 if t == M.MHIP_F32 else 2)), np.uint8)
            dk, dv = c.up(blank, np.uint8), c.up(blank, np.uint8)
            c.gpu.read_q4(1, t, c.up(seqs), c.up(counts), 4, count, dk, dv, width)
            for which, at in ((0, dk), (1, dv)):
                got = torch.from_numpy(g.download(at, blank.shape, np.uint8)).view(TORCH[t])
                want = torch.zeros((4 * count, width), dtype=TORCH[t])
                for i, s in enumerate(seqs):
                    if counts[i]:
                        a, b = c.parts(which, 1, s)
                        want[i * count:i * count + counts[i]] = torch.from_numpy((a + b)[-counts[i]:].reshape(counts[i], -1)).float().to(TORCH[t])
                assert torch.equal(got, want), (counts, which)
    finally:
        c.close()


def test_borders_between_codes(g):
    """Values on and next to every border, groups of one value, of the least steps and of large ones."""
    c = CacheQ4(g, n_layers=1, n_kv_heads=1, head_dim=128, n_pages=64, max_seqs=2, max_blocks=60)
    rng = np.random.default_rng(7)
    try:
        groups = []
        for lo, s in [(-1.0, 0.125), (0.0, 1.0), (-300.0, 40.0), (1.5, 2.0 ** -14), (0.25, 2.0 ** -24 * 3), (-2.0 ** -20, 2.0 ** -23),
                      (-32768.0, 4369.0), (7.0, 0.333251953125), (-0.1, 0.0123)]:
            m, st = np.float32(np.float16(lo)), np.float32(np.float16(s))
            border = (m.astype(np.float64) + (np.arange(15) + 0.5) * np.float64(st)).astype(np.float32)
            for shift in (0, 1, -1):
                x = np.empty(32, np.float32)
                x[:15] = np.nextafter(border, np.float32(np.inf if shift > 0 else -np.inf)) if shift else border
                x[15], x[16] = m, m + 15 * st
                x[17:] = rng.uniform(m, m + 15 * st, 15)
                groups.append(x)
        groups += [np.full(32, x, np.float32) for x in (0.0, -0.0, 1.0, -77.7, 1e-9, 32768.0, -32768.0, 65504.0, 1e30, -1e30)]
        groups += [np.where(np.arange(32) == 5, x, 0.5).astype(np.float32) for x in (np.nan, np.inf, -np.inf, 3e38, 1e-40)]
        groups += [np.full(32, np.nan, np.float32), np.where(np.arange(32) % 2, np.inf, -np.inf).astype(np.float32)]
        groups += [rng.standard_normal(32).astype(np.float32) * np.float32(10.0 ** e) for e in range(-12, 5)]
        while len(groups) % 4:
            groups.append(np.zeros(32, np.float32))
        x = np.array(groups, np.float32).reshape(-1, 128)
        for t in TYPES:
            r = torch.from_numpy(x).to(TORCH[t]).float().numpy()
            odd = not (np.abs(r) <= 32768).all()
            c.extend([1], [len(x)])
            c.write_q4(0, t, [1], [len(x)], x, x[::-1], len(x))
            c.check(M.MHIP_PAGES_NOT_FINITE if odd else 0)
            c.extend([1], [1])
            c.write_q4(0, t, [1], None, np.full((1, 128), 3.0), np.full((1, 128), -32768.0), 1)
            c.check()
            c.free([1])
    finally:
        c.close()


@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_random_calls_keep_the_model(g, shape):
    print("test_random_calls_keep_the_model", SHAPES[shape], flush=True)
    c = CacheQ4(g, **SHAPES[shape])
    rng = np.random.default_rng(shape)
    d = c.d
    try:
        for step in range(22):
            used = [s for s in range(d.max_seqs) if c.len[s]]
            idle = [s for s in range(d.max_seqs) if not c.len[s]]
            left = sum(r == 0 for r in c.refs)
            what = rng.integers(0, 6)
            if what <= 1 or not used:
                seqs = rng.permutation(d.max_seqs)[:rng.integers(1, 4)].tolist()
                room = max(1, left // len(seqs) - 1) * d.page
                counts = [int(rng.integers(0, max(1, min(room, d.max_blocks * d.page - c.len[s], 40)))) for s in seqs]
                if left < sum(-(-n // d.page) + 1 for n in counts):
                    continue
                c.extend(seqs, counts)
                top = max(max(counts), 1)
                for layer in range(d.n_layers):
                    k, v = rows(rng, len(seqs) * top, d.n_kv_heads * d.head_dim)
                    c.write_q4(layer, TYPES[step % 3], seqs, counts, k, v, top)
            elif what == 2 and idle:
                dst = rng.permutation(idle)[:rng.integers(1, len(idle) + 1)].tolist()
                src = [int(rng.choice(used)) for _ in dst]
                deep = bool(rng.integers(0, 2))
                need = sum(len(c.table[a]) if deep else c.len[a] % d.page != 0 for a in src)
                if need <= left:
                    c.fork_weights(src, dst, deep) if step % 2 else c.fork(src, dst, deep)
            elif what == 3:
                c.free(rng.permutation(used)[:rng.integers(1, len(used) + 1)].tolist())
            elif what == 4:
                seqs = rng.permutation(used)[:rng.integers(1, len(used) + 1)].tolist()
                keep = int(rng.integers(1, max(c.len[s] for s in seqs) + 2))
                nb = -(-keep // d.page)
                need = sum(sum(c.refs[p] > 1 for p in c.table[s][:nb]) for s in seqs if c.len[s] > keep)
                if need <= left:
                    c.evict(seqs, keep, int(rng.integers(0, keep + 1)))
            else:
                c.compact()
            c.check()
    finally:
        c.close()


@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (2, 0), (33, 7), (64, 64), (100, 0), (130, 31), (255, 254), (256, 1), (299, 0)])
def test_evict_lengths(g, keep, recent):
    """Long slots to every kind of length, weights with many ties, another slot left alone."""
    c = CacheQ4(g, n_layers=2, n_kv_heads=2, head_dim=64, page=32, n_pages=60, max_blocks=10, max_seqs=5)
    rng = np.random.default_rng(keep)
    try:
        c.fill([0, 1, 2, 3], [300, 257, 300, 40], rng)
        w = rng.integers(0, 5, c.w.shape).astype(np.float32) * np.float32(0.5)
        w[:, 1] = 1.0                                  # all the same
        w[0, 2] = rng.standard_normal(w[0, 2].shape)   # (no attention gives these, but a program may)
        w[1, 2, 0, ::3] = np.nan
        w[1, 2, 1] = np.where(rng.random(c.T) < 0.5, -0.0, 0.0)
        c.set_weights(w)
        c.evict([2, 0, 1], keep, recent)
        c.check()
        c.evict([2, 0, 3, 1], keep, recent)            # (what is short enough stays as it is)
        c.check()
        c.compact()
        c.check()
    finally:
        c.close()


def test_evict_many_tokens(g):
    """More tokens than threads, weights of all sizes, denormals among them."""
    c = CacheQ4(g, n_layers=1, n_kv_heads=2, head_dim=32, page=64, n_pages=200, max_blocks=90, max_seqs=3)
    rng = np.random.default_rng(5)
    try:
        c.fill([2, 0], [5003, 2777], rng)
        w = np.exp(20 * rng.standard_normal(c.w.shape)).astype(np.float32)
        w[0, 0, 1] = rng.integers(1, 5000, c.T).astype(np.uint32).view(np.float32)
        c.set_weights(w)
        c.evict([0, 2], 2500, 300)
        c.check()
        c.evict([0, 2], 1023, 0)
        c.check()
    finally:
        c.close()


def test_evict_forks_of_many_pages(g):
    """More entries than wavefronts keep books, more pages of each than lanes, most of them shared: with each other,
    with a slot that is not in the list, or with none."""
    c = CacheQ4(g, n_layers=1, n_kv_heads=1, head_dim=32, page=16, n_pages=1300, max_blocks=100, max_seqs=14)
    rng = np.random.default_rng(6)
    try:
        c.fill([3, 9, 0, 5], [1490, 1300, 40, 1184], rng)
        c.fork_weights([3, 3, 3, 3, 9, 9, 5, 5, 0], [1, 2, 4, 6, 7, 8, 10, 11, 12])
        c.set_weights(rng.random(c.w.shape).astype(np.float32))
        c.check()
        c.evict([4, 1, 7, 9, 12, 10, 2, 6, 8, 0, 11, 5], 1100, 100)   # (slot 3 keeps its pages)
        c.check()
    finally:
        c.close()


def test_evict_refuses_whole_calls(g):
    """A slot twice, out of range or too long, and too few pages: nothing changes but the error bits."""
    c = CacheQ4(g, n_layers=1, n_kv_heads=1, head_dim=32, page=16, n_pages=12, max_blocks=8, max_seqs=4)
    rng = np.random.default_rng(6)
    try:
        c.fill([0], [120], rng)                        # 8 pages
        c.fork_weights([0], [1])                       # shares 7
        for seqs, most in (([0, 0], 120), ([0, 4], 120), ([-1], 120), ([0], 119), ([1, 0, 1], 128)):
            c.evict(seqs, 50, 5, most, model=False)
            c.check(M.MHIP_PAGES_BAD)
        c.evict([0, 1], 60, 5, model=False)            # 8 shared pages have to be replaced, 3 are free
        c.check(M.MHIP_PAGES_NO_SPACE)
        c.evict([1], 40, 5)                            # 3
        c.check()
        c.evict([0], 40, 5)                            # now its own: none
        c.check()
    finally:
        c.close()


def test_evict_refuses_a_page_out_of_range(g):
    c = CacheQ4(g, n_layers=1, n_kv_heads=1, head_dim=32, max_seqs=3)
    rng = np.random.default_rng(8)
    try:
        c.fill([0, 1], [70, 70], rng)
        table = c.books()[0]
        bad = table.copy()
        bad[1, 3] = c.d.n_pages
        g.check(M.lib().mhip_h2d(g.h, c.gpu.arrays.table, bad.ctypes.data, bad.nbytes), "h2d")
        c.evict([0, 1], 20, 5, model=False)
        assert c.gpu.status()[0] == M.MHIP_PAGES_BAD
        g.check(M.lib().mhip_h2d(g.h, c.gpu.arrays.table, table.ctypes.data, table.nbytes), "h2d")
        c.check()
    finally:
        c.close()


def test_write_and_read_refuse_on_the_device(g):
    """Slots out of range or too short for the call: an error bit, the other rows are done."""
    c = CacheQ4(g, n_layers=1)
    rng = np.random.default_rng(9)
    d = c.d
    width = d.n_kv_heads * d.head_dim
    try:
        c.fill([0, 3], [20, 5], rng)
        k, v = rows(rng, 4, width)
        rk, rv = (c.rows_of(a, 0, M.MHIP_F32)[0] for a in (k, v))
        c.gpu.write_q4(0, M.MHIP_F32, c.up([0, 8, -1, 3]), c.up([1, 1, 1, 1]), 4, 1, c.up(rk, np.uint8),
                       c.up(rv, np.uint8), width, c.d_w)
        for i, s in ((0, 0), (3, 3)):
            b, r = divmod(c.len[s] - 1, d.page)
            for which, a in ((0, k), (1, v)):
                for h in range(d.n_kv_heads):
                    c.put(which, 0, c.table[s][b], h, r, a[i].astype(np.float32).reshape(d.n_kv_heads, -1)[h])
            c.w[0, s, :, c.len[s] - 1] = 0
        c.check(M.MHIP_PAGES_BAD)
        dk = c.up(np.zeros((6, width)), np.float32)
        dv = c.up(np.zeros((6, width)), np.float32)
        c.gpu.read_q4(0, M.MHIP_F32, c.up([3]), c.up([6]), 1, 6, dk, dv, width)  # one token more than there is
        c.check(M.MHIP_PAGES_BAD)
        got = g.download(dk, (6, width), np.float32)
        assert (got[0] == 0).all()
        a, b = c.parts(0, 0, 3)
        assert np.array_equal(got[1:], (a + b).reshape(5, width).astype(np.float32))
    finally:
        c.close()


def test_fork_without_space_leaves_the_weights(g):
    c = CacheQ4(g, n_layers=1, n_kv_heads=1, head_dim=32, n_pages=4, max_seqs=4)
    rng = np.random.default_rng(2)
    try:
        c.fill([0], [50], rng)  # all four pages
        c.fork_weights([0], [2], model=False)
        c.check(M.MHIP_PAGES_NO_SPACE)
        c.fork_weights([0], [0], model=False)
        c.check(M.MHIP_PAGES_BAD)
    finally:
        c.close()


def test_graph_of_store_and_evict(g):
    """A captured step (a token, its rows, an eviction), replayed with eager calls in between."""
    c = CacheQ4(g, n_layers=2, n_kv_heads=2, head_dim=64, n_pages=60, max_blocks=8)
    rng = np.random.default_rng(4)
    d = c.d
    width = d.n_kv_heads * d.head_dim
    L = M.lib()
    try:
        c.fill([0, 1, 2], [60, 33, 61], rng)
        c.fork_weights([2], [5])
        seqs = [5, 0, 2]
        k, v = rows(rng, 3, width)
        (rk, xk), (rv, xv) = (c.rows_of(a, 0, M.MHIP_BF16) for a in (k, v))
        ds, dk, dv = c.up(seqs), c.up(rk, np.uint8), c.up(rv, np.uint8)
        ws = c.up(np.zeros(c.gpu.evict_ws_bytes(3, 60, d.max_blocks * d.page)), np.uint8)
        g.check(L.mhip_sync(g.h), "sync")
        g.check(L.mhip_graph_begin(g.h), "begin")
        c.gpu.extend(ds, None, 3)
        for layer in range(2):
            c.gpu.write_q4(layer, M.MHIP_BF16, ds, None, 3, 1, dk, dv, width, c.d_w)
        c.gpu.evict(c.d_w, ds, 3, 60, 8, d.max_blocks * d.page, ws)
        graph = ctypes.c_void_p()
        g.check(L.mhip_graph_end(g.h, ctypes.byref(graph)), "end")
        eager = c.gpu
        quiet = type("Quiet", (), {"__getattr__": lambda self, name: (lambda *a: None)})()
        for replay in range(4):
            g.check(L.mhip_graph_launch(g.h, graph), "launch")
            quiet.arrays = eager.arrays
            c.gpu = quiet           # the model alone follows the graph
            quiet.evict_ws_bytes = eager.evict_ws_bytes
            c.extend(seqs, None)
            for layer in range(2):
                c.write_q4(layer, M.MHIP_BF16, seqs, None, k, v, 1)
            c.evict(seqs, 60, 8)
            c.gpu = eager
            c.check()
            c.extend([1], None)     # the program's own calls in between
            for layer in range(2):
                a, b = rows(rng, 1, width)
                c.write_q4(layer, M.MHIP_F32, [1], None, a, b, 1)
            c.evict([1], 34, 2)
            c.check()
        L.mhip_graph_destroy(graph)
    finally:
        c.close()


def test_pages_behind_32_bits(g):
    """A pool of more than 2^32 bytes: rows, copies and moves at its end."""
    d = M.PageDims(M.MHIP_Q4, 1, 8, 256, 128, 4 * 1024, 3, 4)  # 160 KiB a page and head: 5 GiB an array
    block = 128 * 256 * 5 // 8
    assert d.n_pages * d.n_kv_heads * block > 1 << 29
    d.n_layers = 9
    assert d.n_layers * d.n_pages * d.n_kv_heads * block > 1 << 32
    p = M.Pages(g, d)
    L = M.lib()
    rng = np.random.default_rng(0)
    held = []

    def up(a, t=np.int32):
        held.append(g.upload(np.ascontiguousarray(a, t)))
        return held[-1]
    try:
        table = np.full((3, 4), -1, np.int32)
        table[1, :2] = [d.n_pages - 1, d.n_pages - 2]
        refs = np.zeros(d.n_pages, np.int32)
        refs[:] = 1                                   # only one page is free, the third from the end
        refs[d.n_pages - 3] = 0
        lens = np.array([0, 200, 0], np.int32)
        for at, a in ((p.arrays.table, table), (p.arrays.refs, refs), (p.arrays.len, lens)):
            g.check(L.mhip_h2d(g.h, at, a.ctypes.data, a.nbytes), "h2d")
        width = 8 * 256
        x = rng.standard_normal((200, width)).astype(np.float32)
        w = up(rng.random(p.weights_bytes() // 4, dtype=np.float32), np.float32)
        out = up(np.zeros((200, width)), np.float32), up(np.zeros((200, width)), np.float32)

        def read(slot, n):
            p.read_q4(8, M.MHIP_F32, up([slot]), up([n]), 1, n, out[0], out[1], width)
            return [g.download(o, (200, width), np.float32)[:n] for o in out]
        p.write_q4(8, M.MHIP_F32, up([1]), up([200]), 1, 200, up(x, np.float32), up(-x, np.float32), width, w)
        k, v = read(1, 200)
        for got, want in ((k, x), (v, -x)):
            c, s, m = codes_of(want.reshape(200, -1, 32))
            assert np.array_equal(got.reshape(200, -1, 32), s.astype(np.float32)[..., None] * c.astype(np.float32) + m.astype(np.float32)[..., None])
        p.fork_weights(w, up([1]), up([2]), 1)        # its partial page goes to the free one
        assert p.status() == (0, 0)
        a, b = read(2, 200)
        assert np.array_equal(a, k) and np.array_equal(b, v)
        refs = g.download(p.arrays.refs, refs.shape, np.int32)
        refs[5] = 0                                   # a page for what slot 2 shares
        g.check(L.mhip_h2d(g.h, p.arrays.refs, refs.ctypes.data, refs.nbytes), "h2d")
        state = np.zeros(16, np.int32)
        g.check(L.mhip_h2d(g.h, p.arrays.state, state.ctypes.data, 64), "h2d")
        ws = up(np.zeros(p.evict_ws_bytes(1, 150, 200)), np.uint8)
        p.evict(w, up([2]), 1, 150, 150, 200, ws)     # the last 150
        assert p.status() == (0, 0)
        a, b = read(2, 150)
        assert np.array_equal(a, k[50:]) and np.array_equal(b, v[50:])
        a, b = read(1, 200)
        assert np.array_equal(a, k) and np.array_equal(b, v)
    finally:
        for h in held:
            g.free(h)
        p.close()


def test_calls_of_more_entries_than_a_workgroup(g):
    """Forks with weights and evictions of more slots than the deciding workgroup keeps in LDS (256) and than it
    has threads (512): short slots, most of which share their first page."""
    c = CacheQ4(g, n_layers=1, n_kv_heads=1, head_dim=32, page=16, n_pages=2000, max_seqs=640, max_blocks=3)
    rng = np.random.default_rng(12)
    try:
        c.fill(list(range(40)), [17 + i % 20 for i in range(40)], rng)
        c.set_weights(rng.integers(0, 9, c.w.shape).astype(np.float32) / 8)
        dst = rng.permutation(np.arange(40, 640)).tolist()
        c.fork_weights([i % 40 for i in range(300)], dst[:300])
        c.check()
        c.fork_weights([(7 * i) % 40 for i in range(300)], dst[300:])
        c.check()
        c.evict(rng.permutation(640)[:300].tolist(), 20, 5)
        c.check()
        c.evict(rng.permutation(640).tolist(), 9, 3)  # every slot, in one page each
        c.check()
        c.evict(rng.permutation(640).tolist() , 9, 3)  # none is longer
        c.check()
        c.evict(dst[:299] + [dst[0]], 4, 0, max_len=48, model=False)  # a slot twice, the last of many
        c.check(M.MHIP_PAGES_BAD)
    finally:
        c.close()
