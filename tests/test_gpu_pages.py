"""The paged cache (mhip_pages_*) against a model that keeps its pages as
Python lists: table, lengths, counts and every byte of the cache after each
call, calls that must change nothing, and replays of a captured graph."""
import ctypes

import numpy as np
import pytest

import motoria_amd as M
from shared_model import TYPES, Cache, rounded

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def g():
    gpu = M.Gpu()
    yield gpu
    gpu.close()


def new_rows(c, rng, n, top):
    shape = (n, top, c.d.n_kv_heads * c.d.head_dim)
    return [rounded(rng.standard_normal(shape), c.d.type)[1].reshape(shape) for _ in (0, 1)]


SHAPES = [dict(), dict(type=M.MHIP_BF16, n_layers=1, n_kv_heads=1, head_dim=16),
          dict(type=M.MHIP_F16, n_layers=3, n_kv_heads=5, head_dim=80, page=32, max_blocks=5),
          dict(n_layers=1, n_kv_heads=4, head_dim=256, page=64, max_blocks=3, n_pages=17),
          dict(type=M.MHIP_BF16, head_dim=128, page=256, max_blocks=2, n_pages=9),
          dict(n_layers=1, n_kv_heads=1, head_dim=16, n_pages=20000, max_blocks=1000)]


@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_random_calls_keep_the_model(g, shape):
    print("test_random_calls_keep_the_model", SHAPES[shape], flush=True)
    c = Cache(g, **SHAPES[shape])
    rng = np.random.default_rng(shape)
    try:
        for step in range(24):
            used = [s for s in range(c.d.max_seqs) if c.len[s]]
            idle = [s for s in range(c.d.max_seqs) if not c.len[s]]
            left = sum(r == 0 for r in c.refs)
            what = rng.integers(0, 5)
            if what <= 1 or not used:
                seqs = rng.permutation(c.d.max_seqs)[:rng.integers(1, 5)].tolist()
                room = max(1, left // len(seqs) - 1) * c.d.page
                counts = [int(rng.integers(0, max(1, min(room, c.d.max_blocks * c.d.page - c.len[s],
                                                         3 * c.d.page))) ) for s in seqs]
                if left < sum(-(-n // c.d.page) + 1 for n in counts):
                    continue
                c.extend(seqs, counts)
                top = max(max(counts), 1)
                for layer in range(c.d.n_layers):
                    k, v = new_rows(c, rng, len(seqs), top)
                    c.write(layer, seqs, counts, k, v, top, pad=[0, 16][step % 2])
            elif what == 2 and idle:
                dst = rng.permutation(idle)[:rng.integers(1, len(idle) + 1)].tolist()
                src = [int(rng.choice(used)) for _ in dst]
                deep = bool(rng.integers(0, 2))
                need = sum(len(c.table[a]) if deep else c.len[a] % c.d.page != 0 for a in src)
                if need <= left:
                    c.fork(src, dst, deep)
            elif what == 3:
                c.free(rng.permutation(used)[:rng.integers(1, len(used) + 1)].tolist())
            else:
                c.compact()
            c.check()
    finally:
        c.close()


def test_one_token_each_and_page_borders(g):
    c = Cache(g, n_layers=1)
    rng = np.random.default_rng(3)
    try:
        c.extend([5, 2], [15, 16])
        for _ in range(3):  # 15 -> 18 and 16 -> 19 tokens: over a page's end
            c.extend([2, 5], None)
            k, v = new_rows(c, rng, 2, 1)
            c.write(0, [2, 5], None, k, v, 1)
            c.check()
        c.fork([2, 2, 5], [0, 1, 7])
        c.extend([0, 1, 2, 7], [1, 13, 14, 1])  # the copies grow apart
        k, v = new_rows(c, rng, 4, 14)
        c.write(0, [0, 1, 2, 7], [1, 13, 14, 1], k, v, 14)
        c.check()
        c.fork([4], [3])  # an empty slot's copy is empty
        c.check()
    finally:
        c.close()


def test_a_call_that_cannot_be_done_changes_nothing(g):
    c = Cache(g, n_pages=6, max_seqs=4, max_blocks=4)
    try:
        c.extend([0, 1], [40, 20])  # 3 + 2 pages of 6
        c.check()
        c.extend([0, 1], [16, 20], model=False)           # 1 + 1 pages, one is left
        c.check(M.MHIP_PAGES_NO_SPACE)
        c.extend([1], [45], model=False)                  # more than max_blocks
        c.check(M.MHIP_PAGES_NO_SPACE)
        c.extend([2], [2 ** 31 - 1], model=False)
        c.check(M.MHIP_PAGES_NO_SPACE)
        for seqs, counts in (([2, 2], [1, 1]), ([-1], [1]), ([4], [1]), ([2, 3], [1, -1])):
            c.extend(seqs, counts, model=False)
            c.check(M.MHIP_PAGES_BAD)
        c.fork([0, 1], [2, 3], model=False)               # two partial pages, one is left
        c.check(M.MHIP_PAGES_NO_SPACE)
        c.fork([0], [2], deep=True, model=False)
        c.check(M.MHIP_PAGES_NO_SPACE)
        for src, dst in (([0], [1]), ([0, 0], [2, 2]), ([0], [4]), ([-1], [2]), ([2], [2]),
                         ([0, 2], [2, 3])):
            c.fork(src, dst, model=False)
            c.check(M.MHIP_PAGES_BAD)
        c.gpu.free(c.up([9, -3]), 2)                       # the others of the list are done
        c.check(M.MHIP_PAGES_BAD)
        c.free([3])                                        # empty: no error
        c.gpu.free(c.up([1, 1, 0, 1]), 4)                  # twice: once
        c.table[0] = c.table[1] = []
        c.len[0] = c.len[1] = 0
        c.refs = [0] * 6
        c.check()
    finally:
        c.close()


def test_write_leaves_other_rows_alone(g):
    """Entries out of range or longer than their slot are skipped, with a bit."""
    c = Cache(g, n_layers=1)
    rng = np.random.default_rng(4)
    try:
        c.extend([1], [3])
        k, v = new_rows(c, rng, 3, 4)
        flat = [c.up(a.reshape(12, -1), c.int) for a in (k, v)]
        w = c.d.n_kv_heads * c.d.head_dim
        c.gpu.write(0, c.up([99, 1, 2]), c.up([4, 4, 1]), 3, 4, *flat, w)
        # slot 1 has 3 tokens: of its 4 rows the first has no place
        for j in range(1, 4):
            for mine, new in ((c.k, k), (c.v, v)):
                mine[0, c.table[1][0], :, j - 1] = new[1, j].reshape(c.d.n_kv_heads, -1)
        c.check(M.MHIP_PAGES_BAD)
    finally:
        c.close()


def test_captured_calls_replay(g):
    """A step's extend and write, a fork and a free as one graph, replayed with
    eager calls between: every replay does what eager calls do."""
    c = Cache(g, type=M.MHIP_BF16, n_layers=2, n_pages=64, max_blocks=8)
    rng = np.random.default_rng(5)
    L = M.lib()
    try:
        c.extend([0, 3], [21, 32])
        k, v = new_rows(c, rng, 2, 1)
        seqs, src, dst = c.up([3, 0]), c.up([0, 3]), c.up([6, 7])
        dk, dv = (c.up(a.reshape(2, -1), c.int) for a in (k, v))
        w = c.d.n_kv_heads * c.d.head_dim
        g.check(L.mhip_graph_begin(g.h), "begin")
        c.gpu.extend(seqs, None, 2)
        for layer in (0, 1):
            c.gpu.write(layer, seqs, None, 2, 1, dk, dv, w)
        c.gpu.fork(src, dst, 2)
        c.gpu.free(dst, 2)
        graph = ctypes.c_void_p()
        g.check(L.mhip_graph_end(g.h, ctypes.byref(graph)), "end")
        for _ in range(4):
            g.check(L.mhip_graph_launch(g.h, graph), "launch")
            c.len[3] += 1
            c.len[0] += 1
            for s in (3, 0):
                if len(c.table[s]) * c.d.page < c.len[s]:
                    c.table[s].append(c.take())
            for i, s in enumerate((3, 0)):
                b, r = divmod(c.len[s] - 1, c.d.page)
                for mine, new in ((c.k, k), (c.v, v)):
                    mine[:, c.table[s][b], :, r] = new[i, 0].reshape(c.d.n_kv_heads, -1)
            free = [p for p in range(c.d.n_pages) if c.refs[p] == 0]
            for s in (0, 3):  # the forked pages keep their bytes when free again
                if c.len[s] % c.d.page:
                    c.copy_rows(c.table[s][-1], free.pop(0), c.len[s] % c.d.page)
            c.check()
            c.extend([1], [5])  # eager work between the replays
            c.check()
        L.mhip_graph_destroy(graph)
    finally:
        c.close()


def test_more_slots_than_one_pass(g):
    """A list longer than the deciding workgroup: 3000 slots of one token, forked
    and freed together."""
    c = Cache(g, n_layers=1, n_kv_heads=1, head_dim=16, n_pages=7000, max_seqs=6000, max_blocks=2)
    try:
        first = list(range(3000))
        c.extend(first, None)
        c.fork(first, [s + 3000 for s in reversed(first)])
        c.check()
        c.free(list(range(0, 6000, 2)))
        c.compact()
        c.check()
    finally:
        c.close()
