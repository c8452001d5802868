"""What the operators of a cache in 4 bits refuse: every argument the host can see is checked
before any device call, so all of it runs without a GPU (and without a context)."""
import ctypes

import pytest

import motoria_amd as M

DIMS = dict(type=M.MHIP_Q4, n_layers=2, n_kv_heads=2, head_dim=64, page=16, n_pages=10, max_seqs=4, max_blocks=5)
BAD_DIMS = [dict(type=3), dict(type=5), dict(head_dim=16), dict(head_dim=80), dict(head_dim=0), dict(head_dim=288),
            dict(n_layers=0), dict(n_kv_heads=257), dict(page=8), dict(n_pages=0), dict(max_seqs=65537), dict(max_blocks=0)]


def cache(**kw):
    d = M.PageDims(**dict(DIMS, **kw))
    return d, M.PageArrays(*[4096 * (i + 1) for i in range(7)])


WRITE = dict(layer=0, type=M.MHIP_F16, seqs=16, count=None, n=2, top=1, k=4096, v=4096, ld=128, weights=None)
READ = {k: v for k, v in WRITE.items() if k != "weights"}
ATTEND = dict(layer=0, type=M.MHIP_F32, heads=4, q=4096, ldq=256, out=4096, ldo=256, seqs=16, count=None, n=2, top=1,
              max_len=80, scale=0.125, weights=None, ws=4096)
EVICT = dict(weights=4096, seqs=16, n=2, keep=20, recent=4, max_len=80, ws=4096)
FORK = dict(weights=4096, src=16, dst=16, n=1, flags=0)


@pytest.mark.parametrize("bad", range(len(BAD_DIMS)))
def test_dimensions(bad):
    L = M.lib()
    d, a = cache(**BAD_DIMS[bad])
    D, A = ctypes.byref(d), ctypes.byref(a)
    assert L.mhip_pages_bytes(D) == 0 and L.mhip_weights_bytes(D) == 0
    assert L.mhip_attention_q4_ws_bytes(D, M.MHIP_F32, 4, 1, 1, 16, 0) == 0
    assert L.mhip_pages_evict_ws_bytes(D, 1, 4, 16) == 0
    assert L.mhip_pages_write_q4(None, D, A, *WRITE.values()) == -1
    assert L.mhip_pages_read_q4(None, D, A, *READ.values()) == -1
    assert L.mhip_attention_q4(None, D, A, *ATTEND.values()) == -1
    assert L.mhip_pages_evict(None, D, A, *EVICT.values()) == -1
    assert L.mhip_pages_fork_weights(None, D, A, *FORK.values()) == -1


@pytest.mark.parametrize("t", [M.MHIP_F32, M.MHIP_F16, M.MHIP_BF16])
def test_other_caches(t):
    """These calls are of caches in 4 bits, and those of other caches refuse them."""
    L = M.lib()
    d, a = cache(type=t)
    D, A = ctypes.byref(d), ctypes.byref(a)
    assert L.mhip_weights_bytes(D) == 0
    assert L.mhip_attention_q4_ws_bytes(D, t, 4, 1, 1, 16, 0) == 0
    assert L.mhip_pages_evict_ws_bytes(D, 1, 4, 16) == 0
    assert L.mhip_pages_write_q4(None, D, A, *WRITE.values()) == -1
    assert L.mhip_pages_read_q4(None, D, A, *READ.values()) == -1
    assert L.mhip_attention_q4(None, D, A, *ATTEND.values()) == -1
    assert L.mhip_pages_evict(None, D, A, *EVICT.values()) == -1
    assert L.mhip_pages_fork_weights(None, D, A, *FORK.values()) == -1
    d, a = cache()
    D, A = ctypes.byref(d), ctypes.byref(a)
    assert L.mhip_pages_write(None, D, A, 0, 16, None, 2, 1, 4096, 4096, 128) == -1
    assert L.mhip_attention_shared_ws_bytes(D, 4, 2, 1, 0, 80) == 0
    assert L.mhip_attention_shared(None, D, A, 0, 4, 4096, 256, 4096, 256, 16, None, 2, 1, 0, 0, 80, 1.0, 4096) == -1


def test_sizes():
    L = M.lib()
    d, _ = cache()
    pool = 2 * 10 * 2 * 16 * 64 * 5 // 8
    assert L.mhip_pages_bytes(ctypes.byref(d)) == 2 * pool + 5 * 256
    assert L.mhip_weights_bytes(ctypes.byref(d)) == 2 * 4 * 2 * 80 * 4
    a = M.PageArrays()
    assert L.mhip_pages_carve(ctypes.byref(d), 1 << 20, ctypes.byref(a)) == 0
    assert a.k == 1 << 20 and a.v == a.k + pool and a.table == a.v + pool
    # sizes that no number of bytes holds
    d, _ = cache(n_layers=65536, n_kv_heads=256, max_seqs=65536, max_blocks=1 << 26)
    assert L.mhip_weights_bytes(ctypes.byref(d)) == 0
    assert L.mhip_pages_evict_ws_bytes(ctypes.byref(d), 65536, 1 << 30, 1 << 30) == 0


def test_rows():
    L = M.lib()
    d, a = cache()
    D, A = ctypes.byref(d), ctypes.byref(a)
    bad = [dict(layer=-1), dict(layer=2), dict(type=-1), dict(type=3), dict(type=M.MHIP_Q4), dict(n=5), dict(n=-1),
           dict(seqs=None), dict(top=-1), dict(ld=127), dict(ld=132), dict(k=None), dict(v=None), dict(k=4100),
           dict(v=4104), dict(top=1 << 23)]
    for b in bad:
        assert L.mhip_pages_write_q4(None, D, A, *dict(WRITE, **b).values()) == -1, b
        assert L.mhip_pages_read_q4(None, D, A, *dict(READ, **b).values()) == -1, b
    assert L.mhip_pages_write_q4(None, D, A, *dict(WRITE, weights=4104).values()) == -1
    for i in range(7):  # a null array
        n = M.PageArrays(*[0 if j == i else 4096 * (j + 1) for j in range(7)])
        assert L.mhip_pages_write_q4(None, D, ctypes.byref(n), *WRITE.values()) == -1
    # nothing to do is no error
    for none in (dict(n=0, seqs=None, k=None, v=None), dict(top=0, k=None, v=None)):
        assert L.mhip_pages_write_q4(None, D, A, *dict(WRITE, **none).values()) == 0
        assert L.mhip_pages_read_q4(None, D, A, *dict(READ, **none).values()) == 0


def test_attention():
    L = M.lib()
    d, a = cache()
    D, A = ctypes.byref(d), ctypes.byref(a)
    bad = [dict(layer=-1), dict(layer=2), dict(type=-1), dict(type=4), dict(heads=3), dict(heads=0), dict(heads=131072),
           dict(q=None), dict(out=None), dict(seqs=None), dict(ws=None), dict(ldq=255), dict(ldo=255), dict(ldq=258),
           dict(ldo=258), dict(q=4100), dict(out=4104), dict(ws=4096 + 16), dict(weights=4104), dict(n=5), dict(n=-1),
           dict(top=-1), dict(top=1 << 24), dict(max_len=-1), dict(max_len=81), dict(scale=0.0), dict(scale=-1.0),
           dict(scale=float("nan")), dict(scale=2.0 ** 65), dict(scale=2.0 ** -65)]
    for b in bad:
        assert L.mhip_attention_q4(None, D, A, *dict(ATTEND, **b).values()) == -1, b
    for args in ((M.MHIP_F32, 3, 2, 1, 80, 0), (M.MHIP_F32, 4, 5, 1, 80, 0), (M.MHIP_F32, 4, 0, 1, 80, 0),
                 (M.MHIP_F32, 4, 2, 0, 80, 0), (M.MHIP_F32, 4, 2, 1, 81, 0), (3, 4, 2, 1, 80, 0),
                 (M.MHIP_F32, 4, 4, 1 << 22, 80, 0)):
        assert L.mhip_attention_q4_ws_bytes(D, *args) == 0, args
    assert L.mhip_attention_q4_ws_bytes(D, M.MHIP_F32, 4, 2, 1, 80, 0) > 0
    assert (L.mhip_attention_q4_ws_bytes(D, M.MHIP_F32, 4, 2, 1, 80, 1) >
            L.mhip_attention_q4_ws_bytes(D, M.MHIP_F32, 4, 2, 1, 80, 0))
    for none in (dict(n=0), dict(top=0)):
        assert L.mhip_attention_q4(None, D, A, *dict(ATTEND, **none).values()) == 0


def test_evict():
    L = M.lib()
    d, a = cache()
    D, A = ctypes.byref(d), ctypes.byref(a)
    bad = [dict(weights=None), dict(weights=4104), dict(seqs=None), dict(ws=None), dict(ws=4096 + 128), dict(n=5),
           dict(n=-1), dict(keep=0), dict(keep=-3), dict(recent=-1), dict(recent=21), dict(max_len=-1), dict(max_len=81)]
    for b in bad:
        assert L.mhip_pages_evict(None, D, A, *dict(EVICT, **b).values()) == -1, b
    for args in ((0, 20, 80), (5, 20, 80), (2, 0, 80), (2, 20, 81), (2, 20, -1)):
        assert L.mhip_pages_evict_ws_bytes(D, *args) == 0, args
    assert L.mhip_pages_evict_ws_bytes(D, 2, 20, 80) > 0
    assert L.mhip_pages_evict_ws_bytes(D, 2, 1 << 30, 80) > 0  # a budget that no slot exceeds
    assert L.mhip_pages_evict(None, D, A, *dict(EVICT, n=0, seqs=None).values()) == 0


def test_fork():
    L = M.lib()
    d, a = cache()
    D, A = ctypes.byref(d), ctypes.byref(a)
    for b in (dict(weights=None), dict(weights=4104), dict(src=None), dict(dst=None), dict(n=5), dict(n=-1), dict(flags=2)):
        assert L.mhip_pages_fork_weights(None, D, A, *dict(FORK, **b).values()) == -1, b
    assert L.mhip_pages_fork_weights(None, D, A, *dict(FORK, n=0).values()) == 0
