"""What the operators for a batch refuse: every argument the host can see is
checked before any device call, so all of it runs without a GPU (and without a
context)."""
import ctypes

import pytest

import motoria_amd as M

DIMS = dict(type=M.MHIP_F16, n_layers=2, n_kv_heads=2, head_dim=64, page=16, n_pages=10, max_seqs=4, max_blocks=5)
BAD_DIMS = [dict(type=3), dict(type=-1), dict(n_layers=0), dict(n_layers=65537), dict(n_kv_heads=0),
            dict(n_kv_heads=257), dict(head_dim=0), dict(head_dim=24), dict(head_dim=272), dict(page=8),
            dict(page=48), dict(page=512), dict(page=0), dict(n_pages=0), dict(n_pages=(1 << 20) + 1),
            dict(max_seqs=0), dict(max_seqs=65537), dict(max_blocks=0), dict(max_blocks=(1 << 26) + 1)]


def cache(**kw):
    d = M.PageDims(**dict(DIMS, **kw))
    a = M.PageArrays(*[4096 * (i + 1) for i in range(7)])
    return d, a


@pytest.mark.parametrize("bad", range(len(BAD_DIMS)))
def test_dimensions(bad):
    L = M.lib()
    d, a = cache(**BAD_DIMS[bad])
    D, A = ctypes.byref(d), ctypes.byref(a)
    assert L.mhip_pages_bytes(D) == 0 and L.mhip_pages_plan_bytes(D) == 0
    assert L.mhip_attention_shared_ws_bytes(D, 4, 1, 1, 0, 16) == 0
    assert L.mhip_pages_carve(D, 4096, A) == -1
    for rc in (L.mhip_pages_clear(None, D, A), L.mhip_pages_extend(None, D, A, 16, None, 1),
               L.mhip_pages_write(None, D, A, 0, 16, None, 1, 1, 4096, 4096, 4096),
               L.mhip_pages_fork(None, D, A, 16, 16, 1, 0), L.mhip_pages_free(None, D, A, 16, 1),
               L.mhip_pages_compact(None, D, A), L.mhip_pages_status(None, D, A, (ctypes.c_int * 2)()),
               L.mhip_attention_shared(None, D, A, 0, 4, 4096, 256, 4096, 256, 16, None, 1, 1, 0, 0, 16, 1.0, 4096)):
        assert rc == -1


def test_sizes():
    L = M.lib()
    d, _ = cache()
    pool = 2 * 10 * 2 * 16 * 64 * 2
    assert L.mhip_pages_plan_bytes(ctypes.byref(d)) == (16 + 40 + 4) * 4
    assert L.mhip_pages_bytes(ctypes.byref(d)) == 2 * pool + 5 * 256
    a = M.PageArrays()
    assert L.mhip_pages_carve(ctypes.byref(d), 1 << 20, ctypes.byref(a)) == 0
    assert a.k == 1 << 20 and a.v == a.k + pool and a.table == a.v + pool
    assert L.mhip_pages_carve(ctypes.byref(d), (1 << 20) + 16, ctypes.byref(a)) == -1
    assert L.mhip_pages_carve(ctypes.byref(d), None, ctypes.byref(a)) == -1


def test_pages():
    L = M.lib()
    d, a = cache()
    D, A = ctypes.byref(d), ctypes.byref(a)
    for i in range(7):  # a null array
        b = M.PageArrays(*[0 if j == i else 4096 * (j + 1) for j in range(7)])
        assert L.mhip_pages_extend(None, D, ctypes.byref(b), 16, None, 1) == -1
    b = M.PageArrays(4104, *[4096 * (j + 2) for j in range(6)])
    assert L.mhip_pages_clear(None, D, ctypes.byref(b)) == -1  # not on 16 bytes
    for args in ((16, None, 5), (None, None, 1), (16, None, -1)):
        assert L.mhip_pages_extend(None, D, A, *args) == -1
    good = dict(layer=0, seqs=16, count=None, n=2, top=1, k=4096, v=4096, ld=128)
    for bad in (dict(layer=-1), dict(layer=2), dict(n=5), dict(n=-1), dict(seqs=None), dict(top=-1), dict(ld=127),
                dict(ld=132), dict(k=None), dict(v=None), dict(k=4100), dict(v=4104)):
        assert L.mhip_pages_write(None, D, A, *dict(good, **bad).values()) == -1, bad
    for args in ((None, 16, 1, 0), (16, None, 1, 0), (16, 16, 5, 0), (16, 16, -1, 0), (16, 16, 1, 2)):
        assert L.mhip_pages_fork(None, D, A, *args) == -1
    for args in ((None, 1), (16, -1)):
        assert L.mhip_pages_free(None, D, A, *args) == -1
    assert L.mhip_pages_status(None, D, A, None) == -1
    # nothing to do is no error
    assert L.mhip_pages_extend(None, D, A, None, None, 0) == 0
    assert L.mhip_pages_write(None, D, A, 0, None, None, 0, 1, None, None, 128) == 0
    assert L.mhip_pages_fork(None, D, A, None, None, 0, 0) == 0
    assert L.mhip_pages_free(None, D, A, None, 0) == 0


def test_attention():
    L = M.lib()
    d, a = cache()
    D, A = ctypes.byref(d), ctypes.byref(a)
    good = dict(layer=0, heads=4, q=4096, ldq=256, out=4096, ldo=256, seqs=16, count=None, n=2, top=1,
                prefix_seq=0, prefix=16, max_len=64, scale=0.1, ws=4096)
    for bad in (dict(layer=-1), dict(layer=2), dict(heads=0), dict(heads=3), dict(q=None), dict(q=4104),
                dict(ldq=255), dict(ldq=260), dict(out=None), dict(out=4098), dict(ldo=240), dict(seqs=None),
                dict(n=-1), dict(n=5), dict(top=-2), dict(prefix=-1), dict(prefix=65), dict(prefix_seq=-1),
                dict(prefix_seq=4), dict(max_len=81), dict(max_len=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=1e-30), dict(scale=1e30),
                dict(scale=float("nan")), dict(scale=float("inf")), dict(ws=None), dict(ws=4096 + 128)):
        assert L.mhip_attention_shared(None, D, A, *dict(good, **bad).values()) == -1, bad
    for none in (dict(n=0), dict(top=0)):
        assert L.mhip_attention_shared(None, D, A, *dict(good, **none).values()) == 0
    size = lambda **kw: L.mhip_attention_shared_ws_bytes(  # noqa: E731
        D, *dict(dict(heads=4, n=2, top=1, prefix=16, max_len=64), **kw).values())
    assert size() > 0
    for bad in (dict(heads=3), dict(n=0), dict(n=5), dict(top=0), dict(prefix=-1), dict(prefix=70), dict(max_len=81)):
        assert size(**bad) == 0


def test_rows():
    L = M.lib()
    good = dict(type=0, out=4096, ldo=64, codes=4096, scales=4096, group=32, x=4096, ldx=128, rows=64, cols=128, n=3,
                ws=4096)
    for bad in (dict(type=3), dict(type=-1), dict(out=None), dict(ldo=63), dict(codes=None), dict(codes=4104),
                dict(scales=None), dict(scales=4097), dict(group=16), dict(group=0), dict(group=256), dict(x=None),
                dict(rows=(1 << 30) + 1, ldo=(1 << 30) + 1), dict(cols=(1 << 24) + 32, ldx=(1 << 24) + 32),
                dict(x=4100), dict(ldx=127), dict(ldx=130), dict(rows=-1), dict(cols=-32), dict(cols=100),
                dict(cols=0), dict(n=-1), dict(ws=None), dict(ws=4112), dict(out=4098)):
        assert L.mhip_matvec_q4(None, *dict(good, **bad).values()) == -1, bad
    for none in (dict(n=0), dict(rows=0)):
        assert L.mhip_matvec_q4(None, *dict(good, **none).values()) == 0
    for args in ((3, 64, 1), (0, 0, 1), (0, 33, 1), (0, 64, 0)):
        assert L.mhip_matvec_q4_ws_bytes(*args) == 0
    assert L.mhip_quantize_q4(None, 16, 4, 100, 32, 16, 16) == -1
    assert L.mhip_quantize_q4(None, None, 4, 128, 32, 16, 16) == -1
    assert L.mhip_dequantize_q4(None, 16, 16, 4, 128, 31, 16) == -1
    assert L.mhip_dequantize_q4(None, 16, 16, 4, 128, 32, None) == -1


def test_launches_have_less_than_2_32_threads():
    L = M.lib()
    d, a = cache(max_blocks=1 << 22)
    D, A = ctypes.byref(d), ctypes.byref(a)
    assert L.mhip_pages_write(None, D, A, 0, 16, None, 4, 1 << 22, 4096, 4096, 128) == -1
    assert L.mhip_pages_free(None, D, A, 16, 1 << 24) == -1
    size = lambda top, heads, prefix, longest: L.mhip_attention_shared_ws_bytes(  # noqa: E731
        D, heads, 2, top, prefix, longest)
    call = lambda top, heads, prefix, longest: L.mhip_attention_shared(  # noqa: E731
        None, D, A, 0, heads, 4096, heads * 64, 4096, heads * 64, 16, None, 2, top, 0, prefix, longest, 0.1, 4096)
    assert size((1 << 23) - 1, 4, 0, 1 << 12) > 0
    for args in ((1 << 23, 4, 0, 1 << 12), ((1 << 23) - 1, 4, 0, 1 << 26), ((1 << 23) - 1, 4, 1 << 26, 1 << 26)):
        assert size(*args) == 0 and call(*args) == -1, args
    rows = (1 << 28) + 1
    assert L.mhip_matvec_q4(None, 0, 4096, rows, 4096, 4096, 32, 4096, 32, rows, 32, 1, 4096) == -1
    rows = (1 << 28) - 1  # 2^36 weights
    assert L.mhip_matvec_q4(None, 0, 4096, rows, 4096, 4096, 32, 4096, 256, rows, 256, 1, 4096) == -1
    assert L.mhip_dequantize_q4(None, 16, 16, rows, 256, 32, 16) == -1
    assert L.mhip_quantize_q4(None, 16, rows, 256, 32, 16, 16) == -1
