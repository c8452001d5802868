"""The largest calls that the operators for a batch take: what lies beyond is
refused before any device call (no GPU, no context)."""
import ctypes

import pytest

import motoria_amd as M


@pytest.mark.parametrize("n", [1, 8, 9, 64])
@pytest.mark.parametrize("rows", [(1 << 28) - 31, (1 << 28) - 1, 1 << 28])
def test_rows_of_a_product(rows, n):
    """Two tiles of 16 rows are a workgroup of 512: with 2^28 rows 2^32 threads."""
    for t in (M.MHIP_F32, M.MHIP_F16, M.MHIP_BF16):
        assert M.lib().mhip_matvec_q4(None, t, 4096, rows, 4096, 4096, 32, 4096, 32, rows, 32, n, 4096) == -1


# rows, query heads, key/value heads, slots, tokens of each
ROWS = [((1 << 26) - 4, 4, 4, 1, (1 << 24) - 1), ((1 << 26) - 4, 2, 1, 2, (1 << 24) - 1),
        ((1 << 26) - 3, 1, 1, 1, (1 << 26) - 3), ((1 << 26) - 2, 2, 2, 1, (1 << 25) - 1),
        ((1 << 26) - 1, 1, 1, 1, (1 << 26) - 1)]


@pytest.mark.parametrize("rows, heads, kv, n, top", ROWS)
def test_rows_of_attention(rows, heads, kv, n, top):
    """Where parts are joined four rows are a workgroup of 256: 2^26 - 4 rows at most."""
    L = M.lib()
    d = M.PageDims(M.MHIP_F16, 1, kv, 64, 16, 10, 4, 1 << 22)
    a = M.PageArrays(*[4096 * (i + 1) for i in range(7)])
    D, A = ctypes.byref(d), ctypes.byref(a)
    assert rows == heads * n * top
    assert L.mhip_attention_shared_ws_bytes(D, heads, n, top, 0, 64) > 0  # one part: nothing to join
    size = L.mhip_attention_shared_ws_bytes(D, heads, n, top, 16, 64)
    assert (size > 0) == (rows <= (1 << 26) - 4)
    if not size:
        assert L.mhip_attention_shared(None, D, A, 0, heads, 4096, heads * 64, 4096, heads * 64, 16, None, n, top, 0, 16,
                                       64, 0.1, 4096) == -1


def test_workspace_of_calls_that_are_refused():
    """No workspace for what no product takes: more than 2^24 columns, more than
    65535 x 64 tokens."""
    size = M.lib().mhip_matvec_q4_ws_bytes
    for t in (M.MHIP_F32, M.MHIP_F16, M.MHIP_BF16):
        assert size(t, 1 << 24, 1) > 0 and size(t, 64, 65535 * 64) > 0
        for cols, n in (((1 << 24) + 32, 1), (64, 65535 * 64 + 1), ((1 << 31) - 32, 1), (32, (1 << 31) - 1)):
            assert size(t, cols, n) == 0, (t, cols, n)
            if n > 65535 * 64:
                assert M.lib().mhip_matvec_q4(None, t, 4096, 64, 4096, 4096, 32, 4096, cols, 64, cols, n, 4096) == -1
