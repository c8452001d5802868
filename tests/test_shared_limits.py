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
