"""mhip_matvec_q4 where tests/test_gpu_rows_q4.py does not go: the largest
numbers of tokens, and values of any size on every way that a call can take."""
import numpy as np
import pytest

import motoria_amd as M
from shared_model import TYPES, q4_tolerance, q4_weights, rounded
from test_gpu_rows_q4 import product, weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def g():
    gpu = M.Gpu()
    yield gpu
    gpu.close()


@pytest.mark.parametrize("t", [M.MHIP_F32, M.MHIP_BF16])
def test_more_tokens_than_a_launch(g, t):
    """More than 65535 workgroups' tokens (fp32 32 each, 16-bit 64)."""
    n = 65535 * 32 + 45 if t == M.MHIP_F32 else 65535 * 64
    print("test_more_tokens_than_a_launch", n, flush=True)
    rng = np.random.default_rng(1)
    codes, scales = weights(rng, 3, 32, 32)
    v = rng.standard_normal((n, 32), dtype=np.float32)
    got = product(g, t, codes, scales, 32, v)
    w, xv = q4_weights(codes, scales, 32), rounded(v, t)[0].reshape(n, 32)
    o = xv @ w.T
    assert (np.abs(got - o) <= q4_tolerance(w, xv, o, t)).all()
