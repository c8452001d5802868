"""mhip_matvec_q4 where tests/test_gpu_rows_q4.py does not go: the largest
numbers of tokens, and values of any size on every way that a call can take."""
import numpy as np
import pytest

import motoria_amd as M
from shared_model import TYPES, q4_tolerance, q4_weights, rounded, values
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


# rows, tokens: operands formed in the workgroup, straight from x or from the
# workspace (in groups of 32 and 64 tokens), and through LDS
WAYS = [(50, 3), (50, 12), (5000, 16), (50, 40), (70, 100), (24600, 20)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("size", [1e-35, 1e-30, 1e-6, 300.0, 1e30, 1e37])
@pytest.mark.parametrize("way", range(len(WAYS)))
def test_any_size_of_x(g, way, size, t):
    """x of any size that its type has: sums of 128 codes times x may be larger than
    fp32 goes where the weights' sums are not."""
    if t == M.MHIP_F16 and not 1e-7 < size < 1e4:
        pytest.skip("not an fp16 value")
    rows, n = WAYS[way]
    print("test_any_size_of_x", WAYS[way], size, t, flush=True)
    rng = np.random.default_rng(30 + way)
    codes, scales = weights(rng, rows, 1152, 128)
    v = rng.standard_normal((n, 1152)) * size
    v[1] = 0.0
    got = product(g, t, codes, scales, 128, v)
    w, xv = q4_weights(codes, scales, 128), rounded(v, t)[0]
    o = xv @ w.T
    assert (got[1] == 0).all()
    # (values, products and results below a type's normal range round to its smallest step: fp16
    # 2^-24, and fp32's and bf16's are nothing beside 1e-35 x 2^-24)
    step = 2.0 ** -24 if t == M.MHIP_F16 else 0.0
    assert (np.abs(got - o) <= q4_tolerance(w, xv, o, t) + step).all()


@pytest.mark.parametrize("t", [M.MHIP_F32, M.MHIP_BF16])
@pytest.mark.parametrize("way", range(len(WAYS)))
def test_values_far_apart(g, way, t):
    """One column 2^25 times the others, with weights of zero in some rows: those
    rows' sums are of the small values alone, and still right."""
    rows, n = WAYS[way]
    rng = np.random.default_rng(40 + way)
    codes, scales = weights(rng, rows, 1024, 32)
    codes[:32, 100] &= 0xf0  # column 200 of the first 32 rows
    v = rng.standard_normal((n, 1024))
    v[:, 200] = 2.0 ** 25
    got = product(g, t, codes, scales, 32, v)
    w, xv = q4_weights(codes, scales, 32), rounded(v, t)[0]
    o = xv @ w.T
    assert (np.abs(got - o) <= q4_tolerance(w, xv, o, t)).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("way", range(len(WAYS)))
def test_values_that_are_not_finite(g, way, t):
    """A token with a NaN or an infinity is NaN or infinite in every row whose
    weight there is not zero (NaN where it is); other tokens are as without."""
    rows, n = WAYS[way]
    rng = np.random.default_rng(50 + way)
    codes, scales = weights(rng, rows, 1184, 32)
    codes[3, 15] = codes[3, 15] & 0xf0  # row 3, column 30: zero
    v = rng.standard_normal((n, 1184))
    v[0, 30], v[n // 2, 1100], v[n - 1, 30] = np.inf, np.nan, -np.inf
    got = product(g, t, codes, scales, 32, v)
    w, xv = q4_weights(codes, scales, 32), rounded(v, t)[0]
    ends = [0, n - 1]
    with np.errstate(all="ignore"):
        o = np.where(w[None, :, 30] == 0, np.nan, np.sign(w[None, :, 30]) * xv[ends][:, 30:31])
    assert np.array_equal(np.isnan(got[ends]), np.isnan(o)) and np.isnan(got[n // 2]).all()
    ok = ~np.isnan(o)
    assert np.array_equal(got[ends][ok], o[ok])
    fine = [i for i in range(n) if i not in (0, n // 2, n - 1)]
    o = xv[fine] @ w.T
    assert (np.abs(got[fine] - o) <= q4_tolerance(w, xv[fine], o, t)).all()


# rows, cols, group, tokens
SPLIT = [(200, 2048, 32, 12), (5000, 1024, 64, 16), (130, 4096, 128, 40), (64, 2080, 32, 100), (300, 1024, 32, 5)]


@pytest.mark.parametrize("x", range(len(SPLIT)))
def test_roundings_of_fp32_do_not_add_up(g, x):
    """fp32 x enters with both its halves: taken together, results are within 2^-23 of
    their sums' sizes (half of one, the halves' and the sums' roundings, which
    average out; without the second half 2^-12 of each value, over the root of cols)."""
    rows, cols, group, n = SPLIT[x]
    rng = np.random.default_rng(60 + x)
    codes, scales = weights(rng, rows, cols, group)
    v = rng.standard_normal((n, cols)) * np.exp(rng.standard_normal(cols))
    got = product(g, M.MHIP_F32, codes, scales, group, v)
    w, xv = q4_weights(codes, scales, group), rounded(v, M.MHIP_F32)[0]
    o = xv @ w.T
    assert np.linalg.norm(got - o) <= np.linalg.norm(np.abs(xv) @ np.abs(w).T) * 2.0 ** -23


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows, cols, group, n", [(70, 1024, 32, 1), (12400, 256, 64, 2), (100, 512, 128, 12),
                                                  (5000, 768, 32, 40), (24600, 256, 64, 20)])
def test_pointers_aligned_as_their_types(g, rows, cols, group, n, t):
    """Scales on 2 bytes and results on their own size, between other data."""
    rng = np.random.default_rng(70)
    codes, scales = weights(rng, rows, cols, group)
    v, raw = rounded(rng.standard_normal((n, cols)), t)
    dt, esz = raw.dtype, raw.dtype.itemsize
    guard = np.full(n * rows + 2, 0x5a5a, dt)
    mem = [g.upload(codes), g.upload(np.concatenate([np.full(1, np.nan, np.float16), scales.ravel()])),
           g.upload(np.ascontiguousarray(raw.reshape(n, cols))), g.upload(guard), g.malloc(M.matvec_q4_ws_bytes(t, cols, n))]
    try:
        M.matvec_q4(g, t, mem[3] + esz, rows, mem[0], mem[1] + 2, group, mem[2], cols, rows, cols, n, mem[4])
        got = g.download(mem[3], guard.shape, dt)
    finally:
        for p in mem:
            g.free(p)
    assert got[0] == guard[0] and got[-1] == guard[-1]
    out = values(got[1:-1], t).reshape(n, rows)
    w, xv = q4_weights(codes, scales, group), v.reshape(n, cols)
    o = xv @ w.T
    assert (np.abs(out - o) <= q4_tolerance(w, xv, o, t)).all()
