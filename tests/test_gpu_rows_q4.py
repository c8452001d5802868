"""4-bit products (mhip_matvec_q4) and their quantization against 64 bits: types,
groups, odd sizes and strides, token counts around the tiles, values far apart
and not finite, repeats."""
import numpy as np
import pytest
import torch

import motoria_amd as M
from shared_model import TYPES, esize, q4_tolerance, q4_weights, rounded, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def g():
    gpu = M.Gpu()
    yield gpu
    gpu.close()


def product(g, t, codes, scales, group, x, padx=0, pado=0):
    """(out float64, guard untouched checked) for x float64 [n][cols]."""
    n, cols = x.shape
    rows = codes.shape[0]
    dt = np.int32 if t == M.MHIP_F32 else np.int16
    raw = np.full((n, cols + padx), 0x7f80 if t else 0x7f800000, dt)
    raw[:, :cols] = rounded(x, t)[1].reshape(n, cols)
    guard = np.full((n + 1, rows + pado), 0x5a5a, dt)
    mem = [g.upload(codes), g.upload(scales), g.upload(raw), g.upload(guard),
           g.malloc(M.matvec_q4_ws_bytes(t, cols, n))]
    try:
        M.matvec_q4(g, t, mem[3], rows + pado, mem[0], mem[1], group, mem[2], cols + padx, rows, cols, n,
                    mem[4])
        got = g.download(mem[3], guard.shape, dt)
        M.matvec_q4(g, t, mem[3], rows + pado, mem[0], mem[1], group, mem[2], cols + padx, rows, cols, n,
                    mem[4])
        assert np.array_equal(got, g.download(mem[3], guard.shape, dt)), "a repeat differs"
    finally:
        for p in mem:
            g.free(p)
    assert np.array_equal(got[n:], guard[n:]) and np.array_equal(got[:, rows:], guard[:, rows:])
    return values(got[:n, :rows], t)


def weights(rng, rows, cols, group):
    codes = rng.integers(0, 256, (rows, cols // 2)).astype(np.uint8)
    scales = (0.01 * (0.5 + rng.random((rows, cols // group)))).astype(np.float16)
    return codes, scales


# rows, cols, group, tokens
SIZES = [(1, 32, 32, 1), (17, 96, 32, 1), (16, 128, 128, 2), (33, 320, 64, 3), (100, 2048, 32, 1),
         (1000, 2080, 32, 7), (512, 1024, 64, 16), (48, 1152, 128, 17), (70, 4096, 32, 15), (129, 3200, 128, 33),
         (40, 8192, 64, 5), (31, 64, 64, 64), (257, 1056, 32, 65), (64, 2304, 128, 130), (20, 16448, 64, 2),
         (33000, 160, 32, 1), (32771, 256, 64, 20), (32768, 1408, 128, 40), (40000, 32, 32, 13)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("x", range(len(SIZES)))
def test_against_64_bits(g, x, t):
    rows, cols, group, n = SIZES[x]
    print("test_against_64_bits", SIZES[x], t, flush=True)
    rng = np.random.default_rng(x)
    codes, scales = weights(rng, rows, cols, group)
    v = rng.standard_normal((n, cols)) * np.exp(rng.standard_normal(cols))
    got = product(g, t, codes, scales, group, v, padx=8 * (x % 3), pado=x % 4)
    w, xv = q4_weights(codes, scales, group), rounded(v, t)[0]
    o = xv @ w.T
    assert (np.abs(got - o) <= q4_tolerance(w, xv, o, t)).all()
    if t == M.MHIP_F32:  # roundings do not add up: their root, 2^-24 sqrt(cols) at most, and x's own
        assert np.linalg.norm(got - o) <= np.linalg.norm(np.abs(xv) @ np.abs(w).T) * 2.0 ** -23


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("size", [1e-30, 1e-6, 1.0, 300.0, 1e30])
def test_any_size_of_x(g, t, size):
    """x of sizes that fp16 does not have (16-bit x only in its own type's range),
    a token of zeros and one far larger than the others."""
    if t == M.MHIP_F16 and not 1e-7 < size < 1e4:
        pytest.skip("not an fp16 value")
    rng = np.random.default_rng(5)
    codes, scales = weights(rng, 50, 2176, 64)
    v = rng.standard_normal((4, 2176)) * size
    v[1] = 0.0
    v[2] *= 30.0
    got = product(g, t, codes, scales, 64, v)
    w, xv = q4_weights(codes, scales, 64), rounded(v, t)[0]
    o = xv @ w.T
    assert (got[1] == 0).all()
    # (fp16 x and products below its normal range round to its smallest step)
    step = 2.0 ** -24 if t == M.MHIP_F16 else 0.0
    assert (np.abs(got - o) <= q4_tolerance(w, xv, o, t) + step).all()


@pytest.mark.parametrize("t", [M.MHIP_F32, M.MHIP_BF16])
def test_values_far_apart(g, t):
    """One column 2^25 times the others, with weights of zero in some rows: those
    rows' sums are of the small values alone, and still right."""
    rng = np.random.default_rng(6)
    codes, scales = weights(rng, 64, 1024, 32)
    codes[:32, 100] &= 0xf0  # column 200 of the first 32 rows
    v = rng.standard_normal((3, 1024))
    v[:, 200] = 2.0 ** 25
    got = product(g, t, codes, scales, 32, v)
    w, xv = q4_weights(codes, scales, 32), rounded(v, t)[0]
    o = xv @ w.T
    assert (np.abs(got - o) <= q4_tolerance(w, xv, o, t)).all()


@pytest.mark.parametrize("t", TYPES)
def test_values_that_are_not_finite(g, t):
    """A token with a NaN or an infinity is NaN or infinite in every row whose
    weight there is not zero (NaN where it is); other tokens are as without."""
    rng = np.random.default_rng(7)
    codes, scales = weights(rng, 40, 1184, 32)
    codes[3, 15] = codes[3, 15] & 0xf0  # row 3, column 30: zero
    v = rng.standard_normal((5, 1184))
    v[1, 30], v[2, 1100], v[3, 30] = np.inf, np.nan, -np.inf
    got = product(g, t, codes, scales, 32, v)
    w, xv = q4_weights(codes, scales, 32), rounded(v, t)[0]
    with np.errstate(all="ignore"):
        o = np.where(w[None, :, 30] == 0, np.nan, np.sign(w[None, :, 30]) * xv[[1, 3]][:, 30:31])
    assert np.array_equal(np.isnan(got[[1, 3]]), np.isnan(o)) and np.isnan(got[2]).all()
    ok = ~np.isnan(o)
    assert np.array_equal(got[[1, 3]][ok], o[ok])
    fine = [0, 4]
    o = xv[fine] @ w.T
    assert (np.abs(got[fine] - o) <= q4_tolerance(w, xv[fine], o, t)).all()


@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantize(g, group):
    """Codes and scales as the definition gives them, weights back, and the
    weights' error: half a step, and the scale's rounding times 7."""
    rng = np.random.default_rng(group)
    rows, cols = 37, 384
    w = (rng.standard_normal((rows, cols)) * 0.02).astype(np.float32)
    w[0, :group] = 0.0
    w[1, :group] = 1e-9      # the scale rounds to 0
    w[2, 0] = 7e8            # the scale is as large as fp16 goes
    w[3, :group] = np.linspace(-0.7, 0.7, group)
    mem = [g.upload(w), g.malloc(rows * cols // 2), g.malloc(rows * cols // group * 2), g.malloc(w.nbytes)]
    try:
        g.check(M.lib().mhip_quantize_q4(g.h, mem[0], rows, cols, group, mem[1], mem[2]), "quantize")
        g.check(M.lib().mhip_dequantize_q4(g.h, mem[1], mem[2], rows, cols, group, mem[3]), "dequantize")
        codes = g.download(mem[1], (rows, cols // 2), np.uint8)
        scales = g.download(mem[2], (rows, cols // group), np.float16)
        back = g.download(mem[3], (rows, cols), np.float32)
    finally:
        for p in mem:
            g.free(p)
    b = w.reshape(rows, -1, group)
    top = np.abs(b).max(2)
    want = np.minimum(top / np.float32(7), np.float32(65504)).astype(np.float16)
    assert np.array_equal(scales, want)
    s = want.astype(np.float32)[..., None]
    q = np.where(s > 0, np.rint(b / np.where(s > 0, s, 1)), 0).clip(-8, 7).reshape(rows, cols)
    got = q4_weights(codes, np.ones_like(scales), group)
    assert np.array_equal(got, q)
    assert np.array_equal(back, (q.reshape(b.shape) * s).reshape(rows, cols).astype(np.float32))
    off = np.abs(back - w).reshape(b.shape)[3:]
    assert (off <= (0.5 + 7 * 2.0 ** -10) * s[3:]).all()


@pytest.mark.parametrize("n", [1, 20])
def test_offsets_beyond_32_bits(g, n):
    """Codes of over 2^32 bytes, zero but for the last rows."""
    rows, cols, group = (1 << 19) + 3, 16512, 128
    rng = np.random.default_rng(9)
    codes, scales = weights(rng, 3, cols, group)
    x, raw = rounded(rng.standard_normal((n, cols)), M.MHIP_BF16)
    L = M.lib()
    size, ssize = rows * (cols // 2), rows * (cols // group) * 2
    assert size > 1 << 32
    mem = [g.malloc(size), g.malloc(ssize), g.upload(raw.reshape(n, cols)), g.malloc(n * rows * 2),
           g.malloc(M.matvec_q4_ws_bytes(M.MHIP_BF16, cols, n))]
    try:
        g.check(L.mhip_zero(g.h, mem[0], size), "zero")
        g.check(L.mhip_zero(g.h, mem[1], ssize), "zero")
        g.check(L.mhip_h2d(g.h, mem[0] + size - codes.nbytes, codes.ctypes.data, codes.nbytes), "h2d")
        g.check(L.mhip_h2d(g.h, mem[1] + ssize - scales.nbytes, scales.ctypes.data, scales.nbytes), "h2d")
        M.matvec_q4(g, M.MHIP_BF16, mem[3], rows, mem[0], mem[1], group, mem[2], cols, rows, cols, n, mem[4])
        out = values(g.download(mem[3], (n, rows), np.int16), M.MHIP_BF16)
    finally:
        for p in mem:
            g.free(p)
    assert (out[:, :-3] == 0).all()
    w = q4_weights(codes, scales, group)
    o = x @ w.T
    assert (np.abs(out[:, -3:] - o) <= q4_tolerance(w, x, o, M.MHIP_BF16)).all()


# rows, cols, group, tokens: around the choices of many tokens
MANY = [(24600, 256, 32, 17), (24577, 1312, 32, 32), (24576, 2304, 128, 20), (5000, 512, 64, 16), (4112, 800, 32, 9),
        (4100, 1056, 32, 33), (200, 512, 64, 100), (100, 2080, 32, 96), (5000, 256, 128, 64)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("pad", [0, 8, 32])  # rows of x that start in other halves of their lines
@pytest.mark.parametrize("x", range(len(MANY)))
def test_many_tokens(g, x, pad, t):
    rows, cols, group, n = MANY[x]
    print("test_many_tokens", MANY[x], pad, t, flush=True)
    rng = np.random.default_rng(100 + x)
    codes, scales = weights(rng, rows, cols, group)
    v = rng.standard_normal((n, cols)) * np.exp(rng.standard_normal(cols))
    got = product(g, t, codes, scales, group, v, padx=pad, pado=x % 3)
    w, xv = q4_weights(codes, scales, group), rounded(v, t)[0]
    o = xv @ w.T
    assert (np.abs(got - o) <= q4_tolerance(w, xv, o, t)).all()
