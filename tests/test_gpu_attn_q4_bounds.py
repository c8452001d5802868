"""What attention over a cache in 4 bits promises of its roundings (include/mia_hip.h), against 64 bits, on
inputs whose scores are known so well that the roundings of weights and values are what is left."""
import numpy as np
import pytest

import motoria_amd as M
from q4_model import CacheQ4, attend
from shared_model import TYPES
from test_gpu_attn_q4 import call

pytestmark = pytest.mark.gpu
HALF = {  # of a value in [1, 2), and the least exponent
    M.MHIP_F32: (2.0 ** -24, -126), M.MHIP_F16: (2.0 ** -11, -14), M.MHIP_BF16: (2.0 ** -8, -126),
}


@pytest.fixture(scope="module")
def g():
    gpu = M.Gpu()
    yield gpu
    gpu.close()


def half_step(t, x):
    """Half a step of type t at x, and not more (relative to a value it is up to twice smaller)."""
    half, least = HALF[t]
    return np.exp2(np.maximum(np.floor(np.log2(np.abs(x) + 1e-300)), least)) * half


def bound(t, see, sizes, err, tiles):
    """How far an output may be off before its own rounding.
    A score: products of 32 elements, each summed by the matrix cores within 32 cuts of 2^-23 of the largest
    size, then a product with s and a sum (2^-23), and the m in one more; fp32 queries enter within 2^-22. Its
    weight is off by twice that (its own and the reference's), two exponentials' 2^-21 and the sums'. Weights enter
    within 2^-22 of their size or 2^-36 of the row's largest, their products with s as well or, all of them, within
    2^-20 (16-bit rows 2^-16) of the sum they belong to. Sums over the tokens: a wavefront adds
    32 at a time (2^-22 of the sum so far each), then wavefronts and parts are joined (2^-20)."""
    v, sc, both = sizes
    e = err * (34 * 2.0 ** -23 + (2.0 ** -22 if t == M.MHIP_F32 else 0))
    weight = 2 * e + 2.0 ** -21 + 2.0 ** -22
    sums = tiles * 2.0 ** -22 + 2.0 ** -20
    group = np.repeat(sc.reshape(*sc.shape[:-1], -1, 32).max(-1), 32, -1)
    few = 2.0 ** -20 if t == M.MHIP_F32 else 2.0 ** -16
    # (the greatest of a group's sums is 7 / 15 of the sum of 15 s w at least: its codes are 0 and 14 or 15 in each token,
    # and those of these tests are spread evenly)
    return weight * v + sums * both + few * 15 / 7 * group + 2.0 ** -21 * both


def check(c, t, heads, q, seqs, counts, top, max_len, scale, tiles):
    """Rows held to the bound and one rounding. Returns how far they are off in units of the tolerance."""
    d = c.d
    got = call(c, 0, t, heads, q, seqs, counts, top, max_len, scale, weights=False)
    x = c.rows_of(q, 0, t)[1].astype(np.float64).reshape(len(seqs) * top, heads, d.head_dim)
    for i, s in enumerate(seqs):
        n = top if counts is None else counts[i]
        k, v = c.parts(0, 0, s), c.parts(1, 0, s)
        for j in range(n):
            see = c.len[s] - n + j + 1
            o, w, sizes, err = attend(x[i * top + j], [a[:see] for a in k], [a[:see] for a in v], scale)
            largest = np.abs((v[0] + v[1])[:see]).max() if see else 0.0
            off = bound(t, see, sizes, err, tiles) + see * 2.0 ** -36 * largest
            row = got[i * top + j]
            tol = off + half_step(t, np.abs(o) + off) + 2.0 ** -25
            over = np.abs(row - o) / tol
            print("row", s, j, "of", see, "worst", over.max(), "of the tolerance", flush=True)
            assert (over <= 1).all(), (s, j, np.abs(row - o).max(), over.max(), (over > 1).mean())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("heads,kv,hd,length,count", [(4, 1, 32, 100, 2), (16, 2, 64, 200, 1), (20, 1, 32, 130, 3), (4, 1, 160, 77, 1)])
def test_one_rounding(g, t, heads, kv, hd, length, count):
    """A row's output is its formula's, rounded once: scores of a few units, from one element of each query, so
    that what scores are off by is far below the output's step."""
    print("test_one_rounding", t, heads, kv, hd, length, count, flush=True)
    c = CacheQ4(g, n_layers=1, n_kv_heads=kv, head_dim=hd, page=16, n_pages=40, max_blocks=16, max_seqs=2)
    rng = np.random.default_rng(heads + hd)
    try:
        c.extend([0], [length])
        k, v = (rng.standard_normal((length, kv * hd)) for _ in (0, 1))
        c.write_q4(0, t, [0], [length], k, v, length)
        q = np.zeros((count, heads, hd))
        q[:, np.arange(heads), rng.integers(0, hd, heads)] = 1.5
        check(c, t, heads, q.reshape(count, -1), [0], [count], count, length, 1.0, length // 128 + 1)
    finally:
        c.close()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [32, 128])
def test_scores_of_queries_of_far_apart_sizes(g, t, hd):
    """A query with one element of 512 at a code of 1, one at a code of 0 and the others of about 2^-14 at codes
    of 15: all that is small has to reach the score. Seen by the weights, which are fp32. A score is off by 33 cuts
    of 2^-23 of its largest product (34 with the product with s); what is small is 2^-14 of it in all."""
    print("test_scores_of_queries_of_far_apart_sizes", t, hd, flush=True)
    n = 60
    c = CacheQ4(g, n_layers=1, n_kv_heads=1, head_dim=hd, page=16, max_seqs=2)
    try:
        step = np.linspace(2.0 ** -10, 1, n).astype(np.float16).astype(np.float32)  # a token's s, 15 of which are fp16's too
        code = np.full(hd, 15.0, np.float32)
        code[0], code[1] = 1, 0
        code[32::32] = 0  # (a least value of 0 in every group)
        c.extend([0], [n])
        k = step[:, None] * code
        c.write_q4(0, t, [0], [n], k, np.zeros_like(k), n)
        q = np.full((1, hd), 2.0 ** -14 * 1.5, np.float32)
        q[0, 0], q[0, 1], q[0, 32::32] = 512, 0, 0
        scale = 2.0 ** -6
        x = c.rows_of(q, 0, t)[1].astype(np.float64).reshape(1, hd)
        ks, km = c.parts(0, 0, 0)
        assert (km == 0).all() and (ks[:, 0, 0] > 0).all()
        start = np.zeros_like(c.w)
        c.set_weights(start)
        call(c, 0, t, 1, q, [0], None, 1, 144, scale)
        got = g.download(c.d_w, c.w.shape, np.float32)[0, 0, 0, :n].astype(np.float64)
        _, w, _, err = attend(x, (ks, km), c.parts(1, 0, 0), scale)
        less = np.abs(ks[:, 0, 2:] @ x[0, 2:] * scale).max()
        e = err * (34 * 2.0 ** -23 + (2.0 ** -22 if t == M.MHIP_F32 else 0))
        tol = 2 * e + 2.0 ** -21 + 2.0 ** -20
        assert less > 3 * tol  # (a score without them is seen)
        assert (np.abs(got / w[:, 0] - 1) <= tol).all(), np.abs(got / w[:, 0] - 1).max() / tol
    finally:
        c.close()
