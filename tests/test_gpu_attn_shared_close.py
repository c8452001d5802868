"""mhip_attention_shared held to one rounding of its result: the softmax's
weights enter the product with v as fp32 would have them, whatever the cache's
type."""
import numpy as np
import pytest
import torch

import motoria_amd as M
from shared_model import TORCH, TYPES, Cache, attention, attention_tolerance, rounded
from test_gpu_attn_shared import fill, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def g():
    gpu = M.Gpu()
    yield gpu
    gpu.close()


def one_rounding(q, k, v, o, scale, t):
    """How far a row of type t may be off: what attention_tolerance allows fp32
    rows, each weight's own error, and half a step of the result.

    A 16-bit cache's weight is held in two pieces. The first leaves at most half a
    step (h = eps / 2 of the weight), the second half a step of that: h^2, in the weight and
    in the sum. fp16 pieces have no step below 2^-24 and are kept 2^6 times larger: at
    most 2^-31 of the reference's weight of 1 for each token, and the sum of the weights
    is 1 or more. The result is rounded from a value that is off by all
    that: half a step where the larger of the two lies."""
    eps = torch.finfo(TORCH[t]).eps
    off = attention_tolerance(q, k, v, o, scale, M.MHIP_F32)
    if len(k) == 0 or t == M.MHIP_F32:
        return off
    g = q.shape[0] // k.shape[1]
    top = np.abs(v).max(0).repeat(g, 0)
    off = off + 2 * (eps / 2) ** 2 * top
    if t == M.MHIP_F16:
        off = off + 2 * len(k) * 2.0 ** -31 * top
    return off + eps / 2 * 2.0 ** np.floor(np.log2(np.maximum(np.abs(o) + off, 2.0 ** -14)))


def check(c, q, heads, seqs, counts, top, prefixes, max_len, scale, layer=0):
    qv = rounded(q, c.d.type)[0].reshape(len(q), heads, -1)
    rows, tol = np.zeros(qv.shape), np.zeros(qv.shape)
    for i, s in enumerate(seqs):
        for j in range(counts[i]):
            lim = max(0, c.len[s] - counts[i] + j + 1)
            k, v, x = c.rows("k", layer, s, lim), c.rows("v", layer, s, lim), i * top + j
            rows[x] = attention(qv[x], k, v, scale)
            tol[x] = one_rounding(qv[x], k, v, rows[x], scale, c.d.type)
    for prefix in prefixes:
        got, bits = run(c, q, heads, seqs, counts, top, prefix, max_len, scale, layer=layer, pad=16)
        assert bits == 0
        off = np.abs(got - rows) - tol
        print(prefix, "beyond", (off > 0).sum(), "of", off.size, "by", off.max(), flush=True)
        assert off.max() <= 0


# heads, kv heads, head size, page, lengths (slot 0 first), prefix, tokens a slot
LAYOUTS = [
    (8, 2, 64, 16, [3, 4, 7, 9], 0, 1),
    (32, 4, 128, 16, [300, 300, 412, 555, 301], 300, 1),
    (10, 2, 80, 64, [130, 200, 131], 128, 3),
    (5, 1, 256, 128, [260, 300, 257, 514], 256, 1),
    (32, 4, 128, 16, [900] * 7, 850, 2),
    (24, 8, 64, 16, [2600, 2599], 2049, 1),
]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("x", range(len(LAYOUTS)))
def test_one_rounding(g, x, t):
    heads, kv, hd, page, lens, prefix, top = LAYOUTS[x]
    print("test_one_rounding", LAYOUTS[x], t, flush=True)
    rng = np.random.default_rng(200 + x)
    blocks = -(-max(lens) // page) + 1
    c = Cache(g, type=t, n_layers=1, n_kv_heads=kv, head_dim=hd, page=page, max_blocks=blocks,
              max_seqs=len(lens) + 1, n_pages=blocks * len(lens) + 2)
    try:
        fill(c, lens, prefix, rng)
        seqs = rng.permutation(len(lens)).tolist()
        counts = [int(n) for n in rng.integers(1, top + 1, len(seqs))]
        q = rng.standard_normal((len(seqs) * top, heads * hd)) * 2
        check(c, q, heads, seqs, counts, top, {prefix, 0}, max(lens), 1 / np.sqrt(hd))
    finally:
        c.close()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("scale", [2.0 ** -5, 2.0 ** -4, 2.0 ** -3, 2.0 ** -2, 0.5, 1.0])
def test_scores_a_step_apart(g, scale, t):
    """Two scores one step of fp32 apart, which is 8 behind the scale: the second is
    a weight of e^8 beside the first's 1, in whichever order they come, in one tile or
    two. Both scores are whole numbers that fp32 has (2^26 / scale, and a step more),
    all others are 0 and weigh nothing; what is left are the exponentials (2^-21 each
    and their arguments' roundings, 16 x 2^-23), the pieces and the output."""
    if t == M.MHIP_F16 and scale < 2.0 ** -4:
        pytest.skip("the first key, 2^11 / scale, is not an fp16 value")
    c = Cache(g, type=t, n_layers=1, n_kv_heads=1, head_dim=64, max_blocks=20, max_seqs=1, n_pages=20)
    try:
        n, rng = 200, np.random.default_rng(21)
        c.extend([0], [n])
        q = np.zeros((1, 64))
        q[0, :2] = 2.0 ** 15, 8.0
        top = 2.0 ** 26 / scale
        c.v = rounded(rng.standard_normal(c.v.shape), t)[1].reshape(c.v.shape)
        for first, second in ((0, 64), (64, 0), (3, 190), (70, 75), (1, 17)):
            k = np.zeros(c.k.shape)
            for at, step in ((first, 0.0), (second, top * 2.0 ** -23 / 8)):
                k[0, c.table[0][at // 16], 0, at % 16, :2] = top / 2 ** 15, step
            c.k = rounded(k, t)[1].reshape(c.k.shape)
            c.load()
            k, v = c.rows("k", 0, 0, n), c.rows("v", 0, 0, n)
            assert scale * (k[second, 0] - k[first, 0]) @ q[0] == 8
            o = attention(q.reshape(1, 64), k, v, scale)
            eps = 0.0 if t == M.MHIP_F32 else torch.finfo(TORCH[t]).eps
            tol = np.abs(v).max() * (2.0 ** -18 + 2 * (eps / 2) ** 2 + n * 2.0 ** -30) + eps / 2 * np.abs(o)
            for prefix in (0, 64, 100):
                got, bits = run(c, q, 1, [0], None, 1, prefix, n, scale)
                print(first, second, prefix, got[0, 0, :2], o[0, :2], flush=True)
                assert bits == 0 and (np.abs(got[0] - o) <= tol).all()
    finally:
        c.close()
