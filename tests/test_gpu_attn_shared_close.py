"""mhip_attention_shared held to one rounding of its result: the softmax's
weights enter the product with v as fp32 would have them, whatever the cache's
type."""
import numpy as np
import pytest
import torch

import motoria_amd as M
from shared_model import TORCH, TYPES, Cache, attention, attention_tolerance, rounded
from test_gpu_attn_shared import close, fill, run

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
    # behind a prefix that ends inside a page and a tile: tiles of 64 rows of heads of 129 to
    # 256, and of 128 rows of 16-bit heads up to 64 and 128
    (16, 2, 256, 32, [340, 341, 350, 339, 400, 338, 339, 361], 338, 1),
    (8, 1, 144, 16, [203, 210, 204, 300, 203, 203, 251, 203], 203, 1),
    (12, 1, 208, 64, [450, 449, 500, 449], 449, 2),
    (8, 1, 64, 16, [310 + 3 * i for i in range(20)], 310, 1),
    (8, 1, 48, 16, [77 + i for i in range(18)], 77, 1),
    (8, 1, 112, 32, [500 + 9 * i for i in range(9)], 500, 2),
    (16, 2, 128, 16, [3020] * 20, 3007, 1),
    (16, 1, 64, 16, [310 + 3 * i for i in range(20)], 310, 1),
    (16, 1, 48, 16, [77 + i for i in range(18)], 77, 1),
    (16, 1, 128, 32, [500 + 9 * i for i in range(9)], 500, 2),
    (20, 1, 80, 64, [1100 + 2 * i for i in range(14)], 1090, 1),
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


# heads, head size, slots
TILES = [(8, 64, 20), (8, 128, 18), (8, 80, 17), (8, 32, 24), (10, 112, 4), (4, 256, 9), (8, 144, 3), (16, 208, 6),
         (2, 96, 7), (16, 64, 20), (16, 128, 17), (20, 80, 14)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("x", range(len(TILES)))
def test_values_that_are_not_finite(g, x, bad, t):
    """Infinities and NaN among the values, for every tile of rows and padded heads: where
    all rows see them, where short slots end before them in the same tile, in
    some slots' own tokens, and behind every end."""
    heads, hd, n = TILES[x]
    print("test_values_that_are_not_finite", TILES[x], bad, t, flush=True)
    rng = np.random.default_rng(300 + x)
    c = Cache(g, type=t, n_layers=1, n_kv_heads=1, head_dim=hd, max_blocks=16, max_seqs=n + 1, n_pages=17 * (n + 1))
    try:
        prefix = 150
        c.extend([0], [prefix])
        c.fork([0] * (n - 1), list(range(2, n + 1)))
        c.extend([1], [40])  # the prefix's first 40 tokens and no more
        for mine in (c.k, c.v):
            for b in range(3):
                mine[:, c.table[1][b]] = mine[:, c.table[0][b]]
        c.extend([0] + list(range(2, n + 1)), [5] + [3 + 2 * (i % 30) for i in range(2, n + 1)])
        worst = rounded(np.array([bad]), t)[1][0]
        for s in range(n + 1):
            b, r = divmod(c.len[s], 16)
            if r:
                c.k[:, c.table[s][b], :, r:] = worst
                c.v[:, c.table[s][b], :, r:] = worst
        c.load()
        q = rng.standard_normal((n + 1, heads * hd))
        seqs = rng.permutation(n + 1).tolist()
        own = [s for s in range(2, n + 1) if s % 3 == 0]
        for seen in ((), (100,), (50,), (20, 120)):
            was = c.v.copy()
            for at in seen:
                # (a page that slot 1 does not share is its own copy)
                for s in (0, 1):
                    if at < c.len[s]:
                        c.v[0, c.table[s][at // 16], 0, at % 16, (at + s) % hd] = worst
            for s in own:
                b, r = divmod(c.len[s] - 1, 16)
                c.v[0, c.table[s][b], 0, r, 1] = worst
            c.load()
            qv = rounded(q, t)[0].reshape(n + 1, heads, hd)
            rows, tol = np.zeros(qv.shape), np.zeros(qv.shape)
            for i, s in enumerate(seqs):
                k, v = c.rows("k", 0, s, c.len[s]), c.rows("v", 0, s, c.len[s])
                rows[i] = attention(qv[i], k, v, 0.1)
                fine = np.where(np.isfinite(v), v, 0.0)
                tol[i] = one_rounding(qv[i], k, fine, attention(qv[i], k, fine, 0.1), 0.1, t)
            # (slot 1 is a copy of the prefix only where nothing in it differs)
            with_prefix = (prefix, 99, 0) if not any(at < 40 for at in seen) else (0,)
            for p in with_prefix:
                got, bits = run(c, q, heads, seqs, None, 1, p, 230, 0.1)
                assert bits == 0
                close(got, rows, tol)
            c.v = was
    finally:
        c.close()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("prefix, lens", [(0, [21000]), (20000, [20000, 20007]), (17001, [17100, 17001, 40])])
def test_more_parts_than_lanes(g, prefix, lens, t):
    """One head over a long context: a row's results come from more than 64 parts."""
    rng = np.random.default_rng(22)
    blocks = -(-max(lens) // 256) + 1
    c = Cache(g, type=t, n_layers=1, n_kv_heads=1, head_dim=48, page=256, max_blocks=blocks, max_seqs=len(lens) + 1,
              n_pages=blocks + 4)
    try:
        fill(c, lens, prefix, rng)
        if lens[-1] < prefix:  # a slot that holds the prefix's first tokens and no more
            for mine in (c.k, c.v):
                mine[:, c.table[len(lens) - 1][0]] = mine[:, c.table[0][0]]
            c.load()
        seqs = list(range(len(lens)))
        q = rng.standard_normal((len(lens), 2 * 48)) * 2
        check(c, q, 2, seqs, [1] * len(lens), 1, {prefix, 0}, max(lens), 0.15)
    finally:
        c.close()


def test_many_slots(g):
    """More slots than workgroups that run at once, behind a prefix and alone."""
    rng = np.random.default_rng(23)
    n = 700
    c = Cache(g, type=M.MHIP_BF16, n_layers=1, n_kv_heads=2, head_dim=32, max_blocks=6, max_seqs=n, n_pages=6 * n)
    try:
        c.extend([0], [40])
        c.fork([0] * (n - 1), list(range(1, n)))
        c.extend(list(range(n)), [1 + i % 37 for i in range(n)])
        seqs = rng.permutation(n).tolist()
        q = rng.standard_normal((n, 4 * 32))
        check(c, q, 4, seqs, [1] * n, 1, {40, 0}, 77, 0.2)
    finally:
        c.close()


@pytest.mark.parametrize("t", TYPES)
def test_prompt_chunks(g, t):
    """Many tokens a slot, of different numbers: a prompt's first chunk, one behind a
    prefix and one that begins inside it."""
    rng = np.random.default_rng(24)
    c = Cache(g, type=t, n_layers=1, n_kv_heads=2, head_dim=64, max_blocks=20, max_seqs=4, n_pages=60)
    try:
        c.extend([0], [150])
        c.fork([0, 0], [1, 3])
        c.extend([1, 2, 3], [77, 130, 1])
        for mine in (c.k, c.v):  # slot 2 begins with the prefix's tokens
            for b in range(9):
                if b < len(c.table[2]) - 1:
                    mine[:, c.table[2][b]] = mine[:, c.table[0][b]]
        c.load()
        seqs, counts, top = [1, 3, 0], [77, 1, 130], 133
        q = rng.standard_normal((3 * top, 6 * 64))
        check(c, q, 6, seqs, counts, top, {0, 150, 90}, 227, 0.125)
        check(c, q, 6, [2, 1, 3], [130, 100, 0], top, {0, 112}, 227, 0.125)
    finally:
        c.close()
