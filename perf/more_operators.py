"""Performance cases of the operators for a long context: a paged key/value
cache held in 4 bits, attention over it, and its eviction by accumulated
attention weight.

kinds
  store  mhip_pages_write_q4 + mhip_pages_read_q4: new tokens' keys and values
         into the cache, and back out of it as the values they have there
  attend mhip_attention_q4: one layer's attention of a batch over its slots,
         with or without adding the attention weights up per token
  evict  mhip_pages_evict: slots that have grown past their budget keep the
         tokens of the greatest weight, in every layer and head

A value of the cache is s c + m: a code c of 0 .. 15 and, for 32 values of a
token and head, s and m in fp16 (G = head_dim / 32 of each). A page of one
layer and head is one run of bytes:
  keys    codes   words [page][4 g][G j]: elements 32 j + 8 g .. + 7, the even ones
                  in the low half's nibbles, the odd ones in the high half's
          s       [page / 4][G][4 tokens]
          m       [page][G]
  values  codes   bytes [page / 4][16 c][G j][4]: elements 32 j + 2 c (low) and the
                  next (high) of tokens 0, 2, 1, 3 of the four
          s, m    [page / 4][G][4 tokens] each

Element types are those of the rows in and out: "f32", "f16", "bf16".
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (2, torch.bfloat16)}
Q4 = 4
_keep = {}


def listed():
    return [
        # a decode step of three sequences: the smallest rows
        {"name": "store 3 tokens", "kind": "store", "type": "f32", "kv": 4, "hd": 128, "page": 16,
         "seqs": 3, "count": 1, "len": 75},
        # a decode step of a full batch
        {"name": "store 64 tokens", "kind": "store", "type": "bf16", "kv": 4, "hd": 128, "page": 32,
         "seqs": 64, "count": 1, "len": 700},
        # prompts of several sequences at once, ragged, other heads
        {"name": "store prompts", "kind": "store", "type": "f16", "kv": 8, "hd": 64, "page": 64,
         "seqs": 7, "count": 1900, "len": 2100},
        # two short sequences: the smallest attention
        {"name": "attend 2 short", "kind": "attend", "type": "f32", "heads": 32, "kv": 4, "hd": 128,
         "page": 16, "seqs": 2, "count": 1, "len": 85, "gone": 0, "weights": False},
        # the library's own activations over middling conversations, one slot without a sequence
        {"name": "attend 16 of 2900 f32", "kind": "attend", "type": "f32", "heads": 32, "kv": 4,
         "hd": 128, "page": 16, "seqs": 16, "count": 1, "len": 2900, "gone": 1, "weights": False},
        # long conversations, every slot's cache is read
        {"name": "attend 32 of 8000", "kind": "attend", "type": "bf16", "heads": 32, "kv": 4,
         "hd": 128, "page": 16, "seqs": 32, "count": 1, "len": 8000, "gone": 0, "weights": False},
        # the same with a budget: weights are added up for the eviction to come
        {"name": "attend 32 of 8000, weights", "kind": "attend", "type": "bf16", "heads": 32, "kv": 4,
         "hd": 128, "page": 32, "seqs": 32, "count": 1, "len": 8000, "gone": 0, "weights": True},
        # several drafted tokens a sequence, other heads, weights
        {"name": "attend 21 x 4 drafted", "kind": "attend", "type": "f16", "heads": 24, "kv": 8,
         "hd": 64, "page": 64, "seqs": 21, "count": 4, "len": 1888, "gone": 2, "weights": True},
        # a chunk of a long prompt behind what is there already
        {"name": "attend chunk 500 of 6000", "kind": "attend", "type": "bf16", "heads": 32, "kv": 4,
         "hd": 128, "page": 64, "seqs": 1, "count": 500, "len": 6000, "gone": 0, "weights": False},
        # short sequences with a small budget, some sharing their first pages
        {"name": "evict 4 short", "kind": "evict", "kv": 4, "hd": 128, "page": 16, "layers": 2,
         "seqs": 4, "len": 300, "keep": 100, "recent": 32},
        # a batch with other heads that has grown past its budget
        {"name": "evict 12 of 1500", "kind": "evict", "kv": 8, "hd": 64, "page": 64, "layers": 6,
         "seqs": 12, "len": 1500, "keep": 777, "recent": 128},
        # one long conversation is halved in every layer
        {"name": "evict 8000 to 4000", "kind": "evict", "kv": 4, "hd": 128, "page": 32, "layers": 48,
         "seqs": 1, "len": 8000, "keep": 4000, "recent": 256},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return w["bytes"] + w["flops"] / 100


def draw(rng):
    c = _draw(rng)
    most = max(_cost(x) for x in listed() if x["kind"] == c["kind"])
    while _cost(c) > most:                                   # fewer sequences, then fewer layers, shorter ones
        if c["seqs"] > 1:
            c["seqs"] = (c["seqs"] + 1) // 2
        elif c.get("layers", 1) > 1:
            c["layers"] = (c["layers"] + 1) // 2
        else:
            c["len"] = max(c["len"] // 2, c.get("count", 0), c.get("keep", 0) + 1)
            if c.get("count", 1) > 1:
                c["count"] = (c["count"] + 1) // 2
    return c


def _draw(rng):
    kind = rng.choice(["store", "attend", "attend", "attend", "evict"])
    kv = rng.choice([1, 2, 4, 8])
    c = {"kind": kind, "kv": kv, "hd": rng.choice([32, 64, 96, 128, 256]), "page": rng.choice([16, 32, 64, 128])}
    if kind == "evict":
        size = _log(rng, 20, 6000)
        keep = rng.randint(1, max(1, size * 3 // 4))
        return dict(c, layers=_log(rng, 1, 12), seqs=_log(rng, 1, 12), len=size, keep=keep,
                    recent=rng.randint(0, keep))
    c["type"] = rng.choice(["f32", "f16", "bf16"])
    if kind == "store":
        count = rng.choice([1, _log(rng, 2, 1000)])
        return dict(c, seqs=_log(rng, 1, 64 if count == 1 else 8), count=count, len=count + _log(rng, 1, 500))
    chunk = rng.choice([False, False, False, True])
    count = _log(rng, 2, 400) if chunk else rng.choice([1, 1, 1, rng.randint(2, 5)])
    return dict(c, heads=kv * rng.choice([1, 2, 4, 5, 8]), seqs=_log(rng, 1, 3 if chunk else 48), count=count,
                len=count + _log(rng, 1, 5000), gone=rng.choice([0, 0, 1]), weights=rng.choice([False, True]))


# ---- inputs ------------------------------------------------------------------------------

def _gen(*key):
    g = torch.Generator("cuda")
    g.manual_seed(sum((int(k) + 1) * p for k, p in zip(key, (1000003, 7919, 104729))))
    return g


def _ints(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def _books(s, table, lens, refs, pages):
    """Table, lengths and counts of references in one buffer (and 16 words that
    the library keeps), with a copy to start from."""
    seqs, blocks = table.shape
    s["cut"] = (seqs * blocks, seqs * blocks + seqs, seqs * blocks + seqs + pages)
    s["start"] = torch.cat([_ints(table.reshape(-1)), _ints(lens), _ints(refs),
                            torch.zeros(16, dtype=torch.int32, device="cuda")])
    s["books"] = s["start"].clone()
    s["seqs"], s["blocks"], s["pages"] = seqs, blocks, pages


def _views(s, books):
    a, b, c = s["cut"]
    return books[:a].view(s["seqs"], s["blocks"]), books[a:b], books[b:c]


def _halves(t):
    """fp16 values as bytes, two in the last place."""
    return t.contiguous().view(torch.uint8).view(*t.shape, 2)


def _pool(case, layers, pages, seed):
    """The cache's two arrays of bytes, [layers][pages][kv][block]: codes, s
    around 0.15, m around -7.5 s, so that values spread around zero by about one."""
    page, hd = case["page"], case["hd"]
    out = []
    for which in (1, 2):
        g = _gen(seed, which)
        shape = (layers, pages, case["kv"])
        pool = torch.randint(0, 256, (*shape, page * hd * 5 // 8), device="cuda", generator=g, dtype=torch.uint8)
        n = page * hd // 32
        s = 0.05 + 0.2 * torch.rand(*shape, n, device="cuda", generator=g)
        m = s * (-7.5 + torch.randn(*shape, n, device="cuda", generator=g))
        # (which token an s and an m belong to is all the same for values made at random)
        pool[..., page * hd // 2:] = torch.cat([_halves(s.half()), _halves(m.half())], -2).flatten(-2)
        out.append(pool)
    return out


def _lens(rng, n, least, top):
    """n lengths from a third of `top` (at least `least`) up, the last of them `top` itself."""
    return np.concatenate([rng.randint(max(least, top // 3), top + 1, n - 1), [top]]).astype(np.int64)


def prepare(case, seed):
    rng = np.random.RandomState(seed % (1 << 31))
    kind, page, n = case["kind"], case["page"], case["seqs"]
    count = case.get("count", 0)
    lens = _lens(rng, n, max(count, 1), case["len"])
    gone = rng.permutation(n)[:min(case.get("gone", 0), n - 1)]
    gone = gone[gone != n - 1]
    lens[gone] = 0
    used = -(-lens // page)
    blocks = -(-case["len"] // page) + 1
    pages = n * (blocks - 1) + 3
    if kind == "evict":
        pages += n * (-(-case["keep"] // page))              # for what has to leave shared pages
    order, at = rng.permutation(pages), 0
    table, refs = np.full((n, blocks), -1), np.zeros(pages, np.int64)
    for i in range(n):
        shared = 0
        if kind == "evict" and i % 3 == 2:                   # forks of one sequence
            shared = int(min(lens[i - 1], lens[i]) // page // 2)
            table[i, :shared] = table[i - 1, :shared]
        k = int(used[i]) - shared
        table[i, shared:used[i]] = order[at:at + k]
        at += k
        refs[table[i, :used[i]]] += 1
    s = {"case": case, "top": int(lens.max())}
    _books(s, table, lens, refs, pages)
    layers = case.get("layers", 1)
    s["k"], s["v"] = _pool(case, layers, pages, seed)
    s["list"] = _ints(rng.permutation(n))
    # a few tokens draw most of the attention
    w = torch.randn(layers, n, case["kv"], blocks * page, device="cuda", generator=_gen(seed, 3))
    s["weights"] = torch.exp(2.0 * w) * 0.05
    if kind == "evict":
        return s
    typ = TYPES[case["type"]][1]
    s["count"] = _ints(np.concatenate([rng.randint(1, count + 1, n - 1), [count]]))
    if kind == "store":
        shape = (2, n * count, case["kv"] * case["hd"])
        x = torch.randn(shape, device="cuda", generator=_gen(seed, 4))
        # keys have channels that are far larger than the others
        x = x * torch.exp(0.7 * torch.randn(shape[-1], device="cuda", generator=_gen(seed, 5)))
        s["new"] = x.to(typ)
        s["back"] = torch.zeros_like(s["new"])
    else:
        q = torch.randn(n * count, case["heads"] * case["hd"], device="cuda", generator=_gen(seed, 4)) * 2.0
        s["q"] = q.to(typ)
        s["out"] = torch.empty_like(s["q"])
    return s


# ---- the plain forms -----------------------------------------------------------------------

def _parts(s, which):
    """Views of an array's bytes by token: codes, s and m, each
    [layers][pages][kv][fours][4 tokens][bytes of a token]."""
    page, hd = s["case"]["page"], s["case"]["hd"]
    a, b, four, g = page * hd // 2, page * hd // 16, page // 4, hd // 32
    x = s[which]
    scale = x[..., a:a + b].unflatten(-1, (four, g, 4, 2)).transpose(-3, -2)
    if which == "k":
        return (x[..., :a].unflatten(-1, (four, 4, hd // 2)), scale, x[..., a + b:].unflatten(-1, (four, 4, g, 2)))
    return (x[..., :a].unflatten(-1, (four, hd // 2, 4)).transpose(-2, -1), scale,
            x[..., a + b:].unflatten(-1, (four, g, 4, 2)).transpose(-3, -2))


def _place(s, which, pos):
    """Where the codes of a page's token `pos` are among its four: in order for
    keys, 0, 2, 1, 3 for values."""
    r = pos % 4
    return r if which == "k" else (r % 2) * 2 + r // 2


def _half(b):
    """fp16 values of two bytes each in the last place, as fp32."""
    return b.contiguous().view(torch.float16)[..., 0].float()


def _get(s, which, layer, pages, pos, head):
    """fp32 values [...][hd] of the tokens at `pos` of `pages` (and of `head`), all of one shape."""
    codes, scale, low = _parts(s, which)
    g, at = s["case"]["hd"] // 32, (layer, pages, head, pos // 4)
    c = codes[(*at, _place(s, which, pos))]
    two = torch.stack([c & 15, c >> 4], -1)                    # [...][bytes][2]
    if which == "k":
        # byte b of a word: nibbles 2b and 2b + 1, which are elements 4b and 4b + 2 (b < 2) or, in
        # the odd ones, 4 (b - 2) + 1 and 4 (b - 2) + 3
        c = two.unflatten(-2, (4, g, 2, 2)).movedim((-5, -4, -3, -2, -1), (-4, -5, -1, -3, -2))
    else:
        c = two.unflatten(-2, (16, g)).transpose(-3, -2)
    c = c.reshape(*c.shape[:pos.dim()], g, 32).float()
    sc, mn = _half(scale[(*at, pos % 4)]), _half(low[(*at, pos % 4)])
    return (sc[..., None] * c + mn[..., None]).flatten(-2)


def _put(s, which, layer, pages, pos, head, x):
    """Quantizes fp32 x [...][hd] into the tokens at `pos` of `pages`."""
    codes, scale, low = _parts(s, which)
    g, at = s["case"]["hd"] // 32, (layer, pages, head, pos // 4)
    x = x.unflatten(-1, (g, 32))
    m = x.amin(-1).half()
    sc = ((x.amax(-1) - m.float()) / torch.full((), 15.0, device="cuda")).half()
    step = sc.double()[..., None]
    c = torch.floor((x.double() - m.double()[..., None]) / step + 0.5)
    c = torch.where(step > 0, c, torch.zeros_like(c)).clamp(0, 15).to(torch.uint8)
    if which == "k":
        c = c.unflatten(-1, (4, 2, 2, 2)).movedim((-5, -4, -3, -2, -1), (-4, -5, -2, -1, -3))
    else:
        c = c.unflatten(-1, (16, 2)).transpose(-3, -2)
    c = c.reshape(*c.shape[:pos.dim()], s["case"]["hd"] // 2, 2)
    codes[(*at, _place(s, which, pos))] = c[..., 0] | c[..., 1] << 4
    scale[(*at, pos % 4)] = _halves(sc)
    low[(*at, pos % 4)] = _halves(m)


def _plain_store(s):
    c = s["case"]
    table, lens, _ = _views(s, s["books"])
    page, seqs, count = c["page"], s["list"].long(), s["count"].long()
    have = lens[seqs].long()
    i, j = torch.nonzero(torch.arange(c["count"], device="cuda")[None] < count[:, None], as_tuple=True)
    at = have[i] - count[i] + j
    pages = table[seqs[i], at // page].long()[:, None].expand(-1, c["kv"])
    head = torch.arange(c["kv"], device="cuda")[None].expand_as(pages)
    pos = (at % page)[:, None].expand_as(pages)
    row = i * c["count"] + j
    for y, which in enumerate("kv"):
        _put(s, which, 0, pages, pos, head, s["new"][y, row].float().unflatten(-1, (c["kv"], c["hd"])))
        s["back"][y, row] = _get(s, which, 0, pages, pos, head).flatten(-2).to(s["back"].dtype)
    s["weights"][0, seqs[i], :, at] = 0
    return {"back": s["back"], "weights": s["weights"]}


def _plain_attend(s):
    c = s["case"]
    n, count, kv, hd, page = c["seqs"], c["count"], c["kv"], c["hd"], c["page"]
    table, lens, _ = _views(s, s["books"])
    seqs, g, top = s["list"].long(), c["heads"] // kv, s["top"]
    t = torch.arange(top, device="cuda")
    pages = table[seqs][:, t // page].clamp(min=0).long()[:, None].expand(n, kv, top)
    head = torch.arange(kv, device="cuda")[None, :, None].expand(n, kv, top)
    pos = (t % page)[None, None].expand(n, kv, top)
    j = torch.arange(count, device="cuda")[None]
    lim = torch.where(j < s["count"][:, None], lens[seqs][:, None] - s["count"][:, None] + j + 1, 0)
    seen = t < lim[..., None]                                                # [n][count][tokens]
    seen = seen[:, None, :, None].expand(n, kv, count, g, top).reshape(n, kv, count * g, top)
    q = s["q"].float().view(n, count, kv, g, hd).transpose(1, 2).reshape(n, kv, count * g, hd)
    k = _get(s, "k", 0, pages, pos, head)
    score = torch.where(seen, (q @ k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(hd)), float("-inf"))
    high = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(high), torch.zeros_like(high), high))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-38)
    o = (p @ _get(s, "v", 0, pages, pos, head)).view(n, kv, count, g, hd).transpose(1, 2)
    out = {"out": o.reshape(n * count, c["heads"] * hd).to(s["q"].dtype)}
    if c["weights"]:
        s["weights"][0, seqs, :, :top] += p.sum(2)
        out["weights"] = s["weights"]
    return out


def _plain_evict(s):
    c = s["case"]
    page, keep = c["page"], c["keep"]
    s["books"].copy_(s["start"])
    table, lens, refs = _views(s, s["books"])
    seqs = s["list"].long()
    seqs = seqs[lens[seqs] > keep]
    have = lens[seqs].long()
    # what stays, in every layer and head: the last ones, then by weight, the first of equal ones
    t = torch.arange(s["top"], device="cuda")
    w = s["weights"][:, seqs, :, :s["top"]]                                  # [layers][n][kv][tokens]
    late = (t >= have[:, None] - c["recent"])[None, :, None]
    past = (t >= have[:, None])[None, :, None]
    rank = torch.where(late, float("inf"), w)
    rank = torch.where(past, -1.0, rank)
    stay = torch.sort(rank, dim=-1, descending=True, stable=True)[1][..., :keep].sort(-1)[0]
    # a page that others hold too is replaced
    nb = -(-keep // page)
    old = table[seqs].long()
    to = old[:, :nb].clone()
    shared = refs[to] > 1
    to[shared] = torch.nonzero(refs == 0)[:, 0][:int(shared.sum())]
    layer = torch.arange(w.shape[0], device="cuda")[:, None, None, None].expand_as(stay)
    head = torch.arange(c["kv"], device="cuda")[None, None, :, None].expand_as(stay)
    entry = torch.arange(len(seqs), device="cuda")[None, :, None, None].expand_as(stay)
    front = torch.arange(keep, device="cuda")[None, None, None].expand_as(stay)
    from_page, to_page = old[entry, stay // page], to[entry, front // page]
    a, b = stay % page, front % page
    for which in "kv":
        for y, x in enumerate(_parts(s, which)):
            ra, rb = (_place(s, which, a), _place(s, which, b)) if y == 0 else (a % 4, b % 4)
            x[layer, to_page, head, b // 4, rb] = x[layer, from_page, head, a // 4, ra]
    s["weights"][layer, seqs[entry], head, front] = s["weights"][layer, seqs[entry], head, stay]
    gone = torch.cat([old[old >= 0], to[shared]])
    kept = torch.cat([torch.zeros_like(old[old >= 0]), torch.ones_like(to[shared])])
    refs.index_add_(0, gone, (kept * 2 - 1).int())
    held = to[~shared]
    refs.index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    table[seqs] = -1
    table[seqs, :nb] = to.int()
    lens[seqs] = keep
    return _caches(s)


# ---- the library's calls ---------------------------------------------------------------------

def _handle(s):
    """The program's handle of a cache: its dimensions, arrays and workspace."""
    import motoria_amd as M
    if "gpu" not in _keep:
        _keep["gpu"] = M.Gpu()
    g = _keep["gpu"]
    if "cache" not in s:
        c = s["case"]
        d = M.PageDims(Q4, s["k"].shape[0], c["kv"], c["hd"], c["page"], s["pages"], s["seqs"], s["blocks"])
        s["plan"] = torch.empty(M.pages_plan_bytes(d), dtype=torch.uint8, device="cuda")
        at, (a, b, e) = s["books"].data_ptr(), s["cut"]
        s["cache"] = M.Pages(g, d, k=s["k"].data_ptr(), v=s["v"].data_ptr(), table=at, len=at + 4 * a,
                             refs=at + 4 * b, state=at + 4 * e, plan=s["plan"].data_ptr())
    return M, g, s["cache"]


def _own(s):
    c = s["case"]
    M, g, cache = _handle(s)
    n, seqs, weights = c["seqs"], s["list"].data_ptr(), s["weights"].data_ptr()
    if c["kind"] == "evict":
        if "ws" not in s:
            s["ws"] = torch.empty(cache.evict_ws_bytes(n, c["keep"], s["top"]), dtype=torch.uint8, device="cuda")
        g.check(M.lib().mhip_d2d(g.h, s["books"].data_ptr(), s["start"].data_ptr(), s["books"].numel() * 4),
                "mhip_d2d")
        cache.evict(weights, seqs, n, c["keep"], c["recent"], s["top"], s["ws"].data_ptr())
        return _caches(s)
    typ, count = TYPES[c["type"]][0], s["count"].data_ptr()
    if c["kind"] == "store":
        width = c["kv"] * c["hd"]
        new, back = s["new"], s["back"]
        cache.write_q4(0, typ, seqs, count, n, c["count"], new[0].data_ptr(), new[1].data_ptr(), width, weights)
        cache.read_q4(0, typ, seqs, count, n, c["count"], back[0].data_ptr(), back[1].data_ptr(), width)
        return {"back": back, "weights": s["weights"]}
    if "ws" not in s:
        s["ws"] = torch.empty(cache.attention_q4_ws_bytes(typ, c["heads"], n, c["count"], s["top"], c["weights"]),
                              dtype=torch.uint8, device="cuda")
    width = c["heads"] * c["hd"]
    cache.attention_q4(0, typ, c["heads"], s["q"].data_ptr(), width, s["out"].data_ptr(), width, seqs, count, n,
                       c["count"], s["top"], 1.0 / math.sqrt(c["hd"]), weights if c["weights"] else None,
                       s["ws"].data_ptr())
    return {"out": s["out"], "weights": s["weights"]} if c["weights"] else {"out": s["out"]}


# ---- the interface ----------------------------------------------------------------------------

def _caches(s):
    """A cache after an eviction: what is moved is moved whole, so its bytes are compared."""
    return {"books": _views(s, s["books"]), "k": s["k"], "v": s["v"], "weights": s["weights"]}


def run(s):
    if own:
        return _own(s)
    return {"store": _plain_store, "attend": _plain_attend, "evict": _plain_evict}[s["case"]["kind"]](s)


def work(case):
    kind, n, kv, hd = case["kind"], case["seqs"], case["kv"], case["hd"]
    row = kv * hd * 5 // 4                                   # a token's key and value in the cache, one layer
    mine = n * case["len"] * 2 // 3                          # lengths run from a third of the longest up
    if kind == "evict":
        keep = min(case["keep"], case["len"]) * n
        return {"bytes": case["layers"] * (mine * kv * 4 + keep * kv * 4 + 2 * keep * row), "flops": 0}
    size, count = TYPES[case["type"]][1].itemsize, case["count"]
    if kind == "store":
        tokens = n * (count + 1) // 2
        return {"bytes": tokens * (4 * kv * hd * size + 2 * row + kv * 4), "flops": 0}
    pairs = count * mine
    rows = 2 * n * count * case["heads"] * hd * size
    return {"bytes": mine * (row + (kv * 8 if case["weights"] else 0)) + rows, "flops": 4 * pairs * case["heads"] * hd}


# ---- the same in 64 bits ------------------------------------------------------------------------

def _read(s, which, layer, slot, n):
    """float64 [n][kv][hd] of a slot's first n tokens, one element's byte at a time by its address."""
    c = s["case"]
    page, hd, g = c["page"], c["hd"], c["hd"] // 32
    table, _, _ = _views(s, s["start"])
    pages = table[slot, :-(-n // page)].long()
    raw = s[which][layer, pages]                                                     # [pages][kv][block]
    t = torch.arange(page, device="cuda")[:, None]
    d = torch.arange(hd, device="cuda")[None]
    if which == "k":
        word = t * (hd // 8) + (d % 32 // 8) * g + d // 32
        nibble = d % 8 // 2 + 4 * (d % 2)
        byte, high = word * 4 + nibble // 2, nibble % 2
        low_at = page * hd * 9 // 16 + 2 * (t * g + d // 32)
    else:
        byte = (t // 4 * 16 + d % 32 // 2) * g * 4 + d // 32 * 4 + torch.tensor([0, 2, 1, 3], device="cuda")[t % 4]
        high = d % 2
        low_at = page * hd * 9 // 16 + 2 * ((t // 4 * g + d // 32) * 4 + t % 4)
    scale_at = page * hd // 2 + 2 * ((t // 4 * g + d // 32) * 4 + t % 4)
    code = (raw[:, :, byte].int() >> (4 * high.int())) & 15

    def half(at):
        bits = raw[:, :, at].int() + 256 * raw[:, :, at + 1].int()
        e, f = bits // 1024 % 32, (bits % 1024).double()
        v = torch.where(e > 0, (1024 + f) * torch.exp2((e - 25).double()), f * 2.0 ** -24)
        return torch.where(bits >= 32768, -v, v)
    x = half(scale_at) * code.double() + half(low_at)
    return x.transpose(1, 2).reshape(-1, c["kv"], hd)[:n]


def exact(case, seed):
    s = prepare(case, seed)
    kind, kv, hd = case["kind"], case["kv"], case["hd"]
    _, lens, _ = _views(s, s["start"])
    if kind == "store":
        # every group of 32 by the definition, and the weights of what is new at nothing
        back = torch.zeros(s["new"].shape, dtype=torch.float64, device="cuda")
        for i, (slot, n) in enumerate(zip(s["list"].tolist(), s["count"].tolist())):
            rows = slice(i * case["count"], i * case["count"] + n)
            x = s["new"][:, rows].double().reshape(2, n, -1, 32)
            low = x.amin(-1, keepdim=True).half().double()
            step = ((x.amax(-1, keepdim=True) - low) / 15).float().half().double()
            level = torch.zeros_like(x)
            for k in range(15):
                level += (x - low >= (k + 0.5) * step).double()
            back[:, rows] = (low + step * level).reshape(2, n, -1)
            s["weights"][0, slot, :, int(lens[slot]) - n:int(lens[slot])] = 0
        return {"back": back, "weights": s["weights"].double()}
    if kind == "attend":
        group, count = case["heads"] // kv, s["count"].tolist()
        q = s["q"].double().view(case["seqs"], case["count"], kv, group, hd)
        out, weights = torch.zeros_like(q), s["weights"].double()
        for i, slot in enumerate(s["list"].tolist()):
            have = int(lens[slot])
            if have == 0:
                continue
            k, v = _read(s, "k", 0, slot, have), _read(s, "v", 0, slot, have)
            first = have - count[i]
            dark = torch.arange(have, device="cuda")[None] > first + torch.arange(count[i], device="cuda")[:, None]
            for h in range(kv):
                for y in range(group):
                    e = q[i, :count[i], h, y] @ k[:, h].T.contiguous() / math.sqrt(hd)
                    p = torch.softmax(e.masked_fill(dark, float("-inf")), -1)
                    out[i, :count[i], h, y] = p @ v[:, h]
                    weights[0, slot, h, :have] += p.sum(0)
        r = {"out": out.view(s["q"].shape)}
        return dict(r, weights=weights) if case["weights"] else r
    # one slot, layer and head after the other; whole bytes move, so the result is exact as it is
    keep, recent = case["keep"], case["recent"]
    weights = s["weights"].double().cpu().numpy().copy()
    for slot in s["list"].tolist():
        have = int(lens[slot])
        if have <= keep:
            continue
        for layer in weights:
            for a in layer[slot]:
                order = np.lexsort((np.arange(have - recent), -a[:have - recent]))[:keep - recent]
                stay = np.concatenate([np.sort(order), np.arange(have - recent, have)])
                a[:keep] = a[stay]
    return {"books": [None, None, None], "k": None, "v": None, "weights": torch.from_numpy(weights).cuda()}
