"""Performance cases of the operators for a batch of sequences that share a
prompt: the pages of a key/value cache, attention that reads the shared
prefix once for the whole batch, and products with 4-bit weights.

kinds
  fork    mhip_pages_fork + mhip_pages_free: children of running sequences (a
          prompt answered several times), released again
  append  mhip_pages_extend + mhip_pages_write: a step's new tokens get their
          pages and every layer's key/value rows
  compact mhip_pages_free + mhip_pages_compact: sequences that ended leave,
          the rest moves to the front of the pool
  attn    mhip_attention_shared: one layer's attention of a batch whose
          sequences start with the same tokens
  rows    mhip_matvec_q4: a weight matrix in 4 bits with group scales, times a
          few tokens

Element types are those of the key/value cache and of the rows in and out:
"f32" (the library's activations), "f16" and "bf16".
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (2, torch.bfloat16)}
_keep = {}


def listed():
    return [
        # four answers to a short question: the smallest call of the cache
        {"name": "fork 4", "kind": "fork", "type": "f32", "layers": 2, "kv": 4, "hd": 128,
         "page": 16, "parents": 1, "children": 4, "len": 75},
        # a server's queue forked at once, every layer's partial pages copied
        {"name": "fork 48", "kind": "fork", "type": "bf16", "layers": 48, "kv": 4, "hd": 128,
         "page": 16, "parents": 5, "children": 48, "len": 300},
        # a decode step of 64 sequences through 8 layers
        {"name": "append 64", "kind": "append", "type": "bf16", "layers": 8, "kv": 4, "hd": 128,
         "page": 16, "seqs": 64, "len": 700, "count": 1},
        # half of a server's sequences end, the pool shrinks
        {"name": "compact 48 layers", "kind": "compact", "type": "bf16", "layers": 48, "kv": 4,
         "hd": 128, "page": 16, "seqs": 25, "len": 200},
        # three short sequences with a short common start: the smallest batch
        {"name": "attn 3 short", "kind": "attn", "type": "f32", "heads": 32, "kv": 4, "hd": 128,
         "page": 16, "seqs": 3, "count": 1, "prefix": 48, "own": 37, "gone": 0},
        # the library's own cache type behind a system prompt
        {"name": "attn 16 of 2500", "kind": "attn", "type": "f32", "heads": 32, "kv": 4,
         "hd": 128, "page": 16, "seqs": 16, "count": 1, "prefix": 2500, "own": 400, "gone": 1},
        # a full batch over a long document
        {"name": "attn 64 of 8000", "kind": "attn", "type": "bf16", "heads": 32, "kv": 4,
         "hd": 128, "page": 32, "seqs": 64, "count": 1, "prefix": 8000, "own": 300, "gone": 0},
        # several drafted tokens a sequence, other heads
        {"name": "attn 21 x 4 drafted", "kind": "attn", "type": "f16", "heads": 24, "kv": 8,
         "hd": 64, "page": 64, "seqs": 21, "count": 4, "prefix": 1111, "own": 777, "gone": 2},
        # long conversations that share nothing: every sequence's cache is read
        {"name": "attn 32 unshared", "kind": "attn", "type": "bf16", "heads": 32, "kv": 4,
         "hd": 128, "page": 16, "seqs": 32, "count": 1, "prefix": 0, "own": 8000, "gone": 0},
        # one token through a key projection: the smallest product
        {"name": "rows 512 x 2048", "kind": "rows", "type": "f32", "rows": 512, "cols": 2048,
         "group": 32, "tokens": 1},
        # one token through the output head
        {"name": "rows head", "kind": "rows", "type": "f32", "rows": 151936, "cols": 2048,
         "group": 32, "tokens": 1},
        # a batch through the query projection
        {"name": "rows 64 tokens", "kind": "rows", "type": "bf16", "rows": 4096, "cols": 2048,
         "group": 128, "tokens": 64},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["fork", "append", "compact", "attn", "attn", "attn", "rows", "rows", "rows"])
    typ = rng.choice(["f32", "f16", "bf16"])
    if kind == "rows":
        group = rng.choice([32, 64, 128])
        return {"kind": kind, "type": typ, "rows": _log(rng, 48, 20000),
                "cols": group * _log(rng, 1, 4096 // group), "group": group,
                "tokens": rng.choice([1, 1, _log(rng, 2, 64)])}
    kv = rng.choice([1, 2, 4, 8])
    c = {"kind": kind, "type": typ, "kv": kv, "hd": rng.choice([64, 80, 128, 256]),
         "page": rng.choice([16, 32, 64, 128])}
    if kind == "attn":
        return dict(c, heads=kv * rng.choice([1, 2, 4, 5, 8]), seqs=_log(rng, 1, 64),
                    count=rng.choice([1, 1, 1, rng.randint(2, 5)]),
                    prefix=rng.choice([0, _log(rng, 16, 6000)]), own=_log(rng, 1, 800),
                    gone=rng.choice([0, 0, 1]))
    c["layers"] = _log(rng, 1, 12)
    if kind == "fork":
        return dict(c, parents=rng.randint(1, 4), children=_log(rng, 1, 32),
                    len=_log(rng, 1, 500))
    c = dict(c, seqs=_log(rng, 2, 48), len=_log(rng, 1, 300))
    return dict(c, count=rng.choice([1, rng.randint(2, 20)])) if kind == "append" else c


# ---- inputs ------------------------------------------------------------------------------

def _gen(*key):
    g = torch.Generator("cuda")
    g.manual_seed(sum((int(k) + 1) * p for k, p in zip(key, (1000003, 7919, 104729))))
    return g


def _ints(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def _pool(case, layers, pages, seed):
    """The cache's two arrays: [layers][pages][kv][page][hd]."""
    shape = (layers, pages, case["kv"], case["page"], case["hd"])
    t = TYPES[case["type"]][1]
    return [torch.randn(shape, device="cuda", generator=_gen(seed, k), dtype=t) for k in (1, 2)]


def _books(s, table, lens, refs, pages):
    """Table, lengths and counts of references in one buffer (and 16 words that
    the library keeps), with a copy to start from."""
    seqs, blocks = table.shape
    s["cut"] = (seqs * blocks, seqs * blocks + seqs, seqs * blocks + seqs + pages)
    s["start"] = torch.cat([_ints(table.reshape(-1)), _ints(lens), _ints(refs),
                            torch.zeros(16, dtype=torch.int32, device="cuda")])
    s["books"], s["after"] = s["start"].clone(), s["start"].clone()
    s["seqs"], s["blocks"], s["pages"] = seqs, blocks, pages


def _views(s, books):
    a, b, c = s["cut"]
    return books[:a].view(s["seqs"], s["blocks"]), books[a:b], books[b:c]


def _lens(rng, n, top):
    """n lengths up to `top`, the last of them `top` itself."""
    return np.concatenate([rng.randint(max(1, top // 3), top + 1, n - 1), [top]]).astype(np.int64)


def _cache(case, seed):
    """A pool in use: sequences of mixed lengths on scattered pages, some of
    them sharing their first pages."""
    rng = np.random.RandomState(seed % (1 << 31))
    kind, page = case["kind"], case["page"]
    n = case["parents"] if kind == "fork" else case["seqs"]
    lens = _lens(rng, n, case["len"])
    used = -(-lens // page)
    more = -(-case.get("count", 0) // page) + 1
    blocks = int(used.max()) + more
    slots = n + case.get("children", 0)
    pages = n * -(-case["len"] // page) + (n + case.get("children", 0)) * more + 7
    order = rng.permutation(pages)
    table, refs, at = np.full((slots, blocks), -1), np.zeros(pages, np.int64), 0
    for i in range(n):
        shared = 0
        if kind != "fork" and i % 3 == 2:
            shared = int(min(lens[i - 1], lens[i]) // page // 2)
            table[i, :shared] = table[i - 1, :shared]
        k = int(used[i]) - shared
        table[i, shared:used[i]] = order[at:at + k]
        at += k
        refs[table[i, :used[i]]] += 1
    s = {"case": case, "rng": rng}
    _books(s, table, np.concatenate([lens, np.zeros(slots - n, np.int64)]), refs, pages)
    s["k"], s["v"] = _pool(case, case["layers"], pages, seed)
    return s


def prepare(case, seed):
    kind = case["kind"]
    if kind == "rows":
        r, c, t = case["rows"], case["cols"], TYPES[case["type"]][1]
        g = _gen(seed, 3)
        codes = torch.randint(0, 256, (r, c // 2), device="cuda", generator=g, dtype=torch.uint8)
        scales = (0.02 / 3 * (0.5 + torch.rand(r, c // case["group"], device="cuda", generator=g))).half()
        x = torch.randn(case["tokens"], c, device="cuda", generator=g)
        x = (x * torch.exp(0.5 * torch.randn(c, device="cuda", generator=g))).to(t)
        out = torch.empty(case["tokens"], r, device="cuda", dtype=t)
        return {"case": case, "codes": codes, "scales": scales, "x": x, "out": out}
    if kind == "attn":
        return _batch(case, seed)
    s = _cache(case, seed)
    rng, n = s["rng"], case["parents"] if kind == "fork" else case["seqs"]
    if kind == "fork":
        s["src"] = _ints(rng.randint(0, n, case["children"]))
        s["dst"] = _ints(n + rng.permutation(case["children"]))
    elif kind == "append":
        s["list"] = _ints(rng.permutation(n))
        top = case["count"]
        s["count"] = _ints(np.concatenate([rng.randint(1, top + 1, n - 1), [top]]))
        shape = (case["layers"], 2, n, top, case["kv"] * case["hd"])
        s["new"] = torch.randn(shape, device="cuda", generator=_gen(seed, 4), dtype=s["k"].dtype)
    else:
        s["list"] = _ints(rng.permutation(n)[:(n + 1) // 2])
    return s


def _batch(case, seed):
    """A batch behind a common prefix (in slot 0's pages as in everybody's),
    every sequence with tokens of its own on scattered pages. The first
    `gone` entries of the batch are slots without a sequence."""
    rng = np.random.RandomState(seed % (1 << 31))
    n, page, prefix, count = case["seqs"], case["page"], case["prefix"], case["count"]
    lens = prefix + _lens(rng, n, max(case["own"], count))
    lens = np.maximum(lens, count)
    used, full = -(-lens // page), prefix // page
    blocks = int(used.max())
    pages = full + int((used - full).sum()) + 3
    order, at = rng.permutation(pages), full
    table, refs = np.full((n, blocks), -1), np.zeros(pages, np.int64)
    for i in range(n):
        k = int(used[i]) - full
        table[i, :full] = order[:full]
        table[i, full:used[i]] = order[at:at + k]
        at += k
        refs[table[i, :used[i]]] += 1
    batch = rng.permutation(n)
    gone = batch[:min(case["gone"], n - 1)]
    gone = gone[gone != 0]
    s = {"case": case}
    lens = np.where(np.isin(np.arange(n), gone), 0, lens)
    _books(s, table, lens, refs, pages)
    s["k"], s["v"] = _pool(case, 1, pages, seed)
    # the tokens of the prefix behind its last full page are in everybody's page
    part = prefix - full * page
    if part:
        at = torch.from_numpy(table[:, full]).cuda()
        for p in (s["k"], s["v"]):
            p[0, at, :, :part] = p[0, at[:1], :, :part].clone()
    s["list"] = _ints(batch)
    s["count"] = _ints(np.concatenate([rng.randint(1, count + 1, n - 1), [count]]))
    s["top"] = int(lens.max())
    width = case["heads"] * case["hd"]
    q = torch.randn(n * count, width, device="cuda", generator=_gen(seed, 5)) * 2.0
    s["q"] = q.to(s["k"].dtype)
    s["out"] = torch.empty_like(s["q"])
    return s


# ---- the plain forms -----------------------------------------------------------------------

def _plain_free(table, lens, refs, seqs):
    rows = table[seqs]
    held = rows[rows >= 0].long()
    refs.index_add_(0, held, -torch.ones_like(held, dtype=torch.int32))
    table[seqs] = -1
    lens[seqs] = 0


def _plain_fork(s):
    table, lens, refs = _views(s, s["books"])
    page, src, dst = s["case"]["page"], s["src"].long(), s["dst"].long()
    have = lens[src].long()
    full, part = have // page, have % page
    rows = table[src]
    keep = torch.arange(s["blocks"], device="cuda")[None] < full[:, None]
    held = rows[keep].long()
    refs.index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    some = torch.nonzero(part > 0)[:, 0]
    new = torch.nonzero(refs == 0)[:, 0][:some.numel()]
    old = rows[some, full[some]].long()
    child = torch.where(keep, rows, torch.full_like(rows, -1))
    child[some, full[some]] = new.int()
    refs[new] = 1
    table[dst] = child
    lens[dst] = have.int()
    mine = torch.arange(page, device="cuda")[None] < part[some][:, None]
    mine = mine[None, :, None, :, None]
    for p in (s["k"], s["v"]):
        p[:, new] = torch.where(mine, p[:, old], p[:, new])
    s["after"].copy_(s["books"])
    _plain_free(table, lens, refs, dst)


def _plain_append(s):
    s["books"].copy_(s["start"])
    table, lens, refs = _views(s, s["books"])
    page, seqs, count = s["case"]["page"], s["list"].long(), s["count"].long()
    have = lens[seqs].long()
    b0, b1 = (have + page - 1) // page, (have + count + page - 1) // page
    need = b1 - b0
    new = torch.nonzero(refs == 0)[:, 0][:int(need.sum())]
    row = torch.repeat_interleave(torch.arange(len(seqs), device="cuda"), need)
    col = b0[row] + torch.arange(len(new), device="cuda") - (torch.cumsum(need, 0) - need)[row]
    table[seqs[row], col] = new.int()
    refs[new] = 1
    lens[seqs] = (have + count).int()
    i, j = torch.nonzero(torch.arange(s["case"]["count"], device="cuda")[None] < count[:, None], as_tuple=True)
    at = have[i] + j
    where = table[seqs[i], at // page].long()
    rows = s["new"][:, :, i, j].reshape(s["new"].shape[0], 2, len(i), s["case"]["kv"], s["case"]["hd"])
    s["k"][:, where, :, at % page] = rows[:, 0].transpose(0, 1)
    s["v"][:, where, :, at % page] = rows[:, 1].transpose(0, 1)


def _plain_compact(s):
    s["books"].copy_(s["start"])
    table, lens, refs = _views(s, s["books"])
    _plain_free(table, lens, refs, s["list"].long())
    live = refs > 0
    n = int(live.sum())
    hole, mover = torch.nonzero(~live[:n])[:, 0], torch.nonzero(live[n:])[:, 0] + n
    for p in (s["k"], s["v"]):
        p[:, hole] = p[:, mover]
    to = torch.arange(s["pages"], device="cuda", dtype=torch.int32)
    to[mover] = hole.int()
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], table))
    refs[hole] = refs[mover]
    refs[mover] = 0


def _plain_attn(s):
    c = s["case"]
    n, count, kv, hd, page = c["seqs"], c["count"], c["kv"], c["hd"], c["page"]
    table, lens, _ = _views(s, s["books"])
    seqs, g = s["list"].long(), c["heads"] // kv
    top = -(-s["top"] // page)
    at = table[seqs, :top].clamp(min=0).long()
    k, v = (p[0][at].transpose(1, 2).reshape(n, kv, top * page, hd).float() for p in (s["k"], s["v"]))
    q = s["q"].float().view(n, count, kv, g, hd).transpose(1, 2).reshape(n, kv, count * g, hd)
    j = torch.arange(count, device="cuda")[None]
    lim = torch.where(j < s["count"][:, None], lens[seqs][:, None] - s["count"][:, None] + j + 1, 0)
    seen = torch.arange(top * page, device="cuda") < lim[..., None]           # [n][count][tokens]
    seen = seen[:, None, :, None].expand(n, kv, count, g, top * page).reshape(n, kv, count * g, top * page)
    score = (q @ k.transpose(2, 3)) * (1.0 / math.sqrt(hd))
    score = score.masked_fill(~seen, float("-inf"))
    high = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(high), torch.zeros_like(high), high))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-38)
    o = (p @ v).view(n, kv, count, g, hd).transpose(1, 2).reshape(n * count, c["heads"] * hd)
    return o.to(s["q"].dtype)


def _plain_rows(s):
    codes, group = s["codes"], s["case"]["group"]
    low, high = codes & 15, codes >> 4
    w = torch.stack([low, high], -1).view(codes.shape[0], -1).to(torch.int8)
    w = torch.where(w > 7, w - 16, w).float()
    w = (w.view(codes.shape[0], -1, group) * s["scales"].float()[..., None]).view(codes.shape[0], -1)
    return (s["x"].float() @ w.T).to(s["x"].dtype)


# ---- the library's calls ---------------------------------------------------------------------

def _gpu():
    import motoria_amd as M
    if "gpu" not in _keep:
        _keep["gpu"] = M.Gpu()
    return M, _keep["gpu"]


def _handle(s):
    """The program's handle of a cache: its dimensions, arrays and workspace."""
    M, g = _gpu()
    if "cache" not in s:
        c = s["case"]
        d = M.PageDims(TYPES[c["type"]][0], s["k"].shape[0], c["kv"], c["hd"], c["page"], s["pages"],
                       s["seqs"], s["blocks"])
        s["plan"] = torch.empty(M.pages_plan_bytes(d), dtype=torch.uint8, device="cuda")
        at, (a, b, e) = s["books"].data_ptr(), s["cut"]
        s["cache"] = M.Pages(g, d, k=s["k"].data_ptr(), v=s["v"].data_ptr(), table=at, len=at + 4 * a,
                             refs=at + 4 * b, state=at + 4 * e, plan=s["plan"].data_ptr())
    return M, g, s["cache"]


def _copy(M, g, to, at):
    g.check(M.lib().mhip_d2d(g.h, to.data_ptr(), at.data_ptr(), to.numel() * to.element_size()), "mhip_d2d")


def _own(s):
    c = s["case"]
    kind = c["kind"]
    if kind == "rows":
        M, g = _gpu()
        if "ws" not in s:
            s["ws"] = torch.empty(M.matvec_q4_ws_bytes(TYPES[c["type"]][0], c["cols"], c["tokens"]),
                                  dtype=torch.uint8, device="cuda")
        M.matvec_q4(g, TYPES[c["type"]][0], s["out"].data_ptr(), c["rows"], s["codes"].data_ptr(),
                    s["scales"].data_ptr(), c["group"], s["x"].data_ptr(), c["cols"], c["rows"], c["cols"],
                    c["tokens"], s["ws"].data_ptr())
        return s["out"]
    M, g, cache = _handle(s)
    if kind == "attn":
        if "ws" not in s:
            s["ws"] = torch.empty(cache.attention_ws_bytes(c["heads"], c["seqs"], c["count"], c["prefix"],
                                                           s["top"]), dtype=torch.uint8, device="cuda")
        width = c["heads"] * c["hd"]
        cache.attention(0, c["heads"], s["q"].data_ptr(), width, s["out"].data_ptr(), width,
                        s["list"].data_ptr(), s["count"].data_ptr(), c["seqs"], c["count"], 0, c["prefix"],
                        s["top"], 1.0 / math.sqrt(c["hd"]), s["ws"].data_ptr())
        return s["out"]
    if kind == "fork":
        cache.fork(s["src"].data_ptr(), s["dst"].data_ptr(), c["children"])
        _copy(M, g, s["after"], s["books"])
        cache.free(s["dst"].data_ptr(), c["children"])
        return _caches(s)
    _copy(M, g, s["books"], s["start"])
    if kind == "append":
        n, top, width = c["seqs"], c["count"], c["kv"] * c["hd"]
        seqs, count = s["list"].data_ptr(), s["count"].data_ptr()
        cache.extend(seqs, count, n)
        at, step = s["new"].data_ptr(), n * top * width * s["new"].element_size()
        for layer in range(c["layers"]):
            cache.write(layer, seqs, count, n, top, at + 2 * layer * step, at + (2 * layer + 1) * step, width)
    else:
        cache.free(s["list"].data_ptr(), s["list"].numel())
        cache.compact()
    return _caches(s)


# ---- the interface ----------------------------------------------------------------------------

def _caches(s):
    out = {"books": _views(s, s["books"]), "k": s["k"], "v": s["v"]}
    if s["case"]["kind"] == "fork":
        out["forked"] = _views(s, s["after"])
    return out


def run(s):
    if own:
        return _own(s)
    kind = s["case"]["kind"]
    if kind == "rows":
        return _plain_rows(s)
    if kind == "attn":
        return _plain_attn(s)
    {"fork": _plain_fork, "append": _plain_append, "compact": _plain_compact}[kind](s)
    return _caches(s)


def work(case):
    kind, size = case["kind"], TYPES[case["type"]][1].itemsize
    if kind == "rows":
        r, c, t = case["rows"], case["cols"], case["tokens"]
        return {"bytes": r * c // 2 + r * (c // case["group"]) * 2 + t * (r + c) * size,
                "flops": 2 * r * c * t}
    row = case["kv"] * case["hd"] * size * 2                # a token's key and value, one layer
    if kind == "attn":
        n, count = case["seqs"], case["count"]
        mine = n * max(case["own"], count) * 2 // 3          # lengths run from a third of the longest up
        pairs = count * (n * case["prefix"] + mine)
        return {"bytes": (case["prefix"] + mine) * row + 2 * n * count * case["heads"] * case["hd"] * size,
                "flops": 4 * pairs * case["heads"] * case["hd"]}
    if kind == "fork":
        moved = case["children"] * (case["page"] // 2 if case["len"] >= case["page"] else case["len"])
        meta = case["children"] * -(-case["len"] // case["page"]) * 16
    elif kind == "append":
        moved, meta = case["seqs"] * (case["count"] + 1) // 2, case["seqs"] * 16
    else:
        moved = case["seqs"] * case["len"] * 2 // 3 // 4     # half the pages stay, half of those move
        meta = case["seqs"] * -(-case["len"] // case["page"]) * 16
    return {"bytes": 2 * moved * row * case["layers"] + meta, "flops": 0}


# ---- the same in 64 bits ------------------------------------------------------------------------

class _Book:
    """A cache's table, lengths and counts as Python values, one page at a time."""

    def __init__(self, s):
        table, lens, refs = (t.cpu().tolist() for t in _views(s, s["start"]))
        self.s, self.table, self.lens, self.refs = s, table, lens, refs
        self.page = s["case"]["page"]
        self.k, self.v = s["k"].clone(), s["v"].clone()

    def take(self):
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def release(self, seqs):
        for i in seqs:
            for p in self.table[i]:
                if p >= 0:
                    self.refs[p] -= 1
            self.table[i], self.lens[i] = [-1] * len(self.table[i]), 0

    def copy(self, a, b, rows):
        for p in (self.k, self.v):
            p[:, b, :, :rows] = p[:, a, :, :rows]

    def books(self):
        return _ints(self.table), _ints(self.lens), _ints(self.refs)


def exact(case, seed):
    kind, s = case["kind"], prepare(case, seed)
    if kind == "rows":
        value = torch.tensor([0, 1, 2, 3, 4, 5, 6, 7, -8, -7, -6, -5, -4, -3, -2, -1], device="cuda",
                             dtype=torch.float64)
        x, c = s["x"].double(), s["codes"].int()
        out = torch.zeros(case["tokens"], case["rows"], dtype=torch.float64, device="cuda")
        for b in range(case["cols"] // case["group"]):
            a = b * case["group"]
            part = c[:, a // 2:(a + case["group"]) // 2]
            dot = x[:, a:a + case["group"]:2] @ value[part % 16].T
            dot = dot + x[:, a + 1:a + case["group"]:2] @ value[part // 16].T
            out += dot * s["scales"][:, b].double()
        return out
    if kind == "attn":
        table, lens, _ = _views(s, s["start"])
        group, count = case["heads"] // case["kv"], s["count"].tolist()
        q = s["q"].double().view(case["seqs"], case["count"], case["heads"], case["hd"])
        out = torch.zeros_like(q)
        for i, slot in enumerate(s["list"].tolist()):
            have = int(lens[slot])
            if have == 0:
                continue
            at = table[slot, :-(-have // case["page"])].long()
            k, v = (p[0, at].double().permute(1, 0, 2, 3).flatten(1, 2)[:, :have] for p in (s["k"], s["v"]))
            for j in range(count[i]):
                top = have - count[i] + j + 1
                for h in range(case["kv"]):
                    e = q[i, j, h * group:(h + 1) * group] @ k[h, :top].T / math.sqrt(case["hd"])
                    out[i, j, h * group:(h + 1) * group] = torch.softmax(e, -1) @ v[h, :top]
        return out.view(s["q"].shape)
    b = _Book(s)
    if kind == "fork":
        dst = s["dst"].tolist()
        for i, j in zip(s["src"].tolist(), dst):
            full, part = divmod(b.lens[i], b.page)
            b.table[j][:full], b.lens[j] = b.table[i][:full], b.lens[i]
            for p in b.table[i][:full]:
                b.refs[p] += 1
            if part:
                b.table[j][full] = b.take()
                b.copy(b.table[i][full], b.table[j][full], part)
        forked = b.books()
        b.release(dst)
        return {"books": b.books(), "k": b.k, "v": b.v, "forked": forked}
    if kind == "append":
        for i, (slot, n) in enumerate(zip(s["list"].tolist(), s["count"].tolist())):
            for j in range(n):
                block, row = divmod(b.lens[slot], b.page)
                if row == 0:
                    b.table[slot][block] = b.take()
                b.lens[slot] += 1
                new = s["new"][:, :, i, j].unflatten(-1, (case["kv"], case["hd"]))
                b.k[:, b.table[slot][block], :, row] = new[:, 0]
                b.v[:, b.table[slot][block], :, row] = new[:, 1]
    else:
        b.release(s["list"].tolist())
        n = sum(r > 0 for r in b.refs)
        movers = [p for p in range(n, len(b.refs)) if b.refs[p] > 0]
        for hole, p in zip([h for h in range(n) if b.refs[h] == 0], movers):
            b.copy(p, hole, b.page)
            b.refs[hole], b.refs[p] = b.refs[p], 0
            b.table = [[hole if e == p else e for e in r] for r in b.table]
    return {"books": b.books(), "k": b.k, "v": b.v}
