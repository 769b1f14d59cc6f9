"""Timed cases of drafted tokens and windows over the paged KV cache, in plain torch
form and as the package's kernels.

tree     ancestors, places and rotary positions of trees of drafted tokens, from each
         token's parent
drafts   attention of the tokens of such trees over the pages of their lanes: each
         sees its ancestors and the context before the tree
window   attention with a sliding window and a few first tokens that stay visible
turn     rotary positions with one or several axes (time, height, width), apart from
         the tokens' places in the cache
keep     the drafts that the model agrees with: their keys and values move up behind
         the context, and the pages behind them are given back

listed() are the cases, draw() gives others of the same ranges, prepare() the tensors
a serving program holds before the call, run() one pass, work() what a pass cannot do
without, exact() its result in 64 bits.  The layout of pages is that of
perf/operators.py; head counts are those of bench.py's shapes and of narrower ones.
"""
import math

import torch

own = False

DEV = "cuda:0"
D, T = 128, 16
KV = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn}
CODE = {"fp16": 1, "bf16": 2, "fp8": 3}  # the package's element type numbers
HEADS = [(4, 4), (32, 32), (32, 8), (16, 8), (64, 8), (8, 1), (20, 20), (12, 3)]


def listed():
    return [
        # one step's trees of a few conversations: latency
        _tree("tree few", requests=4, tokens=8),
        # many lanes with deep searches
        _tree("tree batch", requests=256, tokens=300),
        # a few conversations, a handful of drafts each: latency
        _drafts("drafts few", "bf16", requests=4, tokens=8, q_heads=32, kv_heads=8, own_lo=40,
                own_hi=700),
        # a full batch, each lane with a tree of up to 64 drafts
        _drafts("drafts batch", "bf16", requests=32, tokens=64, q_heads=32, kv_heads=8, own_lo=1024,
                own_hi=8192),
        # two long documents, 8-bit pages, a small tree
        _drafts("drafts long fp8", "fp8", requests=2, tokens=16, q_heads=64, kv_heads=8,
                own_lo=60000, own_hi=131072),
        # a decode step of a model whose layers see their last 4096 tokens
        _window("window step", "bf16", requests=64, tokens=1, q_heads=32, kv_heads=8, own_lo=500,
                own_hi=40000, window=4096, sinks=4),
        # prompts in chunks through such a layer
        _window("window prompts", "fp16", requests=4, tokens=1500, q_heads=32, kv_heads=8, own_lo=1500,
                own_hi=9000, window=1024, sinks=0),
        # a short window over 8-bit pages of three lanes: latency
        _window("window few fp8", "fp8", requests=3, tokens=1, q_heads=64, kv_heads=8, own_lo=900,
                own_hi=9000, window=128, sinks=1),
        # the drafts of 32 lanes get the positions of their depths
        _turn("turn drafts", "bf16", requests=32, tokens=16, q_heads=32, kv_heads=8, axes=1, far=20000),
        # prompts of pictures and text: time, height and width in sections of the pairs
        _turn("turn images", "bf16", requests=6, tokens=2500, q_heads=32, kv_heads=8, axes=3, far=9000),
        # few lanes of a small model, 8-bit pages: latency
        _keep("keep few fp8", "fp8", requests=4, tokens=8, kv_heads=8, layers=4, lo=40, hi=300),
        # a full batch after a step's check
        _keep("keep batch", "bf16", requests=32, tokens=32, kv_heads=8, layers=32, lo=64, hi=256),
    ]


def _tree(name, **kw):
    return dict(name=name, kind="tree", **kw)


def _drafts(name, dtype, **kw):
    c = dict(name=name, kind="drafts", dtype=dtype, group=0, shared=0, window=0, sinks=0)
    c.update(kw)
    return c


def _window(name, dtype, **kw):
    return dict(name=name, kind="window", dtype=dtype, group=0, shared=0, **kw)


def _turn(name, dtype, **kw):
    c = dict(name=name, kind="turn", dtype=dtype, rot=D, layout="halves", mixed=False, q32=False)
    c.update(kw)
    return c


def _keep(name, dtype, **kw):
    return dict(name=name, kind="keep", dtype=dtype, **kw)


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: the kinds above over the sizes between and around the
    listed ones."""
    while True:
        kind = rng.choice(["tree", "drafts", "drafts", "drafts", "window", "window", "window", "turn", "keep"])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp8"])
        hq, hkv = rng.choice(HEADS)
        if kind == "tree":
            c = _tree("", requests=_log(rng, 1, 512), tokens=_log(rng, 1, 1000))
        elif kind == "drafts":
            hi = _log(rng, 16, 131072)
            c = _drafts("", dtype, requests=_log(rng, 1, 128), q_heads=hq, kv_heads=hkv,
                        own_lo=rng.choice([1, max(1, hi // 3), hi]), own_hi=hi, tokens=_log(rng, 1, 300))
            if rng.random() < 0.3:
                c["group"] = rng.randint(2, 32)
                c["shared"] = _log(rng, 1, 1000)
            elif rng.random() < 0.3:
                c["window"], c["sinks"] = _log(rng, 16, 8192), rng.choice([0, 4, 70])
        elif kind == "window":
            hi = _log(rng, 16, 131072)
            c = _window("", dtype, requests=_log(rng, 1, 128), q_heads=hq, kv_heads=hkv,
                        own_lo=rng.choice([1, max(1, hi // 3), hi]), own_hi=hi,
                        tokens=rng.choice([1, 1, rng.randint(2, 8), _log(rng, 2, 2000)]),
                        window=_log(rng, 1, 8192), sinks=rng.choice([0, 1, 4, 4, 64, 200]))
        elif kind == "turn":
            c = _turn("", dtype, requests=_log(rng, 1, 128), tokens=_log(rng, 1, 4000), q_heads=hq,
                      kv_heads=hkv, axes=rng.randint(1, 4), far=_log(rng, 100, 1000000),
                      rot=rng.choice([128, 128, 64, 96, 32, 20]), layout=rng.choice(["halves", "pairs"]),
                      mixed=rng.random() < 0.5, q32=rng.random() < 0.3)
        else:
            lo = _log(rng, 1, 1000)
            c = _keep("", dtype, requests=_log(rng, 1, 128), tokens=_log(rng, 1, 128), kv_heads=hkv,
                      layers=rng.randint(1, 32), lo=lo, hi=lo + _log(rng, 1, 400))
        del c["name"]
        if _cost(c) <= 1.0:
            return c


def _cost(c):
    """Roughly the share of the largest listed case of its kind in time and memory."""
    n, t = c["requests"], c["tokens"]
    if c["kind"] == "tree":
        return n * t * t / (256 * 300 * 300)
    if c["kind"] in ("drafts", "window"):
        most = max(c["own_hi"], t)
        sh = -(-n // c["group"]) * c["shared"] * T if c["group"] else 0
        keys = min(most + c["shared"] * T, c["window"] + c["sinks"] + t + 40 if c["window"] else 1 << 30)
        return max((n * most + sh) * c["kv_heads"] / 2.05e7, n * keys * c["kv_heads"] / 2.2e6,
                   n * t * keys * c["q_heads"] / 5.5e8)
    if c["kind"] == "turn":
        return n * t * (c["q_heads"] + 2 * c["kv_heads"]) / (6 * 2500 * 48)
    es = 1 if c["dtype"] == "fp8" else 2
    return n * ((c["hi"] + t) // T + 2) * c["layers"] * c["kv_heads"] * es / (32 * 20 * 32 * 8 * 2)


# ---- sizes -----------------------------------------------------------------------
def _seeded(seed, what):
    return torch.Generator(device=DEV).manual_seed(8 * seed + what)


def _plan(c, seed):
    """What a program's scheduler knows on the host: new tokens and context of each
    request.  The case gives them, the seed their order."""
    g = torch.Generator().manual_seed(1)
    n = c["requests"]
    order = torch.randperm(n, generator=torch.Generator().manual_seed(8 * seed + 1))

    def some(lo, hi):
        return torch.randint(lo, hi + 1, (n,), generator=g)

    new = some(max(1, c["tokens"] // 2), c["tokens"])
    new[0] = c["tokens"]
    if c["kind"] in ("drafts", "window"):
        kept = torch.maximum(some(c["own_lo"], c["own_hi"]), new)  # own tokens, the new ones last
    elif c["kind"] == "turn":
        kept = some(0, c["far"]) + new
    elif c["kind"] == "tree":
        kept = some(1, 100000) + new
    else:
        kept = some(c["lo"], c["hi"]) + new
    # trees: a token's parent is among the last few before it; and, of the tokens with
    # children, whether the model goes on to one, and to which
    back = (torch.rand((n, c["tokens"]), generator=g) ** 2 * 9).long() + 1
    col = torch.arange(c["tokens"])
    parent = torch.where(col == 0, -1, torch.clamp(col - back, min=0))
    agrees = torch.rand((n, c["tokens"]), generator=g)
    return new[order], kept[order], parent[order], agrees[order]


def _rows(new):
    """Of the batch's rows in order: the request, and the number within it."""
    req = torch.repeat_interleave(torch.arange(new.numel()), new)
    return req, torch.arange(req.numel()) - (new.cumsum(0) - new)[req]


def _ints(x):
    return x.to(torch.int32).to(DEV)


def _starts(new):
    return torch.cat([torch.zeros(1, dtype=torch.long), new.cumsum(0)])


def _values(shape, dtype, seed, what, std):
    """K/V records as the cache holds them: 16-bit values, or codes that fill the
    8-bit range."""
    g = _seeded(seed, what)
    out = torch.empty(shape, dtype=KV[dtype], device=DEV)
    flat = out.view(-1)
    for at in range(0, flat.numel(), 1 << 27):
        part = flat[at:at + (1 << 27)]
        x = torch.randn(part.shape, device=DEV, generator=g)
        part.copy_((x * (96.0 if dtype == "fp8" else std)).clamp_(-448.0, 448.0).to(out.dtype))
    return out


def _masks(parent, new):
    """Ancestors of each token of each tree, itself among them: [n, tokens, tokens]."""
    n, most = parent.shape
    real = torch.arange(most) < new.unsqueeze(1)
    step = torch.zeros((n, most, most + 1))
    step.scatter_(2, torch.where(parent < 0, most, parent).unsqueeze(2), 1.0)
    reach = step[:, :, :most].to(DEV) + torch.eye(most, device=DEV)
    far = 1
    while far < most:
        reach = (torch.matmul(reach, reach) > 0).float()
        far *= 2
    return (reach > 0) & real.to(DEV).unsqueeze(2)


def _words(mask):
    """Bits of the last axis, 64 to an int64."""
    n = mask.shape[-1]
    pad = torch.zeros(mask.shape[:-1] + (-n % 64,), dtype=torch.bool, device=mask.device)
    bits = torch.cat([mask, pad], -1).unflatten(-1, (-1, 64)).long()
    return (bits << torch.arange(64, device=mask.device)).sum(-1)


def prepare(case, seed):
    return {"tree": _prepare_tree, "drafts": _prepare_attend, "window": _prepare_attend,
            "turn": _prepare_turn, "keep": _prepare_keep}[case["kind"]](case, seed)


def _state(c, **kw):
    s = dict(case=c, scales=None, refs=None)
    s.update(kw)
    return s


def _prepare_tree(c, seed):
    new, kept, parent, _ = _plan(c, seed)
    n = c["requests"]
    req, col = _rows(new)
    lanes = torch.randperm(n, generator=torch.Generator().manual_seed(8 * seed + 2))
    length = torch.zeros(n, dtype=torch.long)
    length[lanes] = kept
    rows = req.numel()
    return _state(
        c, lanes=_ints(lanes), length=_ints(length), q_start=_ints(_starts(new)), parent=_ints(parent[req, col]),
        # results
        tree=torch.empty((rows, -(-c["tokens"] // 64)), dtype=torch.int64, device=DEV),
        at=torch.empty(rows, dtype=torch.int32, device=DEV), place=torch.empty(rows, dtype=torch.int32, device=DEV),
        lane=torch.empty(rows, dtype=torch.int32, device=DEV),
        # a cache of one small page: the call reads its lengths
        pool=torch.zeros((1, 1, 1, 2, T, D), dtype=torch.bfloat16, device=DEV),
        table=torch.full((n, 1 + int(kept.max()) // T), -1, dtype=torch.int32, device=DEV),
        # the plain form's padding
        req=req.to(DEV), col=col.to(DEV))


def _prepare_attend(c, seed):
    new, kept, parent, _ = _plan(c, seed)
    n, sh = c["requests"], c["shared"] if c["group"] else 0
    size = c["group"] or 1
    groups = -(-n // size) if c["group"] else 0
    pages = (kept + T - 1) // T
    total = int(pages.sum()) + groups * sh
    ids = torch.randperm(total, device=DEV, generator=_seeded(seed, 2)).to(torch.int32)
    table = torch.full((n, sh + int(pages.max())), -1, dtype=torch.int32, device=DEV)
    if groups:
        table[:, :sh] = ids[:groups * sh].view(groups, sh).repeat_interleave(size, 0)[:n]
    col = torch.arange(int(pages.max()), device=DEV)
    table[:, sh:][col < pages.to(DEV).unsqueeze(1)] = ids[groups * sh:]
    pool = _values((1, total, c["kv_heads"], 2, T, D), c["dtype"], seed, 3, 0.5)
    g = _seeded(seed, 4)
    scales = None
    if c["dtype"] == "fp8":
        scales = 0.5 / 96.0 * (0.75 + 0.5 * torch.rand((1, total, c["kv_heads"], 2), device=DEV, generator=g))
    rows = int(new.sum())
    q = 2.0 * torch.randn((rows, c["q_heads"], D), device=DEV, generator=g)
    start = _starts(new)
    req, nth = _rows(new)
    ends = torch.clamp(torch.arange(groups + 1) * size, max=n)
    tree = None
    if c["kind"] == "drafts":
        tree = _words(_masks(parent, new)[req.to(DEV), nth.to(DEV)]).contiguous()
    # pages from the first that a row of the request sees in its window
    length = sh * T + kept
    first = torch.clamp(length - new - c["window"] + 1, min=0) // T if c["window"] else torch.zeros_like(length)
    return _state(
        c, pool=pool, scales=scales, table=table, length=_ints(length),
        q=q.to(torch.float16 if c["dtype"] == "fp16" else torch.bfloat16),
        lanes=torch.arange(n, dtype=torch.int32, device=DEV),
        q_start=None if c["tokens"] == 1 else _ints(start), tree=tree,
        group_start=_ints(ends) if groups else None,
        shared=torch.full((groups,), sh, dtype=torch.int32, device=DEV) if groups else None,
        # the plain form's padding
        new=new.to(DEV), start=start[:-1].to(DEV), first=first.to(DEV),
        span=int(((length + T - 1) // T - first).max()))


def _prepare_turn(c, seed):
    new, kept, parent, _ = _plan(c, seed)
    n, H, Hq = c["requests"], c["kv_heads"], c["q_heads"]
    req, nth = _rows(new)
    rows = req.numel()
    first = kept - new
    p0, p1 = first // T, (kept + T - 1) // T
    count = p1 - p0
    total = int(count.sum())
    ids = torch.randperm(total, device=DEV, generator=_seeded(seed, 2)).to(torch.int32)
    table = torch.full((n, int(p1.max())), -1, dtype=torch.int32, device=DEV)
    lane_of = torch.repeat_interleave(torch.arange(n), count)
    page = torch.arange(total) - torch.repeat_interleave(count.cumsum(0) - count, count)
    table[lane_of.to(DEV), (p0[lane_of] + page).to(DEV)] = ids
    if c["axes"] == 1:  # a tree's tokens: behind the context by their depth
        deep = torch.zeros_like(parent)
        for t in range(1, min(c["tokens"], 64)):
            deep[:, t] = deep.gather(1, parent[:, t:t + 1]).squeeze(1) + 1
        at = (first[req] + deep[req, nth]).unsqueeze(0)
    else:  # pictures of 20 x 31 patches, one behind the other
        picture, y, x = nth // 620, nth // 31 % 20, nth % 31
        at = torch.stack([first[req] // (a + 1) + picture * 31 + (0, y, x, x + y)[a] for a in range(c["axes"])])
    half = c["rot"] // 2
    pairs = torch.arange(half)
    axis = pairs % c["axes"] if c["mixed"] else pairs * c["axes"] // half
    g = _seeded(seed, 4)
    x = torch.randn((rows, (Hq + 2 * H) * D), device=DEV, generator=g)
    x = x.to(torch.float16 if c["dtype"] == "fp16" else torch.bfloat16)  # a fused projection's rows
    q, k, v = x.split([Hq * D, H * D, H * D], 1)
    fp8 = c["dtype"] == "fp8"
    freq = 1000000.0 ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64) / c["rot"])
    return _state(
        c, pool=_values((1, total, H, 2, T, D), c["dtype"], seed, 3, 0.5), table=table,
        scales=torch.ones((1, total, H, 2), device=DEV) if fp8 else None,
        length=_ints(kept), q=q.view(rows, Hq, D), k=k.view(rows, H, D), v=v.view(rows, H, D),
        lane=_ints(req), pos=_ints(first[req] + nth), at=_ints(at), axis=_ints(axis), inv_freq=freq.to(DEV),
        kv_scale=4.0 / 448.0 * (0.75 + 0.5 * torch.rand((H, 2), device=DEV, generator=g)) if fp8 else None)


def _prepare_keep(c, seed):
    new, kept, parent, agrees = _plan(c, seed)
    n, most = c["requests"], c["tokens"]
    pages = (kept + T - 1) // T
    live = int(pages.sum())
    total = live + n
    ids = torch.randperm(total, device=DEV, generator=_seeded(seed, 2)).to(torch.int32)
    table = torch.full((n, int(pages.max()) + 1), -1, dtype=torch.int32, device=DEV)
    col = torch.arange(table.shape[1], device=DEV)
    table[col < pages.to(DEV).unsqueeze(1)] = ids[:live]
    refs = torch.zeros(total, dtype=torch.int32, device=DEV)
    refs[ids[:live].long()] = 1
    # tokens: siblings differ; the model's choice is one of a token's children, or another
    g = torch.Generator().manual_seed(8 * seed + 5)
    draft = torch.randint(0, 1000, (n, most), generator=g) * most + torch.arange(most)
    chosen = torch.randint(0, 1000, (n, most), generator=g) * most - 32000 * most
    for t in range(most - 1, 0, -1):  # the first child whose turn it is, else the last
        p = parent[:, t]
        r = torch.arange(n)
        take = (t < new) & (agrees[r, p] < 0.85) & ((chosen[r, p] < 0) | (agrees[r, t] < 0.5))
        chosen[r[take], p[take]] = draft[take, t]
    req, nth = _rows(new)
    shape = (c["layers"], total, c["kv_heads"], 2)
    scales = None
    if c["dtype"] == "fp8":  # one scale for a layer and kv head, as what is appended has
        scales = torch.rand((c["layers"], 1, c["kv_heads"], 2), device=DEV, generator=_seeded(seed, 6))
        scales = (0.5 + scales).expand(shape).contiguous()
    rows = req.numel()
    return _state(
        c, pool=_values(shape + (T, D), c["dtype"], seed, 3, 0.5), scales=scales, table=table, refs=refs,
        length=_ints(kept), lanes=torch.arange(n, dtype=torch.int32, device=DEV), q_start=_ints(_starts(new)),
        parent=_ints(parent[req, nth]), draft=_ints(draft[req, nth]), chosen=_ints(chosen[req, nth]),
        new=_ints(new), path=torch.empty(rows, dtype=torch.int32, device=DEV),
        kept=torch.empty(n, dtype=torch.int32, device=DEV), next=torch.empty(n, dtype=torch.int32, device=DEV),
        # the plain form's padding
        req=req.to(DEV), col=nth.to(DEV))


# ---- a pass ------------------------------------------------------------------------
def run(state):
    s, kind = state, state["case"]["kind"]
    c = s["case"]
    if own:
        p = _pages(s)
        if kind == "tree":
            p.tree(s["lanes"], s["parent"], s["tree"], at=s["at"], place=s["place"], lane=s["lane"],
                   q_start=s["q_start"])
            return [s["tree"], s["at"], s["place"], s["lane"]]
        if kind in ("drafts", "window"):
            out = torch.empty_like(s["q"])
            p.attend(0, s["q"], out, s["lanes"], q_start=s["q_start"], group_start=s["group_start"],
                     shared=s["shared"], window=c["window"], sinks=c["sinks"], tree=s["tree"])
            return out
        if kind == "turn":
            q = s["q"]
            q_out = torch.empty(q.shape, dtype=torch.float32 if c["q32"] else q.dtype, device=DEV)
            p.append(0, s["lane"], s["pos"], k=s["k"], v=s["v"], q=q, q_out=q_out, inv_freq=s["inv_freq"],
                     pairs=c["layout"] == "pairs", kv_scale=s["kv_scale"], at=s["at"],
                     axis=None if c["axes"] == 1 else s["axis"])
            return [q_out, s["pool"]] + ([s["scales"]] if s["scales"] is not None else [])
        p.accept(s["lanes"], s["draft"], s["chosen"], s["path"], s["kept"], s["next"], q_start=s["q_start"],
                 parent=s["parent"])
        p.reserve(s["lanes"], s["new"] - s["kept"])  # room for the next drafts
        return _held(s)
    if kind == "tree":
        return _plain_tree(s)
    if kind in ("drafts", "window"):
        return _plain_attend(s)
    if kind == "turn":
        return _plain_turn(s)
    _plain_keep(s)
    _plain_reserve(s, s["new"] - s["kept"])
    return _held(s)


def _held(s):
    return [s["path"], s["kept"], s["next"], s["table"], s["length"], s["refs"], s["pool"]] + \
        ([s["scales"]] if s["scales"] is not None else [])


def _pages(s):
    """The package's handle on the program's tensors, made once for them."""
    if "pages" not in s:
        import ferry_amd as F
        s["pages"] = F.Pages(s["pool"], s["table"], s["length"], refs=s["refs"], scales=s["scales"],
                             dtype=CODE[s["case"].get("dtype", "bf16")])
    return s["pages"]


# ---- the plain forms -------------------------------------------------------------------
def _plain_tree(s):
    """Ancestors by doubling: those of a token and of its ancestors."""
    c = s["case"]
    n, most = c["requests"], c["tokens"]
    req, col = s["req"], s["col"]
    start = s["q_start"].long()
    reach = torch.zeros((n, most, most), device=DEV)
    reach[req, col, col] = 1.0
    has = s["parent"] >= 0
    reach[req[has], col[has], s["parent"][has].long()] = 1.0
    far = 1
    while far < most:
        reach = (torch.matmul(reach, reach) > 0).float()
        far *= 2
    mask = reach[req, col] > 0
    s["tree"].copy_(_words(mask))
    lane = s["lanes"][req]
    base = s["length"][lane.long()] - (start[1:] - start[:-1])[req]
    s["place"].copy_(base + col)
    s["at"].copy_(base + mask.sum(1) - 1)
    s["lane"].copy_(lane)
    return [s["tree"], s["at"], s["place"], s["lane"]]


def _tokens(s, ids):
    """fp32 keys and values [n, Hkv, pages * 16, 128] of the pages ids [n, pages]."""
    pool = s["pool"][0]
    at = ids.clamp(min=0).long()
    if pool.dtype == torch.float8_e4m3fn:
        x = pool.view(torch.uint8)[at].view(pool.dtype).float() * s["scales"][0][at][..., None, None]
    else:
        x = pool[at].float()
    n, pages, H = x.shape[:3]
    x = x.permute(3, 0, 2, 1, 4, 5).reshape(2, n, H, pages * T, D)
    return x[0], x[1]


def _plain_attend(s):
    c = s["case"]
    n, H, Hq = c["requests"], c["kv_heads"], c["q_heads"]
    G, new, most = Hq // H, s["new"], c["tokens"]
    step = torch.arange(most, device=DEV)
    row = s["start"].unsqueeze(1) + step  # the batch, padded to the longest request
    real = step < new.unsqueeze(1)
    row = torch.where(real, row, 0)
    x = s["q"].float()[row].view(n, most, H, G, D).permute(0, 2, 1, 3, 4).reshape(n, H, most * G, D)
    x = x / math.sqrt(D)
    # the pages that count: the window's, or all, and those of the sinks
    col = s["first"].unsqueeze(1) + torch.arange(s["span"], device=DEV)
    at = (col.unsqueeze(2) * T + torch.arange(T, device=DEV)).view(n, -1)
    ahead = -(-c["sinks"] // T)
    wide = s["table"].shape[1]
    if ahead:
        early = torch.arange(ahead, device=DEV).expand(n, -1)
        col = torch.cat([early, col], 1)
        at = torch.cat([torch.arange(ahead * T, device=DEV).expand(n, -1), at], 1)
    k, v = _tokens(s, s["table"].gather(1, col.clamp(max=wide - 1)))
    length = s["length"].unsqueeze(1)
    v = torch.where((at < length).view(n, 1, -1, 1), v, 0.0)
    base = length - new.unsqueeze(1)
    if s["tree"] is not None:
        word = s["tree"][row]  # [n, most, words]
        bit = (at - base).clamp(0, 64 * word.shape[2] - 1)
        drafted = (word.gather(2, (bit // 64).unsqueeze(1).expand(-1, most, -1)) >> (bit % 64).unsqueeze(1)) & 1
        inside = (at >= base) & (at < length)
        sees = (at < base).unsqueeze(1) | (inside.unsqueeze(1) & (drafted > 0))
        deep = torch.zeros((n, most), dtype=torch.long, device=DEV)
        for w in range(word.shape[2]):
            deep += ((word[:, :, w:w + 1] >> torch.arange(64, device=DEV)) & 1).sum(2)
        place = base + deep - 1  # by depth
        within = (at >= base).unsqueeze(1)
    else:
        place = base + step
        sees = at.unsqueeze(1) <= place.unsqueeze(2)
        within = torch.zeros_like(sees)
    if c["window"]:
        near = at.unsqueeze(1) > (place - c["window"]).unsqueeze(2)
        sees = sees & (near | within | (at < c["sinks"]).unsqueeze(1))
        if ahead:  # a page of the sinks may be one of the window's too
            twice = at[:, ahead * T:] < ahead * T
            sees[:, :, ahead * T:] &= ~twice.unsqueeze(1)
    sees = sees.repeat_interleave(G, 1).unsqueeze(1)
    a = torch.matmul(x, k.transpose(2, 3).contiguous())
    a = torch.where(sees, a, -math.inf)
    a = torch.exp(a - a.amax(-1, keepdim=True))
    o = torch.matmul(a, v) / a.sum(-1, keepdim=True)
    o = o.view(n, H, most, G, D).transpose(1, 2).reshape(n, most, Hq, D)
    return o[real].to(s["q"].dtype)


def _plain_turn(s):
    c = s["case"]
    lane, pos = s["lane"].long(), s["pos"].long()
    angle = s["at"][s["axis"].long()].t().double() * s["inv_freq"]
    cos = torch.cos(angle).float().unsqueeze(1)
    sin = torch.sin(angle).float().unsqueeze(1)

    def turn(x):
        r, x = c["rot"], x.float()
        if c["layout"] == "pairs":
            a, b = x[..., 0:r:2], x[..., 1:r:2]
            y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = x[..., :r // 2], x[..., r // 2:r]
            y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([y, x[..., r:]], -1)

    page = s["table"][lane, pos // T].long()
    kv = torch.stack([turn(s["k"]), s["v"].float()], 2)  # [rows, H, 2, D]
    pool = s["pool"]
    if s["scales"] is not None:
        s["scales"][0, page] = s["kv_scale"]
        codes = (kv / s["kv_scale"].unsqueeze(-1)).clamp(-448.0, 448.0).to(pool.dtype)
        pool.view(torch.uint8)[0, page, :, :, pos % T] = codes.view(torch.uint8)
    else:
        pool[0, page, :, :, pos % T] = kv.to(pool.dtype)
    q = turn(s["q"])
    return [q if c["q32"] else q.to(s["q"].dtype), pool] + ([s["scales"]] if s["scales"] is not None else [])


def _plain_keep(s):
    c = s["case"]
    n, most = c["requests"], c["tokens"]
    req, col, start = s["req"], s["col"], s["q_start"].long()[:-1]

    def padded(x, fill):
        y = torch.full((n, most), fill, dtype=torch.long, device=DEV)
        y[req, col] = x.long()
        return y

    parent, draft, chosen = padded(s["parent"], -2), padded(s["draft"], -1), padded(s["chosen"], -1)
    number = torch.arange(most, device=DEV)
    now = torch.zeros(n, dtype=torch.long, device=DEV)
    going = torch.ones(n, dtype=torch.bool, device=DEV)
    path = torch.full((n, most), -1, dtype=torch.long, device=DEV)
    path[:, 0] = 0
    for i in range(1, most):
        fits = (parent == now.unsqueeze(1)) & (draft == chosen.gather(1, now.unsqueeze(1))) & (number > now.unsqueeze(1))
        child = torch.where(fits, number, most).amin(1)
        going = going & (child < most)
        now = torch.where(going, child, now)
        path[:, i] = torch.where(going, child, -1)
    kept = (path >= 0).sum(1)
    base = s["length"].long() - s["new"].long()
    # keys and values of all kept tokens, read before any is written
    r, i = torch.nonzero((path >= 0) & (path != number), as_tuple=True)
    frm, to = base[r] + path[r, i], base[r] + i
    table = s["table"].long()
    raw = s["pool"].view(torch.uint8) if c["dtype"] == "fp8" else s["pool"]
    raw[:, table[r, to // T], :, :, to % T] = raw[:, table[r, frm // T], :, :, frm % T]
    out = torch.where(path >= 0, path + start.unsqueeze(1), -1)
    s["path"].copy_(out[req, col])
    s["kept"].copy_(kept)
    s["next"].copy_(chosen.gather(1, now.unsqueeze(1)).squeeze(1))
    # the pages behind go
    left = base + kept
    number = torch.arange(table.shape[1], device=DEV)
    drop = (number >= ((left + T - 1) // T).unsqueeze(1)) & (table >= 0)
    ids = table[drop]
    s["refs"].index_add_(0, ids, torch.full_like(ids, -1, dtype=torch.int32))
    s["table"].copy_(torch.where(drop, -1, s["table"]))
    s["length"].copy_(left)


def _plain_reserve(s, tokens):
    """The lanes grow by new pages, the lowest free ids in the lanes' order (no page is
    in use twice here)."""
    had = s["length"].long()
    now = had + tokens
    need = (now + T - 1) // T - (had + T - 1) // T
    ids = torch.nonzero(s["refs"] == 0).view(-1)[:int(need.sum())]
    lane = torch.repeat_interleave(torch.arange(need.numel(), device=DEV), need)
    nth = torch.arange(ids.numel(), device=DEV) - (need.cumsum(0) - need)[lane]
    s["table"][lane, (had[lane] + T - 1) // T + nth] = ids.to(torch.int32)
    s["refs"][ids] = 1
    s["length"].copy_(now)


# ---- what a pass cannot do without -----------------------------------------------------
def work(case):
    c = case
    new, kept, parent, agrees = _plan(c, 0)
    n, rows = c["requests"], int(new.sum())
    es = 1 if c.get("dtype") == "fp8" else 2
    if c["kind"] == "tree":
        return {"bytes": rows * (4 + 8 * -(-c["tokens"] // 64) + 12) + n * 12, "flops": 0.0}
    if c["kind"] in ("drafts", "window"):
        H, Hq = c["kv_heads"], c["q_heads"]
        base = kept - new
        sh = c["shared"] * T if c["group"] else 0
        groups = -(-n // c["group"]) if c["group"] else 0
        read, seen = kept.double(), rows * sh + (new * (base + 1)).double().sum()
        if c["kind"] == "window":  # whose rows see one token more each
            seen += (new * (new - 1) / 2).sum()
        if c["window"]:
            most = c["window"] + c["sinks"]
            read = torch.clamp(read, max=most + int(new.max()))
            seen = torch.minimum(torch.full((rows,), float(most)), (base[_rows(new)[0]] + _rows(new)[1] + 1).float()).sum()
        return {"bytes": (float(read.sum()) + groups * sh) * H * 2 * D * es + rows * Hq * D * 4 + n * 4,
                "flops": 4.0 * D * Hq * float(seen)}
    if c["kind"] == "turn":
        q = c["q_heads"] * D * (6 if c["q32"] else 4)
        return {"bytes": rows * (q + 2 * c["kv_heads"] * D * (2 + es) + 8 + 4 * c["axes"]),
                "flops": rows * 3.0 * c["rot"] * (c["q_heads"] + c["kv_heads"])}
    moved = _moves(c)
    return {"bytes": moved * c["layers"] * c["kv_heads"] * 2 * D * es * 2 + rows * 16 + n * 24, "flops": 0.0}


def _moves(c):
    """Tokens of a keep case that change their place."""
    new, _, parent, agrees = _plan(c, 0)
    moved = 0
    for r in range(c["requests"]):
        takes = {}  # as the model's choices are made
        for t in range(int(new[r]) - 1, 0, -1):
            p = int(parent[r, t])
            if agrees[r, p] < 0.85 and (p not in takes or agrees[r, t] < 0.5):
                takes[p] = t
        now, i = 0, 0
        while now in takes:
            now, i = takes[now], i + 1
            moved += now != i
    return moved


# ---- in 64 bits -------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"tree": _exact_tree, "drafts": _exact_attend, "window": _exact_attend, "turn": _exact_turn,
            "keep": _exact_keep}[case["kind"]](case, s)


def _exact_tree(c, s):
    start, parent = s["q_start"].tolist(), s["parent"].tolist()
    length, lanes = s["length"].tolist(), s["lanes"].tolist()
    words = s["tree"].shape[1]
    tree, at, place, lane = [], [], [], []
    for r, ln in enumerate(lanes):
        a, b = start[r], start[r + 1]
        base = length[ln] - (b - a)
        seen = []
        for t in range(b - a):
            p = parent[a + t]
            seen.append((seen[p] if p >= 0 else 0) | 1 << t)
            row = [seen[t] >> 64 * w & (1 << 64) - 1 for w in range(words)]
            tree.append([x - (1 << 64) if x >> 63 else x for x in row])
            at.append(base + bin(seen[t]).count("1") - 1)
            place.append(base + t)
            lane.append(ln)
    return [torch.tensor(tree, dtype=torch.int64)] + [torch.tensor(x, dtype=torch.int32) for x in (at, place, lane)]


def _exact_attend(c, s):
    n, H, G = c["requests"], c["kv_heads"], c["q_heads"] // c["kv_heads"]
    table, length = s["table"].cpu(), s["length"].cpu().tolist()
    new = s["new"].cpu().tolist()
    q = s["q"].double()
    out = torch.empty(q.shape, dtype=torch.float64, device=DEV)
    at = 0
    for r in range(n):
        size, m = length[r], new[r]
        base = size - m
        token = torch.arange(size, device=DEV)
        if s["tree"] is None:
            place = torch.arange(base, size, device=DEV)
            visible = token <= place.unsqueeze(1)
            drafted = torch.zeros_like(visible)
        else:
            drafted = torch.zeros((m, size), dtype=torch.bool, device=DEV)
            bits = torch.tensor([[x >> b & 1 for x in row for b in range(64)][:m] for row in s["tree"][at:at + m].tolist()],
                                dtype=torch.bool, device=DEV)
            drafted[:, base:] = bits
            visible = drafted | (token < base)
            place = base - 1 + bits.sum(1)
        if c["window"]:
            visible &= drafted | (token > place.unsqueeze(1) - c["window"]) | (token < c["sinks"])
        some = torch.nonzero(visible.any(0)).view(-1)  # the tokens that a row sees
        visible = visible[:, some].repeat_interleave(G, 0)
        ids = table[r, :-(-size // T)].long().to(DEV)
        for h in range(H):
            raw = s["pool"][0].view(torch.uint8) if c["dtype"] == "fp8" else s["pool"][0]
            page, slot = ids[some // T], some % T
            kv = raw[page, h, :, slot]
            kv = (kv.view(s["pool"].dtype) if c["dtype"] == "fp8" else kv).double()
            if c["dtype"] == "fp8":
                kv = kv * s["scales"][0][page, h].double().unsqueeze(2)
            k, v = kv[:, 0].contiguous(), kv[:, 1].contiguous()
            x = q[at:at + m, h * G:(h + 1) * G].reshape(-1, D)
            for i in range(0, x.shape[0], 1024):  # rows at a time
                p = torch.softmax((x[i:i + 1024] @ k.t() * D ** -0.5).masked_fill(~visible[i:i + 1024], -math.inf), 1)
                x[i:i + 1024] = p @ v
            out[at:at + m, h * G:(h + 1) * G] = x.view(m, G, D)
        at += m
    return out


def _exact_turn(c, s):
    r = c["rot"]
    angle = torch.stack([s["at"][a].double() * w for a, w in zip(s["axis"].tolist(), s["inv_freq"])], 1)
    phase = torch.polar(torch.ones_like(angle), angle).unsqueeze(1)

    def turned(x):  # each pair is a complex number
        y = x.double().clone()
        if c["layout"] == "pairs":
            z = torch.complex(y[..., 0:r:2], y[..., 1:r:2]) * phase
            y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
        else:
            z = torch.complex(y[..., :r // 2], y[..., r // 2:r]) * phase
            y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
        return y

    lane, pos = s["lane"].cpu().long(), s["pos"].cpu().long()
    page = s["table"].cpu()[lane, pos // T].long()
    place = (page * T + pos % T).to(DEV)
    P, H = s["pool"].shape[1:3]
    flat = s["pool"][0].double().permute(0, 3, 1, 2, 4).reshape(P * T, H, 2, D)  # by token
    k, v = turned(s["k"]), s["v"].double()
    if s["scales"] is not None:
        scale = s["kv_scale"].double()
        k, v = [(x / scale[:, i].view(1, H, 1)).clamp(-448.0, 448.0).to(KV["fp8"]).double() for i, x in enumerate((k, v))]
        s["scales"][0, page.unique().to(DEV)] = s["kv_scale"]
    flat[place, :, 0], flat[place, :, 1] = k, v
    pool = flat.view(P, T, H, 2, D).permute(0, 2, 3, 1, 4).contiguous().unsqueeze(0)
    return [turned(s["q"]), pool] + ([s["scales"].double()] if s["scales"] is not None else [])


def _exact_keep(c, s):
    """The same on Python lists, token by token."""
    start, parent = s["q_start"].tolist(), s["parent"].tolist()
    draft, chosen = s["draft"].tolist(), s["chosen"].tolist()
    table, length, refs = s["table"].tolist(), s["length"].tolist(), s["refs"].tolist()
    raw = s["pool"].view(torch.uint8) if c["dtype"] == "fp8" else s["pool"]
    path, kept, following = [], [], []
    for r in range(c["requests"]):
        a, b = start[r], start[r + 1]
        base, line = length[r] - (b - a), [a]
        for t in range(a + 1, b):
            if a + parent[t] == line[-1] and draft[t] == chosen[line[-1]]:
                line.append(t)
        for i, t in enumerate(line):
            to, frm = base + i, base + t - a
            if to != frm:
                raw[:, table[r][to // T], :, :, to % T] = raw[:, table[r][frm // T], :, :, frm % T].clone()
        path += line + [-1] * (b - a - len(line))
        kept.append(len(line))
        following.append(chosen[line[-1]])
        for i in range(-(-(base + len(line)) // T), -(-length[r] // T)):
            refs[table[r][i]] -= 1
            table[r][i] = -1
        length[r] = base + len(line)
    free = [i for i, x in enumerate(refs) if x == 0]
    for r in range(c["requests"]):
        after = length[r] + start[r + 1] - start[r] - kept[r]
        for i in range(-(-length[r] // T), -(-after // T)):
            table[r][i] = free.pop(0)
            refs[table[r][i]] = 1
        length[r] = after
    out = [torch.tensor(x, dtype=torch.int32) for x in (path, kept, following, table, length, refs)]
    return out + [s["pool"]] + ([s["scales"].double()] if s["scales"] is not None else [])
