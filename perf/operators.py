"""Timed cases of the paged KV cache: the operators that fill, share and read the
pages of a batch of requests, in plain torch form and as the package's kernels.

attend   attention of new query tokens over the pages of their lanes; requests
         of a group share their leading pages, which count once for all of them
append   rotary positions of new tokens' queries and keys, and the write of keys
         and values into the lanes' pages
fork     lanes copied by reference, then grown by a token each: pages in use
         twice are copied before they are written
turnover half of the lanes end, the pool is compacted, new lanes take the room,
         for one half and then for the other

A page is one K and one V record of [16 tokens][128] per layer and kv head, the
block layout of the host tier.  listed() are the cases, draw() gives others of the
same ranges, prepare() the tensors a serving program holds before the call,
run() one pass, work() what a pass cannot do without, exact() its result in 64
bits.  Head counts are those of bench.py's shapes and of narrower ones.
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
        # a few short conversations: one token each, latency only
        _attend("attend few", "bf16", requests=4, q_heads=32, kv_heads=8, own_lo=40, own_hi=700),
        # one user's long document in two conversations: few rows, long axis
        _attend("attend long", "bf16", requests=2, q_heads=32, kv_heads=8, own_lo=90000,
                own_hi=131072),
        # many samples of one long prompt, each a little way on
        _attend("attend samples", "bf16", requests=64, group=64, shared=2048, q_heads=32,
                kv_heads=8, own_lo=1, own_hi=512),
        # the shared-prefix shape: 8 groups of 16 agents, 8-bit pages
        _attend("attend agents fp8", "fp8", requests=128, group=16, shared=517, q_heads=32,
                kv_heads=8, own_lo=16, own_hi=1024),
        # chunks of prompts that start with the same instructions
        _attend("attend chunks", "fp16", requests=6, group=3, shared=256, q_heads=32, kv_heads=8,
                own_lo=1024, own_hi=4096, tokens=1024),
        # a decode step's new token in each of 64 lanes
        _append("append step", "bf16", requests=64, tokens=1, q_heads=32, kv_heads=8, far=20000),
        # prompts of a dozen requests; a part of the head turns, neighbours in pairs
        _append("append prompts", "bf16", requests=12, tokens=2048, q_heads=32, kv_heads=8,
                rot=64, layout="pairs", far=60000),
        # prompts far into contexts of up to a million tokens, 8-bit pages
        _append("append far fp8", "fp8", requests=5, tokens=1500, q_heads=32, kv_heads=32,
                far=1000000, stretch=8.0, q32=True),
        # a prompt sampled 24 times
        _fork("fork samples", "bf16", parents=1, children=24, layers=8, kv_heads=8, lo=700, hi=900),
        # beams of a batch go on from their best
        _fork("fork beams", "fp16", parents=16, children=2, layers=16, kv_heads=8, lo=200, hi=1200),
        # a batch turns over in a pool that serves eight layers
        _turnover("turnover", "bf16", requests=48, layers=8, kv_heads=8, lo=200, hi=1900),
        # a few short lanes of a small model, 8-bit pages: latency
        _turnover("turnover few", "fp8", requests=6, layers=4, kv_heads=8, lo=30, hi=500),
    ]


def _attend(name, dtype, **kw):
    c = dict(name=name, kind="attend", dtype=dtype, group=0, shared=0, tokens=1)
    c.update(kw)
    return c


def _append(name, dtype, **kw):
    c = dict(name=name, kind="append", dtype=dtype, rot=D, layout="halves", stretch=1.0, q32=False)
    c.update(kw)
    return c


def _fork(name, dtype, **kw):
    return dict(name=name, kind="fork", dtype=dtype, **kw)


def _turnover(name, dtype, **kw):
    return dict(name=name, kind="turnover", dtype=dtype, **kw)


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: the kinds above over the sizes between and around the
    listed ones."""
    while True:
        kind = rng.choice(["attend"] * 4 + ["append"] * 2 + ["fork", "turnover"])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp8"])
        hq, hkv = rng.choice(HEADS)
        if kind == "attend":
            hi = _log(rng, 16, 131072)
            c = _attend("", dtype, requests=_log(rng, 1, 128), q_heads=hq, kv_heads=hkv,
                        own_lo=rng.choice([1, max(1, hi // 3), hi]), own_hi=hi,
                        tokens=rng.choice([1, 1, rng.randint(2, 8), _log(rng, 2, 1024)]))
            if rng.random() < 0.5:
                c["group"] = rng.randint(2, 64)
                c["shared"] = _log(rng, 1, 4096)
        elif kind == "append":
            c = _append("", dtype, requests=_log(rng, 1, 128), tokens=_log(rng, 1, 4096), q_heads=hq,
                        kv_heads=hkv, rot=rng.choice([128, 128, 64, 96, 32, 20]),
                        layout=rng.choice(["halves", "pairs"]), far=_log(rng, 100, 1000000),
                        stretch=rng.choice([1.0, 4.0, 8.0, 32.0]), q32=rng.random() < 0.3)
        elif kind == "fork":
            lo = _log(rng, 1, 3000)
            c = _fork("", dtype, parents=_log(rng, 1, 32), children=_log(rng, 1, 32),
                      layers=rng.randint(1, 32), kv_heads=hkv, lo=lo, hi=lo + _log(rng, 1, 2000))
        else:
            lo = _log(rng, 1, 3000)
            c = _turnover("", dtype, requests=_log(rng, 2, 128), layers=rng.randint(1, 32),
                          kv_heads=hkv, lo=lo, hi=lo + _log(rng, 1, 2000))
        del c["name"]
        if _cost(c) <= 1.0:
            return c


def _cost(c):
    """Roughly the share of the largest listed case of its kind in time and memory."""
    es = 1 if c["dtype"] == "fp8" else 2
    if c["kind"] == "attend":
        n, t = c["requests"], c["tokens"]
        groups = -(-n // c["group"]) if c["group"] else 0
        most = max(c["own_hi"], t)
        kept = n * most + groups * c["shared"] * T
        seen = n * t * (most + c["shared"] * T)
        return max(kept * c["kv_heads"] / 2.1e6, seen * c["q_heads"] / 1.6e9)
    if c["kind"] == "append":
        rows = c["requests"] * c["tokens"]
        return rows * (c["q_heads"] + 2 * c["kv_heads"]) / (12 * 2048 * 48)
    lanes = c["parents"] if c["kind"] == "fork" else c["requests"]
    pages = lanes * (c["hi"] // T + 1) + (c["parents"] * c["children"] if c["kind"] == "fork" else 0)
    return pages * c["layers"] * c["kv_heads"] * es / (48 * 119 * 64 * 2)


# ---- sizes -----------------------------------------------------------------------
def _seeded(seed, what):
    return torch.Generator(device=DEV).manual_seed(8 * seed + what)


def _lengths(c, seed):
    """Per-lane sizes on the host, what a program's scheduler knows: the case gives
    them, the seed their order."""
    g = torch.Generator().manual_seed(1)
    n = c["parents"] if c["kind"] == "fork" else c["requests"]
    order = torch.randperm(n, generator=torch.Generator().manual_seed(8 * seed + 1))

    def some(lo, hi):
        return torch.randint(lo, hi + 1, (n,), generator=g)

    if c["kind"] == "attend":
        new = some(1, c["tokens"])
        new[0] = c["tokens"]
        # own tokens, the new ones last
        return new[order], torch.maximum(some(c["own_lo"], c["own_hi"]), new)[order]
    if c["kind"] == "append":
        new = some(max(1, c["tokens"] // 2), c["tokens"])
        new[0] = c["tokens"]
        return new[order], some(0, c["far"])[order]
    return some(c["lo"], c["hi"])[order], None


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


def prepare(case, seed):
    return {"attend": _prepare_attend, "append": _prepare_append, "fork": _prepare_fork,
            "turnover": _prepare_turnover}[case["kind"]](case, seed)


def _state(c, **kw):
    s = dict(case=c, scales=None, refs=None)
    s.update(kw)
    return s


def _prepare_attend(c, seed):
    new, kept = _lengths(c, seed)
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
    start = torch.cat([torch.zeros(1, dtype=torch.long), new.cumsum(0)])
    ends = torch.clamp(torch.arange(groups + 1) * size, max=n)
    return _state(
        c, pool=pool, scales=scales, table=table, length=(sh * T + kept).to(torch.int32).to(DEV),
        q=q.to(torch.float16 if c["dtype"] == "fp16" else torch.bfloat16),
        lanes=torch.arange(n, dtype=torch.int32, device=DEV),
        q_start=None if c["tokens"] == 1 else start.to(torch.int32).to(DEV),
        group_start=ends.to(torch.int32).to(DEV) if groups else None,
        shared=torch.full((groups,), sh, dtype=torch.int32, device=DEV) if groups else None,
        # the plain form's padding
        new=new.to(DEV), start=start[:-1].to(DEV), own_pages=int(pages.max()))


def _frequencies(c):
    """Angles per token of the rotated pairs (float64), and the factor on the
    rotated values.  A stretched context keeps the fast pairs, slows the slow ones by
    the stretch and blends linearly between 32 and 1 turns over 8192 tokens."""
    i = torch.arange(0, c["rot"], 2, dtype=torch.float64)
    f = 500000.0 ** (-i / c["rot"])
    if c["stretch"] == 1.0:
        return f, 1.0
    turns = 8192.0 * f / (2.0 * math.pi)
    keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
    return f * keep + f / c["stretch"] * (1.0 - keep), 0.1 * math.log(c["stretch"]) + 1.0


def _prepare_append(c, seed):
    new, first = _lengths(c, seed)
    n, rows = c["requests"], int(new.sum())
    H, Hq = c["kv_heads"], c["q_heads"]
    p0, p1 = first // T, (first + new + T - 1) // T
    count = p1 - p0
    total = int(count.sum())
    ids = torch.randperm(total, device=DEV, generator=_seeded(seed, 2)).to(torch.int32)
    table = torch.full((n, int(p1.max())), -1, dtype=torch.int32, device=DEV)
    lane_of = torch.repeat_interleave(torch.arange(n), count)
    nth = torch.arange(total) - torch.repeat_interleave(count.cumsum(0) - count, count)
    table[lane_of.to(DEV), (p0[lane_of] + nth).to(DEV)] = ids
    lane = torch.repeat_interleave(torch.arange(n), new)
    pos = torch.arange(rows) - (new.cumsum(0) - new)[lane] + first[lane]
    g = _seeded(seed, 4)
    x = torch.randn((rows, (Hq + 2 * H) * D), device=DEV, generator=g)
    x = x.to(torch.float16 if c["dtype"] == "fp16" else torch.bfloat16)  # a fused projection's rows
    q, k, v = x.split([Hq * D, H * D, H * D], 1)
    freq, factor = _frequencies(c)
    fp8 = c["dtype"] == "fp8"
    return _state(
        c, pool=_values((1, total, H, 2, T, D), c["dtype"], seed, 3, 0.5), table=table,
        scales=torch.ones((1, total, H, 2), device=DEV) if fp8 else None,
        length=(first + new).to(torch.int32).to(DEV), q=q.view(rows, Hq, D), k=k.view(rows, H, D),
        v=v.view(rows, H, D), lane=lane.to(torch.int32).to(DEV), pos=pos.to(torch.int32).to(DEV),
        inv_freq=freq.to(DEV), factor=factor,
        kv_scale=4.0 / 448.0 * (0.75 + 0.5 * torch.rand((H, 2), device=DEV, generator=g)) if fp8 else None)


def _prepare_fork(c, seed):
    kept, _ = _lengths(c, seed)
    n, m = c["parents"], c["parents"] * c["children"]
    pages = (kept + T - 1) // T
    live = int(pages.sum())
    total = live + m + 5
    ids = torch.randperm(total, device=DEV, generator=_seeded(seed, 2)).to(torch.int32)
    table = torch.full((n + m, int(pages.max()) + 1), -1, dtype=torch.int32, device=DEV)
    col = torch.arange(table.shape[1], device=DEV)
    table[:n][col < pages.to(DEV).unsqueeze(1)] = ids[:live]
    refs = torch.zeros(total, dtype=torch.int32, device=DEV)
    refs[ids[:live].long()] = 1
    length = torch.zeros(n + m, dtype=torch.int32, device=DEV)
    length[:n] = kept.to(torch.int32).to(DEV)
    src = torch.arange(m, device=DEV) % n
    return _state(c, pool=_values((c["layers"], total, c["kv_heads"], 2, T, D), c["dtype"], seed, 3, 0.5),
                  scales=_page_scales(c, total, seed), table=table, length=length, refs=refs,
                  src=src.to(torch.int32), dst=torch.arange(n, n + m, dtype=torch.int32, device=DEV),
                  one=torch.ones(m, dtype=torch.int32, device=DEV))


def _page_scales(c, total, seed):
    if c["dtype"] != "fp8":
        return None
    return torch.rand((c["layers"], total, c["kv_heads"], 2), device=DEV, generator=_seeded(seed, 5))


def _prepare_turnover(c, seed):
    kept, _ = _lengths(c, seed)
    n = c["requests"]
    even, odd = torch.arange(0, n, 2), torch.arange(1, n, 2)
    pages = (kept + T - 1) // T
    total = int(pages.sum()) + int(pages.sum()) // 8 + 1
    # even lanes hold the low pages, odd ones those behind them
    order = torch.cat([even, odd])
    lane_of = torch.repeat_interleave(order, pages[order])
    nth = torch.arange(lane_of.numel()) - torch.repeat_interleave(
        pages[order].cumsum(0) - pages[order], pages[order])
    table = torch.full((n, int(pages.max())), -1, dtype=torch.int32, device=DEV)
    table[lane_of.to(DEV), nth.to(DEV)] = torch.arange(lane_of.numel(), dtype=torch.int32, device=DEV)
    refs = torch.zeros(total, dtype=torch.int32, device=DEV)
    refs[:lane_of.numel()] = 1
    halves = [h.to(torch.int32).to(DEV) for h in (even, odd)]
    length = kept.to(torch.int32).to(DEV)
    return _state(c, pool=_values((c["layers"], total, c["kv_heads"], 2, T, D), c["dtype"], seed, 3, 0.5),
                  scales=_page_scales(c, total, seed), table=table, length=length, refs=refs,
                  halves=halves, grow=[length[h.long()].clone() for h in halves])


# ---- a pass ------------------------------------------------------------------------
def run(state):
    s, kind = state, state["case"]["kind"]
    if own:
        p = _pages(s)
        if kind == "attend":
            out = torch.empty_like(s["q"])
            p.attend(0, s["q"], out, s["lanes"], q_start=s["q_start"], group_start=s["group_start"],
                     shared=s["shared"])
            return out
        if kind == "append":
            c, q = s["case"], s["q"]
            q_out = torch.empty(q.shape, dtype=torch.float32 if c["q32"] else q.dtype, device=DEV)
            p.append(0, s["lane"], s["pos"], k=s["k"], v=s["v"], q=q, q_out=q_out,
                     inv_freq=s["inv_freq"], factor=s["factor"], pairs=c["layout"] == "pairs",
                     kv_scale=s["kv_scale"])
            return [q_out, s["pool"]] + ([s["scales"]] if s["scales"] is not None else [])
        if kind == "fork":
            p.trim(s["dst"])
            p.fork(s["src"], s["dst"])
            p.reserve(s["dst"], s["one"])
        else:
            a, b = s["halves"]
            p.trim(a)
            p.compact()
            p.reserve(a, s["grow"][0])
            p.trim(b)
            p.compact()
            p.reserve(b, s["grow"][1])
        return _held(s)
    if kind == "attend":
        return _plain_attend(s)
    if kind == "append":
        return _plain_append(s)
    if kind == "fork":
        _trim(s, s["dst"])
        _plain_fork(s, s["src"], s["dst"])
        _reserve(s, s["dst"], s["one"])
    else:
        a, b = s["halves"]
        _trim(s, a)
        _compact(s)
        _reserve(s, a, s["grow"][0])
        _trim(s, b)
        _compact(s)
        _reserve(s, b, s["grow"][1])
    return _held(s)


def _held(s):
    return [s["table"], s["length"], s["refs"], s["pool"]] + ([s["scales"]] if s["scales"] is not None else [])


def _pages(s):
    """The package's handle on the program's tensors, made once for them."""
    if "pages" not in s:
        import ferry_amd as F
        s["pages"] = F.Pages(s["pool"], s["table"], s["length"], refs=s["refs"], scales=s["scales"],
                             dtype=CODE[s["case"]["dtype"]])
    return s["pages"]


# ---- the plain forms -------------------------------------------------------------------
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
    G, sh, size = Hq // H, c["shared"] if c["group"] else 0, c["group"] or 1
    new, start, most = s["new"], s["start"], c["tokens"]
    step = torch.arange(most, device=DEV)
    row = start.unsqueeze(1) + step  # the batch, padded to the longest request
    real = step < new.unsqueeze(1)
    row = torch.where(real, row, 0)
    x = s["q"].float()[row].view(n, most, H, G, D).permute(0, 2, 1, 3, 4).reshape(n, H, most * G, D)
    x = x / math.sqrt(D)
    # a token sees the tokens up to itself
    limit = (s["length"] - new).unsqueeze(1) + step + 1
    limit = limit.repeat_interleave(G, 1).view(n, 1, most * G, 1)
    k, v = _tokens(s, s["table"][:, sh:sh + s["own_pages"]])
    at = sh * T + torch.arange(k.shape[2], device=DEV)
    live = (at < s["length"].unsqueeze(1)).view(n, 1, -1, 1)
    v = torch.where(live, v, 0.0)
    a = torch.matmul(x, k.transpose(2, 3).contiguous())
    a = torch.where(at < limit, a, -math.inf)
    top = a.amax(-1, keepdim=True)
    if sh:
        groups = -(-n // size)
        k2, v2 = _tokens(s, s["table"][::size, :sh])
        pad = torch.zeros((groups * size, H, most * G, D), device=DEV)
        pad[:n] = x
        x2 = pad.view(groups, size, H, most * G, D).transpose(1, 2).reshape(groups, H, -1, D)
        b = torch.matmul(x2, k2.transpose(2, 3).contiguous())

        def split(t):  # [groups, H, size * rows, m] -> [n, H, rows, m]
            return t.view(groups, H, size, most * G, -1).transpose(1, 2).reshape(groups * size, H, most * G, -1)[:n]

        top = torch.maximum(top, split(b.amax(-1, keepdim=True)))
        pad_top = torch.zeros((groups * size, H, most * G, 1), device=DEV)
        pad_top[:n] = top
        b = torch.exp(b - pad_top.view(groups, size, H, most * G, 1).transpose(1, 2).reshape(groups, H, -1, 1))
        a = torch.exp(a - top)
        o = torch.matmul(a, v) + split(torch.matmul(b, v2))
        o = o / (a.sum(-1, keepdim=True) + split(b.sum(-1, keepdim=True)))
    else:
        a = torch.exp(a - top)
        o = torch.matmul(a, v) / a.sum(-1, keepdim=True)
    o = o.view(n, H, most, G, D).transpose(1, 2).reshape(n, most, Hq, D)
    return o[real].to(s["q"].dtype)


def _plain_append(s):
    c = s["case"]
    lane, pos = s["lane"].long(), s["pos"].long()
    angle = pos.double().unsqueeze(1) * s["inv_freq"]
    cos = (torch.cos(angle) * s["factor"]).float().unsqueeze(1)
    sin = (torch.sin(angle) * s["factor"]).float().unsqueeze(1)

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


def _trim(s, lanes):
    """The lanes end: their pages lose a reference each."""
    lanes = lanes.long()
    ids = s["table"][lanes]
    ids = ids[ids >= 0].long()
    s["refs"].index_add_(0, ids, torch.full_like(ids, -1, dtype=torch.int32))
    s["table"][lanes] = -1
    s["length"][lanes] = 0


def _plain_fork(s, src, dst):
    """dst lanes get src lanes' pages by reference."""
    src, dst = src.long(), dst.long()
    rows = s["table"][src]
    ids = rows[rows >= 0].long()
    s["refs"].index_add_(0, ids, torch.ones_like(ids, dtype=torch.int32))
    s["table"][dst] = rows
    s["length"][dst] = s["length"][src]


def _copy_pages(s, to, frm):
    pool = s["pool"]
    raw = pool.view(torch.uint8) if pool.dtype == torch.float8_e4m3fn else pool
    raw[:, to] = raw[:, frm]
    if s["scales"] is not None:
        s["scales"][:, to] = s["scales"][:, frm]


def _reserve(s, lanes, tokens):
    """The lanes grow: a last page that is begun and in use twice is copied, then new
    pages follow, the lowest free ids in the lanes' order."""
    lanes = lanes.long()
    table, refs = s["table"], s["refs"]
    had = s["length"][lanes].long()
    now = had + tokens
    last = table[lanes, torch.clamp((had - 1) // T, min=0)].long()
    begun = had % T != 0
    # of a page's users the last in the list may keep it, if no other lane holds it
    users = torch.zeros_like(refs).index_add_(0, last[begun], torch.ones_like(last[begun], dtype=torch.int32))
    order = torch.where(begun, last, -1)
    by = torch.sort(order, stable=True)
    final = torch.ones_like(begun)
    final[by.indices[:-1]] = by.values[:-1] != by.values[1:]
    at = last.clamp(min=0)
    alone = final & (users[at] == refs[at])
    copy = begun & ~alone
    fresh = (now + T - 1) // T - (had + T - 1) // T
    need = copy.long() + fresh
    ids = torch.nonzero(refs == 0).view(-1)[:int(need.sum())]
    lane_of = torch.repeat_interleave(torch.arange(len(lanes), device=DEV), need)
    nth = torch.arange(ids.numel(), device=DEV) - (need.cumsum(0) - need)[lane_of]
    col = (had[lane_of] // T) + nth + torch.where(begun & ~copy, 1, 0)[lane_of]
    if bool(copy.any()):
        _copy_pages(s, ids[(need.cumsum(0) - need)[copy]], last[copy])
        refs.index_add_(0, last[copy], torch.full_like(last[copy], -1, dtype=torch.int32))
    table[lanes[lane_of], col] = ids.to(torch.int32)
    refs[ids] = 1
    s["length"][lanes] = now.to(torch.int32)


def _compact(s):
    """Live pages move into the lowest ids: those behind into the gaps, in order."""
    live = s["refs"] > 0
    n = int(live.sum())
    to = torch.nonzero(~live[:n]).view(-1)
    frm = torch.nonzero(live[n:]).view(-1) + n
    _copy_pages(s, to, frm)
    s["refs"][to] = s["refs"][frm]
    s["refs"][frm] = 0
    where = torch.arange(live.numel() + 1, dtype=torch.int32, device=DEV)
    where[-1] = -1
    where[frm] = to.to(torch.int32)
    s["table"].copy_(where[s["table"].long()])


# ---- what a pass cannot do without -----------------------------------------------------
def work(case):
    c = case
    es = 1 if c["dtype"] == "fp8" else 2
    H = c["kv_heads"]
    if c["kind"] == "attend":
        n, Hq = c["requests"], c["q_heads"]
        rows = c["tokens"] if n == 1 else c["tokens"] + (n - 1) * (c["tokens"] + 1) / 2
        kept = n * (c["own_lo"] + c["own_hi"]) / 2
        sh = c["shared"] * T if c["group"] else 0
        groups = -(-n // c["group"]) if c["group"] else 0
        seen = rows * (kept / n + sh - (rows / n - 1) / 2)
        return {"bytes": (kept + groups * sh) * H * 2 * D * es + rows * Hq * D * 4 + n * 4,
                "flops": 4.0 * D * Hq * max(seen, rows)}
    if c["kind"] == "append":
        rows = c["tokens"] + (c["requests"] - 1) * 0.75 * c["tokens"]
        q = c["q_heads"] * D * (6 if c["q32"] else 4)
        return {"bytes": rows * (q + 2 * H * D * (2 + es)), "flops": rows * 3.0 * c["rot"] * (c["q_heads"] + H)}
    page = c["layers"] * H * 2 * T * D * es
    mid = (c["lo"] + c["hi"]) / 2 / T + 0.5
    if c["kind"] == "fork":
        m = c["parents"] * c["children"]
        return {"bytes": m * (15 / 16) * 2 * page + m * mid * 12, "flops": 0.0}
    return {"bytes": c["requests"] * mid * (2 * page + 16), "flops": 0.0}


# ---- in 64 bits -------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attend":
        return _exact_attend(case, s)
    if case["kind"] == "append":
        return _exact_append(case, s)
    return _exact_pages(case, s)


def _exact_attend(c, s):
    n, H, G = c["requests"], c["kv_heads"], c["q_heads"] // c["kv_heads"]
    table, length = s["table"].cpu(), s["length"].cpu().tolist()
    new = s["new"].cpu().tolist()
    q = s["q"].double()
    out = torch.empty(q.shape, dtype=torch.float64, device=DEV)
    at = 0
    for r in range(n):
        size = length[r]
        ids = table[r, :-(-size // T)].long().to(DEV)
        visible = torch.arange(size - new[r], size, device=DEV).unsqueeze(1) >= torch.arange(size, device=DEV)
        visible = visible.repeat_interleave(G, 0)
        for h in range(H):
            kv = s["pool"][0].view(torch.uint8)[ids, h].view(s["pool"].dtype) if c["dtype"] == "fp8" else s["pool"][0][ids, h]
            kv = kv.double()
            if c["dtype"] == "fp8":
                kv = kv * s["scales"][0][ids, h].double().view(-1, 2, 1, 1)
            k, v = kv[:, 0].reshape(-1, D)[:size], kv[:, 1].reshape(-1, D)[:size]
            x = q[at:at + new[r], h * G:(h + 1) * G].reshape(-1, D)
            for i in range(0, x.shape[0], 1024):  # rows at a time
                p = torch.softmax((x[i:i + 1024] @ k.t() * D ** -0.5).masked_fill(~visible[i:i + 1024], -math.inf), 1)
                x[i:i + 1024] = p @ v
            out[at:at + new[r], h * G:(h + 1) * G] = x.view(new[r], G, D)
        at += new[r]
    return out


def _exact_append(c, s):
    r = c["rot"]
    phase = torch.polar(torch.full_like(s["inv_freq"], s["factor"]).expand(s["pos"].numel(), -1).contiguous(),
                        s["pos"].double().unsqueeze(1) * s["inv_freq"]).unsqueeze(1)

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


def _exact_pages(c, s):
    """The same calls on Python lists; the pool is moved page by page at the end."""
    table = [[i for i in row if i >= 0] for row in s["table"].tolist()]
    length, refs = s["length"].tolist(), s["refs"].tolist()
    holds = list(range(len(refs)))  # the page whose bytes page i has now

    def trim(lanes):
        for lane in lanes:
            for i in table[lane]:
                refs[i] -= 1
            table[lane], length[lane] = [], 0

    def reserve(lanes, tokens):
        free = [i for i, r in enumerate(refs) if r == 0]
        before, copies = holds[:], []
        for lane, t in zip(lanes, tokens):
            if length[lane] % T and refs[table[lane][-1]] > 1:
                copies.append((free[0], table[lane][-1]))
                refs[table[lane][-1]] -= 1
                table[lane][-1] = free.pop(0)
                refs[table[lane][-1]] = 1
            length[lane] += t
            while len(table[lane]) * T < length[lane]:
                table[lane].append(free.pop(0))
                refs[table[lane][-1]] = 1
        for to, frm in copies:
            holds[to] = before[frm]

    def compact():
        live = [i for i, r in enumerate(refs) if r]
        gaps = [i for i in range(len(live)) if not refs[i]]
        moved = dict(zip([i for i in live if i >= len(live)], gaps))
        for frm, to in moved.items():
            holds[to], refs[to], refs[frm] = holds[frm], refs[frm], 0
        for lane, row in enumerate(table):
            table[lane] = [moved.get(i, i) for i in row]

    if c["kind"] == "fork":
        src, dst = s["src"].tolist(), s["dst"].tolist()
        trim(dst)
        for a, b in zip(src, dst):
            for i in table[a]:
                refs[i] += 1
            table[b], length[b] = table[a][:], length[a]
        reserve(dst, s["one"].tolist())
    else:
        for half, grow in zip(s["halves"], s["grow"]):
            trim(half.tolist())
            compact()
            reserve(half.tolist(), grow.tolist())
    at = torch.tensor(holds, device=DEV)
    wide = s["table"].shape[1]
    rows = torch.tensor([row + [-1] * (wide - len(row)) for row in table], dtype=torch.int32)
    raw = s["pool"].view(torch.uint8) if c["dtype"] == "fp8" else s["pool"]
    pool = raw[:, at].view(s["pool"].dtype)
    out = [rows, torch.tensor(length, dtype=torch.int32), torch.tensor(refs, dtype=torch.int32), pool]
    return out + ([s["scales"][:, at]] if s["scales"] is not None else [])
