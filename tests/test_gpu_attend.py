"""Attention over the pages of a paged KV cache on the GPU against softmax
attention in float64.

Tolerance, for a row with weights p and values v, A = sum p |v|, S = the largest
sum over dims of |scale q k| of a token: the output's own rounding (half a step
u of its type); each weight rounded to the 16-bit type (u A); a score's fp32 sum
of 128 products, moving its weight and the weights' sum (2 x 130 x 2^-24 S A); the
fp32 exponentials, sums over n tokens and the joins of parts
((n / 8 + 64) x 2^-24 A)."""
import numpy as np
import pytest
import torch

import ferry_amd as F

pytestmark = pytest.mark.gpu

T, D = 16, 128
TORCH = {F.F32: torch.float32, F.F16: torch.float16, F.BF16: torch.bfloat16, F.FP8: torch.float8_e4m3fn}
U = {F.F32: 2.0 ** -24, F.F16: 2.0 ** -11, F.BF16: 2.0 ** -8, F.FP8: 2.0 ** -8}


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Case:
    """A batch: lens[r] tokens in request r's lane, the last new[r] of them its
    query rows; groups of (members, shared pages) take the requests in order."""

    def __init__(self, dt, Hq, H, lens, new=None, groups=(), layers=1, layer=0, seed=0, q_std=2.0, spare=3):
        self.dt, self.Hq, self.H, self.layer = dt, Hq, H, layer
        n = len(lens)
        self.lens = list(lens)
        self.new = [1] * n if new is None else list(new)
        g = self.g = torch.Generator(device="cuda").manual_seed(seed)
        pages = [-(-x // T) for x in lens]
        rng = np.random.default_rng(seed)
        total = sum(pages) + sum(s for _, s in groups) + spare
        ids = rng.permutation(total).tolist()
        lanes = rng.permutation(n + 2)[:n]
        wide = max(pages + [1]) + 2 + max([s for _, s in groups], default=0)
        table = np.full((n + 2, wide), -1, np.int32)
        at = 0
        for m, s in groups:  # a group's table starts with its shared pages
            common = [ids.pop() for _ in range(s)]
            for r in range(at, at + m):
                table[lanes[r], :s] = common
            at += m
        for r, x in enumerate(pages):
            have = int((table[lanes[r]] >= 0).sum())
            for i in range(have, x):
                table[lanes[r], i] = ids.pop()
        length = np.zeros(n + 2, np.int32)
        length[lanes] = lens
        shape = (layers, total, H, 2, T, D)
        x = torch.randn(shape, device="cuda", generator=g)
        scales = None
        if dt == F.FP8:
            x = (x * 96.0).clamp_(-448.0, 448.0)
            scales = 0.5 / 96.0 * (0.5 + torch.rand(shape[:3] + (2,), device="cuda", generator=g))
            scales[..., 1] *= 10.0 ** (2.0 * torch.rand(shape[:3], device="cuda", generator=g) - 1.0)
        else:
            x *= 0.5
        self.p = F.Pages(x.to(TORCH[dt]), ints(table), ints(length), scales=scales)
        self.qt = self.p.q_dtype
        self.rows = sum(self.new)
        self.q = (q_std * torch.randn((self.rows, Hq, D), device="cuda", generator=g)).to(self.qt)
        self.lanes = lanes
        self.groups = list(groups)
        self.start = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)

    def args(self, decode=None):
        decode = all(x == 1 for x in self.new) if decode is None else decode
        a = dict(lanes=ints(self.lanes))
        if not decode:
            a["q_start"] = ints(self.start)
        if self.groups:
            a["group_start"] = ints(np.concatenate([[0], np.cumsum([m for m, _ in self.groups])]))
            a["shared"] = ints([s for _, s in self.groups])
        return a

    def run(self, stream=None, **kw):
        a = {**self.args(), **kw}
        out = torch.full_like(self.q, 9.0)
        lse = torch.full((self.rows, self.Hq), 9.0, device="cuda")
        self.p.attend(self.layer, self.q, out, lse=lse, stream=stream, **a)
        torch.cuda.synchronize()
        self.p.check()
        return out, lse

    def tokens(self, r, head):
        """K and V of request r's tokens as float64 [len, 128]."""
        n = self.lens[r]
        ids = self.p.table[int(self.lanes[r]), :-(-n // T)].long()
        raw = self.p.pool.view(torch.uint8)[self.layer][ids, head]
        x = raw.view(TORCH[self.dt]).double()
        if self.dt == F.FP8:
            x = x * self.p.scales[self.layer][ids, head].double().view(-1, 2, 1, 1)
        return x[:, 0].reshape(-1, D)[:n], x[:, 1].reshape(-1, D)[:n]

    def check(self, out, lse, scale=D ** -0.5):
        G, u = self.Hq // self.H, U[self.dt]
        worst = 0.0
        for r, n in enumerate(self.lens):
            a, b = self.start[r], self.start[r + 1]
            for h in range(self.H):
                k, v = self.tokens(r, h)
                for row in range(a, b):
                    see = n - (b - a) + (row - a) + 1
                    o = out[row, h * G:(h + 1) * G].double()
                    e = lse[row, h * G:(h + 1) * G].double()
                    if see <= 0:
                        assert not torch.any(o) and torch.all(e == -np.inf)
                        continue
                    q = self.q[row, h * G:(h + 1) * G].double()
                    s = scale * (q @ k[:see].t())
                    want_e = torch.logsumexp(s, 1)
                    p = torch.exp(s - want_e.unsqueeze(1))
                    want, A = p @ v[:see], p @ v[:see].abs()
                    S = (abs(scale) * (q.abs() @ k[:see].abs().t())).max(1, keepdim=True).values
                    soft = (2 * 130 * S + see / 8 + 64) * 2.0 ** -24
                    bound = u * want.abs() + A * (u + soft) * (1 + u) + 2.0 ** -25
                    assert torch.all(torch.isfinite(o))
                    worst = max(worst, float(((o - want).abs() / bound).max()))
                    assert torch.all((e - want_e).abs() <= 2 * soft.squeeze(1) + 2.0 ** -23 * want_e.abs())
        assert worst <= 1.0, worst


DTYPES = [F.BF16, F.F16, F.FP8, F.F32]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("Hq,H", [(8, 2), (1, 1), (4, 4), (64, 8), (12, 3), (5, 1), (32, 1), (160, 2)])
def test_single_tokens(dt, Hq, H):
    c = Case(dt, Hq, H, [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 100, 129, 400], seed=Hq)
    c.check(*c.run())


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("groups,lens", [
    ([(5, 3)], [48, 49, 70, 200, 64]),
    ([(3, 1), (2, 9), (1, 4)], [17, 30, 90, 150, 290, 65]),
    ([(2, 4)], [70, 65, 9, 100]),            # the others outside every group
    ([(4, 0), (2, 2)], [7, 20, 33, 64, 32, 40]),  # nothing shared
    ([(3, 20)], [330, 10, 300]),             # a member that ends inside the shared pages
    ([(40, 7)], [112 + i for i in range(40)]),
])
def test_groups(dt, groups, lens):
    c = Case(dt, 8, 2, lens, groups=groups, seed=len(lens))
    out, lse = c.run()
    c.check(out, lse)
    if dt == F.F32:
        return
    # the same without the groups, within both sides' tolerance
    alone = c.args()
    alone.pop("group_start"), alone.pop("shared")
    a, b = torch.empty_like(c.q), torch.empty_like(lse)
    c.p.attend(c.layer, c.q, a, lse=b, **alone)
    c.check(a, b)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("Hq,H", [(8, 2), (3, 3), (16, 1)])
@pytest.mark.parametrize("new,lens,groups", [
    ([1, 2, 3, 5], [1, 40, 64, 130], []),
    ([33, 1, 70], [33, 90, 100], []),
    ([130], [300], []),
    ([7, 0, 4, 0], [7, 20, 64, 0], []),          # requests with no new tokens
    ([2, 5, 1, 30], [130, 131, 129, 170], [(4, 8)]),
    ([40, 20], [50, 100], [(2, 2)]),             # new tokens inside the shared pages
    ([64, 64, 9], [128, 192, 80], [(2, 4)]),
])
def test_several_tokens(dt, Hq, H, new, lens, groups):
    c = Case(dt, Hq, H, lens, new=new, groups=groups, seed=sum(new))
    c.check(*c.run())


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("n,len_,groups", [(1, 5000, []), (2, 3001, []), (9, 2100, [(9, 128)]), (33, 1500, [(30, 90)])])
def test_long_contexts(dt, n, len_, groups):
    c = Case(dt, 8, 2, [len_ + 7 * i for i in range(n)], groups=groups, seed=n)
    c.check(*c.run())


@pytest.mark.parametrize("dt", [F.BF16, F.FP8])
def test_many_requests(dt):
    rng = np.random.default_rng(1)
    lens = rng.integers(1, 60, 1500)
    c = Case(dt, 2, 1, lens, groups=[(int(m), 0) for m in [3] * 100] + [(1, 0)] * 7, seed=9)
    c.check(*c.run())


@pytest.mark.parametrize("dt", [F.BF16, F.F16, F.FP8])
def test_long_runs_of_wide_tiles(dt):
    # so much work that a workgroup takes many steps of a 128-row tile: page ids and fp8
    # scales come in windows of 16 steps.  A sample of requests and heads is checked.
    rng = np.random.default_rng(2)
    n, Hq, H = 64, 32, 8
    lens = [int(x) for x in rng.integers(900, 2300, n)]
    c = Case(dt, Hq, H, lens, new=[32 + int(x) for x in rng.integers(-20, 20, n)], seed=8)
    out, lse = c.run()
    for r in rng.permutation(n)[:10]:
        for h in rng.permutation(H)[:2]:
            near_rows(c, out, lse, int(r), int(h))


@pytest.mark.parametrize("dt", [F.BF16, F.F16, F.FP8])
def test_wide_tiles_of_few_pages(dt):
    # empty requests, rows that see nothing, tiles of 1 to 5 steps, a part of a tile's rows
    lens = [0, 3, 16, 40, 64, 65, 127, 128, 129, 200, 256, 300]
    new = [40, 40, 33, 40, 64, 20, 127, 100, 33, 33, 130, 70]
    c = Case(dt, 4, 1, lens, new, seed=3)
    lanes = c.lanes.copy()
    c.check(*c.run())
    c.lanes[4] = -1  # a request without a lane: its rows are empty
    c.lens[4] = 0
    out, lse = c.run()
    c.lanes = lanes
    c.check(out, lse)


def near_rows(c, out, lse, r, h, scale=D ** -0.5):
    """All rows of one request and kv head at once."""
    G, u, n = c.Hq // c.H, U[c.dt], c.lens[r]
    a, b = c.start[r], c.start[r + 1]
    k, v = c.tokens(r, h)
    q = c.q[a:b, h * G:(h + 1) * G].double()
    s = scale * (q @ k.t())
    S = abs(scale) * (q.abs() @ k.abs().t())
    see = n - (b - a) + torch.arange(b - a, device="cuda") + 1
    hidden = (torch.arange(n, device="cuda")[None] >= see[:, None])[:, None]
    s = s.masked_fill(hidden, -np.inf)
    S = S.masked_fill(hidden, 0.0).amax(-1, keepdim=True)
    want_e = torch.logsumexp(s, -1, keepdim=True)
    p = torch.exp(s - want_e)
    want, A = p @ v, p @ v.abs()
    soft = (2 * 130 * S + see[:, None, None] / 8 + 64) * 2.0 ** -24
    bound = u * want.abs() + A * (u + soft) * (1 + u) + 2.0 ** -25
    o = out[a:b, h * G:(h + 1) * G].double()
    worst = float(((o - want).abs() / bound).max())
    assert worst <= 1.0, (r, h, worst)
    e = lse[a:b, h * G:(h + 1) * G, None].double()
    assert torch.all((e - want_e).abs() <= 2 * soft + 2.0 ** -23 * want_e.abs())


def test_layers_scale_and_strides():
    c = Case(F.BF16, 6, 3, [20, 77], new=[3, 5], layers=3, layer=2, seed=4)
    big = torch.zeros((c.rows, 11, D), dtype=c.qt, device="cuda")
    big[:, 2:8] = c.q
    out = torch.zeros((6, c.rows + 1, D + 8), dtype=c.qt, device="cuda")[:, 1:, :D].transpose(0, 1)
    lse = torch.zeros((c.rows, 6), device="cuda")
    c.p.attend(2, big[:, 2:8], out, scale=0.2, lse=lse, **c.args())
    torch.cuda.synchronize()
    c.check(out, lse, scale=0.2)
    odd = torch.zeros(c.rows * 6 * D + 1, dtype=c.qt, device="cuda")[1:].view(c.rows, 6, D)
    odd.copy_(c.q)  # not 16-byte aligned
    odd_out = torch.zeros(c.rows * 6 * D + 1, dtype=c.qt, device="cuda")[1:].view(c.rows, 6, D)
    c.p.attend(2, odd, odd_out, scale=0.2, lse=lse, **c.args())
    torch.cuda.synchronize()
    c.check(odd_out, lse, scale=0.2)


@pytest.mark.parametrize("dt", DTYPES)
def test_negative_and_large_scores(dt):
    c = Case(dt, 4, 2, [40, 100, 1], seed=3, q_std=30.0)
    c.check(*c.run())
    c = Case(dt, 4, 2, [40, 100, 1], seed=3, q_std=1.0)
    c.q = -c.q.abs()
    c.check(*c.run(scale=-1.0), scale=-1.0)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_values_that_no_row_sees(dt, bad):
    """Behind a lane's end, and in pages no lane has, anything may stand."""
    c = Case(dt, 8, 2, [1, 17, 30, 47, 64, 130], new=[1, 2, 9, 1, 1, 40], groups=[(2, 0), (2, 1)], seed=2)
    want = c.run()
    pool = c.p.pool
    held = torch.zeros(pool.shape[1], T, dtype=torch.bool, device="cuda")
    for r, n in enumerate(c.lens):
        at = torch.arange(n, device="cuda")
        held[c.p.table[int(c.lanes[r])][at // T].long(), at % T] = True
    x = torch.full((1,), bad if dt != F.FP8 else float("nan"), device="cuda").to(TORCH[dt])
    raw, code = pool.view(torch.uint8), x.view(torch.uint8)
    es = code.numel()
    raw = raw.view(*pool.shape[:-1], D, es)
    mask = (~held)[None, :, None, None, :, None, None].expand(raw.shape)
    raw.copy_(torch.where(mask, code.view(1, 1, 1, 1, 1, 1, es), raw))
    got = c.run()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    c.check(*got)


@pytest.mark.parametrize("dt", [F.BF16, F.F16, F.F32])
@pytest.mark.parametrize("new,G", [(4, 1), (9, 4), (70, 4)])
def test_values_that_later_rows_see(dt, new, G):
    """A new token's NaN and infinity reach the rows from it on, not those before."""
    n = 100
    c = Case(dt, 2 * G, 2, [n, 40], new=[new, 1], seed=new)
    plain = c.run()[0]
    at = n - 3  # a token that the last rows see
    page = int(c.p.table[int(c.lanes[0]), at // T])
    c.p.pool[0, page, 0, 1, at % T, 5] = float("nan")
    c.p.pool[0, page, 0, 1, at % T, 77] = float("inf")
    c.p.pool[0, page, 1, 0, at % T, 3] = float("nan")
    out = c.run()[0]
    first = new - 3  # rows from here on see it
    assert torch.all(torch.isfinite(out[:first])) and torch.equal(out[new:], plain[new:])
    tail = out[first:new]
    assert torch.all(torch.isnan(tail[:, :G, 5])) and torch.all(tail[:, :G, 77] == float("inf"))
    assert torch.all(torch.isnan(tail[:, G:]))
    # Everything else is what a finite value there gives, within the tolerance above
    # (both are that near to the formula): the token's page may be summed in another
    # order, for the rows before it too.
    c.p.pool[0, page, 0, 1, at % T, 5] = c.p.pool[0, page, 0, 1, at % T, 77] = 0.0
    c.p.pool[0, page, 1, 0, at % T, 3] = 0.0
    fine, lse = c.run()
    c.check(torch.where(torch.isfinite(out), out, fine), lse)


def test_requests_without_a_lane_and_rows_behind_the_last():
    c = Case(F.BF16, 8, 2, [20, 30, 40, 50], new=[2, 3, 1, 2], seed=8)
    out, lse = c.run()
    c.check(out, lse)
    lanes = np.array(c.lanes).copy()
    lanes[1] = -1
    q = torch.cat([c.q, c.q])  # a padded batch
    got = torch.full_like(q, 3.0)
    c.p.attend(0, q, got, **{**c.args(), "lanes": ints(lanes)})
    torch.cuda.synchronize()
    c.p.check()
    assert torch.equal(got[:2], out[:2]) and not torch.any(got[2:5]) and torch.equal(got[5:8], out[5:8])
    assert torch.all(got[8:] == 3.0)


def test_what_is_out_of_range_is_reported():
    c = Case(F.F16, 4, 2, [20, 30], seed=8)
    for what in ("lane", "page", "length", "offsets"):
        a, keep = c.args(), None
        table, length = c.p.table.clone(), c.p.length.clone()
        if what == "lane":
            a["lanes"] = ints([int(c.lanes[0]), 99])
        elif what == "page":
            c.p.table[int(c.lanes[1]), 0] = 1 << 30
        elif what == "length":
            c.p.length[int(c.lanes[1])] = 16 * c.p.table.shape[1] + 5
            c.p.table[int(c.lanes[1])] = 0
        else:
            a["q_start"] = ints([0, 5, 1])
        out = torch.zeros_like(c.q)
        c.p.attend(0, c.q, out, **a)
        with pytest.raises(F.FerryError) as e:
            c.p.check()
        assert e.value.code == -3
        assert torch.all(torch.isfinite(out))
        c.p.table.copy_(table), c.p.length.copy_(length)
    c.check(*c.run())


def test_a_pool_past_four_gibibytes():
    H, P = 8, 70000
    c = Case(F.BF16, 16, H, [70, 33], seed=1)
    p = F.Pages.empty(1, H, P, 4, 8, F.BF16)
    n = c.p.pool.shape[1]
    p.pool[:, P - n:] = c.p.pool
    p.table[:, :c.p.table.shape[1]] = torch.where(c.p.table >= 0, c.p.table + (P - n), c.p.table)
    p.length.copy_(c.p.length)
    want = c.run()
    c.p = p
    got = c.run()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dt", [F.BF16, F.FP8])
def test_the_same_bits_in_every_call(dt):
    """On another stream, captured, and beside another graph of the same cache."""
    c = Case(dt, 8, 2, [900, 1000, 70, 2000], groups=[(2, 50)], seed=12)
    want, want_lse = c.run()
    c.check(want, want_lse)
    s = torch.cuda.Stream()
    got, lse = c.run(stream=s)
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
    d = Case(dt, 8, 2, [100, 33], new=[30, 4], seed=13)
    other = d.run()[0]
    a, b = c.args(), d.args()
    outs = [torch.empty_like(c.q), torch.empty_like(d.q)]
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    for g, k, kw, o in zip(graphs, (c, d), (a, b), outs):
        with torch.cuda.graph(g, stream=s):
            k.p.attend(0, k.q, o, **kw)
    t = torch.cuda.Stream()
    for i in range(4):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(t):
            graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], other)
        c.run()


@pytest.mark.parametrize("dt,new,groups", [(F.BF16, 1, ((6, 9),)), (F.FP8, 40, ()), (F.F16, 9, ((6, 9),)), (F.F32, 3, ())])
def test_the_output_in_the_queries_place(dt, new, groups):
    c = Case(dt, 8, 2, [300, 1500, 144, 200, 700, 160], [new] * 6, groups, seed=6)
    out, lse = c.run()
    q = c.q.clone()
    c.p.attend(0, q, q, **c.args())
    torch.cuda.synchronize()
    assert torch.equal(q, out)


def test_calls_on_two_streams_at_once():
    # one cache, two batches, each call with its own scratch
    a = Case(F.BF16, 16, 4, [900, 4000, 77, 2048], [50, 1, 77, 3], seed=9)
    q = torch.randn((4, 16, 128), device="cuda", generator=a.g).to(a.qt)
    lanes, first = ints(a.lanes), ints(a.start)
    want = [torch.empty_like(a.q), torch.empty_like(q)]
    a.p.attend(0, a.q, want[0], lanes, q_start=first)
    a.p.attend(0, q, want[1], lanes)
    torch.cuda.synchronize()
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[torch.zeros_like(x) for x in want] for _ in range(6)]
    torch.cuda.synchronize()
    for x, y in got:
        a.p.attend(0, a.q, x, lanes, q_start=first, stream=s[0])
        a.p.attend(0, q, y, lanes, stream=s[1])
    torch.cuda.synchronize()
    a.p.check()
    for x, y in got:
        assert torch.equal(x, want[0]) and torch.equal(y, want[1])


def test_no_rows():
    c = Case(F.BF16, 8, 2, [20], seed=1)
    e = c.q[:0]
    c.p.attend(0, e, e.clone(), ints([]))
    c.p.attend(0, e, e.clone(), ints(c.lanes), q_start=ints([0, 0]))
    c.p.check()


def test_refusals_on_the_host():
    c = Case(F.FP8, 8, 2, [20], seed=1)
    out = torch.empty_like(c.q)
    with pytest.raises(ValueError, match="dtype"):
        c.p.attend(0, c.q.float(), out, ints(c.lanes))
    with pytest.raises(ValueError, match="shape"):
        c.p.attend(0, c.q, out[:, :4], ints(c.lanes))
    with pytest.raises(F.FerryError, match="multiple"):
        c.p.attend(0, c.q[:, :7], out[:, :7], ints(c.lanes))
    with pytest.raises(F.FerryError, match="one token"):
        c.p.attend(0, torch.cat([c.q, c.q]), torch.cat([out, out]), ints(c.lanes))
    with pytest.raises(F.FerryError, match="layer"):
        c.p.attend(1, c.q, out, ints(c.lanes))
    with pytest.raises(ValueError, match="shared"):
        c.p.attend(0, c.q, out, ints(c.lanes), group_start=ints([0, 1]))


def test_the_queries_place_with_other_strides_is_refused():
    c = Case(F.BF16, 8, 2, [20, 30], seed=1)
    both = torch.zeros((2, 2, 8, 128), device="cuda", dtype=c.qt)
    with pytest.raises(F.FerryError, match="other strides"):
        c.p.attend(0, both[0], both[:, 0], ints(c.lanes))


@pytest.mark.parametrize("dt", [F.BF16, F.F16, F.FP8])
def test_wide_tiles_of_odd_strides_layers_and_scales(dt):
    # query and output rows that are not 16-byte aligned, another layer, a negative scale
    c = Case(dt, 10, 2, [200, 90, 1030], new=[60, 33, 41], layers=3, layer=2, seed=12, q_std=1.0)
    n = 10 * 128 + 3
    q = torch.zeros(c.rows * n + 1, device="cuda", dtype=c.qt)[1:].view(c.rows, n)[:, :1280].unflatten(1, (10, 128))
    out = torch.full((c.rows * n + 5,), 3.0, device="cuda", dtype=c.qt)
    rows = out[5:].view(c.rows, n)
    q.copy_(c.q)
    lse = torch.empty((c.rows, 10), device="cuda")
    a = c.args()
    c.p.attend(2, q, rows[:, :1280].unflatten(1, (10, 128)), lse=lse, scale=-0.11, **a)
    torch.cuda.synchronize()
    c.p.check()
    c.check(rows[:, :1280].unflatten(1, (10, 128)), lse, scale=-float(np.float32(0.11)))
    assert torch.all(rows[:, 1280:] == 3.0) and torch.all(out[:5] == 3.0)  # between the rows: left


def test_wide_tiles_past_four_gibibytes():
    H, P = 8, 70000
    c = Case(F.F16, 16, H, [170, 133], new=[80, 40], seed=1)
    p = F.Pages.empty(1, H, P, 4, 16, F.F16)
    n = c.p.pool.shape[1]
    p.pool[:, P - n:] = c.p.pool
    p.table[:, :c.p.table.shape[1]] = torch.where(c.p.table >= 0, c.p.table + (P - n), c.p.table)
    p.length.copy_(c.p.length)
    want = c.run()
    c.p = p
    got = c.run()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dt", [F.BF16, F.FP8])
def test_wide_tiles_with_pages_out_of_range(dt):
    # they are read as page 0 and reported
    c = Case(dt, 4, 1, [300, 120], new=[50, 40], seed=5)
    lane = int(c.lanes[0])
    kept = c.p.table[lane].clone()
    c.p.table[lane, 3] = c.p.pool.shape[1]
    c.p.table[lane, 7] = -5
    out, lse = torch.full_like(c.q, 9.0), torch.empty((c.rows, 4), device="cuda")
    c.p.attend(0, c.q, out, lse=lse, **c.args())
    with pytest.raises(F.FerryError, match="RANGE"):
        c.p.check()
    c.p.table[lane] = kept
    c.p.table[lane, 3] = c.p.table[lane, 7] = 0
    c.check(out, lse)


@pytest.mark.parametrize("dt", [F.BF16, F.FP8])
def test_several_values_that_later_rows_see(dt):
    # NaN in steps next to each other and apart, in 128-row tiles that one workgroup takes whole
    n, H, new = 64, 8, 500
    lens = [int(x) for x in np.random.default_rng(1).integers(560, 700, n)]
    c = Case(dt, H, H, lens, new=[new] * n, seed=4)
    nan = torch.full((1,), float("nan"), device="cuda").to(TORCH[dt])
    raw = c.p.pool.view(torch.uint8).view(*c.p.pool.shape[:-1], D, nan.element_size())
    spots = []
    for r, h, back, d in [(3, 0, 130, 5), (3, 0, 129, 9), (3, 0, 60, 5), (3, 0, 2, 64), (17, 5, 300, 127),
                          (17, 5, 240, 0), (17, 5, 1, 1), (40, 7, 499, 33), (40, 7, 420, 33), (40, 7, 380, 2)]:
        t = lens[r] - back
        at = (0, int(c.p.table[int(c.lanes[r]), t // T]), h, 1, t % T, d)
        spots.append((r, h, back, d, at, raw[at].clone()))
        raw[at] = nan.view(torch.uint8)
    out, lse = c.run()
    for *_, at, was in spots:
        raw[at] = was
    fine = c.run()[0]
    bad = torch.zeros_like(out, dtype=torch.bool)
    for r, h, back, d, *_ in spots:
        bad[c.start[r] + new - back:c.start[r + 1], h, d] = True
    assert torch.equal(torch.isnan(out), bad)
    out = torch.where(bad, fine, out)
    for r, h in [(3, 0), (17, 5), (40, 7), (3, 1), (41, 7), (63, 2)]:
        near_rows(c, out, lse, r, h)


@pytest.mark.parametrize("dt", [F.BF16, F.F16, F.FP8])
@pytest.mark.parametrize("new", [1, 2])
def test_wide_groups_whose_members_end_within_the_shared_pages(dt, new):
    lens = [700, 100, 481, 33, 480, 16, 1, 479, 512, 2, 640, 320, 0, 496, 15, 17] * 3
    c = Case(dt, 8, 2, lens, new=[new] * len(lens), groups=[(16, 30), (31, 30), (1, 2)], seed=new)
    c.check(*c.run())


def test_more_groups_than_are_looked_up_in_lds():
    n = 1300  # 650 groups of two, the last requests in none
    rng = np.random.default_rng(5)
    lens = [int(x) for x in rng.integers(1, 60, n + 7)]
    c = Case(F.BF16, 2, 1, lens, groups=[(2, int(x)) for x in rng.integers(0, 3, n // 2)], seed=2)
    c.check(*c.run())


@pytest.mark.parametrize("dt", [F.BF16, F.F16, F.FP8])
@pytest.mark.parametrize("rows", [33, 64, 96, 128])
def test_the_first_steps_of_partly_filled_wide_tiles(dt, rows):
    # Wavefronts without rows go ahead of those whose products read the first step's K, and
    # load what comes after it.  1 to 5 steps a tile, whole ones and ends; the same bits in
    # every call.
    lens = [max(rows, n) for n in (1, 64, 65, 100, 128, 129, 192, 200, 256, 257, 320)]
    c = Case(dt, 8, 8, lens, [rows] * len(lens), seed=rows)
    want, lse = c.run()
    for r in range(len(lens)):
        for h in range(8):
            near_rows(c, want, lse, r, h)
    for _ in range(20):
        got = c.run()
        assert torch.equal(got[0], want) and torch.equal(got[1], lse)


def spoil(c, at):
    """NaN and (not fp8) infinity in V of the tokens at[r] of requests r, kv head 0, dims 5
    and 77; returns what undoes it."""
    dims = [(5, float("nan"))] + ([] if c.dt == F.FP8 else [(77, float("inf"))])
    es = c.p.pool.element_size()
    raw = c.p.pool.view(torch.uint8).view(*c.p.pool.shape[:-1], D, es)
    was = raw.clone()
    for r, t in at.items():
        page = int(c.p.table[int(c.lanes[r]), t // T])
        for d, x in dims:
            raw[c.layer, page, 0, 1, t % T, d] = \
                torch.full((1,), x, device="cuda").to(TORCH[c.dt]).view(torch.uint8)
    return lambda: raw.copy_(was)


def check_spoiled(c, out, lse, at, fine):
    """Rows that see token at[r] have its NaN and infinity, and nothing else of them: all
    else is what a finite value there gives, which `fine` has in the spoiled places."""
    G = c.Hq // c.H
    nan, inf = torch.zeros_like(out, dtype=torch.bool), torch.zeros_like(out, dtype=torch.bool)
    for r, t in at.items():
        a, b = int(c.start[r]), int(c.start[r + 1])
        first = max(a, b - (c.lens[r] - t))
        nan[first:b, :G, 5] = True
        inf[first:b, :G, 77] = c.dt != F.FP8
    assert torch.equal(torch.isnan(out), nan)
    assert torch.equal(out == float("inf"), inf)
    c.check(torch.where(nan | inf, fine, out), lse)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("new,G", [(1, 1), (8, 4), (5, 6)])
def test_values_not_finite_in_every_page(dt, new, G):
    # a request for each page of lanes of 16, 32, 100 and 700 tokens, all in one call
    lens = [n for n in (16, 32, 100, 700) for _ in range(-(-n // T))]
    where = [p for n in (16, 32, 100, 700) for p in range(-(-n // T))]
    c = Case(dt, 2 * G, 2, lens, new=[new] * len(lens), seed=new)
    fine = c.run()[0]
    at = {r: min(n - 1, T * p + 9) for r, (n, p) in enumerate(zip(lens, where))}
    undo = spoil(c, at)
    out, lse = c.run()
    # ... and a call for each, whose work is cut into runs of a step
    one, one_lse = torch.zeros_like(out), torch.zeros_like(lse)
    for r in range(len(lens)):
        a, b = int(c.start[r]), int(c.start[r + 1])
        c.p.attend(0, c.q[a:b], one[a:b], ints(c.lanes[r:r + 1]), q_start=ints([0, new]), lse=one_lse[a:b])
    torch.cuda.synchronize()
    undo()
    check_spoiled(c, out, lse, at, fine)
    check_spoiled(c, one, one_lse, at, fine)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("new,G", [(1, 4), (2, 5), (3, 16)])
def test_values_not_finite_in_every_shared_page(dt, new, G):
    # a group for each shared page, 3 members each; the last member of some ends within them
    shared = [1, 2, 2] + [7] * 7 + [40] * 5
    where = [0, 0, 1] + list(range(7)) + [0, 13, 26, 38, 39]
    lens, at = [], {}
    for s, p in zip(shared, where):
        n = len(lens)
        lens += [T * s + 30, T * s, max(new, T * s - 21)]
        for r in range(n, n + 3):
            if lens[r] > T * p + 9:
                at[r] = T * p + 9
    c = Case(dt, 2 * G, 2, lens, new=[new] * len(lens), groups=[(3, s) for s in shared], seed=new)
    fine = c.run()[0]
    undo = spoil(c, at)
    out, lse = c.run()
    undo()
    check_spoiled(c, out, lse, at, fine)


def behind_a_free_page(c):
    """The same case with a page in front that no lane holds."""
    p = c.p
    c.p = F.Pages(torch.cat([p.pool[:, :1].view(torch.uint8), p.pool.view(torch.uint8)], 1).view(p.pool.dtype),
                  torch.where(p.table >= 0, p.table + 1, p.table), p.length,
                  scales=torch.cat([p.scales[:, :1], p.scales], 1))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("new,groups", [([1, 2, 9, 1, 7, 8, 3], [(2, 0), (2, 1)]),
                                        ([33, 40, 64, 128, 150, 35, 9], []),
                                        ([9, 9, 12, 9, 9, 9, 9], [(5, 2), (2, 5)])])
def test_scales_that_no_row_sees(new, groups, bad):
    # of pages that no lane holds, page 0 among them, and of a lane's pages behind its end
    c = Case(F.FP8, 8, 2, [33, 40, 64, 130, 150, 81, 95], new=new, groups=groups, seed=2, spare=40)
    behind_a_free_page(c)
    want = c.run()
    held = torch.zeros(c.p.pool.shape[1], dtype=torch.bool, device="cuda")
    for r, n in enumerate(c.lens):
        row = c.p.table[int(c.lanes[r])]
        held[row[:-(-n // T)].long()] = True
        more = (~held).nonzero()[-1 - r]  # a page reserved behind them
        row[-(-n // T)] = more[0]
    c.p.scales[:, ~held] = bad
    got = c.run()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    c.check(*got)


@pytest.mark.parametrize("which,bad", [(0, float("nan")), (1, float("nan")), (1, float("inf"))])
@pytest.mark.parametrize("new,G", [(4, 4), (8, 4), (30, 1), (70, 4), (300, 2)])
def test_scales_that_later_rows_see(new, G, which, bad):
    # of K (which 0) or V: nothing of them in the rows before their page's first token
    n = 400
    c = Case(F.FP8, 2 * G, 2, [n, 60, n], new=[new, 1, new], seed=new)
    fine, lse = c.run()
    c.check(fine, lse)
    keep = c.p.scales.clone()
    for r, back in ((0, 3), (2, new // 2), (2, new - 1)):
        page = c.p.table[int(c.lanes[r]), (n - back) // T]
        c.p.scales[0, page, 0, which] = bad
    out, got_lse = c.run()
    c.p.scales.copy_(keep)
    sees = torch.zeros_like(out, dtype=torch.bool)
    for r, back in ((0, 3), (2, new - 1)):
        first = (n - back) // T * T  # the page's first token
        a, b = int(c.start[r]), int(c.start[r + 1])
        sees[max(a, b - (n - first)):b, :G] = True
    assert torch.all(torch.isnan(out[sees]) if bad != bad else ~torch.isfinite(out[sees]))
    assert torch.all(torch.isfinite(out[~sees]))
    hit = sees[:, :, 0]
    c.check(torch.where(sees, fine, out), torch.where(hit, lse, got_lse))


@pytest.mark.parametrize("shared,new", [(7, 1), (7, 3), (30, 1), (30, 3)])
def test_scales_in_shared_pages_that_some_members_see(shared, new):
    lens = [16 * shared + 20, 16 * shared - 17, 16 * shared - 40, 16 * shared, new, 40]
    c = Case(F.FP8, 16, 2, lens, new=[new] * 6, groups=[(5, shared)], seed=shared)
    fine, lse = c.run()
    page = shared - 2  # tokens that the members of 16 (shared - 2) or fewer do not see
    c.p.scales[0, c.p.table[int(c.lanes[0]), page], 0, 1] = float("nan")
    out, _ = c.run()
    sees = torch.zeros_like(out, dtype=torch.bool)
    for r, m in enumerate(lens[:5]):
        a, b = int(c.start[r]), int(c.start[r + 1])
        sees[max(a, b - max(0, m - 16 * page)):b, :8] = True
    assert sees.any() and not sees.all() and torch.equal(torch.isnan(out), sees)
    c.check(torch.where(sees, fine, out), lse)


@pytest.mark.parametrize("dt", [F.F16, F.BF16])
@pytest.mark.parametrize("n,new", [(1 << 18, 1), (1 << 17, 128)])
def test_a_long_tail_of_small_weights(dt, n, new):
    # A token of weight 1 at the start of what each maximum is taken over (the pages of a
    # wavefront, or all), all others 2^-25.5, which fp16 does not hold: together they are
    # 2^-8.5 of it or more, and their values are of one sign and most of the output.  As many
    # requests of the lane as there are workgroups, so that one takes the whole lane.
    reqs, tops = 512, 4 if new == 1 else 1
    g = torch.Generator(device="cuda").manual_seed(new)
    pool = torch.zeros((1, n // T, 1, 2, T, D), dtype=TORCH[dt], device="cuda")
    pool[0, :, 0, 1] = -(0.5 + torch.rand((n // T, T, D), device="cuda", generator=g)).to(TORCH[dt])
    pool[0, :tops, 0, 0, 0, 0] = 12.5
    pool[0, :tops, 0, 1, 0] = 2.0 ** -6
    p = F.Pages(pool, torch.arange(n // T, dtype=torch.int32, device="cuda")[None], ints([n]))
    q = torch.zeros((reqs * new, 1, D), dtype=TORCH[dt], device="cuda")
    q[:, 0, 0] = 16.0
    out, lse = torch.empty_like(q), torch.empty((reqs * new, 1), device="cuda")
    p.attend(0, q, out, ints([0] * reqs), q_start=ints([new * i for i in range(reqs + 1)]), lse=lse)
    torch.cuda.synchronize()
    p.check()
    k, v = pool[0, :, 0, 0].reshape(n, D).double(), pool[0, :, 0, 1].reshape(n, D).double()
    s = D ** -0.5 * (k[:, 0] * 16.0)
    u = U[dt]
    for row in range(0, reqs * new, max(1, reqs * new // 50) + 1):
        see = n - new + row % new + 1
        want_e = torch.logsumexp(s[:see], 0)
        w = torch.exp(s[:see] - want_e)
        want, A = w @ v[:see], w @ v[:see].abs()
        soft = (2 * 130 * float(s.max()) + see / 8 + 64) * 2.0 ** -24
        # the bound above, and half of fp16's smallest step per weight: 2^-32 of the largest one
        bound = u * want.abs() + A * (u + soft) * (1 + u) + 2.0 ** -25 + see * 2.0 ** -32 / tops * 1.5
        assert torch.all((out[row, 0].double() - want).abs() <= bound)
        assert abs(float(lse[row, 0]) - float(want_e)) <= 2 * soft + 2.0 ** -23 * abs(float(want_e))


def test_more_rows_than_a_launch_joins():
    # A launch of the join has fewer than 2^32 threads.  Two requests of more than 2^28 rows
    # together: the first one's rows see next to nothing, the second's are the last and see so
    # much that several workgroups share them.  In the queries' place: 69 GB.
    Hq, n, len_ = 128, (1 << 21) + 1000, 1 << 22
    g = torch.Generator(device="cuda").manual_seed(3)
    pool = torch.randn((1, len_ // T, 1, 2, T, D), device="cuda", generator=g)
    pool[:, :, :, 1] += 1.0
    pool = pool.to(torch.bfloat16)
    p = F.Pages(pool, torch.arange(len_ // T, dtype=torch.int32, device="cuda").repeat(2, 1), ints([40, len_]))
    q = torch.full((n, Hq, D), 3.0, dtype=torch.bfloat16, device="cuda")
    last = n - 7  # the rest: behind the last request
    rows = torch.randn((Hq, D), device="cuda", generator=g).to(torch.bfloat16)
    q[last - 1] = rows
    lse = torch.zeros((n, Hq), device="cuda")
    p.attend(0, q, q, ints([0, 1]), q_start=ints([0, last - 1, last]), lse=lse)
    torch.cuda.synchronize()
    p.check()
    k, v = pool[0, :, 0, 0].reshape(-1, D).float(), pool[0, :, 0, 1].reshape(-1, D).float()
    for h in range(0, Hq, 9):
        s = (D ** -0.5 * (k @ rows[h].float())).double()
        want_e = torch.logsumexp(s, 0)
        w = torch.exp(s - want_e)
        want, A = (w[None].float() @ v)[0].double(), (w[None].float() @ v.abs())[0].double()
        # the bound of this file; the products above are fp32 too
        S = float((D ** -0.5 * (k.abs() @ rows[h].float().abs())).max())
        soft = 2 * (2 * 130 * S + len_ / 8 + 64) * 2.0 ** -24
        assert torch.all((q[last - 1, h].double() - want).abs() <= 2.0 ** -8 * (want.abs() + 2 * A) + A * soft)
        assert abs(float(lse[last - 1, h] - want_e)) <= 2 * soft + 2.0 ** -23 * float(want_e)
    assert not q[:last - 41].any() and torch.all(q[last:] == 3.0)
    assert torch.all(torch.isfinite(q[last - 41:last - 1])) and torch.all(lse[last - 41:last - 1] > -np.inf)
