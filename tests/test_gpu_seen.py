"""Attention over pages where a row sees a part of what is before it (a sliding
window with sinks, a tree of drafted tokens) against softmax attention in
float64 over the tokens that it sees.

Tolerance: that of attention over all of a lane (test_gpu_attend), with the number
of tokens that the row sees."""
import ctypes as C

import numpy as np
import pytest
import torch

import ferry_amd as F

from test_gpu_attend import D, DTYPES, T, TORCH, U, Case, ints

pytestmark = pytest.mark.gpu


def tree_of(rng, n, back=5, roots=False):
    """Parents of n drafted tokens and, as [n, n], who sees whom."""
    parent = [-1] + [max(0, i - int(rng.integers(1, back + 1))) for i in range(1, n)]
    if roots:
        parent = [-1 if rng.random() < 0.2 else p for p in parent]
    sees = np.zeros((n, n), bool)
    for i, p in enumerate(parent):
        if p >= 0:
            sees[i] = sees[p]
        sees[i, i] = True
    return parent, sees


def words_of(masks, words):
    """Bits of all rows' masks as an int64 tensor [rows, words]."""
    out = []
    for m in masks:
        wide = np.zeros((m.shape[0], 64 * words), np.uint8)
        wide[:, :m.shape[1]] = m
        out.append(np.packbits(wide, axis=1, bitorder="little").view(np.int64).reshape(m.shape[0], words))
    return torch.from_numpy(np.concatenate(out)).cuda()


class Seen(Case):
    """A batch whose rows see `masks` of their request's new tokens, or a window."""

    def __init__(self, dt, Hq, H, lens, new=None, window=0, sinks=0, masks=None, words=None, **kw):
        super().__init__(dt, Hq, H, lens, new, **kw)
        self.window, self.sinks, self.masks = window, sinks, masks
        self.words = None
        if masks is not None:
            self.words = words_of(masks, words or -(-max(self.new) // 64))

    def args(self, decode=None):
        return dict(super().args(decode), window=self.window, sinks=self.sinks, tree=self.words)

    def visible(self, r):
        """[rows of request r, tokens of its lane]"""
        size, n = self.lens[r], self.new[r]
        base = size - n
        tok = np.arange(size)
        if self.masks is None:
            place = base + np.arange(n)
            drafted = np.zeros((n, size), bool)
            see = tok <= place[:, None]
        else:
            drafted = np.zeros((n, size), bool)
            drafted[:, base:] = self.masks[r]
            see = drafted | (tok < base)
            place = base - 1 + self.masks[r].sum(1)
        if self.window:
            see &= drafted | (tok > place[:, None] - self.window) | (tok < self.sinks)
        return see

    def check(self, out, lse, scale=D ** -0.5):
        G, u = self.Hq // self.H, U[self.dt]
        worst = 0.0
        for r in range(len(self.lens)):
            a, b = self.start[r], self.start[r + 1]
            if a == b:
                continue
            see = torch.from_numpy(self.visible(r)).cuda().repeat_interleave(G, 0)
            some = see.any(1)
            count = see.sum(1, keepdim=True)
            for h in range(self.H):
                k, v = self.tokens(r, h)
                o = out[a:b, h * G:(h + 1) * G].double().reshape(-1, D)
                e = lse[a:b, h * G:(h + 1) * G].double().reshape(-1)
                assert not torch.any(o[~some]) and torch.all(e[~some] == -np.inf)
                if not some.any():
                    continue
                q = self.q[a:b, h * G:(h + 1) * G].double().reshape(-1, D)
                seen_by_any = see.any(0)
                k, v, m = k[seen_by_any], v[seen_by_any], see[some][:, seen_by_any]
                q, o, e, n = q[some], o[some], e[some], count[some]
                s = (scale * (q @ k.t())).masked_fill(~m, -np.inf)
                want_e = torch.logsumexp(s, 1)
                p = torch.exp(s - want_e.unsqueeze(1))
                want, A = p @ v, p @ v.abs()
                S = (abs(scale) * (q.abs() @ k.abs().t())).masked_fill(~m, 0.0).max(1, keepdim=True).values
                soft = (2 * 130 * S + n / 8 + 64) * 2.0 ** -24
                bound = u * want.abs() + A * (u + soft) * (1 + u) + 2.0 ** -25
                assert torch.all(torch.isfinite(o))
                worst = max(worst, float(((o - want).abs() / bound).max()))
                assert torch.all((e - want_e).abs() <= 2 * soft.squeeze(1) + 2.0 ** -23 * want_e.abs())
        assert worst <= 1.0, worst


LENS = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 100, 129, 400]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("Hq,H", [(8, 2), (1, 1), (64, 8), (160, 2)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (2, 1), (16, 4), (17, 16), (40, 70), (64, 0), (100, 17), (5000, 4)])
def test_windows_of_single_tokens(dt, Hq, H, window, sinks):
    c = Seen(dt, Hq, H, LENS, window=window, sinks=sinks, seed=window)
    c.check(*c.run())


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("Hq,H", [(8, 2), (3, 3)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (33, 4), (64, 130), (150, 1), (129, 64)])
@pytest.mark.parametrize("new,lens", [
    ([2, 1, 3, 2], [2, 40, 300, 17]), ([5, 0, 7, 1], [5, 9, 500, 100]), ([70, 33, 1, 128], [70, 600, 700, 300]),
])
def test_windows_of_several_tokens(dt, Hq, H, window, sinks, new, lens):
    c = Seen(dt, Hq, H, lens, new, window=window, sinks=sinks, seed=window)
    c.check(*c.run())


@pytest.mark.parametrize("dt", [F.BF16, F.F16, F.FP8])
@pytest.mark.parametrize("window,sinks", [(1000, 4), (257, 0), (640, 200)])
def test_windows_of_long_prompts(dt, window, sinks):
    c = Seen(dt, 8, 2, [1500, 2300, 700], [900, 300, 700], window=window, sinks=sinks, seed=1)
    c.check(*c.run())


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("new", [1, 9, 40])
def test_windows_over_long_contexts(dt, new):
    c = Seen(dt, 8, 2, [9000, 5000, 4111], [new] * 3, window=4096, sinks=4, seed=new)
    c.check(*c.run())


def test_a_window_that_holds_everything_is_causal():
    for new in (1, 6, 50):
        a = Seen(F.BF16, 8, 2, [700, 90, 64], [new] * 3, seed=2)
        out, lse = a.run()
        a.window, a.sinks = 2 ** 31 - 1, 2 ** 31 - 1
        a.check(*a.run())
        got, _ = a.run()
        assert torch.all((got.float() - out.float()).abs() <= 2.0 ** -6 * out.float().abs() + 2.0 ** -8)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("Hq,H", [(8, 2), (1, 1), (64, 8)])
@pytest.mark.parametrize("new,lens", [
    ([1, 2, 3, 4], [1, 2, 40, 300]), ([8, 5, 8], [8, 77, 500]), ([17, 64, 33], [17, 128, 613]),
    ([65, 130, 2], [65, 333, 90]), ([200], [1000]),
])
def test_trees(dt, Hq, H, new, lens):
    rng = np.random.default_rng(len(new))
    masks = [tree_of(rng, n)[1] for n in new]
    c = Seen(dt, Hq, H, lens, new, masks=masks, seed=lens[0])
    c.check(*c.run())


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("new,lens", [([6, 3, 1, 9], [6, 90, 1, 25]), ([40, 70, 128], [40, 300, 128])])
def test_any_bits(dt, new, lens):
    # bits that no tree has: rows of none, of later tokens only, of all; and bits behind
    # the request's tokens, which do not count
    rng = np.random.default_rng(3)
    masks = [rng.random((n, n)) < 0.3 for n in new]
    for m in masks:
        m[0] = False
        m[-1] = True
    masks[0][1] = np.arange(new[0]) == new[0] - 1
    c = Seen(dt, 8, 2, lens, new, masks=masks, words=3, seed=5)
    full = [np.concatenate([m, np.ones((m.shape[0], 192 - m.shape[1]), bool)], 1) for m in masks]
    c.words = words_of(full, 3)
    c.check(*c.run())


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 2), (20, 17), (100, 4), (64, 64)])
@pytest.mark.parametrize("new,lens", [([4, 7, 1], [4, 77, 300]), ([33, 64, 100], [50, 400, 731])])
def test_trees_in_windows(dt, window, sinks, new, lens):
    rng = np.random.default_rng(window)
    masks = [tree_of(rng, n, back=3, roots=True)[1] for n in new]
    masks[-1][0] = False  # a row of no drafts: its window ends before them
    c = Seen(dt, 8, 2, lens, new, window=window, sinks=sinks, masks=masks, seed=7)
    c.check(*c.run())


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("groups,new", [([(3, 9)], [4, 7, 1, 12]), ([(2, 3), (2, 20)], [5, 1, 30, 2]), ([(4, 5)], [1, 1, 1, 1])])
def test_trees_of_groups(dt, groups, new):
    # forked lanes with trees of their own behind what they share
    rng = np.random.default_rng(4)
    masks = [tree_of(rng, n)[1] for n in new]
    shared = [s for m, s in groups for _ in range(m)] + [0] * 4
    lens = [shared[i] * T + 5 * i + new[i] for i in range(4)]
    c = Seen(dt, 8, 2, lens, new, masks=masks, groups=groups, seed=8)
    c.check(*c.run())


@pytest.mark.parametrize("dt", DTYPES)
def test_shared_pages_that_reach_into_the_drafts(dt):
    # a group may name more pages than all members hold before their drafts
    rng = np.random.default_rng(6)
    new = [5, 20, 3]
    masks = [tree_of(rng, n)[1] for n in new]
    c = Seen(dt, 8, 2, [6 * T, 6 * T, 6 * T], new, masks=masks, groups=[(3, 6)], seed=9)
    c.check(*c.run())


@pytest.mark.parametrize("dt", DTYPES)
def test_long_contexts_with_trees(dt):
    rng = np.random.default_rng(2)
    new = [16, 64]
    masks = [tree_of(rng, n)[1] for n in new]
    c = Seen(dt, 8, 2, [5000, 3001], new, masks=masks, seed=3)
    c.check(*c.run())


@pytest.mark.parametrize("dt", [F.BF16, F.FP8])
def test_many_requests(dt):
    rng = np.random.default_rng(9)
    n = 700
    lens = rng.integers(1, 90, n).tolist()
    c = Seen(dt, 4, 1, lens, window=20, sinks=3, seed=1)
    c.check(*c.run())
    new = [int(rng.integers(1, min(x, 9) + 1)) for x in lens]
    masks = [tree_of(rng, x)[1] for x in new]
    c = Seen(dt, 4, 1, lens, new, masks=masks, seed=2)
    c.check(*c.run())


@pytest.mark.parametrize("dt", [F.BF16, F.FP8])
@pytest.mark.parametrize("n", [90, 600])
def test_many_requests_of_wide_tiles(dt, n):
    rng = np.random.default_rng(n)
    new = rng.integers(20, 50, n).tolist()
    lens = [int(x + rng.integers(0, 150)) for x in new]
    c = Seen(dt, 4, 1, lens, new, masks=[tree_of(rng, x)[1] for x in new], seed=3)
    c.check(*c.run())
    c = Seen(dt, 4, 1, lens, new, window=40, sinks=3, seed=4)
    c.check(*c.run())


def spoil(c, dt, value, rows):
    """Put `value` into K and V of tokens: rows of (request, token)."""
    raw = c.p.pool.view(torch.uint8) if dt == F.FP8 else c.p.pool
    x = torch.tensor(value, device="cuda").to(TORCH[dt])
    x = x.view(torch.uint8) if dt == F.FP8 else x
    for r, t in rows:
        page = int(c.p.table[int(c.lanes[r]), t // T])
        raw[c.layer, page, :, :, t % T] = x


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("new,G", [(1, 4), (5, 6), (40, 4)])
def test_values_that_no_row_sees(dt, bad, new, G):
    if dt == F.FP8 and bad == float("inf"):
        bad = float("nan")
    # before the window, between the sinks and it
    c = Seen(dt, 2 * G, 2, [400, 130], [new, new], window=60, sinks=5, seed=3)
    hidden = [(r, t) for r in range(2) for t in np.flatnonzero(~c.visible(r).any(0))]
    assert len(hidden) > 100
    want = [x.clone() for x in c.run()]
    spoil(c, dt, bad, hidden)
    got = c.run()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("new,G", [(6, 1), (9, 4), (70, 4)])
def test_values_that_some_rows_see(dt, bad, new, G):
    """Rows that do not see them have their result all the same."""
    if dt == F.FP8 and bad == float("inf"):
        bad = float("nan")
    rng = np.random.default_rng(5)
    for kind in ("window", "tree", "both"):
        kw = {}
        if kind != "tree":
            kw.update(window=30, sinks=3)
        if kind != "window":
            kw["masks"] = [tree_of(rng, new, back=3)[1] for _ in range(2)]
        c = Seen(dt, 2 * G, 2, [300, 99], [new, new], seed=4, **kw)
        places = [(0, 300 - new + 1), (0, 271 - new), (1, 98)]
        out, lse = c.run()
        before = c.p.pool.clone()
        spoil(c, dt, bad, places)
        got, got_lse = c.run()
        c.p.pool.copy_(before)
        clean = torch.ones(c.rows, dtype=torch.bool, device="cuda")
        for r, t in places:
            hit = torch.from_numpy(np.flatnonzero(c.visible(r)[:, t])).cuda() + int(c.start[r])
            clean[hit] = False
        assert clean.any() and not clean.all()
        assert torch.all(torch.isnan(got[~clean].float()))
        # the others are within the tolerance of the formula without those tokens
        clean = clean.view(-1, 1)
        c.check(torch.where(clean.unsqueeze(2), got, out), torch.where(clean, got_lse, lse))


@pytest.mark.parametrize("which,bad", [(0, float("nan")), (1, float("nan")), (1, float("inf"))])
@pytest.mark.parametrize("new,G", [(1, 4), (8, 4), (40, 4)])
def test_scales_of_pages_that_no_row_sees(new, G, which, bad):
    c = Seen(F.FP8, 2 * G, 2, [500, 333], [new, new], window=70, sinks=20, seed=6)
    out, lse = [x.clone() for x in c.run()]
    for r in range(2):
        see = c.visible(r).any(0)
        for page in range(-(-c.lens[r] // T)):
            if not see[page * T:(page + 1) * T].any():
                c.p.scales[c.layer, int(c.p.table[int(c.lanes[r]), page]), :, which] = bad
    got = c.run()
    assert torch.equal(got[0], out) and torch.equal(got[1], lse)


def test_pages_before_the_window_need_not_be_there():
    # a window's program may have given back what is before it
    c = Seen(F.BF16, 8, 2, [2000, 700], window=128, sinks=4, seed=1)
    want = [x.clone() for x in c.run()]
    for r, n in enumerate(c.lens):
        c.p.table[int(c.lanes[r]), 1:(n - 128) // T] = -1
    got = c.run()  # checks that nothing was found
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dt", [F.BF16, F.F16, F.FP8])
@pytest.mark.parametrize("Hq,H", [(8, 2), (80, 2)])
@pytest.mark.parametrize("new", [1, 9, 40])
@pytest.mark.parametrize("sinks", [4, 20, 100])
@pytest.mark.parametrize("gap", [1, 2, 3, 30])
def test_pages_between_the_sinks_and_the_window_need_not_be_there(dt, Hq, H, new, sinks, gap):
    """`gap` pages that no row sees, in tiles of all forms: their entries are not looked at."""
    window, first = 128, (-(-sinks // T) + gap) * T  # the first row's window starts in the page behind them
    base = first + window + 3
    c = Seen(dt, Hq, H, [base + new, base + new + 5], [new, new], window=window, sinks=sinks, seed=gap)
    assert not any(c.visible(r)[:, -(-sinks // T) * T:first].any() for r in range(2))
    want = [x.clone() for x in c.run()]
    c.check(*want)
    hidden = [(r, t) for r in range(2) for t in range(T * -(-sinks // T), first)]
    spoil(c, dt, float("nan"), hidden)
    table = c.p.table.clone()
    for lane in c.lanes:
        c.p.table[int(lane), -(-sinks // T):first // T] = -1
    got = c.run()  # checks that nothing was found
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    if dt != F.FP8:
        return
    # nor where rows are done one by one, as a scale of the first page behind is not finite
    scale = c.p.scales[c.layer, int(c.p.table[int(c.lanes[0]), first // T]), :, 1]
    finite = scale.clone()
    scale.fill_(float("nan"))
    out, lse = c.run()
    scale.copy_(finite)
    clean = torch.ones((c.rows, 1), dtype=torch.bool, device="cuda")
    clean[:new, 0] = torch.from_numpy(~c.visible(0)[:, first:first + T].any(1)).cuda()
    assert torch.all(torch.isnan(out[~clean[:, 0]].float()))
    c.p.table.copy_(table)
    spoil(c, dt, 0.0, hidden)
    c.check(torch.where(clean.unsqueeze(2), out, want[0]), torch.where(clean, lse, want[1]))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("new", [1, 7, 40, 70])
@pytest.mark.parametrize("window,sinks", [(64, 0), (64, 4), (37, 20)])
@pytest.mark.parametrize("base", [319, 320, 326])
def test_pages_before_the_window_of_all_drafts_need_not_be_there(dt, new, window, sinks, base):
    """The window counts by depth: where every row has a bit, and more so where they
    have many, tokens that a row of none would see are before all windows."""
    rng = np.random.default_rng(base)
    for deep in (0, 30):
        if deep >= new:
            continue
        masks = [tree_of(rng, new, back=2)[1] for _ in range(2)]
        for m in masks:
            m[:, :deep] = True
        c = Seen(dt, 8, 2, [base + new, base + new + 9], [new, new], window=window, sinks=sinks, masks=masks, seed=new)
        want = [x.clone() for x in c.run()]
        c.check(*want)
        for r, lane in enumerate(c.lanes):
            see = c.visible(r).any(0)
            for page in range(-(-sinks // T), base // T):
                if not see[page * T:(page + 1) * T].any():
                    c.p.table[int(lane), page] = -1
        got = c.run()  # checks that nothing was found
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dt", [F.BF16, F.FP8])
@pytest.mark.parametrize("new", [[40, 33], [60] * 6])
def test_a_seen_without_a_window_or_a_tree_is_the_causal_call(dt, new):
    """Structures of zeros: the same kernels, grid and order of sums."""
    c = Seen(dt, 32, 8, [3000 + 7 * i for i in range(len(new))], new, seed=3)
    want = c.run()
    n, need = len(new), C.c_uint64()
    a = c.args()
    d = F.AttendArgs(n_req=n, n_tokens=c.rows, q_heads=32, lanes=a["lanes"].data_ptr(), q_start=a["q_start"].data_ptr(),
                     q=c.q.data_ptr())
    d.q_stride[0] = d.out_stride[0] = 32 * D
    d.q_stride[1] = d.out_stride[1] = D
    assert F.lib.ferry_pages_attend_work_bytes(c.p._r, C.byref(d), C.byref(need)) == 0
    work = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    d.work, d.work_bytes = work.data_ptr(), need.value
    for seen in (None, F.SeenArgs()):
        out, lse = torch.full_like(c.q, 9.0), torch.full((c.rows, 32), 9.0, device="cuda")
        d.out, d.lse = out.data_ptr(), lse.data_ptr()
        rc = F.lib.ferry_pages_attend_seen(c.p._r, 0, C.byref(d), seen and C.byref(seen),
                                           torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        torch.cuda.synchronize()
        c.p.check()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_requests_without_a_lane_and_rows_behind_the_last():
    rng = np.random.default_rng(1)
    new = [5, 3, 4]
    masks = [tree_of(rng, n)[1] for n in new]
    for kw in (dict(window=20, sinks=2), dict(masks=masks)):
        c = Seen(F.BF16, 8, 2, [50, 70, 90], new, seed=2, **kw)
        want, want_lse = c.run()
        lanes = ints([int(c.lanes[0]), -1, int(c.lanes[2])])
        q = torch.cat([c.q, c.q[:2]])
        out = torch.full_like(q, 9.0)
        lse = torch.full((14, 8), 9.0, device="cuda")
        a = c.args()
        if a["tree"] is not None:
            a["tree"] = torch.cat([a["tree"], a["tree"][:2]])
        a["lanes"] = lanes
        c.p.attend(0, q, out, lse=lse, **a)
        torch.cuda.synchronize()
        c.p.check()
        # (the work is cut otherwise without the second request: not the same bits)
        c.check(torch.cat([out[:5], want[5:8], out[8:12]]), torch.cat([lse[:5], want_lse[5:8], lse[8:12]]))
        assert not torch.any(out[5:8]) and torch.all(lse[5:8] == -np.inf)
        assert torch.all(out[12:] == 9.0) and torch.all(lse[12:] == 9.0)


def test_more_tokens_than_the_words_hold():
    # reported; what the bits can name is as it should be
    masks = [np.tril(np.ones((70, 70), bool)), np.tril(np.ones((10, 10), bool))]
    c = Seen(F.BF16, 8, 2, [200, 50], [70, 10], masks=masks, seed=1)
    c.words = c.words[:, :1].contiguous()
    out = torch.empty_like(c.q)
    lse = torch.empty((80, 8), device="cuda")
    c.p.attend(0, c.q, out, lse=lse, **c.args())
    torch.cuda.synchronize()
    with pytest.raises(F.FerryError) as e:
        c.p.check()
    assert e.value.code == -3
    c.masks[0][:, 64:] = False
    c.check(out, lse)


def test_more_new_tokens_than_the_lane_holds():
    c = Seen(F.BF16, 8, 2, [5, 40], [5, 4], masks=[np.tril(np.ones((5, 5), bool)), np.tril(np.ones((4, 4), bool))])
    c.p.length[int(c.lanes[0])] = 3  # its first two tokens are not there
    for args in (c.args(), dict(c.args(), tree=None, window=9)):
        out = torch.full_like(c.q, 9.0)
        lse = torch.full((9, 8), 9.0, device="cuda")
        c.p.attend(0, c.q, out, lse=lse, **args)
        torch.cuda.synchronize()
        c.p.check()
        assert not torch.any(out[:2]) and torch.all(lse[:2] == -np.inf)
        assert torch.all(torch.isfinite(lse[2:]))


def test_strides_layers_scale_and_the_output_in_the_queries_place():
    rng = np.random.default_rng(8)
    for new in (3, 40):
        masks = [tree_of(rng, new)[1] for _ in range(2)]
        for kw in (dict(window=50, sinks=3), dict(masks=masks)):
            c = Seen(F.F16, 12, 3, [300, 77], [new, new], layers=3, layer=2, seed=2, **kw)
            wide = torch.empty((c.rows, 30, 131), dtype=c.qt, device="cuda")
            q = wide[:, 1:25:2, 1:129]
            q.copy_(c.q)
            lse = torch.empty((c.rows, 12), device="cuda")
            c.p.attend(2, q, q, lse=lse, scale=-0.05, **c.args())
            torch.cuda.synchronize()
            c.p.check()
            c.check(q, lse, scale=-0.05)


@pytest.mark.parametrize("dt", [F.BF16, F.FP8])
def test_a_captured_call_follows_lengths_and_bits(dt):
    rng = np.random.default_rng(4)
    new = [6, 6]
    for kw in (dict(window=40, sinks=4), dict(masks=[tree_of(rng, 6)[1] for _ in new])):
        c = Seen(dt, 8, 2, [500, 300], new, seed=5, **kw)
        a = c.args()
        out, lse = torch.empty_like(c.q), torch.empty((c.rows, 8), device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c.p.attend(0, c.q, out, lse=lse, **a)
        for step, lens in enumerate([[500, 300], [499, 17], [33, 299], [6, 6]]):
            c.lens = lens
            for lane, n in zip(c.lanes, lens):
                c.p.length[int(lane)] = n
            if c.masks is not None:
                c.masks = [tree_of(rng, 6)[1] for _ in new]
                a["tree"].copy_(words_of(c.masks, 1))
            graph.replay()
            torch.cuda.synchronize()
            c.check(out, lse)
            e_out, e_lse = torch.empty_like(out), torch.empty_like(lse)
            c.p.attend(0, c.q, e_out, lse=e_lse, **a)
            torch.cuda.synchronize()
            c.p.check()
            assert torch.equal(out, e_out) and torch.equal(lse, e_lse)


def test_two_calls_at_once_and_the_same_bits():
    rng = np.random.default_rng(4)
    c = Seen(F.BF16, 32, 8, [3000, 4000, 100], [30, 1, 20], masks=[tree_of(rng, n)[1] for n in (30, 1, 20)], seed=5)
    w = Seen(F.BF16, 32, 8, [3000, 4000, 100], [30, 1, 20], window=1000, sinks=4, seed=6)
    wants = [x.run() for x in (c, w)]
    args = [x.args() for x in (c, w)]  # of the current stream: they outlive the calls
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        outs = []
        for x, s in zip((c, w), streams):
            out, lse = torch.empty_like(x.q), torch.empty((x.rows, 32), device="cuda")
            torch.cuda.synchronize()
            outs.append((out, lse))
        for x, s, a, (out, lse) in zip((c, w), streams, args, outs):
            x.p.attend(0, x.q, out, lse=lse, stream=s, **a)
        torch.cuda.synchronize()
        for (out, lse), want in zip(outs, wants):
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_a_pool_past_four_gibibytes():
    # 18,000 pages of 8 heads in 16 bits are 1.2 GB; layer 4 of 5 starts behind 4 GiB
    for kw in (dict(window=3000, sinks=4), dict(masks=[np.tril(np.ones((12, 12), bool))] * 2)):
        new = [12, 12]
        c = Seen(F.BF16, 8, 8, [9000, 5000], new, layers=5, layer=4, spare=17200, seed=1, **kw)
        assert 4 * c.p.pool[0].numel() * 2 > 2 ** 32
        c.check(*c.run())
        del c


def test_no_rows():
    c = Seen(F.BF16, 8, 2, [50], window=8)
    q = c.q[:0]
    c.p.attend(0, q, q, ints([]), window=8)
    c.p.attend(0, q, q, ints([]), tree=torch.zeros((0, 1), dtype=torch.int64, device="cuda"))
    c.p.check()


def test_refusals():
    c = Seen(F.BF16, 8, 2, [50, 60])
    out, lanes = torch.empty_like(c.q), ints(c.lanes)
    groups = dict(group_start=ints([0, 2]), shared=ints([1]))
    tree = torch.ones((2, 1), dtype=torch.int64, device="cuda")
    for kw, text in [(dict(window=-1), "negative"), (dict(window=4, sinks=-1), "negative"), (dict(sinks=3), "go with a window"),
                     (dict(window=4, **groups), "no groups")]:
        with pytest.raises(F.FerryError, match=text):
            c.p.attend(0, c.q, out, lanes, **kw)
    for bad in (tree[:1], tree.int(), tree.cpu(), torch.ones((2, 2), dtype=torch.int64, device="cuda")[:, :1], tree[:, :0]):
        with pytest.raises(ValueError, match="tree"):
            c.p.attend(0, c.q, out, lanes, tree=bad)
    with pytest.raises(F.FerryError, match="tree_words"):
        c.p.attend(0, c.q, out, lanes, tree=torch.ones((2, 65), dtype=torch.int64, device="cuda"))
