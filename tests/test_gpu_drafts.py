"""Drafted tokens in the paged KV cache on the GPU: their ancestors, places and
positions, and what stays of them, against the same rules on Python lists; and a
server's steps with them, whose cache in the end is that of the kept tokens alone."""
import ctypes as C

import numpy as np
import pytest
import torch

import ferry_amd as F

from test_gpu_append import near, turned
from test_gpu_axes import turned as turned_at
from test_gpu_attend import TORCH, ints
from test_gpu_seen import Seen, tree_of, words_of

pytestmark = pytest.mark.gpu

T, D = 16, 128
EINVAL, ERANGE, ESTATE = -1, -3, -7


def cache(lens, lanes, H=1, layers=1, dt=F.BF16, spare=4, seed=0, n_lanes=None):
    """Lanes that hold lens tokens in pages of random ids and bytes."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = [-(-n // T) for n in lens]
    n_lanes = n_lanes or max(lanes) + 2
    p = F.Pages.empty(layers, H, sum(pages) + spare, n_lanes, max(pages + [1]) + 2, dt)
    raw = p.pool.view(torch.uint8)
    raw.copy_(torch.randint(0, 256, raw.shape, device="cuda", generator=g, dtype=torch.uint8))
    ids = torch.randperm(p.refs.numel(), generator=torch.Generator().manual_seed(seed)).tolist()
    for lane, n, m in zip(lanes, lens, pages):
        mine = [ids.pop() for _ in range(m)]
        p.table[lane, :m] = ints(mine)
        p.length[lane] = n
        p.refs[ints(mine).long()] = 1
    return p


def run_tree(p, lanes, parents, words, rows=None, start=None):
    flat = [x for q in parents for x in q]
    rows = rows or len(flat)
    flat += [5] * (rows - len(flat))
    tree = torch.full((rows, words), 77, dtype=torch.int64, device="cuda")
    at, place, lane = (torch.full((rows,), 77, dtype=torch.int32, device="cuda") for _ in range(3))
    q_start = np.concatenate([[0], np.cumsum([len(q) for q in parents])]) if start is None else start
    p.tree(ints(lanes), ints(flat), tree, at=at, place=place, lane=lane, q_start=ints(q_start))
    torch.cuda.synchronize()
    return tree, at.tolist(), place.tolist(), lane.tolist()


@pytest.mark.parametrize("sizes", [[1], [2, 0, 3], [63, 64, 65], [8] * 40, [130, 1, 700], [1000], [1300, 5, 4000]])
@pytest.mark.parametrize("back", [1, 3, 40, 100000])
def test_trees_from_parents(sizes, back):
    rng = np.random.default_rng(back + len(sizes))
    n = len(sizes)
    lanes = rng.permutation(n + 1)[:n].tolist()
    before = rng.integers(0, 50, n).tolist()
    p = cache([b + s for b, s in zip(before, sizes)], lanes)
    made = [tree_of(rng, s, back=back, roots=back == 3) if s else ([], np.zeros((0, 0), bool)) for s in sizes]
    words = -(-max(sizes) // 64) + (back == 3)
    tree, at, place, lane = run_tree(p, lanes, [m[0] for m in made], words)
    p.check()
    assert torch.equal(tree, words_of([m[1] for m in made], words))
    assert at == [b - 1 + int(row.sum()) for b, m in zip(before, made) for row in m[1]]
    assert place == [b + i for b, s in zip(before, sizes) for i in range(s)]
    assert lane == [x for x, s in zip(lanes, sizes) for _ in range(s)]


def test_tokens_of_no_request_are_padding():
    p = cache([20, 30], [0, 2])
    tree, at, place, lane = run_tree(p, [0, -1, 2], [[-1, 0], [-1, 0, 1], [-1, 0, 0, 2]], 2, rows=140)
    p.check()
    assert lane == [0] * 2 + [-1] * 3 + [2] * 4 + [-1] * 131
    assert place == [18, 19] + [-1] * 3 + [26, 27, 28, 29] + [-1] * 131
    assert at == [18, 19] + [0] * 3 + [26, 27, 27, 28] + [0] * 131
    assert tree[:, 0].tolist() == [1, 3] + [0] * 3 + [1, 3, 5, 13] + [0] * 131 and not torch.any(tree[:, 1])
    # the first request's tokens need not be the batch's first
    tree, at, place, lane = run_tree(p, [0], [[7], [7], [-1, 0]], 1, rows=5, start=[2, 4])
    p.check()
    assert lane == [-1, -1, 0, 0, -1] and place == [-1, -1, 18, 19, -1] and tree[:, 0].tolist() == [0, 0, 1, 3, 0]


def test_without_offsets_and_without_some_results():
    p = cache([20, 1, 30], [0, 1, 2])
    tree = torch.zeros((3, 1), dtype=torch.int64, device="cuda")
    at = ints([0, 0, 0])
    p.tree(ints([2, 0, 1]), ints([-1, -1, -1]), tree, at=at)
    torch.cuda.synchronize()
    p.check()
    assert tree.tolist() == [[1], [1], [1]] and at.tolist() == [29, 19, 0]


@pytest.mark.parametrize("what", ["parent", "lane", "low", "words", "offsets"])
def test_trees_out_of_range_are_reported(what):
    p = cache([20, 30], [0, 1])
    parents, lanes, words, start = [[-1, 0, 1], [-1, 0, 0]], [0, 1], 1, None
    if what == "parent":
        parents[0] = [-1, 1, -2]  # not before the token: roots
    elif what == "lane":
        lanes = [9, 1]
    elif what == "low":
        p.length[0] = 2
    elif what == "words":
        parents[0] = [-1] + list(range(69))
        p.length[0] = 70
        p.table = torch.zeros((3, 8), dtype=torch.int32, device="cuda")
        p = F.Pages(p.pool, p.table, p.length)
    else:
        start = [0, 5, 3]
    tree, at, place, lane = run_tree(p, lanes, parents, words, start=start)
    with pytest.raises(F.FerryError) as e:
        p.check()
    assert e.value.code == ERANGE
    if what == "parent":
        assert tree[:3, 0].tolist() == [1, 2, 4] and at[:3] == [17, 17, 17]
    elif what in ("lane", "low"):
        assert lane == [-1] * 3 + [1] * 3 and not torch.any(tree[:3])
    elif what == "words":
        assert tree[63, 0] == -1 and tree[69, 0] == -1 and at[:64] == list(range(64))
    if what != "offsets":
        assert tree[-3:, 0].tolist() == [1, 3, 5] and at[-3:] == [27, 28, 28]


def test_a_captured_tree_follows_lengths_and_parents():
    rng = np.random.default_rng(0)
    p = cache([300, 300], [0, 1])
    parent = ints([0] * 140)
    tree = torch.zeros((140, 2), dtype=torch.int64, device="cuda")
    at, place, lane = ints([0] * 140), ints([0] * 140), ints([0] * 140)
    lanes, start = ints([1, 0]), ints([0, 100, 140])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p.tree(lanes, parent, tree, at=at, place=place, lane=lane, q_start=start)
    for lens in ([300, 200], [40, 100], [299, 150]):
        made = [tree_of(rng, 100), tree_of(rng, 40)]
        parent.copy_(ints(made[0][0] + made[1][0]))
        p.length[:2] = ints(lens)
        graph.replay()
        torch.cuda.synchronize()
        p.check()
        assert torch.equal(tree, words_of([m[1] for m in made], 2))
        assert place.tolist() == list(range(lens[1] - 100, lens[1])) + list(range(lens[0] - 40, lens[0]))
        want = [lens[1] - 101 + int(x.sum()) for x in made[0][1]] + [lens[0] - 41 + int(x.sum()) for x in made[1][1]]
        assert at.tolist() == want


# ---- what stays of the drafts ------------------------------------------------------
def walk(parent, draft, chosen):
    line = [0] if draft else []
    for c in range(1, len(draft)):
        if line and parent[c] == line[-1] and draft[c] == chosen[line[-1]]:
            line.append(c)
    return line


class Check:
    """A cache, requests with trees of drafts, and what the rules make of it."""

    def __init__(self, dt, before, sizes, H=2, layers=2, back=4, agree=0.8, seed=0, chain=False, scales="one"):
        rng = np.random.default_rng(seed)
        n = len(sizes)
        self.lanes = rng.permutation(n + 2)[:n].tolist()
        self.before, self.sizes = before, sizes
        lens = [b + s for b, s in zip(before, sizes)]
        self.p = p = cache(lens, self.lanes, H, layers, dt, seed=seed, n_lanes=n + 2)
        if dt == F.FP8:
            raw = p.pool.view(torch.uint8)
            raw.copy_(torch.where((raw & 127) == 127, raw & 126, raw))  # no NaN
            g = torch.Generator(device="cuda").manual_seed(seed)
            s = 0.5 + torch.rand(p.scales.shape, device="cuda", generator=g)
            p.scales.copy_(s[:, :1].expand(s.shape) if scales == "one" else s)
        self.parents, self.draft, self.chosen = [], [], []
        for s in sizes:
            parent = list(range(-1, s - 1)) if chain else tree_of(rng, s, back=back)[0] if s else []
            draft = rng.integers(0, 4, s).tolist()  # siblings may be equal: the first child counts
            chosen = rng.integers(100, 104, s).tolist()
            for c in range(s - 1, 0, -1):
                if rng.random() < agree:
                    chosen[parent[c]] = draft[c]
            self.parents.append(parent)
            self.draft.append(draft)
            self.chosen.append(chosen)
        self.chain = chain
        self.rows = sum(sizes)
        self.start = np.concatenate([[0], np.cumsum(sizes)])

    def buffers(self):
        def flat(x):
            return ints([v for q in x for v in q])
        path = torch.full((self.rows + 3,), 77, dtype=torch.int32, device="cuda")
        return dict(lanes=ints(self.lanes), draft=flat(self.draft), chosen=flat(self.chosen), path=path,
                    kept=torch.full((len(self.sizes),), 77, dtype=torch.int32, device="cuda"),
                    next=torch.full((len(self.sizes),), 77, dtype=torch.int32, device="cuda"),
                    q_start=ints(self.start), parent=None if self.chain else flat(self.parents))

    def lines(self):
        return [walk(*x) for x in zip(self.parents, self.draft, self.chosen)]

    def run_and_check(self, args=None):
        p = self.p
        table, refs = p.table.cpu().numpy(), p.refs.cpu().numpy()
        raw = p.pool.view(torch.uint8)
        want, scales = raw.clone(), p.scales
        lines = self.lines()
        differ = []
        for r, line in enumerate(lines):
            row = table[self.lanes[r]]
            for i, c in enumerate(line):
                to, frm = self.before[r] + i, self.before[r] + c
                if to != frm:
                    a, b = row[frm // T], row[to // T]
                    if scales is not None and not torch.equal(scales[:, a], scales[:, b]):
                        differ.append((frm, to, int(a), int(b)))
                        x = want[:, a, :, :, frm % T].view(torch.float8_e4m3fn).float()
                        x = x * scales[:, a].unsqueeze(-1) / scales[:, b].unsqueeze(-1)
                        want[:, b, :, :, to % T] = x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
                    else:
                        want[:, b, :, :, to % T] = want[:, a, :, :, frm % T].clone()
            left = self.before[r] + len(line)
            for e in range(-(-left // T), -(-(self.before[r] + self.sizes[r]) // T)):
                refs[row[e]] -= 1
                row[e] = -1
        b = args or self.buffers()
        p.accept(**b)
        torch.cuda.synchronize()
        p.check()
        path = b["path"].tolist()
        assert path[self.rows:] == [77] * 3
        for r, line in enumerate(lines):
            a = int(self.start[r])
            assert path[a:a + self.sizes[r]] == [a + c for c in line] + [-1] * (self.sizes[r] - len(line))
        assert b["kept"].tolist() == [len(x) for x in lines]
        assert b["next"].tolist() == [q[x[-1]] if x else -1 for q, x in zip(self.chosen, lines)]
        length = [0] * p.length.numel()
        for lane, bf, line in zip(self.lanes, self.before, lines):
            length[lane] = bf + len(line)
        assert p.length.tolist() == length
        assert np.array_equal(p.table.cpu().numpy(), table)
        assert np.array_equal(p.refs.cpu().numpy(), refs)
        assert torch.equal(raw, want)
        return lines, differ


@pytest.mark.parametrize("dt", [F.BF16, F.F16, F.F32, F.FP8])
@pytest.mark.parametrize("before,sizes", [
    ([0], [1]), ([5, 16, 31], [8, 1, 9]), ([15, 0, 100, 7], [40, 64, 65, 0]), ([33] * 12, [20] * 12), ([1000, 3], [200, 130]),
])
def test_drafts_that_stay(dt, before, sizes):
    for seed in range(3):
        c = Check(dt, before, sizes, H=3, layers=3, seed=seed)
        c.run_and_check()


@pytest.mark.parametrize("dt", [F.BF16, F.FP8])
def test_all_and_none_stay(dt):
    c = Check(dt, [7, 40], [50, 9], agree=1.0, back=1)
    lines, _ = c.run_and_check()
    assert [len(x) for x in lines] == [50, 9]
    c = Check(dt, [7, 40], [50, 9], agree=0.0)
    lines, _ = c.run_and_check()
    assert [len(x) for x in lines] == [1, 1]


def test_chains_and_more_moves_than_are_listed_at_once():
    c = Check(F.BF16, [3, 900], [30, 1], chain=True, agree=0.95)
    c.run_and_check()
    c = Check(F.BF16, [9], [1400], chain=True, agree=1.0, seed=1)
    lines, _ = c.run_and_check()
    assert len(lines[0]) == 1400
    # a line of every other token: 700 moves, each into the place of another's source
    c = Check(F.BF16, [9], [1400], agree=0.0, seed=2)
    c.parents[0] = [-1, 0] + [i - 2 for i in range(2, 1400)]
    for i in range(0, 1398, 2):
        c.chosen[0][i] = 7
        c.draft[0][i + 1], c.draft[0][i + 2] = 8, 7
    lines, _ = c.run_and_check()
    assert lines[0] == list(range(0, 1400, 2))


def test_many_requests_and_layers():
    rng = np.random.default_rng(5)
    n = 3000
    c = Check(F.F16, rng.integers(0, 40, n).tolist(), rng.integers(0, 12, n).tolist(), H=1, layers=1, seed=3)
    c.run_and_check()
    c = Check(F.BF16, [30] * 5, [20] * 5, H=8, layers=40, seed=4)
    c.run_and_check()


def test_pages_of_other_scales_are_rounded_again():
    differing = 0
    for seed in range(4):
        c = Check(F.FP8, [5, 12, 40], [60, 33, 20], seed=seed, scales="many", agree=0.95)
        _, differ = c.run_and_check()
        differing += len(differ)
    for seed in range(3):  # trees whose lines leap over pages
        c = Check(F.FP8, [5, 12, 40], [160, 133, 120], seed=seed, scales="many", agree=0.95, back=40)
        _, differ = c.run_and_check()
        differing += len(differ)
    assert differing


def test_requests_without_a_lane():
    c = Check(F.BF16, [20, 30, 9], [9, 9, 9], seed=6)
    b = c.buffers()
    b["lanes"] = ints([c.lanes[0], -1, c.lanes[2]])
    idle = c.lanes[1]
    row, raw = c.p.table[idle].clone(), c.p.pool.clone()
    c.p.accept(**b)
    torch.cuda.synchronize()
    c.p.check()
    lines = c.lines()
    assert b["kept"].tolist() == [len(lines[0]), 0, len(lines[2])]
    assert b["next"].tolist()[1] == -1 and b["path"][9:18].tolist() == [-1] * 9
    assert torch.equal(c.p.table[idle], row) and int(c.p.length[idle]) == 39
    ids = row[:3].long()
    assert torch.equal(c.p.pool[:, ids].view(torch.int16), raw[:, ids].view(torch.int16))
    # and one whose lane has no new tokens
    e = ints([-5])
    c.p.accept(ints([idle]), ints([]), ints([]), ints([]), e, ints([0]), q_start=ints([0, 0]))
    torch.cuda.synchronize()
    c.p.check()
    assert e.tolist() == [0] and int(c.p.length[idle]) == 39


@pytest.mark.parametrize("what", ["twice", "lane", "offsets", "past", "held", "end"])
def test_a_refused_call_changes_nothing(what):
    c = Check(F.BF16, [20, 3, 50], [9, 8, 7], seed=7)
    b = c.buffers()
    if what == "twice":
        b["lanes"] = ints([c.lanes[0], c.lanes[1], c.lanes[0]])
    elif what == "lane":
        b["lanes"] = ints([c.lanes[0], 5, c.lanes[2]])
    elif what == "offsets":
        b["q_start"] = ints([0, 17, 9, 24])
    elif what == "past":
        b["q_start"] = ints([0, 9, 17, 25])
    elif what == "end":
        b["q_start"] = ints([-1, 9, 17, 24])
    else:
        c.p.length[c.lanes[1]] = 7
    p = c.p
    state = [x.clone() for x in (p.table, p.length, p.refs, p.pool.view(torch.uint8))]
    p.accept(**b)
    torch.cuda.synchronize()
    with pytest.raises(F.FerryError) as e:
        p.check()
    assert e.value.code == EINVAL
    for x, y in zip(state, (p.table, p.length, p.refs, p.pool.view(torch.uint8))):
        assert torch.equal(x, y)
    for name in ("path", "kept", "next"):
        assert torch.all(b[name] == 77)


def test_moves_into_pages_in_use_twice_are_left_out():
    c = Check(F.BF16, [20, 30], [30, 9], agree=1.0, back=2, seed=8)
    lane = c.lanes[0]
    page = int(c.p.table[lane, 1])
    c.p.refs[page] = 2  # as if another lane named it
    before = c.p.pool[:, page].clone()
    b = c.buffers()
    c.p.accept(**b)
    torch.cuda.synchronize()
    with pytest.raises(F.FerryError) as e:
        c.p.check()
    assert e.value.code == ESTATE
    assert torch.equal(c.p.pool[:, page].view(torch.int16), before.view(torch.int16))
    assert b["kept"].tolist() == [len(x) for x in c.lines()]
    # a page that is not there
    c = Check(F.BF16, [20], [30], agree=1.0, back=2, seed=8)
    c.p.table[c.lanes[0], 2] = 10 ** 6
    c.p.accept(**c.buffers())
    torch.cuda.synchronize()
    with pytest.raises(F.FerryError) as e:
        c.p.check()
    assert e.value.code == ESTATE


def test_a_captured_call_follows_the_choices():
    c = Check(F.BF16, [20, 30], [12, 9], seed=9)
    b = c.buffers()
    state = [x.clone() for x in (c.p.table, c.p.length, c.p.refs, c.p.pool.view(torch.uint8))]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.p.accept(**b)
    for seed in (9, 10, 11):
        other = Check(F.BF16, [20, 30], [12, 9], seed=seed)
        other.p, other.lanes = c.p, c.lanes
        for x, y in zip((c.p.table, c.p.length, c.p.refs, c.p.pool.view(torch.uint8)), state):
            x.copy_(y)
        new = other.buffers()
        for k in ("draft", "chosen", "parent"):
            b[k].copy_(new[k])
        b["path"].fill_(77)

        class Replay:
            def __getattr__(self, name):
                return getattr(c.p, name)

            def accept(self, **kw):
                graph.replay()
        other.p = Replay()
        other.run_and_check(b)


def test_refusals():
    c = Check(F.BF16, [20, 30], [5, 9])
    b = c.buffers()
    for name in ("path", "kept", "next"):
        for other in ("lanes", "draft", "chosen", "q_start", "parent"):
            with pytest.raises((F.FerryError, ValueError), match="overlaps|elements"):
                c.p.accept(**{**b, name: b[other]})
    with pytest.raises(F.FerryError, match="overlaps"):
        c.p.accept(**{**b, "kept": b["path"][:2]})
    with pytest.raises(F.FerryError, match="the cache's own"):
        c.p.accept(**{**b, "kept": c.p.length[:2]})
    with pytest.raises(F.FerryError, match="one token"):
        c.p.accept(**{**b, "q_start": None})
    with pytest.raises(ValueError, match="draft"):
        c.p.accept(**{**b, "draft": b["draft"].long()})
    with pytest.raises(F.FerryError, match="refs"):
        F.Pages(c.p.pool, c.p.table, c.p.length).accept(**b)
    many = ints([-1] * 5)
    with pytest.raises(F.FerryError, match="n_lanes"):
        c.p.accept(many, many.clone(), many.clone(), many.clone(), many.clone(), many.clone())
    tree = torch.zeros((2, 1), dtype=torch.int64, device="cuda")
    lanes, parent = ints(c.lanes), ints([-1, -1])
    with pytest.raises(F.FerryError, match="overlaps"):
        c.p.tree(lanes, parent, tree, at=parent)
    with pytest.raises(F.FerryError, match="overlaps"):
        c.p.tree(lanes, parent, tree, at=parent.clone(), lane=tree.view(torch.int32).view(-1)[:2])
    with pytest.raises(F.FerryError, match="overlaps len"):
        c.p.tree(lanes, parent, tree, at=c.p.length)
    with pytest.raises(F.FerryError, match="tree_words"):
        c.p.tree(lanes, parent, torch.zeros((2, 65), dtype=torch.int64, device="cuda"))
    with pytest.raises(F.FerryError, match="one token"):
        c.p.tree(ints(c.lanes[:1]), parent, tree)
    with pytest.raises(ValueError, match="tree"):
        c.p.tree(lanes, parent, tree[:1])
    torch.cuda.synchronize()
    c.p.check()
    assert C.sizeof(F.AcceptArgs) == 72


# ---- a server's steps --------------------------------------------------------------
@pytest.mark.parametrize("dt", [F.BF16, F.FP8, F.F16])
@pytest.mark.parametrize("window", [0, 24])
def test_steps_with_drafts(dt, window):
    """Prompts, then steps: room for a tree in each lane, its rows and positions, the
    write, attention, and what stays of it.  The cache holds the keys and values of the
    kept tokens at their positions, as if they had come one after the other."""
    L, H, HQ, X = 2, 2, 8, torch.bfloat16
    rng = np.random.default_rng(3)
    g = torch.Generator(device="cuda").manual_seed(dt)
    lanes = [2, 0, 3]
    p = F.Pages.empty(L, H, 40, 5, 12, dt)
    freq = F.rope_freqs(F.ROPE_PLAIN, 128)
    inv = torch.from_numpy(freq).cuda()
    kv = 0.01 + 0.01 * torch.rand((H, 2), device="cuda", generator=g) if dt == F.FP8 else None
    held = {a: [] for a in lanes}  # (k, v) [L, H, D] of every token

    def fresh(n):
        return [torch.randn((L, n, h, D), device="cuda", generator=g).to(X) for h in (HQ, H, H)]

    def layers(rows, lane, place, at, **seen):
        q, k, v = fresh(rows)
        qr = torch.empty((L, rows, HQ, D), dtype=p.q_dtype, device="cuda")
        out, lse = torch.empty_like(qr), torch.empty((L, rows, HQ), device="cuda")
        for i in range(L):
            p.append(i, lane, place, k=k[i], v=v[i], q=q[i], q_out=qr[i], inv_freq=inv, kv_scale=kv, at=at)
            p.attend(i, qr[i], out[i], ints(lanes), lse=lse[i], window=window, sinks=3 if window else 0, **seen)
        return q, k, v, qr, out, lse

    def attended(new, masks, qr, out, lse):
        c = Seen.__new__(Seen)
        c.dt, c.Hq, c.H, c.p, c.lanes, c.new, c.masks = dt, HQ, H, p, lanes, new, masks
        c.window, c.sinks = window, 3 if window else 0
        c.lens = p.length[ints(lanes).long()].tolist()
        c.start = np.concatenate([[0], np.cumsum(new)])
        for c.layer in range(L):
            c.q = qr[c.layer]
            c.check(out[c.layer], lse[c.layer])

    prompt = [17, 33, 2]
    start = np.concatenate([[0], np.cumsum(prompt)])
    p.reserve(ints(lanes), ints(prompt))
    lane, place = ints(np.repeat(lanes, prompt)), ints(np.concatenate([np.arange(n) for n in prompt]))
    q, k, v, qr, out, lse = layers(52, lane, place, None, q_start=ints(start))
    torch.cuda.synchronize()
    p.check()
    attended(prompt, None, qr, out, lse)
    for a, s, n in zip(lanes, start, prompt):
        held[a] += [(k[:, t], v[:, t]) for t in range(s, s + n)]

    for step in range(4):
        new = [int(rng.integers(1, 15)) for _ in lanes]
        rows, start = sum(new), np.concatenate([[0], np.cumsum(new)])
        made = [tree_of(rng, n, back=3) for n in new]
        d_lanes, d_start = ints(lanes), ints(start)
        d_parent = ints([x for m in made for x in m[0]])
        tree = torch.empty((rows, 1), dtype=torch.int64, device="cuda")
        at, place, lane = (torch.empty(rows, dtype=torch.int32, device="cuda") for _ in range(3))
        p.reserve(d_lanes, ints(new))
        p.tree(d_lanes, d_parent, tree, at=at, place=place, lane=lane, q_start=d_start)
        q, k, v, qr, out, lse = layers(rows, lane, place, at, q_start=d_start, tree=tree)
        torch.cuda.synchronize()
        p.check()
        depth = np.concatenate([m[1].sum(1) - 1 for m in made])
        position = np.repeat([len(held[a]) for a in lanes], new) + depth
        near(qr.flatten(0, 1), *turned_at(q.flatten(0, 1), np.tile(position, L)[None], np.zeros(64, int), freq, 1.0, False),
             1.0, F.BF16 if dt == F.FP8 else dt)
        attended(new, [m[1] for m in made], qr, out, lse)
        draft = rng.integers(0, 2, rows)
        chosen = rng.integers(0, 2, rows)
        path, kept, following = (torch.empty(n, dtype=torch.int32, device="cuda") for n in (rows, 3, 3))
        p.accept(d_lanes, ints(draft), ints(chosen), path, kept, following, q_start=d_start, parent=d_parent)
        torch.cuda.synchronize()
        p.check()
        for r, a in enumerate(lanes):
            s = int(start[r])
            line = walk(made[r][0], draft[s:s + new[r]].tolist(), chosen[s:s + new[r]].tolist())
            assert path[s:s + len(line)].tolist() == [s + c for c in line] and int(kept[r]) == len(line)
            assert int(following[r]) == chosen[s + line[-1]]
            held[a] += [(k[:, s + c], v[:, s + c]) for c in line]
        for a in lanes:
            n = len(held[a])
            assert int(p.length[a]) == n
            ids = p.table[a, :-(-n // T)].long()
            assert torch.all(p.table[a, -(-n // T):] == -1) and torch.all(p.refs[ids] == 1)
            got = p.pool.view(torch.uint8)[:, ids].view(TORCH[dt]).movedim(1, 3).reshape(L, H, 2, -1, D)[:, :, :, :n]
            for j, f in ((0, freq), (1, freq * 0.0)):
                want = torch.stack([x[j] for x in held[a]], 1)  # [L, n, H, D]
                y, size = turned(want.flatten(0, 1), np.tile(np.arange(n), L), f, 1.0, False)
                for h in range(H):
                    scale = 1.0 if kv is None else float(kv[h, j])
                    near(got[:, h, j].flatten(0, 1), y[:, h], size[:, h], 1.0, dt, scale)
    assert int(p.refs.sum()) == sum(-(-len(x) // T) for x in held.values())
