"""Managing the pages of a paged KV cache on the GPU (reserve, fork, trim,
compact) against the same calls on Python lists: tables, lengths, reference
counts and the pages' bytes are equal after every call, and a call that is
refused changes nothing."""
import numpy as np
import pytest
import torch

import ferry_amd as F

pytestmark = pytest.mark.gpu

EINVAL, ECAPACITY, ESTATE = -1, -4, -7
T = 16


class Lists:
    """The rules of ferry_pages_* on Python lists; holds[i] is the page whose first
    bytes page i has now."""

    def __init__(self, n_pages, n_lanes, max_pages):
        self.table = [[] for _ in range(n_lanes)]
        self.length = [0] * n_lanes
        self.refs = [0] * n_pages
        self.holds = list(range(n_pages))
        self.max_pages = max_pages

    def _named(self, lanes):
        return len(set(lanes)) == len(lanes) and all(0 <= x < len(self.table) for x in lanes)

    def reserve(self, lanes, tokens):
        if not self._named(lanes) or min(tokens) < 0:
            return EINVAL
        if any(self.length[x] + t > self.max_pages * T for x, t in zip(lanes, tokens)):
            return ECAPACITY
        free = [i for i, r in enumerate(self.refs) if r == 0]
        table, refs, holds = [r[:] for r in self.table], self.refs[:], self.holds[:]
        for lane, t in zip(lanes, tokens):
            row = table[lane]
            need = -(-(self.length[lane] + t) // T) - len(row)
            if self.length[lane] % T and refs[row[-1]] > 1:
                if not free:
                    return ECAPACITY
                refs[row[-1]] -= 1
                holds[free[0]] = self.holds[row[-1]]
                row[-1] = free.pop(0)
                refs[row[-1]] = 1
            if need > len(free):
                return ECAPACITY
            for _ in range(need):
                row.append(free.pop(0))
                refs[row[-1]] = 1
        for lane, t in zip(lanes, tokens):
            self.length[lane] += t
        self.table, self.refs, self.holds = table, refs, holds
        return 0

    def fork(self, src, dst, keep=None):
        if not self._named(dst) or any(self.length[d] for d in dst) or set(src) & set(dst) or \
                not all(0 <= s < len(self.table) for s in src):
            return EINVAL
        keep = [self.length[s] for s in src] if keep is None else keep
        if any(not 0 <= k <= self.length[s] for s, k in zip(src, keep)):
            return EINVAL
        for s, d, k in zip(src, dst, keep):
            self.table[d] = self.table[s][:-(-k // T)]
            self.length[d] = k
            for i in self.table[d]:
                self.refs[i] += 1
        return 0

    def trim(self, lanes, keep=None):
        keep = [0] * len(lanes) if keep is None else keep
        if not self._named(lanes) or any(not 0 <= k <= self.length[x] for x, k in zip(lanes, keep)):
            return EINVAL
        for lane, k in zip(lanes, keep):
            n = -(-k // T)
            for i in self.table[lane][n:]:
                self.refs[i] -= 1
            self.table[lane], self.length[lane] = self.table[lane][:n], k
        return 0

    def compact(self):
        live = [i for i, r in enumerate(self.refs) if r]
        n = len(live)
        to = dict(zip([i for i in live if i >= n], [i for i in range(n) if not self.refs[i]]))
        for a, b in to.items():
            self.holds[b], self.refs[b], self.refs[a] = self.holds[a], self.refs[a], 0
        self.table = [[to.get(i, i) for i in row] for row in self.table]
        return n


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Both:
    """A cache and the lists, called alike and compared after every call."""

    def __init__(self, n_pages, n_lanes, max_pages, dtype=F.BF16, layers=2, heads=3, seed=0):
        self.p = F.Pages.empty(layers, heads, n_pages, n_lanes, max_pages, dtype)
        self.l = Lists(n_pages, n_lanes, max_pages)
        g = torch.Generator(device="cuda").manual_seed(seed)
        raw = self.p.pool.view(torch.uint8)
        raw.copy_(torch.randint(0, 256, raw.shape, device="cuda", generator=g, dtype=torch.uint8))
        if self.p.scales is not None:
            self.p.scales.copy_(torch.rand(self.p.scales.shape, device="cuda", generator=g))
            self.scales0 = self.p.scales.clone()
        self.pool0 = raw.clone()

    def same(self):
        torch.cuda.synchronize()
        t = self.p.table.cpu().numpy()
        want = np.full(t.shape, -1, np.int32)
        for r, row in enumerate(self.l.table):
            want[r, :len(row)] = row
        assert np.array_equal(t, want)
        assert self.p.length.tolist() == self.l.length
        assert self.p.refs.tolist() == self.l.refs
        at = torch.tensor(self.l.holds, device="cuda")
        assert torch.equal(self.p.pool.view(torch.uint8), self.pool0[:, at])
        if self.p.scales is not None:
            assert torch.equal(self.p.scales, self.scales0[:, at])

    def call(self, name, *lists):
        want = getattr(self.l, name)(*lists)
        getattr(self.p, name)(*[None if x is None else ints(x) for x in lists])
        if want:
            with pytest.raises(F.FerryError) as e:
                self.p.check()
            assert e.value.code == want
        else:
            self.p.check()
        self.same()
        return want

    def compact(self):
        live = ints([-1])
        want = self.l.compact()
        self.p.compact(live)
        self.p.check()
        self.same()
        assert int(live) == want


@pytest.mark.parametrize("dtype,layers,heads", [(F.BF16, 2, 3), (F.FP8, 3, 2), (F.F32, 1, 1), (F.F16, 1, 8)])
def test_growing_forking_and_ending_lanes(dtype, layers, heads):
    b = Both(80, 9, 20, dtype, layers, heads, seed=layers)
    assert b.call("reserve", [3, 0, 7], [37, 1, 16]) == 0
    assert b.call("reserve", [0], [0]) == 0
    assert b.call("fork", [3, 3, 7, 0], [4, 1, 5, 8]) == 0
    # 3, 4 and 1 share a begun page: the last of the list keeps it
    assert b.call("reserve", [4, 3, 1, 5], [1, 0, 20, 1]) == 0
    assert b.call("fork", [1, 4], [2, 6], [33, 0]) == 0
    assert b.call("reserve", [2, 6, 8], [15, 5, 14]) == 0
    assert b.call("trim", [3, 1], [16, 3]) == 0
    b.compact()
    assert b.call("trim", [7, 4]) == 0
    b.compact()
    b.compact()  # nothing to move
    assert b.call("reserve", [7, 4, 3], [200, 31, 17]) == 0
    assert b.call("trim", list(range(9))) == 0
    b.compact()
    assert not any(b.l.refs)


def test_random_calls():
    rng = np.random.default_rng(7)
    b = Both(150, 40, 12, F.BF16, 1, 1)
    seen = set()
    for step in range(120):
        n = int(rng.integers(1, 12))
        lanes = rng.permutation(40)[:n].tolist()
        what = rng.choice(["reserve", "reserve", "fork", "trim", "compact"])
        if what == "reserve":
            seen.add((what, b.call("reserve", lanes, rng.integers(0, 60, n).tolist())))
        elif what == "fork":
            empty = [x for x in range(40) if not b.l.length[x]][:n]
            src = [x for x in lanes if x not in empty]
            if empty and src:
                src = [src[i % len(src)] for i in range(len(empty))]
                keep = None if step % 2 else [int(rng.integers(0, b.l.length[s] + 1)) for s in src]
                seen.add((what, b.call("fork", src, empty, keep)))
        elif what == "trim":
            keep = None if step % 3 == 0 else [int(rng.integers(0, b.l.length[x] + 1)) for x in lanes]
            seen.add((what, b.call("trim", lanes, keep)))
        else:
            b.compact()
    assert {("reserve", 0), ("reserve", ECAPACITY), ("fork", 0), ("trim", 0)} <= seen


def test_refused_calls_change_nothing():
    b = Both(10, 6, 5, F.BF16, 1, 1)
    assert b.call("reserve", [0, 1], [30, 16]) == 0
    assert b.call("fork", [0], [2]) == 0
    for lanes, tokens, code in [([3, 3], [1, 1], EINVAL), ([6], [1], EINVAL), ([-1], [1], EINVAL),
                                ([3, 4], [1, -1], EINVAL), ([0], [51], ECAPACITY),
                                ([0, 3], [1, 97], ECAPACITY),
                                # a copy and six pages: one more than there are
                                ([2, 3, 4], [2, 64, 48], ECAPACITY)]:
        assert b.call("reserve", lanes, tokens) == code
    assert b.call("reserve", [3, 4], [80, 16]) == 0  # 6 of the 7 free pages
    assert b.call("trim", [3, 4]) == 0
    for src, dst, keep in [([0], [1], None), ([0, 0], [3, 3], None), ([0], [0], None), ([6], [3], None),
                           ([0], [-2], None), ([0], [3], [31]), ([0], [3], [-1]), ([0, 3], [3, 4], None)]:
        assert b.call("fork", src, dst, keep) == EINVAL
    for lanes, keep in [([0, 0], None), ([7], None), ([0], [31]), ([1], [-1])]:
        assert b.call("trim", lanes, keep) == EINVAL
    assert b.call("reserve", [2, 3, 4], [2, 64, 32]) == 0  # all of them


def test_lists_longer_than_a_workgroup_and_many_pages():
    n = 2500
    b = Both(70001, n + 1, 40, F.FP8, 1, 1)
    rng = np.random.default_rng(3)
    order = rng.permutation(n).tolist()
    assert b.call("reserve", order, rng.integers(0, 200, n).tolist()) == 0
    assert b.call("trim", order[::3]) == 0
    assert b.call("fork", [order[1]] * len(order[::3]), order[::3]) == 0
    assert b.call("reserve", order, rng.integers(0, 200, n).tolist()) == 0
    assert b.call("trim", order[::2]) == 0
    b.compact()
    assert b.call("reserve", [n], [640]) == 0


@pytest.mark.parametrize("n", [1, 1024, 1025, 2500])
def test_growing_within_begun_pages(n):
    # no page is taken, with and without lanes that take one
    b = Both(n + 2, n + 1, 2, F.F16, 1, 1)
    order = list(range(n))[::-1]
    assert b.call("reserve", order, [1] * n) == 0
    assert b.call("reserve", order, [15 - i % 3 for i in range(n)]) == 0
    assert b.call("reserve", order, [0] * n) == 0
    assert b.call("reserve", [n] + order[1:], [3] + [0] * (n - 1)) == 0


def test_many_copies_by_a_long_list():
    n = 1500
    b = Both(2 * n, n, 3, F.FP8, 2, 1)
    assert b.call("reserve", [7], [20]) == 0
    assert b.call("fork", [7] * (n - 1), [i for i in range(n) if i != 7]) == 0
    assert b.call("reserve", list(range(n)), [1 + 20 * (i % 2) for i in range(n)]) == 0


def test_a_page_past_four_gibibytes_is_copied():
    # records past 2^32 bytes: forked there, copied on growth, moved back by compact
    H, P = 8, 70000  # 64 KiB a page, 4.6 GB
    p = F.Pages.empty(1, H, P, 3, 4, F.BF16)
    far = P - 1
    p.table[0, :2] = ints([far - 1, far])
    p.length[0] = 20
    p.refs[far - 1:] = 1
    p.refs[0] = 1  # held outside every lane
    g = torch.Generator(device="cuda").manual_seed(1)
    data = torch.randn((2, H, 2, 16, 128), device="cuda", generator=g).to(torch.bfloat16)
    p.pool[0, far - 1:] = data
    p.fork(ints([0]), ints([1]))
    p.refs[1:far - 2] = 1
    p.reserve(ints([1]), ints([1]))
    p.check()
    assert p.table[1, :2].tolist() == [far - 1, far - 2]
    assert torch.equal(p.pool[0, far - 2], data[1])
    p.refs[1:far - 2] = 0
    p.compact()
    p.check()
    assert p.table[:2, :2].tolist() == [[2, 3], [2, 1]]
    assert torch.equal(p.pool[0, 1:4], data[[1, 0, 1]])
    assert p.refs[:5].tolist() == [1, 1, 2, 1, 0]


def test_calls_in_a_captured_graph():
    b = Both(60, 8, 8, F.BF16, 2, 2)
    assert b.call("reserve", [0, 1], [20, 40]) == 0
    src, dst, one = ints([0, 1, 0]), ints([2, 3, 4]), ints([1, 1, 1])
    live = ints([-1])

    def step():
        b.p.trim(dst)
        b.p.fork(src, dst)
        b.p.reserve(dst, one)
        b.p.compact(live)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        step()
    for i in range(4):
        graph.replay()
        b.l.trim([2, 3, 4])
        b.l.fork([0, 1, 0], [2, 3, 4])
        b.l.reserve([2, 3, 4], [1, 1, 1])
        want = b.l.compact()
        b.same()
        assert int(live) == want
        b.p.check()
        if i == 1:  # the program's own calls between replays
            assert b.call("reserve", [5], [33]) == 0
            assert b.call("trim", [0], [17]) == 0


def test_calls_on_another_stream():
    b = Both(60, 8, 8, F.F16, 1, 2)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    lanes, n = ints([1, 2]), ints([17, 30])
    torch.cuda.synchronize()
    b.p.reserve(lanes, n, stream=s)
    b.p.trim(lanes, n, stream=s)
    b.p.compact(stream=s)
    b.l.reserve([1, 2], [17, 30])
    b.l.compact()
    b.same()


def test_refusals_on_the_host():
    p = F.Pages.empty(1, 2, 8, 4, 4, F.BF16)
    with pytest.raises(ValueError, match="dtype"):
        p.reserve(torch.zeros(1, dtype=torch.int64, device="cuda"), ints([1]))
    with pytest.raises(ValueError, match="elements"):
        p.reserve(ints([0, 1]), ints([1]))
    with pytest.raises(F.FerryError, match="n must be"):
        p.reserve(ints([0, 1, 2, 3, 0]), ints([0] * 5))
    bare = F.Pages(p.pool, p.table, p.length)
    with pytest.raises(F.FerryError, match="null refs"):
        bare.trim(ints([0]))
    with pytest.raises(F.FerryError, match="null refs"):
        bare.compact()
    p.reserve(ints([]), ints([]))  # nothing to do
    p.check()


def test_tables_and_counts_that_contradict_each_other():
    p = F.Pages.empty(1, 1, 12, 6, 4, F.BF16)
    p.reserve(ints([0, 1]), ints([40, 33]))  # pages 0 1 2 and 3 4 5
    p.fork(ints([0, 0]), ints([2, 3]))
    p.check()
    p.refs[1] = 0  # in three tables
    p.trim(ints([0, 2, 3]))
    with pytest.raises(F.FerryError) as e:
        p.check()
    assert e.value.code == ESTATE
    # the pages' counts are those of free ones, not of 2^32 - 1 uses
    assert p.refs.tolist() == [0, 0, 0, 1, 1, 1] + [0] * 6
    p.table[1, 1] = 77  # no page of the pool
    for call in (lambda: p.fork(ints([1]), ints([2])), lambda: p.trim(ints([2])), lambda: p.trim(ints([1]))):
        call()
        with pytest.raises(F.FerryError) as e:
            p.check()
        assert e.value.code == ESTATE
    assert p.refs.tolist() == [0, 0, 0, 0, 1, 0] + [0] * 6  # page 4 is in no table any more
    assert not p.length.any() and torch.all(p.table == -1)
    p.refs[4] = 0
    p.reserve(ints([5]), ints([64]))
    p.check()
    assert p.table[5].tolist() == [0, 1, 2, 3]
    # reserve: nothing of the call is done
    p.trim(ints([5]), ints([50]))
    p.table[5, 3] = -1
    p.reserve(ints([4, 5]), ints([20, 1]))
    with pytest.raises(F.FerryError) as e:
        p.check()
    assert e.value.code == ESTATE
    assert p.length.tolist() == [0, 0, 0, 0, 0, 50] and torch.all(p.table[4] == -1)


def test_lists_that_are_the_cache_s_own():
    p = F.Pages.empty(1, 1, 40, 6, 4, F.BF16)
    p.reserve(ints([0, 1, 2]), ints([1, 2, 0]))
    lanes = ints([5, 0, 1, 2, 3, 4])
    for call in (lambda: p.trim(lanes, p.length), lambda: p.trim(p.length[3:]), lambda: p.reserve(p.table[0], lanes),
                 lambda: p.reserve(p.length, lanes), lambda: p.fork(p.refs[30:31], ints([3])),
                 lambda: p.compact(p.refs[39:])):
        with pytest.raises(F.FerryError, match="own table, len or refs"):
            call()
    p.reserve(lanes, p.length)
    assert p.length.tolist() == [1 + 2, 2 + 0, 0, 0, 0, 1]
    p.fork(ints([0, 0]), ints([2, 3]), p.length[:2])
    assert p.length.tolist() == [3, 2, 3, 2, 0, 1]
    p.check()


@pytest.mark.parametrize("n,tokens", [(5, 2000), (1500, 20)])
def test_lanes_that_grow_by_other_lanes_lengths(n, tokens):
    # more than the plan hands out by itself: another launch, whose workgroups write lengths
    # and read how far lanes grow.  The list goes against the lanes' order.
    b = Both(2 * n * (tokens // T + 3), n, 2 * tokens // T + 4, F.FP8, 1, 1)
    order = list(range(n))[::-1]
    first = [tokens - i % 9 for i in range(n)]
    assert b.call("reserve", list(range(n)), first) == 0
    b.p.reserve(ints(order), b.p.length)
    b.l.reserve(order, first)
    b.p.check()
    b.same()


def test_an_error_found_on_another_stream():
    p = F.Pages.empty(1, 1, 8, 4, 4, F.BF16)
    bad, s = ints([9]), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(2):
        with torch.cuda.stream(s):
            torch.cuda._sleep(20_000_000)  # still to come when the check begins
            p.trim(bad)
        with pytest.raises(F.FerryError) as e:
            p.check()
        assert e.value.code == EINVAL
    p.check()


@pytest.mark.parametrize("n,pages", [(1, 256), (1, 257), (16, 200), (17, 129), (64, 64), (65, 64), (900, 3)])
def test_forks_on_both_sides_of_one_launch(n, pages):
    b = Both(3 * pages + 4, n + 3, pages, F.FP8, 1, 1)
    assert b.call("reserve", [n, n + 1, n + 2], [16 * pages, 16 * pages - 7, 5]) == 0
    assert b.call("fork", [n + i % 3 for i in range(n)], list(range(n))[::-1]) == 0


@pytest.mark.parametrize("n", [3, 1100])
def test_growth_past_31_bits_is_refused(n):
    b = Both(n + 20, n, 9, F.BF16, 1, 1)
    assert b.call("reserve", list(range(n)), [1 + i % 16 for i in range(n)]) == 0
    for t in (2 ** 31 - 1, 2 ** 31 - 16, 9 * 16):
        assert b.call("reserve", [2, 1, 0] + list(range(3, n)), [0, t, 0] + [0] * (n - 3)) == ECAPACITY
