"""Attention of drafts and windows where one workgroup takes many steps of a tile in a
row: a tile for each CU, so that the places of K and V in LDS come round, and the page
ids and scales of a tile go on from 64 pages to the next, several times. Against
softmax attention in float64 as in test_gpu_seen, with its tolerance."""
import numpy as np
import pytest
import torch

import ferry_amd as F

from test_gpu_seen import Seen, spoil, tree_of

pytestmark = pytest.mark.gpu

T = 16
DTYPES = [F.BF16, F.F16, F.FP8]


def trees(seed, new):
    rng = np.random.default_rng(seed)
    return [tree_of(rng, n)[1] for n in new]


def clean_rows(c, places):
    """[rows, 1]: whether a row sees none of `places`, (request, token)."""
    clean = torch.ones((c.rows, 1), dtype=torch.bool, device="cuda")
    for r, t in places:
        clean[int(c.start[r]):int(c.start[r + 1]), 0] &= torch.from_numpy(~c.visible(r)[:, t]).cuda()
    return clean


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("lo,hi", [(40, 64), (20, 30), (8, 16)])  # 256, 128 and 32 to 64 rows
def test_runs_of_many_steps_with_trees(dt, lo, hi):
    rng = np.random.default_rng(lo)
    n = 36
    new = rng.integers(lo, hi + 1, n).tolist()
    lens = rng.integers(3000, 5000, n).tolist()
    c = Seen(dt, 32, 8, lens, new, masks=trees(lo, new), seed=lo)
    out, lse = c.run()
    c.check(out, lse)
    again = c.run()
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("new", [24, 40, 64, 80])  # on both sides of the widest tiles' rule
@pytest.mark.parametrize("sinks", [4, 1100])
def test_runs_of_many_steps_with_windows(dt, new, sinks):
    rng = np.random.default_rng(new)
    n = 32
    lens = rng.integers(5300, 6500, n).tolist()
    c = Seen(dt, 32, 8, lens, [new] * n, window=4096, sinks=sinks, seed=new)
    out, lse = c.run()
    c.check(out, lse)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("new", [24, 40, 64])
def test_values_not_finite_late_in_a_run(dt, new):
    """In the last steps of a run of more than 64 pages: rows that do not see them have
    their result all the same."""
    rng = np.random.default_rng(new)
    n = 32
    lens = rng.integers(3000, 4000, n).tolist()
    masks = trees(new, [new] * n)
    c = Seen(dt, 32, 8, lens, [new] * n, masks=masks, seed=new)
    want = [x.clone() for x in c.run()]
    before = c.p.pool.clone()
    places = [(r, lens[r] - new // 2 + r % 3) for r in range(0, n, 3)]
    spoil(c, dt, float("nan"), places)
    got = c.run()
    c.p.pool.copy_(before)
    clean = clean_rows(c, places)
    assert clean.any() and not clean.all()
    assert torch.all(torch.isnan(got[0][~clean[:, 0]].float()))
    c.check(torch.where(clean.unsqueeze(2), got[0], want[0]), torch.where(clean, got[1], want[1]))


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("new", [24, 40, 64])
def test_scales_not_finite_late_in_a_run(new, which):
    """A K or V scale of a page that holds drafts only, late in a run."""
    rng = np.random.default_rng(new)
    n = 32
    lens = rng.integers(3000, 4000, n).tolist()
    masks = trees(new, [new] * n)
    places = []
    for r in range(n):
        page = lens[r] // T - 1  # whole, and behind the context where it is the drafts' own
        if r % 4 == 0 and page * T >= lens[r] - new:
            first = page * T - (lens[r] - new)
            masks[r][:, first:first + T] &= np.arange(new)[:, None] % 2 == 0  # half of the rows see none of it
            places += [(r, page * T + i) for i in range(T)]
    c = Seen(F.FP8, 32, 8, lens, [new] * n, masks=masks, seed=new)
    want = [x.clone() for x in c.run()]
    finite = c.p.scales.clone()
    for r, t in places:
        c.p.scales[c.layer, int(c.p.table[int(c.lanes[r]), t // T]), :, which] = float("nan")
    got = c.run()
    c.p.scales.copy_(finite)
    clean = clean_rows(c, places)
    assert places and clean.any() and not clean.all()
    assert torch.all(torch.isnan(got[0][~clean[:, 0]].float()))
    c.check(torch.where(clean.unsqueeze(2), got[0], want[0]), torch.where(clean, got[1], want[1]))


@pytest.mark.parametrize("dt", DTYPES + [F.F32])
@pytest.mark.parametrize("new", [[257, 300], [700, 65], [4096]])
def test_trees_of_many_words(dt, new):
    """5, 11 and 64 words of bits."""
    c = Seen(dt, 4, 1, [x + 40 for x in new], new, masks=trees(3, new), seed=len(new))
    c.check(*c.run())
    if len(new) > 1:
        c.window, c.sinks = 50, 3
        c.check(*c.run())
