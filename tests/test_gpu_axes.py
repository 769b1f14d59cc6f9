"""Rotary positions on several axes, apart from the tokens' places, against the
formula in float64 (tolerance: test_gpu_append's)."""
import numpy as np
import pytest
import torch

import ferry_amd as F

from test_gpu_append import D, HALF, T, TORCH, Case, freqs, ints, near

pytestmark = pytest.mark.gpu


def turned(x, at, axis, freq, factor, pairs):
    """The formula in float64, and |a| + |b| of each value's pair; at [axes, tokens]."""
    x = x.double().cpu().numpy()
    y, size = x.copy(), np.abs(x)
    r = 2 * len(freq)
    ang = (at[axis].T.astype(np.float64) * freq)[:, None, :]
    c, s = factor * np.cos(ang), factor * np.sin(ang)
    ia = np.arange(0, r, 2) if pairs else np.arange(r // 2)
    ib = ia + 1 if pairs else ia + r // 2
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    size[..., ia] = size[..., ib] = np.abs(a) + np.abs(b)
    return y, size


def check(c, layer, q_out, at, axis, freq, factor, pairs):
    p = c.p
    torch.cuda.synchronize()
    p.check()
    near(q_out, *turned(c.q, at, axis, freq, factor, pairs), factor, {v: k for k, v in TORCH.items()}[q_out.dtype])
    page = p.table.cpu().numpy()[c.lane, c.pos // T].astype(np.int64)
    got = p.pool.view(torch.uint8)[layer][page, :, :, c.pos % T].view(TORCH[c.pt])
    want, size = turned(c.k, at, axis, freq, factor, pairs)
    value = c.v.double().cpu().numpy()
    if c.kv is not None:
        sc = c.kv.double().cpu().numpy()
        near(got[:, :, 0].float(), want, size, factor, c.pt, sc[None, :, :1])
        near(got[:, :, 1].float(), value, np.abs(value), 1.0, c.pt, sc[None, :, 1:])
    else:
        near(got[:, :, 0], want, size, factor, c.pt)
        near(got[:, :, 1], value, np.abs(value), 1.0, c.pt)
    raw = p.pool.view(torch.uint8).clone()
    raw[layer, page, :, :, c.pos % T] = c.before[layer, page, :, :, c.pos % T]
    assert torch.equal(raw, c.before)


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("rot", [2, 6, 20, 32, 96, 128])
@pytest.mark.parametrize("axes", [1, 2, 3, 4])
@pytest.mark.parametrize("xt,pt,ot", [(F.BF16, F.BF16, F.BF16), (F.F16, F.F16, F.F32), (F.BF16, F.FP8, F.BF16),
                                      (F.F32, F.F32, F.F32)])
def test_axes_match_the_formula(xt, pt, ot, axes, rot, pairs):
    c = Case(xt, pt, 6, 3, [1, 16, 37, 333, 64], [1, 3, 37, 40, 1], seed=rot)
    f, df = freqs(rot, base=10000.0)
    rng = np.random.default_rng(axes)
    rows = len(c.pos)
    at = rng.integers(-50, 3000, (axes, rows))
    at[0, :3] = [2 ** 24 - 1, 0, -2 ** 20]
    for axis in (rng.integers(0, axes, rot // 2), np.arange(rot // 2) % axes):
        q_out = torch.empty(c.q.shape, dtype=TORCH[ot], device="cuda")
        c.p.append(1, ints(c.lane), ints(c.pos), k=c.k, v=c.v, q=c.q, q_out=q_out, inv_freq=df, factor=1.25, pairs=pairs,
                   kv_scale=c.kv, at=ints(at), axis=ints(axis))
        check(c, 1, q_out, at, axis, f, 1.25, pairs)
    if axes == 1:  # one axis needs no list, and no second dimension
        again = torch.empty_like(q_out)
        c.p.append(1, ints(c.lane), ints(c.pos), k=c.k, v=c.v, q=c.q, q_out=again, inv_freq=df, factor=1.25, pairs=pairs,
                   kv_scale=c.kv, at=ints(at[0]))
        torch.cuda.synchronize()
        assert torch.equal(again, q_out)


@pytest.mark.parametrize("xt,pt", [(F.BF16, F.BF16), (F.F32, F.FP8)])
def test_positions_that_are_the_places(xt, pt):
    c = Case(xt, pt, 8, 2, [100, 33], [50, 33], seed=1)
    _, df = freqs(64)
    outs, pools = [], []
    for kw in ({}, dict(at=ints(c.pos)), dict(at=ints(np.stack([c.pos, c.pos])), axis=ints(np.arange(32) % 2))):
        out = torch.empty_like(c.q)
        c.p.append(0, ints(c.lane), ints(c.pos), k=c.k, v=c.v, q=c.q, q_out=out, inv_freq=df, kv_scale=c.kv, **kw)
        torch.cuda.synchronize()
        c.p.check()
        outs.append(out)
        pools.append(c.p.pool.clone().view(torch.uint8))
    for x, y in zip(outs[1:], pools[1:]):
        assert torch.equal(x, outs[0]) and torch.equal(y, pools[0])


def test_strides_of_the_axes_queries_alone_and_in_place():
    c = Case(F.F16, F.F16, 6, 3, [40], [40], seed=2)
    f, df = freqs(128)
    rng = np.random.default_rng(0)
    at = rng.integers(0, 500, (3, 40))
    axis = np.arange(64) * 3 // 64
    wide = torch.zeros((3, 101), dtype=torch.int32, device="cuda")
    wide[:, 7:47] = ints(at)
    q = c.q.clone()
    c.p.append(0, None, ints(c.pos), q=q, q_out=q, inv_freq=df, at=wide[:, 7:47], axis=ints(axis))
    torch.cuda.synchronize()
    c.p.check()
    near(q, *turned(c.q, at, axis, f, 1.0, False), 1.0, F.F16)
    assert torch.equal(c.p.pool.view(torch.uint8), c.before)


def test_padding_and_tokens_without_a_place():
    c = Case(F.BF16, F.BF16, 4, 2, [20, 40], [20, 40], seed=3)
    f, df = freqs(32)
    lane, pos = c.lane.copy(), c.pos.copy()
    lane[5] = -1
    pos[9] = 40 if lane[9] == 1 else 20  # behind the lane's end
    at = np.arange(60)[None] + 7
    out = torch.full_like(c.q, 9.0)
    c.p.append(0, ints(lane), ints(pos), k=c.k, v=c.v, q=c.q, q_out=out, inv_freq=df, at=ints(at))
    torch.cuda.synchronize()
    with pytest.raises(F.FerryError) as e:
        c.p.check()
    assert e.value.code == -3
    assert torch.all(out[[5, 9]] == 9.0)
    kept = [i for i in range(60) if i not in (5, 9)]
    near(out[kept], *turned(c.q[kept], at[:, kept], np.zeros(16, int), f, 1.0, False), 1.0, F.BF16)


def test_an_axis_out_of_range_is_reported():
    c = Case(F.BF16, F.BF16, 4, 2, [20], [20], seed=4)
    f, df = freqs(32)
    at = np.stack([np.arange(20), np.arange(20) * 3])
    for bad in (2, -1, 2 ** 31 - 1):
        axis = np.arange(16) % 2
        axis[3] = bad
        out = torch.empty_like(c.q)
        c.p.append(0, ints(c.lane), ints(c.pos), k=c.k, v=c.v, q=c.q, q_out=out, inv_freq=df, at=ints(at), axis=ints(axis))
        torch.cuda.synchronize()
        with pytest.raises(F.FerryError) as e:
            c.p.check()
        assert e.value.code == -3
        axis[3] = 0
        near(out, *turned(c.q, at, axis, f, 1.0, False), 1.0, F.BF16)


def test_a_captured_call_follows_the_positions():
    c = Case(F.BF16, F.BF16, 8, 2, [100], [30], seed=5)
    f, df = freqs(64)
    at, axis = ints(np.zeros((2, 30))), ints(np.arange(32) % 2)
    lane, pos = ints(c.lane), ints(c.pos)
    out = torch.empty_like(c.q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.p.append(0, lane, pos, k=c.k, v=c.v, q=c.q, q_out=out, inv_freq=df, at=at, axis=axis)
    rng = np.random.default_rng(1)
    for _ in range(3):
        new = rng.integers(0, 9000, (2, 30))
        at.copy_(ints(new))
        graph.replay()
        check(c, 0, out, new, np.arange(32) % 2, f, 1.0, False)


def test_refusals():
    c = Case(F.BF16, F.BF16, 4, 2, [20], [20], seed=6)
    _, df = freqs(32)
    out = torch.empty_like(c.q)

    def call(**kw):
        c.p.append(0, ints(c.lane), ints(c.pos), k=c.k, v=c.v, q=c.q, q_out=out, inv_freq=df, **kw)

    at = ints(np.zeros((2, 20)))
    axis = ints(np.zeros(16))
    for bad in (at.cpu(), at.long(), at[:, :19], at.t().contiguous().t(), at[0, 0], at.unsqueeze(0)):
        with pytest.raises(ValueError, match="at: "):
            call(at=bad, axis=axis)
    with pytest.raises(ValueError, match="axis"):
        call(axis=axis)
    with pytest.raises(ValueError, match="axis"):
        call(at=at, axis=axis[:15])
    with pytest.raises(F.FerryError, match="several axes"):
        call(at=at)
    with pytest.raises(F.FerryError, match="n_axes"):
        call(at=ints(np.zeros((5, 20))), axis=axis)
    torch.cuda.synchronize()
    c.p.check()
    assert torch.equal(c.p.pool.view(torch.uint8), c.before)
    assert D == 128 and HALF
