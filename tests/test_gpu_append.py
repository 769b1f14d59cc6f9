"""Rotary positions and the write into pages on the GPU against the formula in
float64.

Tolerance: an angle is reduced in 64 bits, its cosine and sine rounded to fp32
and multiplied by the factor (2^-24 relative each, and 2^-23 for the fp32
functions), a rotated value is two products and a sum (3 x 2^-24): together
under 2^-20 of factor (|a| + |b|).  Then one rounding, half a step of the
output's type."""
import numpy as np
import pytest
import torch

import ferry_amd as F

pytestmark = pytest.mark.gpu

T, D = 16, 128
TORCH = {F.F32: torch.float32, F.F16: torch.float16, F.BF16: torch.bfloat16, F.FP8: torch.float8_e4m3fn}
# half a step relative to the value, and of the smallest (denormal) values
HALF = {F.F32: (2.0 ** -24, 2.0 ** -150), F.F16: (2.0 ** -11, 2.0 ** -25), F.BF16: (2.0 ** -8, 2.0 ** -134),
        F.FP8: (2.0 ** -4, 2.0 ** -10)}


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def turned(x, pos, freq, factor, pairs):
    """The formula in float64, and |a| + |b| of each value's pair."""
    x = x.double().cpu().numpy()
    y, size = x.copy(), np.abs(x)
    r = 2 * len(freq)
    ang = np.asarray(pos, np.float64)[:, None, None] * freq
    c, s = factor * np.cos(ang), factor * np.sin(ang)
    ia = np.arange(0, r, 2) if pairs else np.arange(r // 2)
    ib = ia + 1 if pairs else ia + r // 2
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    size[..., ia] = size[..., ib] = np.abs(a) + np.abs(b)
    return y, size


def near(got, want, size, factor, dt, scale=1.0):
    rel, tiny = HALF[dt]
    got = got.double().cpu().numpy()
    if dt == F.FP8:
        want = np.clip(want / scale, -448.0, 448.0)
        err = size / scale * factor * 2.0 ** -20
    else:
        err = size * factor * 2.0 ** -20
    assert np.all(np.isfinite(got))
    bound = err + rel * (np.abs(want) + err) + tiny
    worst = np.max(np.abs(got - want) / bound)
    assert worst <= 1.0, worst


class Case:
    def __init__(self, xt, pt, Hq, H, lengths, new, layers=2, refs=True, seed=0):
        """Lanes that hold `lengths` tokens, the last `new` of which are appended."""
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        n = len(lengths)
        pages = [-(-x // T) for x in lengths]
        self.p = F.Pages.empty(layers, H, sum(pages) + 3, n, max(pages) + 1, pt)
        p = self.p
        if not refs:
            p = self.p = F.Pages(p.pool, p.table, p.length, scales=p.scales, dtype=pt)
        raw = p.pool.view(torch.uint8)
        raw.copy_(torch.randint(0, 256, raw.shape, device="cuda", generator=self.g, dtype=torch.uint8))
        order = torch.randperm(sum(pages), device="cuda", generator=self.g).to(torch.int32) + 1
        at = 0
        for i, x in enumerate(pages):
            p.table[i, :x] = order[at:at + x]
            at += x
        p.length.copy_(ints(lengths))
        if refs:
            p.refs[order.long()] = 1
        self.lane = np.repeat(np.arange(n), new)
        self.pos = np.concatenate([np.arange(x - k, x) for x, k in zip(lengths, new)]).astype(np.int64)
        rows = len(self.lane)
        perm = np.random.default_rng(seed).permutation(rows)  # tokens in any order
        self.lane, self.pos = self.lane[perm], self.pos[perm]
        self.q, self.k, self.v = (torch.randn((rows, h, D), device="cuda", generator=self.g).to(TORCH[xt])
                                  for h in (Hq, H, H))
        self.xt, self.pt = xt, pt
        self.kv = None
        if pt == F.FP8:
            self.kv = 0.004 + 0.01 * torch.rand((H, 2), device="cuda", generator=self.g)
        self.before = raw.clone()

    def check(self, layer, q_out, freq, factor, pairs, dropped=()):
        p = self.p
        p.check() if not len(dropped) else None
        kept = np.array([i for i in range(len(self.lane)) if i not in set(dropped)])
        if q_out is not None:
            want, size = turned(self.q[kept], self.pos[kept], freq, factor, pairs)
            near(q_out[kept], want, size, factor, {v: k for k, v in TORCH.items()}[q_out.dtype])
        table = p.table.cpu().numpy()
        lane, pos = self.lane[kept], self.pos[kept]
        page = table[lane, pos // T].astype(np.int64)
        got = p.pool.view(torch.uint8)[layer][page, :, :, pos % T]
        got = got.view(TORCH[self.pt])
        want, size = turned(self.k[kept], pos, freq, factor, pairs)
        value = self.v[kept].double().cpu().numpy()
        if self.kv is not None:
            sc = self.kv.double().cpu().numpy()
            near(got[:, :, 0].float(), want, size, factor, self.pt, sc[None, :, :1])
            near(got[:, :, 1].float(), value, np.abs(value), 1.0, self.pt, sc[None, :, 1:])
            for i in set(page.tolist()):
                assert torch.equal(p.scales[layer, i], self.kv)
        else:
            near(got[:, :, 0], want, size, factor, self.pt)
            near(got[:, :, 1], value, np.abs(value), 1.0, self.pt)
        # nothing else of the pool changed
        raw = p.pool.view(torch.uint8).clone()
        raw[layer, page, :, :, pos % T] = self.before[layer, page, :, :, pos % T]
        assert torch.equal(raw, self.before)


def freqs(rot, kind=F.ROPE_PLAIN, **kw):
    f = F.rope_freqs(kind, rot, **kw)
    return f, torch.from_numpy(f).cuda()


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("rot", [2, 6, 20, 32, 64, 96, 128])
@pytest.mark.parametrize("xt,pt,ot", [(F.BF16, F.BF16, F.BF16), (F.F16, F.F16, F.F32), (F.BF16, F.FP8, F.BF16),
                                      (F.F32, F.F32, F.F32), (F.F32, F.BF16, F.F16), (F.F16, F.FP8, F.F16)])
def test_append_matches_the_formula(xt, pt, ot, rot, pairs):
    c = Case(xt, pt, 6, 3, [1, 16, 37, 333, 64], [1, 3, 37, 40, 1], seed=rot)
    f, df = freqs(rot, base=10000.0)
    out = torch.empty(c.q.shape, dtype=TORCH[ot], device="cuda")
    c.p.append(1, ints(c.lane), ints(c.pos), k=c.k, v=c.v, q=c.q, q_out=out, inv_freq=df, factor=1.25,
               pairs=pairs, kv_scale=c.kv)
    torch.cuda.synchronize()
    c.check(1, out, f, 1.25, pairs)


@pytest.mark.parametrize("xt,pt", [(F.BF16, F.BF16), (F.F16, F.FP8), (F.F32, F.F32)])
@pytest.mark.parametrize("Hq,H,rows", [(1, 1, 1), (8, 1, 3), (20, 20, 5), (64, 8, 70), (12, 3, 9)])
def test_head_counts_and_far_positions(xt, pt, Hq, H, rows):
    c = Case(xt, pt, Hq, H, [rows + 7, 3], [rows, 2], layers=1, seed=Hq)
    # the same places with rotary positions far into a long context: lanes of the
    # longest row a table may have
    f, df = freqs(128, F.ROPE_PARTS, base=500000.0, stretch=32.0, trained_ctx=8192.0)
    far = (1 << 20) - 64
    wide = torch.full((2, far // T + 8), -1, dtype=torch.int32, device="cuda")
    wide[:, far // T:far // T + c.p.table.shape[1]] = c.p.table[:, :8]
    p = F.Pages(c.p.pool, wide, c.p.length + far, refs=c.p.refs, scales=c.p.scales, dtype=pt)
    c.p, c.pos = p, c.pos + far
    out = torch.empty_like(c.q)
    p.append(0, ints(c.lane), ints(c.pos), k=c.k, v=c.v, q=c.q, q_out=out, inv_freq=df, kv_scale=c.kv)
    torch.cuda.synchronize()
    c.check(0, out, f, 1.0, False)


@pytest.mark.parametrize("xt,pt", [(F.BF16, F.BF16), (F.F32, F.FP8)])
@pytest.mark.parametrize("how", ["fused", "odd rows", "heads apart", "off by one"])
def test_strides_and_alignment(xt, pt, how):
    Hq, H = 4, 2
    c = Case(xt, pt, Hq, H, [40, 21], [33, 9], seed=5)
    f, df = freqs(64, base=10000.0)
    rows = len(c.lane)

    def place(x):
        h = x.shape[1]
        if how == "fused":
            big = torch.zeros((rows, Hq + 2 * H + 1, D), dtype=x.dtype, device="cuda")
            y = big[:, 1:1 + h]
        elif how == "odd rows":
            y = torch.zeros((rows, h * D + 3), dtype=x.dtype, device="cuda")[:, :h * D].view(rows, h, D)
        elif how == "heads apart":
            y = torch.zeros((h, rows + 2, D), dtype=x.dtype, device="cuda")[:, :rows].transpose(0, 1)
        else:
            y = torch.zeros(rows * h * D + 1, dtype=x.dtype, device="cuda")[1:].view(rows, h, D)
        y.copy_(x)
        return y

    q, k, v, out = place(c.q), place(c.k), place(c.v), place(torch.zeros_like(c.q))
    c.p.append(0, ints(c.lane), ints(c.pos), k=k, v=v, q=q, q_out=out, inv_freq=df, kv_scale=c.kv)
    torch.cuda.synchronize()
    c.check(0, out, f, 1.0, False)


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("rot", [20, 64, 128])
def test_queries_in_place_alone_and_keys_alone(rot, pairs):
    c = Case(F.BF16, F.BF16, 5, 2, [50], [50], seed=2)
    f, df = freqs(rot, base=10000.0)
    out = c.q.clone()
    c.p.append(0, None, ints(c.pos), q=out, q_out=out, inv_freq=df, pairs=pairs)
    torch.cuda.synchronize()
    assert torch.equal(c.p.pool.view(torch.uint8), c.before)
    want, size = turned(c.q, c.pos, f, 1.0, pairs)
    near(out, want, size, 1.0, F.BF16)
    c.p.append(0, ints(c.lane), ints(c.pos), k=c.k, v=c.v, inv_freq=df, pairs=pairs)
    torch.cuda.synchronize()
    c.check(0, None, f, 1.0, pairs)


@pytest.mark.parametrize("pt", [F.F16, F.FP8])
def test_tokens_without_a_place_are_left_out(pt):
    c = Case(F.F16, pt, 4, 2, [20, 40, 16], [4, 40, 1], seed=3)
    f, df = freqs(128, base=10000.0)
    sentinel = 7.0
    # padding; behind the lane's end; no such lane; before its start; a hole in the table
    lane, pos = c.lane.copy(), c.pos.copy()
    drop = [1, 5, 9, 12, 20]
    lane[1] = -1
    lane[5], pos[5] = 0, 20
    lane[9] = 3
    pos[12] = -1
    holes = [i for i in range(len(pos)) if c.lane[i] == 1 and c.pos[i] // T == 1 and i not in drop]
    assert holes
    kept_entry = int(c.p.table[1, 1])
    c.p.table[1, 1] = c.p.pool.shape[1]  # a page the pool does not have
    out = torch.full(c.q.shape, sentinel, dtype=torch.float16, device="cuda")
    c.p.append(0, ints(lane), ints(pos), k=c.k, v=c.v, q=c.q, q_out=out, inv_freq=df, kv_scale=c.kv)
    with pytest.raises(F.FerryError) as e:
        c.p.check()
    assert e.value.code == -3
    c.p.table[1, 1] = kept_entry
    gone = sorted(set(drop) | set(holes))
    assert torch.all(out[gone] == sentinel)
    c.check(0, out, f, 1.0, False, dropped=gone)


def test_padding_alone_is_no_error():
    c = Case(F.BF16, F.BF16, 4, 2, [20], [4], seed=3)
    f, df = freqs(128, base=10000.0)
    lane = c.lane.copy()
    lane[[0, 3]] = -1
    out = torch.zeros_like(c.q)
    c.p.append(0, ints(lane), ints(c.pos), k=c.k, v=c.v, q=c.q, q_out=out, inv_freq=df)
    c.p.check()
    assert not torch.any(out[[0, 3]])
    c.check(0, out, f, 1.0, False, dropped=[0, 3])


def test_a_shared_page_is_not_written():
    c = Case(F.BF16, F.BF16, 4, 2, [20, 33], [20, 33], seed=4)
    f, df = freqs(128, base=10000.0)
    page = int(c.p.table[0, 1])
    c.p.refs[page] = 2
    c.p.append(0, ints(c.lane), ints(c.pos), k=c.k, v=c.v, inv_freq=df)
    with pytest.raises(F.FerryError) as e:
        c.p.check()
    assert e.value.code == -7
    gone = [i for i in range(len(c.lane)) if c.lane[i] == 0 and c.pos[i] >= 16]
    c.check(0, None, f, 1.0, False, dropped=gone)


def test_a_cache_without_counts():
    c = Case(F.BF16, F.BF16, 4, 2, [20, 33], [20, 33], refs=False, seed=4)
    f, df = freqs(128, base=10000.0)
    c.p.append(1, ints(c.lane), ints(c.pos), k=c.k, v=c.v, inv_freq=df)
    torch.cuda.synchronize()
    c.check(1, None, f, 1.0, False)


def test_values_out_of_the_8_bit_range_saturate():
    c = Case(F.F32, F.FP8, 1, 2, [16], [16], layers=1)
    f, df = freqs(2, base=10000.0)
    c.v *= 1e6
    c.v[3] = 0.0
    c.v[5] = 1e-6
    c.p.append(0, ints(c.lane), ints(c.pos), k=c.k, v=c.v, inv_freq=df, kv_scale=c.kv)
    torch.cuda.synchronize()
    c.check(0, None, f, 1.0, False)


@pytest.mark.parametrize("offset", [0, 1])  # 16-byte aligned, and not
def test_quotients_at_the_ends_of_fp32(offset):
    # infinities and quotients past fp32 saturate, NaN stays, zero stays zero, and scales
    # whose inverse is no fp32 number divide all the same
    x = [1e30, -1e30, np.inf, -np.inf, np.nan, 0.0, -0.0, 1e-39, 3e-39, 7e-40, 1e38, 2.0 ** 127]
    for s in (1e-10, 1e-40, 2.0 ** -149, 2.0 ** 127, 1e38, 1.0):
        p = F.Pages.empty(1, 1, 1, 1, 1, F.FP8)
        p.reserve(ints([0]), ints([16]))
        buf = torch.zeros(2 * 128 + offset, device="cuda")
        k, v = buf[offset:offset + 128].view(1, 1, 128), buf[offset + 128:].view(1, 1, 128)
        v[0, 0, :len(x)] = torch.tensor(x)
        p.append(0, ints([0]), ints([3]), k=k, v=v, inv_freq=torch.ones(64, dtype=torch.float64, device="cuda"),
                 kv_scale=torch.tensor([[1.0, s]], device="cuda"))
        torch.cuda.synchronize()
        p.check()
        f = np.float32(s).astype(np.float64)
        with np.errstate(all="ignore"):
            want = np.clip(np.float32(x).astype(np.float64) / f, -448.0, 448.0)
        got = p.pool[0, 0, 0, 1, 3, :len(x)].double().cpu().numpy()
        # half a step of E4M3 (2^-4 relative, 2^-10 below the normal range), and of fp32
        bound = np.abs(want) * (2.0 ** -4 + 2.0 ** -23) + 2.0 ** -10
        assert np.array_equal(np.isnan(got), np.isnan(want)), (s, got)
        ok = ~np.isnan(want)
        assert np.all(np.abs(got - want)[ok] <= bound[ok]), (s, got, want)


def test_a_pool_past_four_gibibytes():
    H, P = 8, 70000
    p = F.Pages.empty(1, H, P, 1, 2, F.BF16)
    p.table[0, 0] = P - 1
    p.length[0] = 3
    k = torch.randn((1, H, D), device="cuda").to(torch.bfloat16)
    _, df = freqs(64, base=10000.0)
    p.append(0, ints([0]), ints([0]), k=k, v=-k, inv_freq=df)
    p.check()
    assert torch.equal(p.pool[0, P - 1, :, 0, 0], k[0]) and torch.equal(p.pool[0, P - 1, :, 1, 0], -k[0])


def test_captured_and_on_another_stream():
    c = Case(F.BF16, F.BF16, 4, 2, [20, 33], [20, 33], seed=6)
    f, df = freqs(64, base=10000.0)
    lane, pos, out = ints(c.lane), ints(c.pos), torch.empty_like(c.q)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        c.p.append(1, lane, pos, k=c.k, v=c.v, q=c.q, q_out=out, inv_freq=df)
    for _ in range(3):
        out.zero_()
        c.p.pool.view(torch.uint8).copy_(c.before)
        graph.replay()
        torch.cuda.synchronize()
        c.check(1, out, f, 1.0, False)
    c.p.pool.view(torch.uint8).copy_(c.before)
    torch.cuda.synchronize()
    c.p.append(0, lane, pos, k=c.k, v=c.v, q=c.q, q_out=out, inv_freq=df, stream=s)
    torch.cuda.synchronize()
    c.check(0, out, f, 1.0, False)


def test_no_tokens():
    c = Case(F.BF16, F.BF16, 4, 2, [20], [4])
    _, df = freqs(64, base=10000.0)
    c.p.append(0, ints([]), ints([]), k=c.k[:0], v=c.v[:0], q=c.q[:0], q_out=c.q[:0].clone(), inv_freq=df)
    c.p.check()
    assert torch.equal(c.p.pool.view(torch.uint8), c.before)


def test_refusals_on_the_host():
    c = Case(F.BF16, F.FP8, 4, 2, [20], [4])
    _, df = freqs(64, base=10000.0)
    lane, pos = ints(c.lane), ints(c.pos)
    with pytest.raises(ValueError, match="shape"):
        c.p.append(0, lane, pos, k=c.k[:, :1], v=c.v, inv_freq=df, kv_scale=c.kv)
    with pytest.raises(ValueError, match="kv_scale"):
        c.p.append(0, lane, pos, k=c.k, v=c.v, inv_freq=df)
    with pytest.raises(ValueError, match="contiguous"):
        c.p.append(0, lane, pos, k=c.k[:, :, ::2].repeat(1, 1, 2).transpose(1, 2).contiguous().transpose(1, 2),
                   v=c.v, inv_freq=df, kv_scale=c.kv)
    with pytest.raises(ValueError, match="dtype"):
        c.p.append(0, lane, pos, k=c.k, v=c.v.float(), inv_freq=df, kv_scale=c.kv)
    with pytest.raises(F.FerryError, match="layer"):
        c.p.append(2, lane, pos, k=c.k, v=c.v, inv_freq=df, kv_scale=c.kv)
    with pytest.raises(F.FerryError, match="other"):
        c.p.append(0, None, pos, q=c.q, q_out=c.q.flatten().as_strided(c.q.shape, (128, 128, 1)), inv_freq=df)


def test_no_frequencies():
    p = F.Pages.empty(1, 1, 1, 1, 1, F.F16)
    with pytest.raises(ValueError, match="inv_freq"):
        p.append(0, ints([0]), ints([0]), q=torch.zeros((1, 1, 128), device="cuda"),
                 q_out=torch.zeros((1, 1, 128), device="cuda"))


def test_more_tokens_than_a_launch_has_workgroups():
    # a workgroup per token, and a launch has fewer than 2^32 threads
    n = (1 << 24) + 40
    p = F.Pages.empty(1, 1, (1 << 20) + 3, 2, 1 << 20)
    p.table[0] = torch.arange(1 << 20, dtype=torch.int32, device="cuda")
    p.table[1, :3] = ints([(1 << 20) + i for i in range(3)])
    p.length.copy_(ints([1 << 24, 40]))
    at = torch.arange(n, dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randint(1, 1 << 14, (n, 1, D), device="cuda", generator=g, dtype=torch.int16).view(torch.bfloat16)
            for _ in range(2))
    p.append(0, at >> 24, at & ((1 << 24) - 1), k=k, v=v,
             inv_freq=torch.zeros(64, dtype=torch.float64, device="cuda"))  # no turn: the same bits
    p.check()
    for i, x in enumerate((k, v)):
        got = p.pool[0, :, 0, i].reshape(-1, D)[:n].view(torch.int16)
        assert torch.equal(got, x.view(torch.int16)[:, 0])
