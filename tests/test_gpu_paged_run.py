"""The calls of the paged KV cache together, as a server makes them: prompts in
ragged chunks, samples forked from a prompt, single tokens from a captured
graph over growing lengths, drafts taken back, lanes that end, and pages handed
to the executor's host tier.

Every token's K and V, read back through the lane's table, are the rotary
formula's within the append's rounding (whatever was forked, copied or moved
since), and every attention output is that of the pages' values in float64."""
import numpy as np
import pytest
import torch

import ferry_amd as F

from test_gpu_append import near, turned
from test_gpu_attend import TORCH, U, Case, ints
from test_gpu_parity import TOL

pytestmark = pytest.mark.gpu

T, D, L, H, HQ = 16, 128, 2, 2, 8
X = torch.bfloat16


class Server:
    """A cache and, for each lane, the K and V that its tokens were made of."""

    def __init__(self, dt, lanes=8, pages=60, max_pages=12):
        self.dt, self.p = dt, F.Pages.empty(L, H, pages, lanes, max_pages, dt)
        self.g = torch.Generator(device="cuda").manual_seed(11 + dt)
        self.freq = F.rope_freqs(F.ROPE_PARTS, 64, stretch=4.0, trained_ctx=64.0)
        self.inv = torch.from_numpy(self.freq).cuda()
        self.kv = 0.01 + 0.01 * torch.rand((H, 2), device="cuda", generator=self.g) if dt == F.FP8 else None
        self.held = [[] for _ in range(lanes)]  # (k, v) [L, H, 128] of every token

    def fresh(self, n):
        return [torch.randn((L, n, h, D), device="cuda", generator=self.g).to(X) for h in (HQ, H, H)]

    def tokens(self, lanes, new, **groups):
        """New tokens of several lanes through all layers, checked."""
        rows = sum(new)
        q, k, v = self.fresh(rows)
        lane = np.repeat(lanes, new)
        pos = np.concatenate([len(self.held[a]) + np.arange(n) for a, n in zip(lanes, new)])
        start = np.concatenate([[0], np.cumsum(new)])
        self.p.reserve(ints(lanes), ints(new))
        qr = torch.empty((L, rows, HQ, D), device="cuda", dtype=self.p.q_dtype)
        out = torch.empty_like(qr)
        lse = torch.empty((L, rows, HQ), device="cuda")
        for i in range(L):
            self.p.append(i, ints(lane), ints(pos), k=k[i], v=v[i], q=q[i], q_out=qr[i], inv_freq=self.inv,
                          factor=1.1, kv_scale=self.kv)
            self.p.attend(i, qr[i], out[i], ints(lanes), q_start=ints(start), lse=lse[i], **groups)
        self.took(lane, pos, q, k, v, qr)
        self.attended(lanes, new, qr, out, lse)

    def took(self, lane, pos, q, k, v, qr):
        torch.cuda.synchronize()
        self.p.check()
        q_type = F.BF16 if self.dt == F.FP8 else self.dt
        near(qr.flatten(0, 1), *turned(q.flatten(0, 1), np.tile(pos, L), self.freq, 1.1, False), 1.1, q_type)
        for t, a in enumerate(lane):
            self.held[a].append((k[:, t], v[:, t]))

    def attended(self, lanes, new, qr, out, lse):
        c = Case.__new__(Case)
        c.dt, c.Hq, c.H, c.p, c.lanes, c.new = self.dt, HQ, H, self.p, lanes, new
        c.lens = [len(self.held[a]) for a in lanes]
        c.start = np.concatenate([[0], np.cumsum(new)])
        for c.layer in range(L):
            c.q = qr[c.layer]
            c.check(out[c.layer], lse[c.layer])

    def same(self):
        """Every lane holds its tokens; no page is lost or used twice."""
        torch.cuda.synchronize()
        self.p.check()
        assert self.p.length.tolist() == [len(x) for x in self.held]
        table = self.p.table.cpu().numpy()
        uses = np.zeros(self.p.refs.numel(), int)
        for a, held in enumerate(self.held):
            n = -(-len(held) // T)
            assert np.all(table[a, n:] == -1)
            np.add.at(uses, table[a, :n], 1)
            if not held:
                continue
            ids = self.p.table[a, :n].long()
            got = self.p.pool.view(torch.uint8)[:, ids].view(TORCH[self.dt]).movedim(1, 3)  # [L, H, 2, n, 16, D]
            got = got.reshape(L, H, 2, n * T, D)[:, :, :, :len(held)].transpose(1, 3)  # [L, token, 2, H, D]
            for j, freq in ((0, self.freq), (1, self.freq * 0.0)):
                want = torch.stack([x[j] for x in held], 1)  # [L, token, H, D]
                y, size = turned(want.flatten(0, 1), np.tile(np.arange(len(held)), L), freq,
                                 1.0 if j else 1.1, False)
                for h in range(H):
                    scale = 1.0 if self.kv is None else float(self.kv[h, j])
                    near(got[:, :, j, h].flatten(0, 1), y[:, h], size[:, h], 1.1, self.dt, scale)
        assert self.p.refs.tolist() == uses.tolist()


@pytest.mark.parametrize("dt", [F.BF16, F.FP8, F.F16, F.F32])
def test_a_server_s_run(dt):
    s = Server(dt)
    s.tokens([0, 1, 2], [75, 33, 1])
    s.tokens([2, 0, 1], [16, 40, 1])
    s.same()
    s.p.fork(ints([0, 0, 0, 1]), ints([3, 4, 5, 6]), ints([115, 115, 115, 32]))
    for a in (3, 4, 5):
        s.held[a] = s.held[0][:]
    s.held[6] = s.held[1][:32]
    s.same()

    # single tokens of all lanes from a captured graph
    lanes = [0, 3, 4, 5, 1, 6, 2]
    B = len(lanes)
    d_lanes, one = ints(lanes), ints([1] * B)
    groups = dict(group_start=ints([0, 4, 6, 7]), shared=ints([7, 2, 0]))
    q, k, v = s.fresh(B)
    qr = torch.empty((L, B, HQ, D), device="cuda", dtype=s.p.q_dtype)
    out, lse = torch.empty_like(qr), torch.empty((L, B, HQ), device="cuda")

    def step():
        pos = s.p.length[d_lanes.long()]
        s.p.reserve(d_lanes, one)
        for i in range(L):
            s.p.append(i, d_lanes, pos, k=k[i], v=v[i], q=q[i], q_out=qr[i], inv_freq=s.inv, factor=1.1,
                       kv_scale=s.kv)
            s.p.attend(i, qr[i], out[i], d_lanes, lse=lse[i], **groups)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for i in range(16):
        for x, y in zip((q, k, v), s.fresh(B)):
            x.copy_(y)
        pos = np.array([len(s.held[a]) for a in lanes])
        if i % 5 == 4:
            step()
        else:
            graph.replay()
        s.took(lanes, pos, q, k.clone(), v.clone(), qr)
        s.attended(lanes, [1] * B, qr, out, lse)
        if i == 3:  # four drafted tokens of two lanes, all but one taken back
            s.tokens([4, 6], [4, 4])
            s.p.trim(ints([4, 6]), ints([len(s.held[a]) - 3 for a in (4, 6)]))
            for a in (4, 6):
                del s.held[a][-3:]
            s.same()
        if i == 8:  # a lane starts again and the pages move
            s.p.trim(ints([2]))
            s.held[2] = []
            s.p.compact()
            s.same()
    s.same()
    s.p.trim(ints(list(range(8))))
    s.held = [[] for _ in s.held]
    s.same()


@pytest.mark.parametrize("dt", [F.F16, F.BF16, F.FP8])
def test_pages_as_the_executor_s_host_tier(dt):
    # a page is the executor's block record: whole pages, handed over and all of them
    # selected, give the paged attention's output
    n, blocks = 3, 6
    s = Server(dt)
    lanes = [5, 0, 3]
    s.tokens(lanes, [blocks * T] * n)
    ex = F.Executor(n, L, H, blocks, blocks + 2, blocks, q_heads=HQ, dtype=dt, host_blocks=n * L * H * blocks)
    host = torch.empty(ex.cfg.host_blocks * ex.block_bytes, dtype=torch.uint8, pin_memory=True)
    ids = s.p.table[ints(lanes).long(), :blocks].long()
    # [L, request, block, H] -> [request, L, H, block]
    host.copy_(s.p.pool.view(torch.uint8)[:, ids].permute(1, 0, 3, 2, 4, 5, 6).reshape(-1))
    scales = None
    if dt == F.FP8:
        scales = torch.empty(2 * ex.cfg.host_blocks, pin_memory=True)
        scales.copy_(s.p.scales[:, ids].permute(1, 0, 3, 2, 4).reshape(-1))
    ex.hosttier_register(host, scales)
    sel = torch.arange(blocks, dtype=torch.int32, device="cuda").repeat(n, L, H, 1).contiguous()
    bufs = ex.alloc_step_buffers()
    ex.fetch_step(sel, bufs)
    q = torch.randn((n, L, HQ, D), device="cuda", generator=s.g).to(s.p.q_dtype)
    sparse = torch.empty((n, L, HQ, D), device="cuda")
    ex.sparse_decode(q.float().contiguous(), bufs["slots"], sparse)
    out = torch.empty_like(q)
    for i in range(L):
        s.p.attend(i, q[:, i], out[:, i], ints(lanes))
    torch.cuda.synchronize()
    s.p.check()
    assert ex.stats()["device_error"] == 0
    ex.close()
    # the executor's bound, relative to a row's largest value; here the weights' and
    # the output's rounding, with sum p |v| at most the largest |v|
    v = s.p.pool[:, ids][..., 1, :, :].double()
    if scales is not None:
        v = v * s.p.scales[:, ids][..., 1, None, None].double()
    want = sparse.double().abs().amax(-1, keepdim=True)
    bound = TOL[dt] * want + U[dt] * (want + v.abs().max()) * 1.01
    assert torch.all((out.double() - sparse.double()).abs() <= bound)


def test_scratch_on_another_stream():
    # memory that the current stream still uses is not handed to another stream's call
    c = Case(F.BF16, 8, 2, [700, 90], seed=4)
    a = c.args()
    out = torch.empty_like(c.q)
    need = F.C.c_uint64()
    args = F.AttendArgs(2, 2, 0, 8, 0.0)
    assert F.lib.ferry_pages_attend_work_bytes(F.C.byref(c.p._d), F.C.byref(args), F.C.byref(need)) == 0
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    x = torch.full((need.value,), 7, dtype=torch.uint8, device="cuda")
    torch.cuda._sleep(20_000_000)
    y = x.clone()
    del x
    c.p.attend(0, c.q, out, stream=s, **a)
    torch.cuda.synchronize()
    assert torch.all(y == 7)
    lse = torch.empty((2, 8), device="cuda")
    c.p.attend(0, c.q, out, lse=lse, stream=0, **a)
    torch.cuda.synchronize()
    c.check(out, lse)
