"""GPU: the calls of the attention half together and as a serving loop makes them: rotary, cache and attention of a
prompt in chunks and then token by token, as a graph, on several streams and lanes, with workspaces that are shared, and
caches whose offsets pass 32 bits.

Tolerances are those of test_gpu_kv.py (the cache's bytes are exact) and test_gpu_attention.py.
"""
from __future__ import annotations

import numpy as np
import pytest

import crosslane_amd as xl
from kv_ref import Cache, attention, page_bytes, turned
from test_gpu_attention import check, filled, work_of
from test_gpu_kv import TYPES, Batch, lane, open_lane, rand_rows, step  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


class Loop:
    """Sequences that grow in one cache: each step writes some rows of each and attends."""

    def __init__(self, lane, lens, P, KV, H, D, kind, axes=1, seed=0):
        self.lane, self.P, self.KV, self.H, self.D, self.kind, self.axes = lane, P, KV, H, D, kind, axes
        self.g = torch.Generator().manual_seed(seed)
        B, cols = len(lens), -(-max(lens) // P)
        self.n_pages = B * cols + 1
        self.table = torch.randperm(self.n_pages, generator=self.g)[: B * cols].view(B, cols).to(torch.int32)
        self.cache = torch.full((self.n_pages, KV, page_bytes(P, D)), 0x7e, dtype=torch.uint8, device="cuda")
        self.ref = Cache(self.cache.cpu().numpy().copy(), P, D)
        self.lens = np.zeros(B, np.int64)
        self.d_table = self.table.cuda()
        self.freqs = (10000.0 ** (-np.arange(D // 2) / (D // 2))).astype(np.float32)
        self.d_freqs = torch.from_numpy(self.freqs).cuda()
        self.sections = (D // 2,) if axes == 1 else (D // 4, D // 8, D // 8)

    def rows(self, counts, behind=0):
        """New rows of q, k and v (parts of the same rows), and a batch for them."""
        T = int(sum(counts)) + behind
        self.lens += counts
        qkv = torch.randn((T, self.H + 2 * self.KV, self.D), generator=self.g).to(TYPES[self.kind])
        self.lens_d = torch.from_numpy(self.lens.astype(np.int32)).cuda()
        self.starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        b = xl.KVBatch(self.cache, self.d_table, self.lens_d, torch.from_numpy(self.starts).cuda(), T, self.D, max_rows=max(1, max(counts)))
        pos = torch.randint(0, 5000, (3, T), generator=self.g, dtype=torch.int32).cuda() if self.axes == 3 else None
        return b, qkv, qkv.cuda(), pos

    def write_ref(self, counts, qkv, pos):
        """The same rows into the reference's cache; q turned and rounded."""
        T = int(sum(counts))
        x = qkv[:T].float().numpy()
        place = np.concatenate([np.arange(ln - n, ln) for n, ln in zip(counts, self.lens)])
        y = turned(x[:, : self.H + self.KV], self.freqs, place[None].astype(np.int32) if pos is None else pos[:, :T].cpu().numpy(),
                   self.sections, False)
        t = 0
        for i, n in enumerate(counts):
            for j in range(n):
                p = int(self.lens[i]) - n + j
                for h in range(self.KV):
                    self.ref.put(int(self.table[i, p // self.P]), h, p % self.P, y[t, self.H + h], x[t, self.H + self.KV + h])
                t += 1
        return torch.from_numpy(y[:, : self.H]).to(TYPES[self.kind])

    def as_batch(self, counts, rows):
        """What `check` wants of a batch."""
        b = object.__new__(Batch)
        b.seqs, b.starts, b.P, b.KV, b.D, b.rows, b.table = list(zip(counts, self.lens.tolist())), self.starts, self.P, self.KV, self.D, rows, \
            self.table.numpy()
        return b


@pytest.mark.parametrize("axes,kind,D,H", [(1, "bf16", 128, 8), (3, "f16", 64, 6)])
def test_prompt_in_chunks_then_tokens(lane, axes, kind, D, H):  # noqa: F811
    step(f"attention loop {axes} {kind}")
    loop = Loop(lane, [150, 90, 60], 16, 2, H, D, kind, axes)
    s = torch.cuda.Stream().cuda_stream
    for counts, behind in (((70, 5, 33), 2), ((45, 60, 0), 0), ((1, 1, 1), 1), ((1, 1, 1), 0), ((3, 2, 4), 0)):
        b, qkv, d, pos = loop.rows(counts, behind)
        T = d.shape[0]
        q_out = torch.full((T, H, D), 7.0, dtype=TYPES[kind], device="cuda")
        out, work = torch.full_like(q_out, 7.0), torch.full((xl.attention_work_bytes(b, H),), 0xFF, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        lane.kv_write_async(b, d[:, H:H + 2], d[:, H + 2:], q=d[:, :H], q_out=q_out, freqs=loop.d_freqs, positions=pos,
                            sections=loop.sections, stream=s)
        lane.attention_async(b, q_out, out, work=work, stream=s)
        lane.sync(s)
        q = loop.write_ref(counts, qkv, pos)
        n = q.shape[0]
        assert torch.equal(q_out[:n].cpu(), q) and (q_out[n:] == 7).all()
        used = np.zeros((loop.n_pages, 16), bool)
        for i, ln in enumerate(loop.lens):
            for j in range(ln):
                used[loop.table[i, j // 16], j % 16] = True
        got, want = Cache(loop.cache.cpu().numpy(), 16, D), loop.ref
        for page in range(loop.n_pages):
            for h in range(2):
                for x, y in zip(got.values(page, h), want.values(page, h)):
                    assert np.array_equal(x[used[page]], y[used[page]])
        q32 = np.zeros((T, H, D), np.float32)
        q32[:n] = q.float().numpy()
        check(loop.as_batch(counts, T), loop.ref, q32, out.double().cpu().numpy(), H, kind, D ** -0.5, 0, 0.0)


@pytest.mark.parametrize("rows,length", [(1, 700), (1, 5000), (4, 900), (90, 2500)])
def test_graph(rows, length):
    """A step of write, attention and read as a graph: replayed with other inputs, eager work between the replays, equal to
    eager calls each time; another graph of the same lane on the same workspace in between."""
    step(f"attention graph {rows} {length}")
    P, KV, H, D, kind = 32, 2, 8, 128, "bf16"
    s = torch.cuda.Stream()
    with open_lane() as ln:
        b = Batch([(rows, length), (rows, length // 2)], P, KV, D)
        filled(b, 1)
        T = b.rows
        qkv = torch.randn((T, H + 2 * KV, D), device="cuda").to(TYPES[kind])
        freqs = torch.rand(D // 2, device="cuda")
        q_out, out, k, v = (torch.zeros((T, n, D), dtype=TYPES[kind], device="cuda") for n in (H, H, KV, KV))
        work = work_of(b, H)

        def one():
            ln.kv_write_async(b.kv, qkv[:, H:H + KV], qkv[:, H + KV:], q=qkv[:, :H], q_out=q_out, freqs=freqs, stream=s.cuda_stream)
            ln.attention_async(b.kv, q_out, out, work=work, stream=s.cuda_stream)
            ln.kv_read_async(b.kv, k, v, stream=s.cuda_stream)

        def other():
            ln.attention_async(b.kv, q_out, out, window=33, softcap=20.0, work=work, stream=s.cuda_stream)

        torch.cuda.synchronize()
        graphs = []
        for f in (one, other):
            f()
            ln.sync(s.cuda_stream)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                f()
            graphs.append(g)
        start = b.whole.clone()
        for turn in range(3):
            qkv.copy_(torch.randn(qkv.shape, device="cuda"))
            lens = torch.tensor([length - 3 * turn, length // 2 - turn], dtype=torch.int32)
            b.d_lens.copy_(lens)
            want = []
            for f in (one, other):
                b.whole.copy_(start)
                torch.cuda.synchronize()
                one()
                f()
                ln.sync(s.cuda_stream)
                want.append([t.clone() for t in (q_out, out, k, v, b.whole)])
            b.whole.copy_(start)
            work.fill_(0xFF)
            torch.cuda.synchronize()
            with torch.cuda.stream(s):
                graphs[0].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(want[0], (q_out, out, k, v, b.whole)))
            with torch.cuda.stream(s):
                graphs[1].replay()
            torch.cuda.synchronize()
            assert torch.equal(want[1][1], out)
        ln.sync(s.cuda_stream)


def test_streams_and_lanes(lane):  # noqa: F811
    """A write on one stream is ordered before the attention on another of the same lane; two lanes attend at once, each with its workspace."""
    step("attention streams")
    P, KV, H, D = 16, 2, 8, 64
    b = Batch([(40, 3000)], P, KV, D)
    c = filled(b, 3)
    k, k32 = rand_rows(40, KV, D, "f16", 1)
    v, v32 = rand_rows(40, KV, D, "f16", 2)
    q, q32 = rand_rows(40, H, D, "f16", 3, 0, 0.5)
    for t, i, p in b.places():
        for h in range(KV):
            c.put(b.table[0, p // P], h, p % P, k32[t, h], v32[t, h])
    s1, s2 = torch.cuda.Stream().cuda_stream, torch.cuda.Stream().cuda_stream
    outs = [torch.zeros((40, H, D), dtype=torch.float16, device="cuda") for _ in range(3)]
    works = [work_of(b, H) for _ in range(2)]
    torch.cuda.synchronize()
    with open_lane() as second:
        lane.kv_write_async(b.kv, k, v, stream=s1)
        lane.attention_async(b.kv, q, outs[0], work=works[0], stream=s2)
        lane.sync(s2)
        lane.attention_async(b.kv, q, outs[1], work=works[0], stream=s1)
        second.attention_async(b.kv, q, outs[2], work=works[1])
        lane.sync(s1)
        second.sync()
    check(b, c, q32, outs[0].double().cpu().numpy(), H, "f16", D ** -0.5, 0, 0.0)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("rows", [1, 80])
def test_offsets_past_32_bits(lane, rows):  # noqa: F811
    """Pages 3 GiB apart, as where the layers of a model take turns in one buffer."""
    step(f"attention, offsets past 32 bits {rows}")
    P, KV, H, D, ln, stride = 16, 1, 4, 64, 100, 3 << 30
    pb, n = page_bytes(P, D), 7
    whole = torch.empty((n - 1) * stride + KV * pb, dtype=torch.uint8, device="cuda")
    cache = torch.as_strided(whole, (n, KV, pb), (stride, pb, 1))
    b = Batch([(rows, ln)], P, KV, D)
    small = b.cache[:n]
    c = filled(b, 5)
    b.table[0, :n] = [6, 0, 3, 5, 1, 2, 4]
    b.d_table.copy_(torch.from_numpy(b.table))
    cache.copy_(torch.from_numpy(c.raw[:n]))
    kv = xl.KVBatch(cache, b.d_table, b.d_lens, b.d_starts, b.rows, D)
    k, k32 = rand_rows(rows, KV, D, "f16", 1)
    v, v32 = rand_rows(rows, KV, D, "f16", 2)
    q, q32 = rand_rows(rows, H, D, "f16", 3, 0, 0.5)
    for t, i, p in b.places():
        c.put(b.table[0, p // P], 0, p % P, k32[t, 0], v32[t, 0])
    out = torch.zeros((rows, H, D), dtype=torch.float16, device="cuda")
    back = [torch.zeros((rows, KV, D), device="cuda") for _ in range(2)]
    work = torch.empty(xl.attention_work_bytes(kv, H), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    lane.kv_write_async(kv, k, v)
    lane.attention_async(kv, q, out, work=work)
    lane.kv_read_async(kv, *back)
    lane.sync()
    assert small.shape[0] == n
    assert np.array_equal(cache.cpu().numpy(), c.raw[:n])
    check(b, c, q32, out.double().cpu().numpy(), H, "f16", D ** -0.5, 0, 0.0)
    for x, j in zip(back, range(2)):
        want = np.stack([c.values(b.table[0, p // P], 0)[j][p % P] for _, _, p in b.places()])
        assert np.abs(x.cpu().numpy()[:, 0] - want).max() <= 2.0 ** -23 * np.abs(want).max()


@pytest.mark.parametrize("seqs,rows", [(300, 1), (37, 20)])
def test_many_sequences(lane, seqs, rows):  # noqa: F811
    step(f"attention, many sequences {seqs}")
    rng = np.random.default_rng(seqs)
    b = Batch([(int(rng.integers(0, rows + 1)), int(rng.integers(0, 120))) for _ in range(seqs - 1)] + [(rows, 130)], 16, 1, 64, behind=3, before=2)
    c = filled(b, 1, 0x7e)
    q, q32 = rand_rows(b.rows, 4, 64, "bf16", 5, 0, 0.5)
    out = torch.full((b.rows, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    k, v = (torch.full((b.rows, 1, 64), 7.0, device="cuda") for _ in range(2))
    work = work_of(b, 4)
    torch.cuda.synchronize()
    lane.attention_async(b.kv, q, out, work=work)
    lane.kv_read_async(b.kv, k, v)
    lane.sync()
    check(b, c, q32, out.double().cpu().numpy(), 4, "bf16", 0.125, 0, 0.0)
    want = np.full((2, b.rows, 64), 7.0)
    for t, i, p in b.places():
        want[:, t] = [x[p % 16] for x in c.values(b.table[i, p // 16], 0)] if p >= 0 else 0
    for x, w in zip((k, v), want):
        assert np.abs(x.cpu().numpy()[:, 0] - w).max() <= 2.0 ** -23 * 40


def long_batch(seed=3):
    """A sequence long enough that its attention is still running when the host enqueues the next call."""
    P, KV, H, D, T = 64, 2, 8, 64, 200
    b = Batch([(T, 20000)], P, KV, D)
    filled(b, seed)
    q, _ = rand_rows(T, H, D, "bf16", 3, 0, 0.5)
    kv = [[rand_rows(T, KV, D, "bf16", 10 * i + j)[0] for j in range(2)] for i in range(3)]
    return b, q, kv, work_of(b, H)


def test_order_across_streams(lane):  # noqa: F811
    """Writes on one stream and attention on another, in turn and without a wait by the caller: the results of one stream."""
    step("attention half, order across streams")
    b, q, kv, work = long_batch()
    start = b.whole.clone()
    s1, s2 = torch.cuda.Stream().cuda_stream, torch.cuda.Stream().cuda_stream
    outs = [[torch.zeros_like(q) for _ in kv] for _ in range(2)]
    backs = [[torch.zeros_like(kv[0][0]) for _ in range(2)] for _ in range(2)]
    torch.cuda.synchronize()
    for streams, o, back in (((s1, s1), outs[0], backs[0]), ((s1, s2), outs[1], backs[1])):
        b.whole.copy_(start)
        torch.cuda.synchronize()
        for (k, v), out in zip(kv, o):
            lane.kv_write_async(b.kv, k, v, stream=streams[1])
            lane.attention_async(b.kv, q, out, work=work, stream=streams[0])
        lane.kv_read_async(b.kv, *back, stream=streams[1])
        lane.sync(streams[0])
        lane.sync(streams[1])
    assert all(torch.equal(x, y) for x, y in zip(outs[0] + backs[0], outs[1] + backs[1]))


def test_sync_waits_for_another_stream(lane):  # noqa: F811
    """A wait for the context's own stream waits for a call that named another one."""
    step("attention half, sync of another stream")
    b, q, kv, work = long_batch()
    s1 = torch.cuda.Stream().cuda_stream
    want, out = torch.zeros_like(q), torch.zeros_like(q)
    torch.cuda.synchronize()
    lane.attention_async(b.kv, q, want, work=work)
    lane.sync()
    lane.attention_async(b.kv, q, out, work=work, stream=s1)
    lane.sync()
    got = out.cpu()   # (torch's own stream does not wait for s1)
    assert torch.equal(got, want.cpu())


def test_order_around_a_capture():
    """A call on another stream while the previous call's stream is captured is refused, unless it is captured too: then it
    becomes part of the same graph, ordered."""
    step("attention half, order around a capture")
    b, q, kv, work = long_batch()
    out, other = torch.zeros_like(q), torch.zeros_like(q)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    with open_lane() as ln:
        torch.cuda.synchronize()
        ln.attention_async(b.kv, q, out, work=work, stream=s1.cuda_stream)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s1):
            ln.kv_write_async(b.kv, *kv[0], stream=s1.cuda_stream)
            with pytest.raises(xl.XLError, match="being captured"):
                ln.attention_async(b.kv, q, other, work=work, stream=s2.cuda_stream)
            s2.wait_stream(s1)
            ln.attention_async(b.kv, q, out, work=work, stream=s2.cuda_stream)
            s1.wait_stream(s2)
        start = b.whole.clone()
        for turn in range(3):
            b.whole.copy_(start)
            torch.cuda.synchronize()
            ln.kv_write_async(b.kv, *kv[turn], stream=s2.cuda_stream)
            ln.attention_async(b.kv, q, other, work=work, stream=s2.cuda_stream)
            ln.sync(s2.cuda_stream)
            want = other.clone()
            b.whole.copy_(start)
            out.zero_()
            for x, y in zip(kv[0], kv[turn]):
                x.copy_(y)
            torch.cuda.synchronize()
            with torch.cuda.stream(s1):
                g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and (other == want).all()
        ln.sync()
