"""GPU: calls of the attention half from a caller that takes streams in turn: the next call waits for the call on the
other stream, not for what the caller has enqueued there behind it."""
from __future__ import annotations

import pytest

from test_gpu_attention import filled, work_of
from test_gpu_kv import Batch, open_lane, rand_rows, step

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

SLEEP = 50_000_000   # cycles: some 20 ms at least


@pytest.mark.parametrize("what", ["attention", "write", "read"])
def test_later_work_is_not_waited_for(what):
    step(f"attention half, streams in turn, {what}")
    b = Batch([(3, 500)], 16, 2, 64)
    filled(b, 1)
    k, _ = rand_rows(b.rows, 2, 64, "f16", 1)
    v, _ = rand_rows(b.rows, 2, 64, "f16", 2)
    q, _ = rand_rows(b.rows, 4, 64, "f16", 3, 0, 0.5)
    outs = [torch.zeros_like(q) for _ in range(3)]
    back = [torch.zeros_like(k) for _ in range(2)]
    work = work_of(b, 4)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    with open_lane() as ln:
        calls = {"attention": lambda s: ln.attention_async(b.kv, q, outs[0], work=work, stream=s.cuda_stream),
                 "write": lambda s: ln.kv_write_async(b.kv, k, v, stream=s.cuda_stream),
                 "read": lambda s: ln.kv_read_async(b.kv, *back, stream=s.cuda_stream)}
        torch.cuda.synchronize()
        ln.kv_write_async(b.kv, k, v, stream=s1.cuda_stream)
        ln.attention_async(b.kv, q, outs[1], work=work, stream=s2.cuda_stream)
        torch.cuda.synchronize()
        calls[what](s1)
        with torch.cuda.stream(s1):
            torch.cuda._sleep(SLEEP)
        slept = s1.record_event()
        ln.attention_async(b.kv, q, outs[2], work=work, stream=s2.cuda_stream)
        s2.synchronize()
        early = not slept.query()
        torch.cuda.synchronize()
        assert torch.equal(outs[2], outs[1]) and early
        ln.sync(s2.cuda_stream)


def test_one_stream_again_after_a_change():
    """After 64 calls on one stream the record is left to the next call again; order and results hold throughout."""
    step("attention half, one stream again")
    b = Batch([(3, 500)], 16, 2, 64)
    filled(b, 1)
    k, _ = rand_rows(b.rows, 2, 64, "f16", 1)
    v, _ = rand_rows(b.rows, 2, 64, "f16", 2)
    back = [torch.zeros_like(k) for _ in range(2)]
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    with open_lane() as ln:
        torch.cuda.synchronize()
        for turn in range(4):
            for n in (1, 63, 64, 65, 70):
                for i in range(n):
                    ln.kv_write_async(b.kv, k, v, stream=s1.cuda_stream)
                ln.kv_read_async(b.kv, *back, stream=s2.cuda_stream)
                ln.sync(s2.cuda_stream)
                assert all((x - y).abs().max() < 0.1 * y.abs().max() for x, y in zip(back, (k, v)))
                for x in back:
                    x.zero_()
                torch.cuda.synchronize()
