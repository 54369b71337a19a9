"""What the calls over a 4-bit cache refuse, on the CPU: arguments are checked before the
context, so a null context shows whether a call got past them (no pointer here is ever read);
and how the kernels address a batch, with the same functions built for the host and
batches that hold anything."""
from __future__ import annotations

import ctypes as C
import os
import random
import shutil
import subprocess

import pytest

import crosslane_amd as xl
from crosslane_amd import lane as L

A = 1 << 24   # addresses, far apart and aligned
PAST = b"null context"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

BATCH = dict(struct_bytes=C.sizeof(L._KVBatch), head_dim=128, kv_heads=2, page_tokens=32, n_pages=10, max_pages=4, n_seqs=3, rows=7,
             max_rows=5, reserved=0, page_stride=2 * 32 * 160, table_stride=4, pages=A, table=2 * A, lens=3 * A, starts=4 * A)
ROTARY = dict(struct_bytes=C.sizeof(L._Rotary), n_freqs=64, n_axes=3, interleaved=0, section=(24, 20, 20), reserved=0,
              positions_stride=7, freqs=5 * A, positions=6 * A)
WRITE = dict(k=7 * A, k_stride=256, v=8 * A, v_stride=256, type=2, rotary=ROTARY, q=9 * A, q_stride=768, q_heads=6, q_out=10 * A,
             q_out_stride=768, stream=None)
READ = dict(k=7 * A, k_stride=256, v=8 * A, v_stride=256, type=0, stream=None)
ATTEND = dict(q=7 * A, q_stride=768, q_heads=6, type=1, scale=0.1, window=0, softcap=0.0, out=8 * A, out_stride=768, work=9 * A,
              work_bytes=A, stream=None)
CALLS = {"xl_kv_write_async": WRITE, "xl_kv_read_async": READ, "xl_attention_async": ATTEND}


def call(name, change):
    change = dict(change)
    batch = {**BATCH, **{k[2:]: change.pop(k) for k in list(change) if k.startswith("b_")}}
    rot = {**ROTARY, **{k[2:]: change.pop(k) for k in list(change) if k.startswith("r_")}}
    args = dict(CALLS[name])
    assert set(change) <= set(args) and set(batch) == set(BATCH) and set(rot) == set(ROTARY)
    if "rotary" in args:
        args["rotary"] = rot
    args.update(change)
    b = L._KVBatch(**batch)
    keep = L._Rotary(**rot)
    values = [C.addressof(keep) if v is rot else v for v in args.values()]
    err = L._Err()
    rc = getattr(xl.lib(), name)(None, C.byref(b), *values, C.byref(err))
    return rc, err.message


@pytest.mark.parametrize("name,change", [
    ("xl_kv_write_async", {}), ("xl_kv_write_async", {"rotary": None, "q": None, "q_out": None}),
    ("xl_kv_write_async", {"q": None, "q_out": None, "q_heads": 0}), ("xl_kv_write_async", {"k": 7 * A + 4, "type": 2}),
    ("xl_kv_write_async", {"r_n_axes": 1, "r_section": (64, 0, 0), "r_positions": None, "r_positions_stride": 0}),
    ("xl_kv_write_async", {"r_section": (0, 64, 0)}), ("xl_kv_write_async", {"r_n_freqs": 1, "r_section": (0, 0, 1)}),
    # parts of the same rows
    ("xl_kv_write_async", {"q": 7 * A, "k": 7 * A + 2 * 768, "v": 7 * A + 2 * 1024, "q_stride": 1280, "k_stride": 1280, "v_stride": 1280}),
    ("xl_kv_read_async", {}), ("xl_attention_async", {}), ("xl_attention_async", {"window": 2 ** 31 - 1}),
    # keys and values as columns of the same rows
    ("xl_kv_read_async", {"v": 7 * A + 4 * 256, "k_stride": 512, "v_stride": 512}), ("xl_kv_read_async", {"k": 8 * A + 4 * 300, "k_stride": 556, "v_stride": 556}), ("xl_attention_async", {"window": 1, "softcap": 30.0}),
    ("xl_attention_async", {"scale": -1.0}), ("xl_attention_async", {"b_page_tokens": 1024, "b_page_stride": 2 * 1024 * 160}),
    ("xl_attention_async", {"b_page_stride": 1 << 40, "b_n_pages": 1}),
], ids=str)
def test_good_arguments_reach_the_context(name, change):
    rc, msg = call(name, change)
    assert rc == 1 and PAST in msg, msg


BATCH_BAD = [({"b_head_dim": 96}, "head_dim"), ({"b_kv_heads": 0}, "kv_heads"), ({"b_kv_heads": 257}, "kv_heads"),
             ({"b_page_tokens": 24}, "page_tokens"), ({"b_page_tokens": 0}, "page_tokens"), ({"b_page_tokens": 1040}, "page_tokens"),
             ({"b_n_pages": 0}, "n_pages"), ({"b_max_pages": 0}, "max_pages"), ({"b_max_pages": (1 << 21) + 1}, "max_pages"),
             ({"b_n_seqs": 0}, "n_seqs"), ({"b_n_seqs": 65536}, "n_seqs"), ({"b_rows": 0}, "rows"), ({"b_rows": (1 << 23) + 1}, "rows"),
             ({"b_max_rows": 0}, "max_rows"), ({"b_max_rows": 8}, "max_rows"), ({"b_reserved": 1}, "reserved"),
             ({"b_page_stride": 2 * 32 * 160 - 16}, "page_stride"), ({"b_page_stride": 2 * 32 * 160 + 8}, "page_stride"),
             ({"b_page_stride": (1 << 40) + 16}, "page_stride"), ({"b_pages": A + 8}, "16-byte"), ({"b_pages": None}, "null"),
             ({"b_table": None}, "null"), ({"b_lens": None}, "null"), ({"b_starts": None}, "null"), ({"b_table": 2 * A + 2}, "table"),
             ({"b_table_stride": 3}, "table"), ({"b_lens": 3 * A + 1}, "lens"), ({"b_starts": 4 * A + 3}, "starts")]
BAD = [(n, c, m) for n in CALLS for c, m in BATCH_BAD] + [
    ("xl_kv_write_async", {"k": None}, "null"), ("xl_kv_write_async", {"v": None}, "null"), ("xl_kv_write_async", {"type": 3}, "f32"),
    ("xl_kv_write_async", {"q": None}, "together"), ("xl_kv_write_async", {"q_out": None}, "together"),
    ("xl_kv_write_async", {"rotary": None}, "without rotary"), ("xl_kv_write_async", {"k_stride": 255}, "stride"),
    ("xl_kv_write_async", {"v": 8 * A + 1}, "aligned"), ("xl_kv_write_async", {"q_heads": 5}, "q_heads"),
    ("xl_kv_write_async", {"q_heads": 0}, "q_heads"), ("xl_kv_write_async", {"q_out_stride": 767}, "stride"),
    ("xl_kv_write_async", {"q_out": 9 * A}, "overlaps"), ("xl_kv_write_async", {"q_out": A + 64}, "overlaps"),
    ("xl_kv_write_async", {"k": A + 1024}, "overlaps"), ("xl_kv_write_async", {"q_out": 6 * A}, "overlaps"),
    ("xl_kv_write_async", {"b_table": A + 64}, "overlaps"),
    ("xl_kv_write_async", {"r_n_freqs": 65, "r_section": (65, 0, 0)}, "n_freqs"), ("xl_kv_write_async", {"r_n_freqs": 0}, "n_freqs"),
    ("xl_kv_write_async", {"r_n_axes": 4}, "n_axes"), ("xl_kv_write_async", {"r_n_axes": 0}, "n_axes"),
    ("xl_kv_write_async", {"r_section": (24, 20, 19)}, "add up"), ("xl_kv_write_async", {"r_section": (84, -40, 20)}, "section"),
    ("xl_kv_write_async", {"r_n_axes": 2}, "section"), ("xl_kv_write_async", {"r_freqs": None}, "null"),
    ("xl_kv_write_async", {"r_positions": None}, "need positions"), ("xl_kv_write_async", {"r_positions_stride": 6}, "positions"),
    ("xl_kv_write_async", {"r_reserved": 2}, "reserved"),
    ("xl_kv_read_async", {"k": None}, "null"), ("xl_kv_read_async", {"type": 3}, "f32"), ("xl_kv_read_async", {"v": 7 * A}, "overlaps"),
    ("xl_kv_read_async", {"v": 7 * A + 1024}, "overlaps"), ("xl_kv_read_async", {"k": 3 * A}, "overlaps"),
    ("xl_kv_read_async", {"v": A}, "overlaps"), ("xl_kv_read_async", {"v_stride": 10}, "stride"),
    ("xl_attention_async", {"q": None}, "null"), ("xl_attention_async", {"out": None}, "null"), ("xl_attention_async", {"type": 0}, "f16"),
    ("xl_attention_async", {"q_heads": 7}, "q_heads"), ("xl_attention_async", {"q_heads": 1026}, "q_heads"),
    ("xl_attention_async", {"scale": float("nan")}, "scale"), ("xl_attention_async", {"softcap": -1.0}, "softcap"),
    ("xl_attention_async", {"softcap": float("inf")}, "softcap"), ("xl_attention_async", {"softcap": 1e-21}, "softcap"),
    ("xl_attention_async", {"softcap": 16385.0}, "softcap"),
    ("xl_kv_read_async", {"v": 7 * A + 4 * 256, "k_stride": 511, "v_stride": 511}, "overlaps"),
    ("xl_kv_read_async", {"v": 7 * A + 4 * 256, "k_stride": 512, "v_stride": 768}, "overlaps"), ("xl_attention_async", {"window": -1}, "window"),
    ("xl_attention_async", {"b_n_seqs": 65535, "b_rows": 1 << 23, "b_max_rows": 1 << 23, "b_kv_heads": 256, "q_heads": 1024,
                            "b_page_stride": 256 * 32 * 160, "q_stride": 1 << 17, "out_stride": 1 << 17}, "workgroups"),
    ("xl_attention_async", {"q_stride": 700}, "stride"), ("xl_attention_async", {"out": 8 * A + 1}, "aligned"),
    ("xl_attention_async", {"work": 9 * A + 128}, "256-byte"), ("xl_attention_async", {"out": 7 * A}, "overlaps"),
    ("xl_attention_async", {"out": A}, "overlaps"),
]


@pytest.mark.parametrize("name,change,message", BAD, ids=str)
def test_refusals(name, change, message):
    rc, msg = call(name, change)
    assert rc == 1 and message.encode() in msg and PAST not in msg, msg


@pytest.mark.parametrize("change", [{"b_struct_bytes": 8}, {"r_struct_bytes": 0}])
def test_struct_sizes(change):
    rc, msg = call("xl_kv_write_async", change)
    assert rc == 5 and b"size mismatch" in msg
    assert L.lib().xl_kv_write_async(None, None, *[None] * 1, 0, None, 0, 0, None, None, 0, 0, None, 0, None, None) == 1


def test_sizes():
    assert xl.kv_page_bytes(32, 128) == 32 * 160 and xl.kv_page_bytes(16, 64) == 16 * 80 and xl.kv_page_bytes(1024, 256) == 1024 * 320
    for bad in ((15, 64), (8, 128), (1040, 64), (32, 96), (0, 64), (-16, 64)):
        assert xl.kv_page_bytes(*bad) == 0
    none = 2 ** 64 - 1
    b = L._KVBatch(**BATCH)
    assert L.lib().xl_attention_work_bytes(C.addressof(b), 6) < none
    assert L.lib().xl_attention_work_bytes(C.addressof(b), 5) == none
    assert L.lib().xl_attention_work_bytes(None, 6) == none


def test_work_is_checked():
    b = {"b_n_seqs": 1, "b_rows": 1, "b_max_rows": 1, "b_max_pages": 1 << 15, "b_table_stride": 1 << 15}
    s = L._KVBatch(**{**BATCH, **{k[2:]: v for k, v in b.items()}})
    need = L.lib().xl_attention_work_bytes(C.addressof(s), 6)
    rc, msg = call("xl_attention_async", {**b, "work_bytes": need})
    assert PAST in msg
    if need:
        rc, msg = call("xl_attention_async", {**b, "work_bytes": need - 1})
        assert b"workspace smaller" in msg
        rc, msg = call("xl_attention_async", {**b, "work": None})
        assert b"workspace smaller" in msg
        rc, msg = call("xl_attention_async", {**b, "work": 8 * A, "work_bytes": need})
        assert b"overlaps" in msg


def test_work_covers_every_window():
    """What xl_attention_work_bytes says is enough with any window."""
    rng = random.Random(5)
    split = 0
    for _ in range(4000):
        dim, kv, page = rng.choice((64, 128, 256)), rng.choice((1, 2, 8)), rng.choice((16, 64, 1024))
        heads, seqs, most = kv * rng.choice((1, 4, 7)), rng.choice((1, 3, 40)), rng.choice((1, 2, 9, 40, 300, 1200))
        rows, cols = rng.randint(most, seqs * most), int(rng.choice((1, 300, 3000, 40000, 400000)) * rng.random() / page) + 1
        b = {"b_head_dim": dim, "b_kv_heads": kv, "b_page_tokens": page, "b_page_stride": kv * xl.kv_page_bytes(page, dim), "b_n_pages": 3,
             "b_max_pages": cols, "b_table_stride": cols, "b_n_seqs": seqs, "b_rows": rows, "b_max_rows": most}
        s = L._KVBatch(**{**BATCH, **{k[2:]: v for k, v in b.items()}})
        need = L.lib().xl_attention_work_bytes(C.addressof(s), heads)
        split += need > 0
        at = [i << 40 for i in range(1, 9)]
        b.update(b_pages=at[0], b_table=at[1], b_lens=at[2], b_starts=at[3])
        rc, msg = call("xl_attention_async", {**b, "q": at[4], "out": at[5], "work": at[6], "q_heads": heads, "q_stride": heads * dim,
                                              "out_stride": heads * dim, "work_bytes": need, "window": rng.choice((0, 1, 500, 2000, 9000, 100000))})
        assert PAST in msg, (b, msg)
    assert split > 1000


def test_lane_refuses_host_tensors_and_wrong_shapes():
    torch = pytest.importorskip("torch")
    lane = object.__new__(xl.Lane)
    lane._ctx = None
    i = torch.zeros((2, 4), dtype=torch.int32)
    cache = torch.zeros((3, 2, 32 * 160), dtype=torch.uint8)
    with pytest.raises(xl.XLError, match="not on the GPU"):
        xl.KVBatch(cache, i, i[:, 0], i[0, :3], 5, 128)
    with pytest.raises(xl.XLError, match="uint8"):
        xl.KVBatch(cache.float(), i, i[:, 0], i[0, :3], 5, 128)
    with pytest.raises(xl.XLError, match="consecutive"):
        xl.KVBatch(cache.transpose(0, 1), i, i[:, 0], i[0, :3], 5, 128)
    batch = object.__new__(xl.KVBatch)
    batch.rows, batch.kv_heads, batch.head_dim, batch._kv_shape = 5, 2, 64, (5, 2, 64)
    k = torch.zeros((5, 2, 64))
    for f in (lambda: lane.kv_read_async(batch, k, k), lambda: lane.kv_write_async(batch, k, k), lambda: lane.attention_async(batch, k, k)):
        with pytest.raises(xl.XLError, match="not on the GPU"):
            f()
    with pytest.raises(xl.XLError, match="shape"):
        lane.kv_read_async(batch, k[:4], k)
    with pytest.raises(xl.XLError, match="consecutive"):
        lane.kv_read_async(batch, torch.zeros((5, 64, 2)).transpose(1, 2), k)


# ---- addressing, on the host ---------------------------------------------------
DRIVER = r"""
#include <cstdio>
#include <cstring>
#include <random>
#include <set>
#include <vector>
#include "xl_kv_index.hpp"
using namespace xl;
static int fails = 0;
#define CHECK(x) do { if (!(x)) { if (fails++ < 5) std::printf("line %d: %s\n", __LINE__, #x); } } while (0)

template <int D> void layout(int page) {   // every place of a page once, inside it, four parts apart
    Slab<D> s(page);
    std::vector<int> seen(s.bytes());
    for (int t = 0; t < page; ++t) {
        for (int c = 0; c < D / 8; ++c) {
            for (int i = 0; i < 4; ++i) ++seen.at(s.k_word(t, c) + i);
            for (int i = 0; i < 2; ++i) { ++seen.at(s.v_half(t, c) + i); ++seen.at(s.v_half(t, c) + 4 + i); }
            CHECK(s.k_word(t, c) % 4 == 0 && s.k_word(t, c) + 4 <= s.k_scales());
            CHECK(s.v_half(t, c) >= s.v_codes() && s.v_half(t, c) + 6 <= s.v_scales());
        }
        for (int g = 0; g < D / 32; ++g) {
            for (int i = 0; i < 4; ++i) ++seen.at(s.k_scale(t, g) + i);
            for (int i = 0; i < 2; ++i) { ++seen.at(s.v_scale(t, g) + i); ++seen.at(s.v_scale(t, g) + 8 + i); }
            CHECK(s.k_scale(t, g) >= s.k_scales() && s.k_scale(t, g) + 4 <= s.v_codes());
        }
    }
    for (int n : seen) CHECK(n == 1);
    CHECK(s.bytes() == page * D * 5 / 4);
}

int main() {
    for (int page = 16; page <= 1024; page += page < 128 ? 16 : 112) { layout<64>(page); layout<128>(page); layout<256>(page); }
    for (int page = 16; page <= 1024; page += 16) {   // pages of runs, up to the last run that a batch may have
        const uint32_t runs = page / 16, inv = kv_page_inverse(page);
        for (uint64_t run = 0; run <= (1u << 22); run += run < 5000 || run > (1u << 22) - 5000 ? 1 : 977) {
            const uint32_t got = inv ? uint32_t((run * inv) >> 32) : uint32_t(run);
            CHECK(got == run / runs);
        }
    }
    std::mt19937 rng(5);
    const auto pick = [&](int lo, int hi) { return int(lo + int64_t(rng() % uint32_t(hi - lo + 1))); };
    for (int turn = 0; turn < 20000; ++turn) {   // batches that hold anything: nothing out of bounds
        const int B = pick(1, 6), page = 16 * pick(1, 5), cols = pick(1, 4), pages = pick(1, 5), rows = pick(1, 40);
        std::vector<int32_t> table(B * (cols + 1)), lens(B), starts(B + 1);
        const bool wild = turn % 2;
        const auto any = [&]() { return rng() % 3 ? pick(-3, 70) : int32_t(rng()); };
        for (auto& v : table) v = wild ? any() : pick(0, pages - 1);
        for (auto& v : lens) v = wild ? any() : pick(0, cols * page);
        for (auto& v : starts) v = wild ? any() : 0;
        if (!wild)
            for (int i = 1; i <= B; ++i) starts[i] = pick(starts[i - 1], rows);
        const int64_t stride = 1ll << 33;
        KvBatch b{nullptr, stride, cols + 1, table.data(), lens.data(), starts.data(), 64, 1, page, pages, cols, B, rows, pick(1, rows),
                  kv_page_inverse(page), nullptr};
        for (int t = 0; t < rows; ++t) {
            const int seq = seq_of(b, t);
            CHECK(seq >= 0 && seq < B);
            if (!wild && t >= starts[0] && t < starts[B]) CHECK(starts[seq] <= t && t < starts[seq + 1]);
        }
        for (int q = 0; q < B; ++q) {
            const SeqRows r = seq_rows(b, q);
            CHECK(r.first >= 0 && r.n >= 0 && r.first + r.n <= rows && r.n <= b.max_rows && r.len >= 0 && r.len <= cols * page);
            const int64_t n = int64_t(starts[q + 1]) - starts[q];
            const bool good = starts[q] >= 0 && n >= 0 && starts[q + 1] <= rows && n <= b.max_rows && lens[q] >= 0 && lens[q] <= cols * page;
            CHECK(good == !r.bad);
            if (good) CHECK(r.first == starts[q] && r.n == n && r.len == lens[q]);
            for (int j = 0; j < r.len; j += 16) {
                int in = -1;
                const int64_t at = page_at(b, q, j / 16, in);
                CHECK(in >= 0 && in < page / 16 && in == j % page / 16);
                const int id = table[q * (cols + 1) + j / page];
                CHECK(id >= 0 && id < pages ? at == id * stride : at == -1);
            }
        }
    }
    std::printf("fails=%d\n", fails);
    return fails != 0;
}
"""


def test_addressing(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("g++ absent")
    src, exe = tmp_path / "kv.cpp", tmp_path / "kv"
    src.write_text(DRIVER)
    r = subprocess.run(["g++", "-O1", "-g", "-std=c++20", "-fsanitize=address,undefined", "-fno-sanitize-recover=undefined",
                        f"-I{os.path.join(ROOT, 'crosslane_amd', 'csrc')}", str(src), "-o", str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    env = {k: v for k, v in os.environ.items() if k != "LD_PRELOAD"}
    r = subprocess.run([str(exe)], capture_output=True, text=True, env=env)
    assert r.returncode == 0, r.stdout + r.stderr
