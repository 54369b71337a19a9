"""The attention half of a block of an 8-bit model, as cases that a timing program runs.

A case is one pass through one of them, on what a serving loop has in hand: a cache of
pages that holds keys and values in 4 bits (groups of 32 with a scale and a smallest
value in 16 bits), and a batch of sequences, each with some rows (new tokens).

  write   rotary positions on q and k, then k and v quantized into the cache; the rows
          are read back, so that what the cache now stands for is returned
  read    tokens of the cache as floats: a prefix that goes to another cache or device
  attend  attention of the rows over the cache: one token a sequence, a few drafted
          ones, or a chunk of a prompt

With `own` false, `run` computes them with elementary torch operations in 32 bits (the
angles of far positions in 64), with `own` true it makes the calls of
`crosslane_amd.Lane`. `exact` evaluates the definitions in 64 bits.

One kv head's part of a page of P tokens, heads of D values, G = D / 32 groups, is
  K codes   P x [4][G] words; word (c, g) has dims 32g + 8c ..+7, dim 2i in nibble i and
            dim 2i+1 in nibble i + 4
  K scales  P x [G][2] float16: scale, smallest value
  V codes   P/4 x [D/8][2][2][2] halfwords: dims 8c + 4h ..+3 of token 4a + 2b + e at
            [a][c][b][h][e], dims in order
  V scales  P/4 x [G][2][4] float16: the scales, then the smallest values, of four tokens
"""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
LIMIT = 32768.0


# ---- the cases ---------------------------------------------------------------
def listed():
    return [
        # one decoded token: latency alone
        {"name": "write_decode", "op": "write", "seqs": 1, "rows": 1, "tokens": 1000, "ragged": 0, "behind": 0, "page": 64,
         "heads": 32, "kv_heads": 8, "dim": 128, "type": "bf16", "axes": 1, "rotated": 128, "interleaved": False},
        # a packed batch of prompts of an image model, part of each head rotated by time, height and width
        {"name": "write_axes", "op": "write", "seqs": 9, "rows": 411, "tokens": 2000, "ragged": 7, "behind": 5, "page": 48,
         "heads": 24, "kv_heads": 4, "dim": 64, "type": "f16", "axes": 3, "rotated": 48, "interleaved": True},
        # a long prefill
        {"name": "write_prefill", "op": "write", "seqs": 4, "rows": 4096, "tokens": 4096, "ragged": 0, "behind": 0,
         "page": 64, "heads": 32, "kv_heads": 8, "dim": 128, "type": "bf16", "axes": 1, "rotated": 128, "interleaved": False},
        # a short prefix, odd in length
        {"name": "read_prefix", "op": "read", "seqs": 1, "rows": 771, "tokens": 771, "ragged": 0, "behind": 0, "page": 16,
         "heads": 8, "kv_heads": 2, "dim": 256, "type": "f16"},
        # the contexts of a batch that moves
        {"name": "read_batch", "op": "read", "seqs": 6, "rows": 30000, "tokens": 30000, "ragged": 3, "behind": 0,
         "page": 64, "heads": 32, "kv_heads": 8, "dim": 128, "type": "bf16"},
        # the first tokens of one conversation: latency alone
        {"name": "decode_one", "op": "attend", "seqs": 1, "rows": 1, "tokens": 200, "ragged": 0, "behind": 0, "page": 64,
         "heads": 32, "kv_heads": 8, "dim": 128, "type": "bf16", "window": 0, "softcap": 0.0},
        # one conversation with a very long context
        {"name": "decode_long", "op": "attend", "seqs": 1, "rows": 1, "tokens": 131072, "ragged": 0, "behind": 0,
         "page": 64, "heads": 32, "kv_heads": 8, "dim": 128, "type": "bf16", "window": 0, "softcap": 0.0},
        # a decode step of many conversations, from a token to 16384
        {"name": "decode_batch", "op": "attend", "seqs": 64, "rows": 1, "tokens": 16384, "ragged": 1, "behind": 0,
         "page": 64, "heads": 64, "kv_heads": 8, "dim": 128, "type": "bf16", "window": 0, "softcap": 0.0},
        # drafted tokens to verify, with a window and capped scores
        {"name": "verify", "op": "attend", "seqs": 24, "rows": 5, "tokens": 9000, "ragged": 5, "behind": 3, "page": 16,
         "heads": 16, "kv_heads": 8, "dim": 256, "type": "f16", "window": 4096, "softcap": 50.0},
        # chunks of prompts behind contexts, odd in all sizes
        {"name": "chunk_ragged", "op": "attend", "seqs": 5, "rows": 517, "tokens": 5000, "ragged": 2, "behind": 1,
         "page": 48, "heads": 15, "kv_heads": 5, "dim": 64, "type": "f16", "window": 0, "softcap": 0.0},
        # one chunk of a long prompt
        {"name": "chunk", "op": "attend", "seqs": 1, "rows": 512, "tokens": 32768, "ragged": 0, "behind": 0, "page": 64,
         "heads": 32, "kv_heads": 8, "dim": 128, "type": "bf16", "window": 0, "softcap": 0.0},
        # a whole prompt at once: what the matrix cores can do
        {"name": "prefill", "op": "attend", "seqs": 1, "rows": 8192, "tokens": 8192, "ragged": 0, "behind": 0, "page": 64,
         "heads": 32, "kv_heads": 8, "dim": 128, "type": "bf16", "window": 0, "softcap": 0.0},
    ]


MOST_VALUES = 64 * 16384 * 8 * 128      # keys of a padded batch
MOST_SCORES = 32 * 8192 * 8192 // 2     # (row, token, head) triples
MOST_ROWS = 16384 * 48 * 128            # values of q, k and v that a write takes


def _log(rng, lo, hi):
    return int(round(lo * (max(hi, lo) / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(("write", "read", "attend", "attend", "attend"))
    dim = rng.choice((64, 128, 128, 256))
    kv = rng.choice((1, 2, 4, 5, 8, 16))
    heads = kv * rng.choice((1, 2, 3, 4, 5, 8, 12, 16))
    page = rng.choice((16, 32, 48, 64, 128, 256))
    case = {"op": op, "ragged": rng.choice((0, rng.randint(1, 999))), "behind": rng.choice((0, 0, 1, 9)), "page": page,
            "heads": heads, "kv_heads": kv, "dim": dim}
    if op == "write":
        most = MOST_ROWS // ((heads + 2 * kv) * dim)
        seqs = _log(rng, 1, min(256, most))
        rows = rng.choice((1, _log(rng, 1, min(16384, most // seqs))))
        axes = rng.choice((1, 1, 2, 3))
        return {**case, "seqs": seqs, "rows": rows, "tokens": rows + _log(rng, 1, 30000) - 1, "type": rng.choice(("f32", "f16", "bf16")),
                "axes": axes, "rotated": rng.choice((dim, dim, dim // 2, dim - 16)), "interleaved": rng.random() < 0.4}
    seqs = _log(rng, 1, 128)
    tokens = _log(rng, 1, min(131072, MOST_VALUES // (seqs * kv * dim)))
    if op == "read":
        rows = max(1, min(tokens, 6 * 30000 * 8 * 128 // (seqs * kv * dim)))
        return {**case, "seqs": seqs, "rows": rows, "tokens": tokens, "type": rng.choice(("f32", "f16", "bf16"))}
    most = MOST_SCORES // (seqs * heads * tokens)
    kind = rng.choice(("decode", "draft", "chunk"))
    rows = 1 if kind == "decode" else rng.randint(2, 12) if kind == "draft" else _log(rng, 13, 8192)
    return {**case, "seqs": seqs, "rows": max(1, min(rows, tokens, most)), "tokens": tokens, "type": rng.choice(("f16", "bf16")),
            "window": rng.choice((0, 0, 0, _log(rng, 1, 8192))), "softcap": rng.choice((0.0, 0.0, 30.0, 50.0))}


def _lengths(case):
    """Rows (new tokens) and lengths (with them) of the sequences; a ragged batch has from one row to `rows`
    and from one token to `tokens`, so that now and then rows come before a sequence's first token."""
    b = case["seqs"]
    if not case["ragged"]:
        return [case["rows"]] * b, [case["tokens"]] * b
    rng = random.Random(case["ragged"])
    rows, lens = [], []
    for i in range(b):
        n = case["rows"] if i == b // 2 else rng.randint(1, case["rows"])
        most = case["tokens"]
        ln = most if i == b // 3 else rng.randint(1, most)
        rows.append(n)
        lens.append(ln if case["op"] == "attend" else max(ln, n))
    return rows, lens


def work(case):
    rows, lens = _lengths(case)
    t, d, kv, h, es = sum(rows), case["dim"], case["kv_heads"], case["heads"], BYTES[case["type"]]
    held = kv * d * 5 // 4      # the cache's bytes of a token, keys and values
    if case["op"] == "write":
        return {"bytes": t * (2 * h * d * es + 2 * kv * d * es + 2 * held + 2 * kv * d * 2), "flops": t * d * (6 * h + 16 * kv)}
    if case["op"] == "read":
        return {"bytes": t * (held + 2 * kv * d * es), "flops": t * d * 4 * kv}
    pairs = read = 0
    for n, ln in zip(rows, lens):
        first = max(0, ln - n)
        w = case["window"] or ln + 1
        pos = np.arange(first, ln, dtype=np.int64)
        pairs += int(np.minimum(pos + 1, w).sum())
        read += ln - max(0, first - w + 1)
    return {"bytes": read * held + 2 * t * h * d * es, "flops": 4 * d * h * pairs}


# ---- inputs ------------------------------------------------------------------
def _parts(page, dim):
    """Where the parts of one kv head's slab begin, and its bytes."""
    codes, scales = page * dim // 2, page * dim // 8
    return 0, codes, codes + scales, 2 * codes + scales, 2 * (codes + scales)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    dt = TYPES[case["type"]]
    rand = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    rows, lens = _lengths(case)
    b, d, kv, h, page = case["seqs"], case["dim"], case["kv_heads"], case["heads"], case["page"]
    t = sum(rows) + case["behind"]
    cols = -(-max(lens) // page)
    pages = sum(-(-n // page) for n in lens) + 3
    s = {"case": case, "batch": None, "work": None, "most": max(rows)}
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["starts"] = torch.tensor(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32), device="cuda")
    # the sequences' pages lie anywhere in the cache; what is behind a sequence's last one is not a page
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    used = torch.arange(cols, device="cuda")[None, :] < ((s["lens"] + (page - 1)) // page)[:, None]
    table = torch.full((b, cols), -1, dtype=torch.int32, device="cuda")
    table[used] = order[: int(used.sum())]
    s["table"] = table
    at = _parts(page, d)
    cache = torch.zeros((pages, kv, at[4]), dtype=torch.uint8, device="cuda")
    s["cache"] = cache
    if case["op"] == "write":
        # q, k and v as one projection leaves them: parts of the same rows; channels of keys differ in size
        qkv = rand(t, h + 2 * kv, d)
        qkv[:, h:h + kv] *= torch.exp(0.5 * rand(kv, d))
        s["qkv"] = qkv.to(dt)
        s["q_out"] = torch.zeros((t, h, d), dtype=dt, device="cuda")
        n = case["rotated"] // 2
        s["freqs"] = torch.exp(torch.arange(n, device="cuda", dtype=torch.float64) * (-math.log(10000.0) / n)).float()
        axes = case["axes"]
        s["sections"] = [n - (axes - 1) * (n // axes)] + [n // axes] * (axes - 1)
        if axes > 1:
            # time goes on with the tokens, height and width lie on a grid
            time = torch.arange(t, device="cuda", dtype=torch.int32) + 17
            s["positions"] = torch.stack([time, time // 31 % 37, time % 31][:axes])
        else:
            s["positions"] = None
        s["k_out"] = torch.zeros((t, kv, d), dtype=torch.float16, device="cuda")
        s["v_out"] = torch.zeros((t, kv, d), dtype=torch.float16, device="cuda")
        return s
    # codes at random; a group reaches from about -2.5 to 2.5, larger for some channels
    groups = d // 32
    for k in range(2):
        codes, scales = cache[:, :, at[2 * k]:at[2 * k + 1]], cache[:, :, at[2 * k + 1]:at[2 * k + 2]]
        codes.copy_(torch.randint(0, 256, codes.shape, generator=g, device="cuda", dtype=torch.uint8))
        scale = 0.3 * torch.exp(0.3 * rand(pages, kv, page, groups)).half()
        small = (-7.5 * scale.float() + 0.2 * rand(pages, kv, page, groups)).half()
        both = torch.stack([scale, small], -1)
        if k:
            both = both.view(pages, kv, page // 4, 4, groups, 2).permute(0, 1, 2, 4, 5, 3)
        scales.copy_(both.contiguous().view(pages, kv, -1).view(torch.uint8))
    if case["op"] == "read":
        s["k_out"] = torch.zeros((t, kv, d), dtype=dt, device="cuda")
        s["v_out"] = torch.zeros((t, kv, d), dtype=dt, device="cuda")
        return s
    # some heads look at everything, some at few tokens
    s["q"] = (rand(t, h, d) * torch.exp(0.6 * rand(h, 1))).to(dt)
    s["out"] = torch.zeros((t, h, d), dtype=dt, device="cuda")
    return s


# ---- the plain forms -----------------------------------------------------------
def _unpacked(s):
    """Keys and values [seqs, kv heads, tokens, dim] in float32, out of the pages; tokens behind a sequence are 0."""
    c = s["case"]
    page, d, kv = c["page"], c["dim"], c["kv_heads"]
    at = _parts(page, d)
    table = s["table"].long()
    b, cols = table.shape
    slab = s["cache"][table.clamp(min=0)]
    groups, lead = d // 32, (b, cols, kv)
    there = torch.arange(cols * page, device="cuda")[None, :] < s["lens"][:, None]
    words = slab[..., at[0]:at[1]].contiguous().view(torch.int32).view(*lead, page, 4, groups, 1)
    shifts = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], dtype=torch.int32, device="cuda")
    codes = ((words >> shifts) & 15).transpose(-3, -2).reshape(*lead, page, groups, 32).float()
    sm = slab[..., at[1]:at[2]].contiguous().view(torch.float16).view(*lead, page, groups, 2, 1).float()
    k = codes * sm[..., 0, :] + sm[..., 1, :]
    halves = slab[..., at[2]:at[3]].contiguous().view(torch.int16).view(*lead, page // 4, d // 8, 2, 2, 2, 1).int()
    shifts = torch.tensor([0, 4, 8, 12], dtype=torch.int32, device="cuda")
    codes = ((halves >> shifts) & 15).permute(0, 1, 2, 3, 5, 7, 4, 6, 8).reshape(*lead, page, groups, 32).float()
    sm = slab[..., at[3]:at[4]].contiguous().view(torch.float16).view(*lead, page // 4, groups, 2, 4).float()
    sm = sm.permute(0, 1, 2, 3, 6, 4, 5).reshape(*lead, page, groups, 2, 1)
    v = codes * sm[..., 0, :] + sm[..., 1, :]
    k, v = (x.reshape(b, cols, kv, page, d).transpose(1, 2).reshape(b, kv, cols * page, d) for x in (k, v))
    zero = ~there[:, None, :, None]
    return k.masked_fill_(zero, 0.0), v.masked_fill_(zero, 0.0)


def _rows_of(s):
    """For the padded batch: each row's index among the T rows, whether it is one, and its position."""
    n = s["starts"][1:] - s["starts"][:-1]
    i = torch.arange(s["most"], device="cuda")[None, :]
    is_row = i < n[:, None]
    at = torch.where(is_row, s["starts"][:-1, None] + i, 0).long()
    return at, is_row, s["lens"][:, None] - n[:, None] + i


def _rotated(x, cos, sin, case):
    r = case["rotated"]
    x = x.float()
    if case["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., : r // 2], x[..., r // 2:r]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, x[..., r:]], -1)


def _held(x):
    """What 4 bits hold of float32 rows [..., dim]: groups of 32 with scale and smallest value in float16."""
    g = x.clamp(-LIMIT, LIMIT).unflatten(-1, (-1, 32))
    small = g.amin(-1, keepdim=True).half().float()
    scale = ((g.amax(-1, keepdim=True) - small) * torch.tensor(1 / 15, dtype=torch.float32, device="cuda")).half().float()
    code = torch.round((g - small) * torch.where(scale > 0, torch.reciprocal(scale), 0.0)).clamp(0, 15)
    return (code * scale + small).flatten(-2)


def _write_plain(s):
    c = s["case"]
    at, is_row, pos = _rows_of(s)
    t, h, kv = s["qkv"].shape[0], c["heads"], c["kv_heads"]
    place = torch.full((t,), -1, dtype=torch.int64, device="cuda")
    place[at[is_row]] = pos[is_row].long()
    here = (place >= 0)[:, None, None]
    n = s["freqs"].numel()
    if s["positions"] is None:
        angle = place.double()[:, None] * s["freqs"].double()
    else:
        axis = torch.repeat_interleave(torch.arange(len(s["sections"]), device="cuda"), torch.tensor(s["sections"], device="cuda"),
                                       output_size=n)
        angle = s["positions"].double()[axis].t() * s["freqs"].double()
    cos, sin = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]
    q = _rotated(s["qkv"][:, :h], cos, sin, c)
    k = _held(_rotated(s["qkv"][:, h:h + kv], cos, sin, c))
    v = _held(s["qkv"][:, h + kv:].float())
    return {"q": torch.where(here, q, 0.0).to(TYPES[c["type"]]), "k": torch.where(here, k, 0.0).half(), "v": torch.where(here, v, 0.0).half()}


def _read_plain(s):
    c = s["case"]
    k, v = _unpacked(s)
    at, is_row, pos = _rows_of(s)
    seq = torch.arange(c["seqs"], device="cuda")[:, None].expand_as(pos)
    out = []
    for x in (k, v):
        y = torch.zeros((s["k_out"].shape[0], c["kv_heads"], c["dim"]), device="cuda")
        y[at[is_row]] = x[seq[is_row], :, pos[is_row].long()]
        out.append(y.to(TYPES[c["type"]]))
    return {"k": out[0], "v": out[1]}


def _attend_plain(s):
    c = s["case"]
    d, kv, h = c["dim"], c["kv_heads"], c["heads"]
    r = h // kv
    k, v = _unpacked(s)
    at, is_row, pos = _rows_of(s)
    b, n = at.shape
    q = s["q"].float()[at].view(b, n, kv, r, d).permute(0, 2, 1, 3, 4).reshape(b, kv, n * r, d)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1.0 / d ** 0.5)
    del k
    if c["softcap"]:
        x = torch.tanh(x / c["softcap"]) * c["softcap"]
    j = torch.arange(x.shape[3], device="cuda")
    seen = j <= pos[:, :, None]
    if c["window"]:
        seen &= j > pos[:, :, None] - c["window"]
    x = x.view(b, kv, n, r, -1)
    hidden = ~seen[:, None, :, None, :]
    x.masked_fill_(hidden, -float("inf"))
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top == -float("inf"), 0.0, top)).exp_()
    total = x.sum(-1, keepdim=True)
    y = torch.matmul(x.view(b, kv, n * r, -1), v).view(b, kv, n, r, d) / torch.where(total == 0, 1.0, total)
    out = torch.zeros_like(s["out"])
    out[at[is_row]] = y.permute(0, 2, 1, 3, 4).reshape(b, n, h, d)[is_row].to(out.dtype)
    return out


# ---- the framework's calls ------------------------------------------------------
_LANE = _STREAM = None


def _lane():
    """The lane and the one stream that the program's calls go to."""
    global _LANE, _STREAM
    if _LANE is None:
        import crosslane_amd as xl
        # the calls use no expert bank: the smallest one
        _LANE = xl.Lane(256, 256, 1, 1, np.full((1, 1, 3), xl.IQ1_M, np.int32))
        _STREAM = torch.cuda.Stream().cuda_stream
    return _LANE, _STREAM


def _run_own(s):
    import crosslane_amd as xl
    lane, stream = _lane()
    c = s["case"]
    h, kv = c["heads"], c["kv_heads"]
    if s["batch"] is None:   # kept with the cache and the buffers of the batch, as a serving loop does
        rows = s["qkv" if c["op"] == "write" else "q" if c["op"] == "attend" else "k_out"].shape[0]
        s["batch"] = xl.KVBatch(s["cache"], s["table"], s["lens"], s["starts"], rows, c["dim"], max_rows=s["most"])
        if c["op"] == "attend":
            s["work"] = torch.empty(xl.attention_work_bytes(s["batch"], h), dtype=torch.uint8, device="cuda")
    if c["op"] == "attend":
        lane.attention_async(s["batch"], s["q"], s["out"], window=c["window"], softcap=c["softcap"], work=s["work"], stream=stream)
        return s["out"]
    if c["op"] == "write":
        qkv = s["qkv"]
        lane.kv_write_async(s["batch"], qkv[:, h:h + kv], qkv[:, h + kv:], q=qkv[:, :h], q_out=s["q_out"], freqs=s["freqs"],
                            positions=s["positions"], sections=s["sections"], interleaved=c["interleaved"], stream=stream)
    lane.kv_read_async(s["batch"], s["k_out"], s["v_out"], stream=stream)
    return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]} if c["op"] == "write" else {"k": s["k_out"], "v": s["v_out"]}


def run(s):
    if own:
        return _run_own(s)
    return {"write": _write_plain, "read": _read_plain, "attend": _attend_plain}[s["case"]["op"]](s)


# ---- the definitions in 64 bits ---------------------------------------------------
def _values64(s, seq, upto):
    """Keys and values [tokens, kv heads, dim] of one sequence's first tokens in float64, each value from its own address."""
    c = s["case"]
    page, d, kv = c["page"], c["dim"], c["kv_heads"]
    at = _parts(page, d)
    flat, slab = s["cache"].reshape(-1), at[4]
    tok = torch.arange(upto, device="cuda")
    base = s["table"][seq].long()[tok // page][:, None, None] * (kv * slab) + torch.arange(kv, device="cuda")[None, :, None] * slab
    t = (tok % page)[:, None, None]
    x = torch.arange(d, device="cuda")[None, None, :]
    half = lambda a: (flat[a].int() | (flat[a + 1].int() << 8)).to(torch.int16).view(torch.float16).double()  # noqa: E731
    nibble = x % 8 // 2 + 4 * (x % 2)
    byte = t * (d // 2) + 4 * ((x % 32 // 8) * (d // 32) + x // 32) + nibble // 2
    a = base + at[1] + (t * (d // 32) + x // 32) * 4
    k = ((flat[base + at[0] + byte].int() >> (4 * (nibble % 2))) & 15).double() * half(a) + half(a + 2)
    byte = (t // 4) * 2 * d + (x // 8) * 16 + (t // 2 % 2) * 8 + (x // 4 % 2) * 4 + (t % 2) * 2 + x % 4 // 2
    a = base + at[3] + ((t // 4) * (d // 32) + x // 32) * 16 + (t % 4) * 2
    v = ((flat[base + at[2] + byte].int() >> (4 * (x % 2))) & 15).double() * half(a) + half(a + 8)
    return k, v


def _held64(x):
    y = torch.empty_like(x)
    for at in range(0, x.shape[-1], 32):
        g = x[..., at:at + 32].clamp(-LIMIT, LIMIT)
        low = g.min(-1, keepdim=True).values.half().double()
        step = ((g.max(-1, keepdim=True).values - low) / 15).half().double()
        code = torch.round((g - low) / torch.where(step == 0, 1.0, step)).clamp(0, 15)
        y[..., at:at + 32] = low + step * torch.where(step == 0, 0.0, code)
    return y


def _exact_write(s):
    c = s["case"]
    h, kv, r = c["heads"], c["kv_heads"], c["rotated"]
    x = s["qkv"].double()
    rows, lens = _lengths(c)
    done, n = torch.zeros_like(x), r // 2
    pairs = [(2 * i, 2 * i + 1) for i in range(n)] if c["interleaved"] else [(i, i + n) for i in range(n)]
    axis = [a for a, m in enumerate(s["sections"]) for _ in range(m)]
    own_place = torch.cat([torch.arange(ln - m, ln, device="cuda") for m, ln in zip(rows, lens)])
    t = own_place.numel()
    done[:t] = x[:t]
    for i, (a, b) in enumerate(pairs):
        place = own_place if s["positions"] is None else s["positions"][axis[i], :t]
        turn = (place.double() * s["freqs"][i].double())[:, None]
        p, q = x[:t, : h + kv, a], x[:t, : h + kv, b]
        done[:t, : h + kv, a] = p * torch.cos(turn) - q * torch.sin(turn)
        done[:t, : h + kv, b] = q * torch.cos(turn) + p * torch.sin(turn)
    return {"q": done[:, :h], "k": _held64(done[:, h:h + kv]), "v": _held64(done[:, h + kv:])}


def _exact_read(s):
    c = s["case"]
    rows, lens = _lengths(c)
    k = torch.zeros((s["k_out"].shape[0], c["kv_heads"], c["dim"]), dtype=torch.float64, device="cuda")
    v, at = torch.zeros_like(k), 0
    for b, (n, ln) in enumerate(zip(rows, lens)):
        a, z = _values64(s, b, ln)
        k[at:at + n], v[at:at + n] = a[ln - n:], z[ln - n:]
        at += n
    return {"k": k, "v": v}


def _exact_attend(s):
    c = s["case"]
    rows, lens = _lengths(c)
    r = c["heads"] // c["kv_heads"]
    out, at = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for b, (n, ln) in enumerate(zip(rows, lens)):
        k, v = _values64(s, b, ln)
        place = torch.arange(ln - n, ln, device="cuda")[:, None]
        tok = torch.arange(ln, device="cuda")[None, :]
        off = (tok > place) | (tok <= place - c["window"] if c["window"] else tok < 0)
        for head in range(c["heads"]):
            x = s["q"][at:at + n, head].double() @ k[:, head // r].t() / math.sqrt(c["dim"])
            if c["softcap"]:
                x = c["softcap"] * torch.tanh(x / c["softcap"])
            x[off] = -math.inf
            p = torch.softmax(x, 1)
            p[off.all(1)] = 0.0
            out[at:at + n, head] = p @ v[:, head // r]
        at += n
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"write": _exact_write, "read": _exact_read, "attend": _exact_attend}[case["op"]](s)
