"""The operators around a block of an 8-bit model, as cases that a timing program runs.

A case is one pass through one of them, on what a serving loop has in hand:

  route   the router of T tokens: softmax or sigmoid scores, a bias for balance,
          groups of experts, top-k, renormalized weights
  norm    what lies between two blocks: the norm of a block's output, its gate,
          the scaled residual, the norm that makes the next block's input
  linear  the product with int8 weights, scales for each token and each output
          channel; the activations arrive as floats and are quantized by the call
          or arrive as int8; `gated`: two matrices and SwiGLU (gate and up)
  normed  norm and linear as a block has them: the next block's input leaves the
          norm as int8 and goes straight into the product

With `own` false, `run` computes them with elementary torch operations in 32 bits
(the router's scores and keys in 64: picks are whole numbers, and keys of two
experts may lie closer than 32 bits tell), with `own` true it makes the calls of
`crosslane_amd.Lane`. `exact` evaluates the definitions in 64 bits.
"""
import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6
MASKED = -1e300    # key of an expert whose logit is -inf
TINY = 1e-20       # added to the sum of the picked scores


# ---- the cases ---------------------------------------------------------------
def listed():
    return [
        # one decoded token's router: latency alone
        {"name": "route_decode", "op": "route", "tokens": 1, "experts": 256, "score": "sigmoid", "groups": 8,
         "top_groups": 4, "group_keys": 2, "picks": 8, "renorm": True, "scale": 2.5, "bias": True, "type": "f32",
         "masked": 0.0},
        # a prefill chunk over many experts without groups, logits as a bf16 product leaves them
        {"name": "route_chunk", "op": "route", "tokens": 2048, "experts": 384, "score": "softmax", "groups": 1,
         "top_groups": 1, "group_keys": 1, "picks": 6, "renorm": True, "scale": 1.0, "bias": False, "type": "bf16",
         "masked": 0.0},
        # a long prefill with groups and bias, some experts switched off for some tokens
        {"name": "route_prefill", "op": "route", "tokens": 8192, "experts": 256, "score": "sigmoid", "groups": 8,
         "top_groups": 4, "group_keys": 2, "picks": 8, "renorm": True, "scale": 2.5, "bias": True, "type": "f32",
         "masked": 0.05},
        # between two blocks of one decoded token
        {"name": "norm_decode", "op": "norm", "tokens": 1, "dim": 5120, "type": "f32", "res_type": "f32", "post": True,
         "gate": "channel", "alpha": 1.0, "pre": True, "pad": 0},
        # an odd width out of a wider buffer, a gate for each token, the residual stream in 32 bits
        {"name": "norm_odd", "op": "norm", "tokens": 771, "dim": 4099, "type": "f16", "res_type": "f32", "post": False,
         "gate": "token", "alpha": 0.5, "pre": True, "pad": 5},
        # a long prefill at the model's width
        {"name": "norm_prefill", "op": "norm", "tokens": 8192, "dim": 5120, "type": "bf16", "res_type": "bf16",
         "post": True, "gate": "channel", "alpha": 1.0, "pre": True, "pad": 0},
        # one decoded token through a projection: the weights' bytes are all there is
        {"name": "linear_decode", "op": "linear", "tokens": 1, "dim": 5120, "rows": 4096, "type": "f32", "gated": False,
         "limit": 0.0, "quantized": False},
        # a batched decode step through gate and up of the real expert's shape
        {"name": "linear_batch", "op": "linear", "tokens": 24, "dim": 5120, "rows": 2304, "type": "bf16", "gated": True,
         "limit": 10.0, "quantized": False},
        # sizes that no tile divides
        {"name": "linear_ragged", "op": "linear", "tokens": 333, "dim": 2301, "rows": 1111, "type": "f16",
         "gated": False, "limit": 0.0, "quantized": False},
        # the down product of a prefill chunk
        {"name": "linear_chunk", "op": "linear", "tokens": 512, "dim": 2304, "rows": 5120, "type": "bf16",
         "gated": False, "limit": 0.0, "quantized": False},
        # gate and up of a long prefill: what the matrix cores can do
        {"name": "linear_prefill", "op": "linear", "tokens": 8192, "dim": 5120, "rows": 4096, "type": "bf16",
         "gated": True, "limit": 0.0, "quantized": True},
        # norm, quantization and projection of a prefill chunk as one block makes them
        {"name": "normed_chunk", "op": "normed", "tokens": 2048, "dim": 4096, "rows": 5120, "type": "bf16",
         "res_type": "bf16", "post": True, "gate": "channel", "alpha": 1.0, "pre": True, "pad": 0, "gated": False,
         "limit": 0.0, "quantized": True},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(("route", "norm", "linear", "linear", "normed"))
    if op == "route":
        groups = rng.choice((1, 1, 2, 4, 8, 16))
        size = _log(rng, 8, 1024 // groups) if groups > 1 else _log(rng, 17, 1024)
        top = rng.randint(1, groups)
        return {"op": op, "tokens": _log(rng, 1, 8192), "experts": groups * size, "score": rng.choice(("softmax", "sigmoid")),
                "groups": groups, "top_groups": top, "group_keys": rng.choice((1, 2)), "picks": rng.randint(1, min(16, top * size)),
                "renorm": rng.random() < 0.7, "scale": rng.choice((1.0, 2.5, 16.0)), "bias": rng.random() < 0.5,
                "type": rng.choice(("f32", "f32", "bf16", "f16")), "masked": rng.choice((0.0, 0.0, 0.1, 0.9))}
    norm = {"post": rng.random() < 0.6, "gate": rng.choice(("none", "channel", "channel", "token")),
            "alpha": rng.choice((1.0, 0.5, 2.25)), "pre": rng.random() < 0.8 or op == "normed", "pad": rng.choice((0, 0, 8, 3))}
    most = 8192 * 5120
    if op == "norm":
        d = _log(rng, 64, 16384)
        return {"op": op, "tokens": _log(rng, 1, min(8192, most // d)), "dim": d, "type": rng.choice(("f32", "bf16", "f16")),
                "res_type": rng.choice(("f32", "f32", "same")), **norm}
    k = _log(rng, 32, 8192)
    n = _log(rng, 16, 9216)
    gated = rng.random() < 0.4
    t = _log(rng, 1, max(1, min(8192, most * 8192 // (k * n * (2 if gated else 1)), most // k)))
    limit = rng.choice((0.0, 7.0, 10.0)) if gated else 0.0
    if op == "normed":
        return {"op": op, "tokens": t, "dim": k, "rows": n, "type": rng.choice(("bf16", "f16")), "res_type": rng.choice(("f32", "same")),
                **norm, "gated": gated, "limit": limit, "quantized": True}
    return {"op": op, "tokens": t, "dim": k, "rows": n, "type": rng.choice(("f32", "bf16", "f16")), "gated": gated, "limit": limit,
            "quantized": rng.random() < 0.3}


def _res_type(case):
    return case["type"] if case["res_type"] == "same" else case["res_type"]


def work(case):
    t, es = case["tokens"], BYTES[case["type"]]
    if case["op"] == "route":
        n = case["experts"]
        return {"bytes": t * n * es + t * case["picks"] * 8 + (4 * n if case["bias"] else 0), "flops": 30 * t * n}
    d = case["dim"]
    nbytes = flops = 0
    if case["op"] in ("norm", "normed"):
        rs = BYTES[_res_type(case)]
        nbytes += t * d * (es + 2 * rs) + (4 * d if case["post"] else 0)
        nbytes += {"none": 0, "channel": d * es, "token": t * d * es}[case["gate"]]
        if case["pre"]:
            nbytes += 4 * d + (t * d * es if case["op"] == "norm" else 0)
        flops += 10 * t * d
    if case["op"] in ("linear", "normed"):
        n, m = case["rows"], 2 if case["gated"] else 1
        if case["op"] == "linear":
            nbytes += t * d + 4 * t if case["quantized"] else t * d * es
        nbytes += m * (n * d + 4 * n) + t * n * es
        flops += 2 * m * t * n * d
    return {"bytes": nbytes, "flops": flops}


# ---- inputs ------------------------------------------------------------------
def _wide(shape, pad, dtype, g, spread=1.0):
    """Rows of normal values, a part of a buffer with `pad` more columns."""
    x = torch.randn((shape[0], shape[1] + pad), generator=g, device="cuda") * spread
    return x.to(dtype)[:, : shape[1]]


def _quantized(x):
    """int8 and a float32 scale for each row."""
    s = x.abs().amax(1) / 127.0
    return torch.round(x / s[:, None]).clamp(-127, 127).to(torch.int8), s


def _weights(n, k, g):
    """int8 rows of normal weights, 16-byte aligned rows, a scale for each; the product of normal rows is about one."""
    w = torch.empty((n, -(-k // 16) * 16), dtype=torch.int8, device="cuda")
    w.zero_()
    scale = torch.empty(n, device="cuda")
    for at in range(0, n, 1024):
        m = min(1024, n - at)
        rows = torch.randn((m, k), generator=g, device="cuda") * torch.exp(0.3 * torch.randn((m, 1), generator=g, device="cuda"))
        w[at:at + m, :k], scale[at:at + m] = _quantized(rows / k ** 0.5)
    return w[:, :k], scale


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    t, dt = case["tokens"], TYPES[case["type"]]
    rand = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    s = {"case": case}
    if case["op"] == "route":
        n, k = case["experts"], case["picks"]
        logits = 2.0 * rand(t, n)
        if case["masked"]:
            off = torch.rand((t, n), generator=g, device="cuda") < case["masked"]
            logits = torch.where(off, torch.full_like(logits, -float("inf")), logits)
        s["logits"] = logits.to(dt)
        s["bias"] = 0.2 * rand(n) if case["bias"] else None
        s["ids"] = torch.zeros((t, k), dtype=torch.int32, device="cuda")
        s["w"] = torch.zeros((t, k), device="cuda")
        return s
    d = case["dim"]
    if case["op"] in ("norm", "normed"):
        rt = TYPES[_res_type(case)]
        s["y"] = _wide((t, d), case["pad"], dt, g, 0.7)
        s["res"] = _wide((t, d), case["pad"], rt, g, 3.0)
        s["post_w"] = 1.0 + 0.1 * rand(d) if case["post"] else None
        s["pre_w"] = 1.0 + 0.1 * rand(d) if case["pre"] else None
        s["gate"] = {"none": lambda: None, "channel": lambda: (0.3 * rand(d)).to(dt),
                     "token": lambda: (0.5 + 0.3 * rand(t, d)).to(dt)}[case["gate"]]()
        s["res_out"] = torch.zeros((t, d), dtype=rt, device="cuda")
        if case["op"] == "norm":
            s["x_out"] = torch.zeros((t, d), dtype=dt, device="cuda") if case["pre"] else None
            return s
    n = case["rows"]
    s["mats"] = [_weights(n, d, g) for _ in range(2 if case["gated"] else 1)]
    if case["op"] == "linear":
        # channels differ in size, as hidden states do
        x = rand(t, d) * torch.exp(0.5 * rand(d))
        if case["quantized"]:
            q, s["x_scale"] = _quantized(x)
            s["x"] = torch.zeros((t, -(-d // 16) * 16), dtype=torch.int8, device="cuda")[:, :d]
            s["x"].copy_(q)
        else:
            s["x"] = x.to(dt)
    else:
        s["x"] = torch.zeros((t, -(-d // 16) * 16), dtype=torch.int8, device="cuda")[:, :d]
        s["x_scale"] = torch.zeros(t, device="cuda")
    s["out"] = torch.zeros((t, n), dtype=dt, device="cuda")
    s["work"] = None
    return s


# ---- the plain forms -----------------------------------------------------------
def _route_plain(s):
    c = s["case"]
    logits = s["logits"].double()
    off = logits == -float("inf")
    if c["score"] == "softmax":
        top = logits.amax(1, keepdim=True)
        p = torch.where(off, 0.0, torch.exp(logits - torch.where(top == -float("inf"), 0.0, top)))
        total = p.sum(1, keepdim=True)
        score = p / torch.where(total == 0, 1.0, total)
    else:
        score = torch.where(off, 0.0, 1.0 / (1.0 + torch.exp(-logits)))
    key = score if s["bias"] is None else score + s["bias"].double()
    key = torch.where(off, MASKED, key)
    t, n = key.shape
    if c["groups"] > 1:
        by_group = key.view(t, c["groups"], n // c["groups"])
        value = torch.sort(by_group, dim=2, descending=True)[0][:, :, : c["group_keys"]].sum(2)
        kept = torch.sort(value, dim=1, descending=True, stable=True)[1][:, : c["top_groups"]]
        inside = torch.zeros_like(value, dtype=torch.bool).scatter_(1, kept, True)
        key = torch.where(inside[:, :, None], by_group, -float("inf")).view(t, n)
    ids = torch.sort(key, dim=1, descending=True, stable=True)[1][:, : c["picks"]]
    w = torch.gather(score, 1, ids)
    if c["renorm"]:
        w = w / (w.sum(1, keepdim=True) + TINY)
    return {"ids": ids.to(torch.int32), "w": (w * c["scale"]).float()}


def _rms(x):
    return x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)


def _norm_plain(s):
    """The new residual and the next block's input, in float32."""
    c = s["case"]
    a = s["y"].float()
    if c["post"]:
        a = _rms(a) * s["post_w"]
    if s["gate"] is not None:
        a = s["gate"].float() * a
    r = c["alpha"] * s["res"].float() + a
    return r, _rms(r) * s["pre_w"] if c["pre"] else None


def _product_plain(s, q, scale):
    """The int8 product in float32 (`q` whole numbers)."""
    c = s["case"]
    y = [(q @ w.float().t()) * scale[:, None] * ws for w, ws in s["mats"]]
    if not c["gated"]:
        return y[0]
    g, u = y
    if c["limit"] > 0:
        g, u = g.clamp(max=c["limit"]), u.clamp(-c["limit"], c["limit"])
    return g / (1.0 + torch.exp(-g)) * u


def _rows_plain(x):
    """Whole numbers -127..127 and a scale for each row of x."""
    scale = x.abs().amax(1) / 127.0
    q = torch.round(x / scale[:, None]).clamp(-127, 127)
    return torch.where(scale[:, None] == 0, 0.0, q), scale


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


def _linear_own(s, x, x_scale, lane, stream):
    c = s["case"]
    (w, ws), (up, ups) = s["mats"][0], s["mats"][1] if c["gated"] else (None, None)
    if s["work"] is None:   # kept with the weights, as a serving loop does
        import crosslane_amd as xl
        need = xl.linear_i8_work_bytes(c["tokens"], c["dim"], c["rows"], gated=c["gated"])
        s["work"] = torch.empty(need, dtype=torch.uint8, device="cuda")
    lane.linear_i8_async(x, w, ws, s["out"], x_scale=x_scale, up=up, up_scale=ups, limit=c["limit"], work=s["work"],
                         stream=stream)


def run(s):
    c = s["case"]
    if own:
        lane, stream = _lane()
        if c["op"] == "route":
            lane.route_scored_async(s["logits"], c["picks"], s["ids"], s["w"], score=c["score"], bias=s["bias"],
                                    groups=c["groups"], top_groups=c["top_groups"], group_keys=c["group_keys"],
                                    renorm=c["renorm"], scale=c["scale"], stream=stream)
            return {"ids": s["ids"], "w": s["w"]}
        if c["op"] == "linear":
            _linear_own(s, s["x"], s.get("x_scale"), lane, stream)
            return s["out"]
        normed = c["op"] == "normed"
        lane.block_norm_async(s["res"], y=s["y"], post_w=s["post_w"], gate=s["gate"], alpha=c["alpha"], pre_w=s["pre_w"],
                              eps=EPS, res_out=s["res_out"], x=None if normed else s["x_out"],
                              q=s["x"] if normed else None, q_scale=s["x_scale"] if normed else None, stream=stream)
        if not normed:
            return {"res": s["res_out"], "x": s["x_out"]}
        _linear_own(s, s["x"], s["x_scale"], lane, stream)
        return {"res": s["res_out"], "out": s["out"]}
    dt = TYPES[c["type"]]
    if c["op"] == "route":
        return _route_plain(s)
    if c["op"] == "linear":
        q, scale = (s["x"].float(), s["x_scale"]) if c["quantized"] else _rows_plain(s["x"].float())
        return _product_plain(s, q, scale).to(dt)
    r, x = _norm_plain(s)
    res = r.to(TYPES[_res_type(c)])
    if c["op"] == "norm":
        return {"res": res, "x": None if x is None else x.to(dt)}
    return {"res": res, "out": _product_plain(s, *_rows_plain(x)).to(dt)}


# ---- the definitions in 64 bits ---------------------------------------------------
def _exact_route(s):
    c = s["case"]
    logits = s["logits"].float().cpu().numpy().astype(np.float64)
    t, n = logits.shape
    on = np.isfinite(logits)
    if c["score"] == "softmax":
        top = np.max(np.where(on, logits, -1e300), axis=1, keepdims=True)
        e = np.exp(np.where(on, logits - top, -np.inf))
        e[~on] = 0.0
        score = e / np.maximum(e.sum(1, keepdims=True), 1e-300)
    else:
        score = np.zeros((t, n))
        score[on] = 1.0 / (1.0 + np.exp(-logits[on]))
    key = score.copy()
    if s["bias"] is not None:
        key += s["bias"].cpu().numpy().astype(np.float64)
    key[~on] = MASKED
    if c["groups"] > 1:
        size = n // c["groups"]
        value = np.empty((t, c["groups"]))
        for j in range(c["groups"]):
            part = np.sort(key[:, j * size:(j + 1) * size], axis=1)
            value[:, j] = part[:, -1] + (part[:, -2] if c["group_keys"] == 2 else 0.0)
        rank = np.argsort(np.argsort(-value, axis=1, kind="stable"), axis=1)
        key[np.repeat(rank >= c["top_groups"], size, axis=1)] = -np.inf
    ids = np.argsort(-key, axis=1, kind="stable")[:, : c["picks"]]
    w = np.take_along_axis(score, ids, 1)
    if c["renorm"]:
        w = w / (w.sum(1, keepdims=True) + TINY)
    return {"ids": ids.astype(np.int32), "w": w * c["scale"]}


def _exact_product(s, q, scale):
    c = s["case"]
    out = [torch.matmul(q, w.double().t()).mul_(scale[:, None]).mul_(ws.double()) for w, ws in s["mats"]]
    if c["gated"]:
        g, u = out
        if c["limit"] > 0:
            g, u = torch.clamp(g, max=c["limit"]), torch.clamp(u, min=-c["limit"], max=c["limit"])
        return g * torch.sigmoid(g) * u
    return out[0]


def _exact_rows(x):
    """Quants and scales of float64 rows; the scale is held in float32, as the operator defines it."""
    scale = (x.abs().max(1).values / 127.0).float().double()
    q = torch.where(scale[:, None] > 0, x / scale[:, None], torch.zeros_like(x)).round()
    return torch.clamp(q, -127, 127), scale


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "route":
        return _exact_route(s)
    if c["op"] == "linear":
        q, scale = (s["x"].double(), s["x_scale"].double()) if c["quantized"] else _exact_rows(s["x"].double())
        return _exact_product(s, q, scale)
    a = s["y"].double()
    if c["post"]:
        a = a / torch.sqrt(a.square().sum(1, keepdim=True) / c["dim"] + EPS) * s["post_w"].double()
    if s["gate"] is not None:
        a = a * s["gate"].double()
    r = s["res"].double() * c["alpha"] + a
    x = None
    if c["pre"]:
        x = r / torch.sqrt(r.square().sum(1, keepdim=True) / c["dim"] + EPS) * s["pre_w"].double()
    if c["op"] == "norm":
        return {"res": r, "x": x}
    return {"res": r, "out": _exact_product(s, *_exact_rows(x))}
