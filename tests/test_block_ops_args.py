"""What the calls around a block of an 8-bit model refuse, on the CPU: arguments
are checked before the context, so a null context shows whether a call got past
them. No pointer here is ever read."""
from __future__ import annotations

import ctypes as C

import pytest

import crosslane_amd as xl
from crosslane_amd import lane as L

A = 1 << 20   # addresses, far apart and aligned
PAST = b"null context"


def call(name, *args):
    err = L._Err()
    rc = getattr(xl.lib(), name)(None, *args, C.byref(err))
    return rc, err.message


ROUTE = dict(logits=A, type=0, T=4, stride=64, bias=None, n=64, score=1, groups=8, top=4, keys=2, k=6, renorm=1, scale=1.0,
             ids=2 * A, w=3 * A, stream=None)
NORM = dict(y=A, y_stride=100, res=2 * A, res_stride=100, gate=None, gate_stride=0, post=3 * A, pre=4 * A, T=4, D=100, type=2,
            res_type=0, alpha=1.0, eps=1e-6, res_out=5 * A, res_out_stride=100, x=6 * A, x_stride=100, q=7 * A, q_stride=112,
            q_scale=8 * A, stream=None)
QUANT = dict(x=A, type=1, T=4, K=100, x_stride=100, q=2 * A, q_stride=112, scale=3 * A, stream=None)
LIN = dict(x=A, x_type=0, x_scale=None, x_stride=100, T=4, K=100, w=2 * A, w_scale=3 * A, up=4 * A, up_scale=5 * A, w_stride=112,
           N=50, limit=0.0, out=6 * A, out_type=2, out_stride=50, work=7 * A, work_bytes=A, stream=None)
CALLS = {"xl_route_scored_async": ROUTE, "xl_block_norm_async": NORM, "xl_quantize_rows_async": QUANT,
         "xl_linear_i8_async": LIN}


@pytest.mark.parametrize("name", sorted(CALLS))
def test_good_arguments_reach_the_context(name):
    rc, msg = call(name, *CALLS[name].values())
    assert rc == 1 and PAST in msg


BAD = [
    ("xl_route_scored_async", {"logits": None}, "null"), ("xl_route_scored_async", {"ids": None}, "null"),
    ("xl_route_scored_async", {"w": None}, "null"), ("xl_route_scored_async", {"type": 3}, "f32"),
    ("xl_route_scored_async", {"T": 0}, "T outside"), ("xl_route_scored_async", {"T": -1}, "T outside"),
    ("xl_route_scored_async", {"n": 0}, "expert count"), ("xl_route_scored_async", {"n": 1025, "stride": 1025, "groups": 1, "top": 1}, "expert count"),
    ("xl_route_scored_async", {"score": 2}, "score"), ("xl_route_scored_async", {"groups": 7}, "groups"),
    ("xl_route_scored_async", {"groups": 0}, "groups"), ("xl_route_scored_async", {"top": 9}, "top_groups"),
    ("xl_route_scored_async", {"top": 0}, "top_groups"), ("xl_route_scored_async", {"keys": 3}, "group_keys"),
    ("xl_route_scored_async", {"groups": 64, "top": 64}, "group_keys"), ("xl_route_scored_async", {"k": 17}, "pick count"),
    ("xl_route_scored_async", {"k": 0}, "pick count"), ("xl_route_scored_async", {"top": 1, "k": 9}, "pick count"),
    ("xl_route_scored_async", {"scale": float("nan")}, "scale"), ("xl_route_scored_async", {"scale": -1.0}, "scale"),
    ("xl_route_scored_async", {"stride": 63}, "stride"), ("xl_route_scored_async", {"logits": A + 2}, "aligned"),
    ("xl_route_scored_async", {"ids": A + 64}, "overlaps"), ("xl_route_scored_async", {"w": 2 * A + 8}, "overlaps"),
    ("xl_block_norm_async", {"y": None, "res": None}, "neither"), ("xl_block_norm_async", {"y": None}, "gate and post"),
    ("xl_block_norm_async", {"res_out": None, "x": None, "q": None, "q_scale": None}, "no output"),
    ("xl_block_norm_async", {"pre": None}, "weights of the norm"), ("xl_block_norm_async", {"q_scale": None}, "together"),
    ("xl_block_norm_async", {"T": 0}, "T outside"), ("xl_block_norm_async", {"D": 0}, "D outside"),
    ("xl_block_norm_async", {"D": 32769}, "D outside"), ("xl_block_norm_async", {"type": 3}, "element types"),
    ("xl_block_norm_async", {"res_type": -1}, "element types"), ("xl_block_norm_async", {"eps": 0.0}, "eps"),
    ("xl_block_norm_async", {"alpha": float("inf")}, "alpha"), ("xl_block_norm_async", {"y_stride": 99}, "stride"),
    ("xl_block_norm_async", {"q_stride": 100}, "multiple of 16"), ("xl_block_norm_async", {"q": 7 * A + 8}, "16-byte"),
    ("xl_block_norm_async", {"gate": 9 * A + 1}, "aligned"), ("xl_block_norm_async", {"gate": 9 * A, "gate_stride": 99}, "stride"),
    ("xl_block_norm_async", {"res_out": 2 * A, "res_out_stride": 101}, "overlaps"),
    ("xl_block_norm_async", {"res_out": 2 * A + 4}, "overlaps"), ("xl_block_norm_async", {"x": A + 2}, "overlaps"),
    ("xl_block_norm_async", {"x": 4 * A}, "overlaps"), ("xl_block_norm_async", {"q": A}, "overlaps"),
    ("xl_quantize_rows_async", {"x": None}, "null"), ("xl_quantize_rows_async", {"type": 3}, "f32"),
    ("xl_quantize_rows_async", {"K": 65537, "x_stride": 1 << 17, "q_stride": 1 << 17}, "K outside"),
    ("xl_quantize_rows_async", {"T": 0}, "T outside"), ("xl_quantize_rows_async", {"q": 2 * A + 1}, "16-byte"),
    ("xl_quantize_rows_async", {"q_stride": 104}, "multiple of 16"), ("xl_quantize_rows_async", {"scale": A + 8}, "overlaps"),
    ("xl_linear_i8_async", {"x": None}, "null"), ("xl_linear_i8_async", {"work": None}, "null"),
    ("xl_linear_i8_async", {"up_scale": None}, "together"), ("xl_linear_i8_async", {"up": None}, "together"),
    ("xl_linear_i8_async", {"x_type": 4}, "x must be"), ("xl_linear_i8_async", {"x_type": 3}, "x_scale"),
    ("xl_linear_i8_async", {"x_scale": 9 * A}, "x_scale"), ("xl_linear_i8_async", {"out_type": 3}, "out must be"),
    ("xl_linear_i8_async", {"T": 0}, "T or N"), ("xl_linear_i8_async", {"N": 0}, "T or N"),
    ("xl_linear_i8_async", {"K": 65537, "x_stride": 1 << 17, "w_stride": 1 << 17}, "K outside"),
    ("xl_linear_i8_async", {"limit": float("nan")}, "limit"), ("xl_linear_i8_async", {"w_stride": 104}, "multiple of 16"),
    ("xl_linear_i8_async", {"w": 2 * A + 4}, "16-byte"), ("xl_linear_i8_async", {"up": 4 * A + 4}, "16-byte"),
    ("xl_linear_i8_async", {"x_type": 3, "x_scale": 9 * A}, "multiple of 16"),
    ("xl_linear_i8_async", {"w_stride": (1 << 20) + 16}, "2^20"), ("xl_linear_i8_async", {"out_stride": 49}, "stride"),
    ("xl_linear_i8_async", {"work_bytes": 0}, "workspace smaller"), ("xl_linear_i8_async", {"work": 7 * A + 16}, "256-byte"),
    ("xl_linear_i8_async", {"out": A}, "overlaps"), ("xl_linear_i8_async", {"work": 6 * A}, "overlaps"),
]


@pytest.mark.parametrize("name,change,message", BAD, ids=lambda v: v if isinstance(v, str) else "-".join(v))
def test_refusals(name, change, message):
    args = dict(CALLS[name])
    assert set(change) <= set(args)
    rc, msg = call(name, *{**args, **change}.values())
    assert rc == 1 and message.encode() in msg and PAST not in msg, msg


@pytest.mark.parametrize("change", [{"res_out": 2 * A}, {"x": A}, {"y": None, "post": None, "type": 0, "x": 6 * A},
                                    {"res": None}, {"gate": 9 * A}, {"gate": 9 * A, "gate_stride": 100},
                                    {"q": None, "q_scale": None}, {"x": None}, {"res_out": None},
                                    {"pre": None, "x": None, "q": None, "q_scale": None}])
def test_block_norm_optional_arguments(change):
    rc, msg = call("xl_block_norm_async", *{**NORM, **change}.values())
    assert rc == 1 and PAST in msg, msg


def test_work_bytes():
    assert xl.linear_i8_work_bytes(1, 1, 1) > 0
    assert xl.linear_i8_work_bytes(7, 4099, 100) >= 7 * 4099 + 7 * 4
    for bad in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (1, 65537, 1), ((1 << 19) + 1, 1, 1)):
        assert xl.linear_i8_work_bytes(*bad) == 0
    need = xl.linear_i8_work_bytes(LIN["T"], LIN["K"], LIN["N"], gated=True)
    rc, msg = call("xl_linear_i8_async", *{**LIN, "work_bytes": need}.values())
    assert PAST in msg
    rc, msg = call("xl_linear_i8_async", *{**LIN, "work_bytes": need - 1}.values())
    assert b"workspace smaller" in msg


def test_lane_refuses_host_tensors_and_wrong_types():
    torch = pytest.importorskip("torch")
    lane = object.__new__(xl.Lane)
    lane._ctx = None
    f = torch.zeros((2, 16))
    with pytest.raises(xl.XLError, match="not on the GPU"):
        lane.quantize_rows_async(f, f.to(torch.int8), torch.zeros(2))
    with pytest.raises(xl.XLError, match="contiguous rows"):
        lane.linear_i8_async(f.t(), f, f, f)
    with pytest.raises(xl.XLError, match="score must be"):
        lane.route_scored_async(f, 2, f, f, score="tanh")
    with pytest.raises(xl.XLError, match="res or y"):
        lane.block_norm_async(None)
