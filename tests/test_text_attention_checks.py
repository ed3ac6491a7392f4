"""What cross_attention and text_attention refuse, the buckets, and the workspace rules, without a GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from selas_amd import _lib
from selas_amd import text_attention as ta

from .text_attention_reference import bucket_map, side_of


def problem(**kw):
    v = dict(q=4096, q_sb=0, q_sh=64, q_sl=256, k=4096, k_sb=0, k_sh=64, k_sl=256, v=4096, v_sb=0, v_sh=64, v_sl=256, out=4096,
             o_sb=0, o_sl=256, lse=0, lengths=0, mask=0, mask_sb=0, start=0, start0=0, table=0, table_sl=4, B=1, H=4, Hk=4,
             Lq=100, Lk=100, Dh=64, buckets=32, max_distance=128, scale=0.125, table_dt=2, both=1, causal=0, reserved=0)
    v.update(kw)
    return ta._PROBLEM.pack(*v.values())


def forward(ws=None, size=0, dtype=_lib.BF16, **kw):
    _lib.call("selas_text_attention", problem(**kw), dtype, ws, size, None)


def backward(grad=4096, g_sb=0, g_sl=256, dq=4096, dk=4096, dv=4096, dtable=4096, ws=None, size=0, dtype=_lib.BF16, **kw):
    _lib.call("selas_text_attention_backward", problem(**{"lse": 4096, **kw}), grad, g_sb, g_sl, dq, dk, dv, dtable, dtype, ws,
              size, None)


def query(name="selas_text_attention_workspace_bytes", dtype=_lib.BF16, **kw):
    n = ctypes.c_int64(-1)
    _lib.call(name, problem(**kw), dtype, ctypes.byref(n))
    return n.value


def test_the_structure_has_the_headers_layout():
    assert ta._PROBLEM.size == 8 * (12 + 3 + 1 + 2 + 1 + 2 + 2 + 8 + 1) + 4 * 4


@pytest.mark.parametrize("kw,match", [({"B": -1}, "shape"), ({"Lq": -1}, "shape"), ({"Lk": -1}, "shape"), ({"Dh": 0}, "shape"),
                                      ({"Hk": 3}, "evenly"), ({"Hk": 0}, "evenly"), ({"scale": 0.0}, "scale"),
                                      ({"scale": -1.0}, "scale"), ({"scale": float("nan")}, "scale"), ({"scale": 1e11}, "scale"),
                                      ({"reserved": 1}, "reserved"), ({"q_sl": -8}, "negative"), ({"o_sb": -4}, "negative"),
                                      ({"mask": 16, "mask_sb": -1}, "negative"), ({"q": 0}, "null"), ({"k": 0}, "null"),
                                      ({"v": 0}, "null"), ({"out": 0}, "null"), ({"table": 16, "table_dt": 7}, "table dtype"),
                                      ({"table": 16, "table_sl": -4}, "negative"), ({"table": 16, "buckets": 31}, "halve"),
                                      ({"table": 16, "buckets": 2}, "two buckets"), ({"table": 16, "max_distance": 8}, "max_distance")])
def test_bad_calls_are_refused(kw, match):
    with pytest.raises(ValueError, match=match):
        forward(**kw)
    with pytest.raises(ValueError, match=match):
        backward(**kw)


@pytest.mark.parametrize("kw,match", [({"Dh": 136}, "head dims"), ({"Dh": 12}, "head dims"), ({"q": 4104}, "16-byte"),
                                      ({"k_sl": 260}, "whole 16"), ({"v_sh": 4}, "whole 16"), ({"out": 4100}, "8-byte"),
                                      ({"o_sl": 258}, "whole 8"), ({"q_sl": 1 << 24}, "2\\^23"), ({"o_sl": 1 << 24}, "2\\^23"),
                                      ({"Lq": 1 << 30}, "2\\^26"), ({"B": 1 << 26}, "2\\^26"),
                                      ({"table": 16, "buckets": 512, "max_distance": 300}, "128 buckets"), ({"table": 16, "max_distance": 513}, "512")])
def test_what_the_kernels_do_not_cover_is_unsupported(kw, match):
    with pytest.raises(_lib.Unsupported, match=match):
        forward(**kw)
    with pytest.raises(_lib.Unsupported, match=match):
        backward(**kw)


def test_types():
    for call in (forward, backward):
        with pytest.raises(_lib.Unsupported, match="bf16 or fp16"):
            call(dtype=_lib.F32)
        with pytest.raises(ValueError, match="dtype"):
            call(dtype=9)


def test_bad_gradients_are_refused():
    for kw in ({"grad": 0}, {"lse": 0}, {"dq": 0}, {"dk": 0}, {"dv": 0}, {"table": 16, "dtable": 0}):
        with pytest.raises(ValueError, match="null"):
            backward(**kw)
    with pytest.raises(ValueError, match="negative"):
        backward(g_sl=-8)
    for kw in ({"grad": 4104}, {"g_sb": 4}, {"g_sl": 1 << 24}, {"dq": 4100}, {"dv": 4100}):
        with pytest.raises(_lib.Unsupported):
            backward(**kw)


def test_empty_calls_launch_nothing():
    forward(B=0, q=0, k=0, v=0, out=0)
    forward(Lq=0, q=0, k=0, v=0, out=0)
    forward(H=0, Hk=0, q=0, k=0, v=0, out=0)
    backward(H=0, Hk=0, q=0, k=0, v=0, out=0, grad=0, lse=0, dq=0, dk=0, dv=0)


def test_a_missing_workspace_is_refused():
    long = dict(Lq=64, Lk=20000)  # few rows over a long axis: the keys are split
    need = query(**long)
    assert need > 0 and need % 4 == 0 and query(Lq=4096, Lk=512, B=8) == 0 and query(Lq=1, Lk=20000) > 0
    name = "selas_text_attention_backward_workspace_bytes"
    for call, kw, size in ((forward, long, need), (backward, {}, query(name)), (backward, long, query(name, **long))):
        assert size > 0
        for ws, given in ((None, 0), (4096, size - 1), (4104, size)):
            with pytest.raises(ValueError, match="workspace"):
                call(ws=ws, size=given, **kw)
    with pytest.raises(ValueError, match="null"):
        _lib.call("selas_text_attention_workspace_bytes", problem(), _lib.BF16, None)


def edges(buckets, distance, both):
    e, n = (ctypes.c_int32 * 128)(), ctypes.c_int64()
    _lib.call("selas_relative_buckets", buckets, distance, both, e, ctypes.byref(n))
    return list(e[:n.value])


@pytest.mark.parametrize("n", [2, 3, 4, 7, 12, 16, 31, 32, 64, 101, 127, 128])
def test_buckets_begin_where_whole_numbers_say(n):
    for distance in sorted({n // 2 + 1, n // 2 + 2, 2 * (n // 2), 4 * (n // 2), 16 * (n // 2), 100, 128, 333, 512}):
        if not n // 2 < distance <= 512:
            continue
        side = side_of(n, distance)
        e = edges(n, distance, 0)
        assert len(e) == n and e[0] == 0
        assert [sum(d >= x for x in e) - 1 for d in range(distance + 1)] == side
        assert edges(2 * n, distance, 1) == e


def test_buckets_of_the_usual_sizes():
    assert edges(32, 128, 1) == [0, 1, 2, 3, 4, 5, 6, 7, 8, 12, 16, 23, 32, 46, 64, 91]
    rel = torch.tensor([-200, -128, -91, -90, -8, -1, 0, 1, 8, 11, 12, 500])
    assert bucket_map(rel, 32, 128, True).tolist() == [15, 15, 15, 14, 8, 1, 0, 17, 24, 24, 25, 31]
    assert bucket_map(rel, 32, 128, False).tolist()[6:] == [0] * 6
    with pytest.raises(ValueError, match="null"):
        _lib.call("selas_relative_buckets", 32, 128, 1, None, None)


def heads(b=2, h=4, l=10, dh=64, dtype=torch.bfloat16):
    return torch.zeros(b, h, l, dh, dtype=dtype)


@pytest.mark.parametrize("args,match", [
    ((heads()[0], heads(), heads()), "are \\[B, heads"), ((heads(), heads(h=3), heads(h=3)), "do not go"),
    ((heads(), heads(b=1), heads(b=1)), "do not go"), ((heads(), heads(dh=72), heads(dh=72)), "do not go"),
    ((heads(), heads(l=5), heads(l=6)), "do not go"), ((heads(), heads(), heads(dtype=torch.float16)), "one type"),
    ((heads(), heads(h=0), heads(h=0)), "do not go"), ((heads(), heads(), heads()), "runs on the GPU")])
def test_shapes_that_do_not_go_together(args, match):
    with pytest.raises(ValueError, match=match):
        ta.cross_attention(*args)


def test_tensors_that_require_grad_are_refused():
    q = heads().requires_grad_()
    with pytest.raises(ValueError, match="cross_attention_backward"):
        ta.cross_attention(q, heads(), heads())
    with pytest.raises(ValueError, match="text_attention_backward"):
        ta.text_attention(heads(), heads(), heads(), torch.zeros(32, 4).requires_grad_())
    with torch.no_grad(), pytest.raises(ValueError, match="runs on the GPU"):
        ta.cross_attention(q, heads(), heads())
