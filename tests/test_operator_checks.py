"""What raw_linear and rope_qk refuse, and the layout rules behind it, without a GPU."""

from __future__ import annotations

import ctypes
import itertools
import struct

import pytest
import torch

from selas_amd import _lib
from selas_amd._layout import distinct, may_meet, same_elements
from selas_amd.linear import RawLinear, raw_linear, raw_linear_batched
from selas_amd.rope import rope_qk

BF, F32 = torch.bfloat16, torch.float32


def elements(t):
    return {t.storage_offset() + sum(i * s for i, s in zip(at, t.stride()))
            for at in itertools.product(*map(range, t.shape))}


def test_distinct_says_whether_elements_share_an_address():
    base = torch.zeros(400)
    for shape, stride in (((3, 4), (4, 1)), ((3, 4), (1, 3)), ((3, 4), (3, 1)), ((3, 4), (0, 1)), ((1, 4), (0, 1)),
                          ((2, 3, 4), (50, 4, 1)), ((2, 3, 4), (4, 8, 1)), ((2, 3, 4), (4, 4, 1)), ((5,), (2,)), ((2, 2), (1, 1))):
        t = base.as_strided(shape, stride)
        want = len(elements(t)) == t.numel()
        assert distinct(t) <= want  # never called distinct wrongly
        assert distinct(t) == want or stride == (3, 1)


def test_may_meet_never_misses_an_overlap():
    base = torch.zeros(2, 6, 24)
    views = [base, base[:, 1:], base[..., :8], base[..., 8:16], base[..., 4:12], base[:, :, 16:], base[0], base[1, 2:, 3:9],
             base[:, 0], base.view(2, 6, 3, 2, 4).permute(2, 0, 3, 1, 4)[0], base.view(2, 6, 3, 2, 4).permute(2, 0, 3, 1, 4)[1],
             base.transpose(0, 1), base.view(12, 24)[:, 20:], base.view(-1)[:5], base.view(-1)[100:]]
    for a, b in itertools.product(views, views):
        meet = bool(elements(a) & elements(b))
        assert may_meet(a, b) or not meet
    q, k = (base.view(2, 6, 3, 2, 4).permute(2, 0, 3, 1, 4)[i] for i in (0, 1))
    assert not may_meet(q, k) and not may_meet(base[..., :8], base[..., 8:16]) and not may_meet(base[..., 8:16], base[..., :8])
    assert not may_meet(base[:0], base) and not may_meet(base, torch.zeros(288)) and may_meet(base[..., :9], base[..., 8:])
    assert same_elements(base[:, 1:], base[:, 1:]) and not same_elements(base[:, 1:], base[:, :-1])


def problem(**kw):
    v = dict(x=4096, x_sb=0, x_sl=64, w=4096, ldw=64, bias=0, gate=0, gate_sb=0, residual=0, r_sb=0, r_sl=0, y=4096, y_sb=0,
             y_sl=64, B=1, L=8, N=64, K=64, bias_dt=2, gate_dt=0, res_dt=0, y_dt=2, act=0, reserved=0)
    v.update(kw)
    return _lib.RAW_LINEAR_PROBLEM.pack(*v.values())


def query(*problems, dtype=_lib.BF16):
    n = ctypes.c_int64(-1)
    _lib.call("selas_raw_linear_workspace_bytes", b"".join(problems), len(problems), dtype, ctypes.byref(n))
    return n.value


def test_structures_have_the_headers_layout():
    assert _lib.RAW_LINEAR_PROBLEM.size == 8 * 18 + 4 * 6 and _lib.ROPE_PART.size == 88


@pytest.mark.parametrize("kw,match", [({"L": -1}, "shape"), ({"N": -1}, "shape"), ({"K": -1}, "shape"), ({"B": -1}, "shape"),
                                      ({"act": 3}, "activation"), ({"act": -1}, "activation"), ({"y_dt": 1}, "f32 or bf16"),
                                      ({"bias": 16, "bias_dt": 1}, "f32 or bf16"), ({"gate": 16, "gate_dt": 7}, "f32 or bf16"),
                                      ({"residual": 16, "res_dt": 1}, "f32 or bf16"), ({"x_sl": -64}, "negative"),
                                      ({"y_sb": -1}, "negative")])
def test_bad_linears_are_refused(kw, match):
    with pytest.raises(ValueError, match=match):
        query(problem(**kw))
    with pytest.raises(ValueError, match=match):
        _lib.call("selas_raw_linear", problem(**kw), 1, _lib.BF16, None, 0, None)


def test_linear_calls_that_launch_nothing():
    with pytest.raises(ValueError, match="up to 4"):
        query(*[problem()] * 5)
    with pytest.raises(ValueError, match="dtype"):
        query(problem(), dtype=9)
    with pytest.raises(_lib.Unsupported, match="bf16 or fp16"):
        query(problem(y_dt=0), dtype=_lib.F32)
    with pytest.raises(_lib.Unsupported, match="2\\^31"):
        query(problem(L=1 << 31))
    with pytest.raises(ValueError, match="null"):
        _lib.call("selas_raw_linear", problem(y=0), 1, _lib.BF16, None, 0, None)
    with pytest.raises(ValueError, match="null"):
        _lib.call("selas_raw_linear", problem(w=0), 1, _lib.BF16, None, 0, None)
    with pytest.raises(ValueError, match="null"):
        _lib.call("selas_raw_linear_workspace_bytes", problem(), 1, _lib.BF16, None)
    # Empty problems are no work, whatever their pointers.
    _lib.call("selas_raw_linear", problem(L=0, x=0, w=0, y=0) + problem(N=0, x=0, w=0, y=0), 2, _lib.BF16, None, 0, None)
    _lib.call("selas_raw_linear", None, 0, _lib.BF16, None, 0, None)


def test_a_missing_workspace_is_refused():
    split = problem(L=512, N=3072, K=12288, x_sl=12288, ldw=12288, y_sl=3072)  # few tiles, long K
    odd = problem(L=300, N=300, K=67, x_sl=67, ldw=67, y_sl=300)               # rows off alignment: copied
    for p in (split, odd):
        need = query(p)
        assert need > 0 and need % 16 == 0
        for ws, size in ((None, 0), (4096, need - 16), (4104, need)):
            with pytest.raises(ValueError, match="workspace"):
                _lib.call("selas_raw_linear", p, 1, _lib.BF16, ws, size, None)
    assert query(odd) == 16 * (300 + 300) * 16  # 67 columns as 128: 16 chunks of 16 bytes a row
    assert query(problem(L=4608, N=3072, K=64, y_sl=3072)) == 0


def test_workspace_depends_on_the_problems_alone():
    a, b = problem(L=512, N=1024, K=12288, x_sl=12288, ldw=12288, y_sl=1024), problem(L=20, N=96, K=4096, x_sl=4096, ldw=4096, y_sl=96)
    assert query(a) == query(a) and query(a, b) >= query(b)


def rope(parts=None, count=2, B=1, L=4, Dh=64, ids=4096, ids_dt=_lib.F32, ids_sb=0, ids_sl=2, dims=(32, 32), theta=1e4, halves=0,
         inverse=0, dtype=_lib.BF16, naxes=None):
    part = _lib.ROPE_PART.pack(4096, 0, 256, 64, 8192, 0, 256, 64, 0, 2, 1)
    _lib.call("selas_rope", part * count if parts is None else parts, count, B, L, Dh, ids, ids_dt, ids_sb, ids_sl,
              len(dims) if naxes is None else naxes, struct.pack(f"@{len(dims)}q", *dims), theta, halves, inverse, dtype, None)


@pytest.mark.parametrize("kw,match", [({"count": 0}, "1 to 3"), ({"count": 4}, "1 to 3"), ({"dims": (), "naxes": 0}, "axes"),
                                      ({"dims": (8,) * 5}, "axes"), ({"B": -1}, "shape"), ({"Dh": 0}, "shape"),
                                      ({"dtype": 5}, "dtype"), ({"ids_dt": _lib.BF16}, "positions"), ({"theta": 0.0}, "theta"),
                                      ({"theta": float("inf")}, "theta"), ({"theta": float("nan")}, "theta"),
                                      ({"dims": (33, 31)}, "even"), ({"dims": (-2, 32)}, "even"), ({"dims": (64, 2)}, "heads 64"),
                                      ({"ids": None}, "positions"), ({"ids_sl": -1}, "positions")])
def test_bad_rotations_are_refused(kw, match):
    with pytest.raises(ValueError, match=match):
        rope(**kw)


def test_bad_rotation_tensors_are_refused():
    good = (4096, 0, 256, 64, 8192, 0, 256, 64, 0, 2, 1)
    for at, value, match in ((0, 0, "null"), (4, 0, "null"), (9, -1, "negative"), (2, -256, "negative"), (7, -1, "negative")):
        bad = list(good)
        bad[at] = value
        with pytest.raises(ValueError, match=match):
            rope(parts=_lib.ROPE_PART.pack(*bad), count=1)
    with pytest.raises(ValueError, match="inverse"):
        rope(parts=_lib.ROPE_PART.pack(*good[:8], 4096, 2, 1), count=1, inverse=1)
    with pytest.raises(_lib.Unsupported, match="head_dim"):
        rope(Dh=258, dims=(32, 32))
    with pytest.raises(_lib.Unsupported, match="alignment"):
        rope(Dh=162, dims=(32, 32))
    with pytest.raises(_lib.Unsupported, match="tokens"):
        rope(B=1 << 16, L=1 << 16)
    rope(parts=_lib.ROPE_PART.pack(0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1), count=1)  # no heads: nothing to do
    rope(L=0, ids=None)


def test_python_refusals_before_any_device_work():
    x, w = torch.zeros(4, 16, dtype=BF), torch.zeros(8, 16, dtype=BF)
    with pytest.raises(ValueError, match="GPU"):
        raw_linear(x, w)
    assert raw_linear_batched([]) == []
    with pytest.raises(ValueError, match="GPU"):
        raw_linear_batched([RawLinear(x, w), RawLinear(x, w, residual=torch.zeros(4, 8))])
    q = torch.zeros(1, 2, 3, 8)
    for args, match in (((q[0], q, torch.zeros(3, 1), (8,)), "B, heads"), ((q, q, torch.zeros(3, 1), (8,)), "GPU")):
        with pytest.raises(ValueError, match=match):
            rope_qk(*args)
    with pytest.raises(ValueError, match="pairs"):
        rope_qk(q, q, torch.zeros(3, 1), (8,), pairs="both")


def tile(m, n, k, *more):
    ps = [problem(L=m, N=n, K=k, x_sl=k, ldw=k, y_sl=n) for m, n, k in ((m, n, k), *more)]
    out = [ctypes.c_int64(-1) for _ in range(3)]
    _lib.call("selas_raw_linear_tile", b"".join(ps), len(ps), _lib.BF16, *map(ctypes.byref, out))
    return tuple(o.value for o in out)


def test_tiles_and_ranges():
    # Full grids run whole wide tiles, narrow ones fill the CUs of smaller grids, long K of few tiles is split.
    assert tile(4608, 3072, 15360) == (256, 256, 1) and tile(4096, 12288, 3072) == (256, 256, 1)
    assert tile(1536, 3072, 3072) == (256, 128, 1)
    assert tile(512, 3072, 3072)[:2] == (128, 128) and tile(512, 3072, 12288)[2] > 1
    assert tile(32, 3072, 3072) == tile(4096, 64, 3072) == tile(0, 64, 64) == (0, 0, 0)
    assert tile(28, 96, 64, (4608, 3072, 15360)) == (256, 256, 1)  # the few rows do not count
    with pytest.raises(ValueError, match="null"):
        _lib.call("selas_raw_linear_tile", problem(), 1, _lib.BF16, None, None, None)
