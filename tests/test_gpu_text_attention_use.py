"""cross_attention and text_attention as a program uses them: views and destinations, streams, graphs, long strides, refusals
that need a GPU, and the two in a row as a text encoder and what reads its states run them."""

from __future__ import annotations

import pytest
import torch

from selas_amd import _lib
from selas_amd.linear import raw_linear
from selas_amd.text_attention import (cross_attention, cross_attention_backward, text_attention, text_attention_backward)

from .conftest import seeded
from .test_gpu_text_attention import BF, F32, FP, heads, inputs, table_of
from .test_gpu_text_attention_backward import grad_of
from .text_attention_reference import Reference, within

pytestmark = pytest.mark.gpu


def step(q, k, v, table, **kw):
    out, lse = text_attention(q, k, v, table, return_lse=True, **kw)
    return out, lse, *text_attention_backward(grad_of(q), q, k, v, out, lse, table, **kw)


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("lq", [1, 100])
def test_inputs_of_any_layout(lq):
    b, h, l, dh = 2, 4, 150, 64
    base = torch.randn(b, l, h, dh, generator=seeded(1)).to(BF).cuda()
    k = base.transpose(1, 2)
    q, table = heads(b, h, lq, dh, 2), table_of(32, h)
    want = step(q, k.contiguous(), k.contiguous(), table, causal=True)
    wide = torch.full((b, l, h, 2 * dh + 8), float("nan"), dtype=BF, device="cuda")
    wide[..., 8:8 + dh] = base
    odd = torch.full((b, l, h, dh + 1), float("nan"), dtype=BF, device="cuda")
    odd[..., 1:] = base
    flat = torch.empty(b * l * h * dh + 3, dtype=BF, device="cuda")[3:].view(b, l, h, dh).copy_(base)
    turned = base.permute(3, 0, 2, 1).contiguous().permute(1, 2, 3, 0)  # channels are the slowest
    for other in (wide[..., 8:8 + dh].transpose(1, 2), odd[..., 1:].transpose(1, 2), flat.transpose(1, 2), turned):
        assert same(step(q, other, other, table, causal=True), want)
    wide_q = torch.zeros(b, h, lq, dh + 4, dtype=BF, device="cuda")
    wide_q[..., :dh] = q
    assert same(step(wide_q[..., :dh], k, k, table, causal=True), want)
    table2 = torch.full((32, 2 * h), float("nan"), dtype=BF, device="cuda")
    table2[:, ::2] = table
    assert same(step(q, k, k, table2[:, ::2], causal=True), want)
    table3 = torch.full((32, h + 3), float("nan"), dtype=BF, device="cuda")
    table3[:, :h] = table
    assert same(step(q, k, k, table3[:, :h], causal=True), want)


def test_one_encoders_states_for_a_whole_batch():
    q, k, v = heads(3, 4, 100, 64, 1), heads(1, 4, 77, 64, 2), heads(1, 4, 77, 64, 3)
    ke, ve = k.expand(3, -1, -1, -1), v.expand(3, -1, -1, -1)
    out, lse = cross_attention(q, ke, ve, return_lse=True)
    assert torch.equal(out, cross_attention(q, ke.contiguous(), ve.contiguous()))
    dq, dk, dv = cross_attention_backward(grad_of(q), q, ke, ve, out, lse)
    ref = Reference(q, ke, ve).backward(grad_of(q))
    for y, (x, e) in zip((dq, dk, dv), ref):  # of each image's view; the sum is the caller's
        within(y, x, e)


def test_destinations():
    q, k, v = inputs(2, 4, 4, 100, 77, 64)
    want = cross_attention(q, k, v)
    wide = torch.full((2, 100, 300), 7.0, dtype=BF, device="cuda")
    out = cross_attention(q, k, v, out=wide[..., 20:276])
    assert out.data_ptr() == wide[..., 20:].data_ptr() and torch.equal(out, want)
    assert bool((wide[..., :20] == 7).all()) and bool((wide[..., 276:] == 7).all())
    rows = torch.full((2, 110, 256), 7.0, dtype=BF, device="cuda")
    cross_attention(q, k, v, out=rows[:, :100])
    assert torch.equal(rows[:, :100], want) and bool((rows[:, 100:] == 7).all())  # rows behind the last stay
    for lq in (1, 100):
        with pytest.raises(ValueError, match="overlaps"):
            cross_attention(q[:, :, :lq], k, v, out=q.transpose(1, 2).view(2, 100, 256)[:, :lq])
    with pytest.raises(ValueError, match="one address"):
        cross_attention(q, k, v, out=wide[:1, :, :256].expand(2, -1, -1))
    for bad in (wide[..., :255], wide.float()[..., :256], wide[..., 1:257], torch.empty(2, 256, 100, dtype=BF, device="cuda").mT):
        with pytest.raises(ValueError, match="out must be"):
            cross_attention(q, k, v, out=bad)


def test_refusals_beside_a_gpu():
    q, k, v = inputs(2, 4, 4, 10, 20, 64)
    for kw, match in ((dict(lengths=torch.ones(3, dtype=torch.int32).cuda()), "lengths"), (dict(lengths=torch.ones(2).cuda()), "lengths"),
                      (dict(mask=torch.ones(2, 20).cuda()), "mask must be bool"), (dict(mask=torch.ones(2, 19, dtype=torch.bool).cuda()), "mask"),
                      (dict(mask=torch.ones(2, 20, dtype=torch.bool)), "runs on the GPU"), (dict(scale=0.0), "scale")):
        with pytest.raises(ValueError, match=match):
            cross_attention(q, k, v, **kw)
    with pytest.raises(ValueError, match="table must be"):
        text_attention(q, k, v, table_of(32, 3))
    for buckets, match in ((0, "no buckets"), (2, "two buckets"), (31, "halve")):
        with pytest.raises(ValueError, match=match):
            text_attention(q, k, v, table_of(buckets, 4))
    with pytest.raises(ValueError, match="q_start"):
        text_attention(q, k, v, q_start=1 << 30)
    with pytest.raises(ValueError, match="q_start"):
        text_attention(q, k, v, q_start=torch.zeros(2).cuda())
    for bad in ((q.float(), k.float(), v.float()), (heads(1, 1, 4, 12, 0),) * 3, (heads(1, 1, 4, 136, 0),) * 3):
        with pytest.raises(_lib.Unsupported):
            cross_attention(*bad)
    out, lse = cross_attention(q, k, v, return_lse=True)
    for grad, o, s in ((out[:1], out, lse), (out.float(), out, lse), (out, out[:, :9], lse), (out, out, lse[:, :3]), (out, out, lse.double())):
        with pytest.raises(ValueError, match="must be"):
            cross_attention_backward(grad, q, k, v, o, s)


def test_empty_sizes():
    for b, h, lq, lk in ((0, 4, 5, 6), (2, 0, 5, 6), (2, 4, 0, 6), (2, 4, 5, 0), (2, 4, 100, 0)):
        q, k, v = inputs(b, h, h, lq, lk, 64)
        table = table_of(32, h)
        out, lse = text_attention(q, k, v, table, return_lse=True)
        assert out.shape == (b, lq, h * 64) and not out.any() and bool((lse == float("-inf")).all())
        got = text_attention_backward(torch.ones_like(out), q, k, v, out, lse, table)
        assert [x.shape for x in got] == [q.shape, k.shape, v.shape, table.shape] and not any(x.any() for x in got)


def test_strides_that_pass_32_bits():
    # Rows 2^23 elements apart: 300 of them span 5 GB. Images 3 GB apart.
    for strides, b, l in (((0, 64, 1 << 23), 1, 300), (((3 << 29) + 64, 64 * 300, 64), 2, 300)):
        h, dh = 2, 64
        size = (b - 1) * strides[0] + (h - 1) * strides[1] + (l - 1) * strides[2] + dh
        k, v = (torch.empty(size, dtype=BF, device="cuda").as_strided((b, h, l, dh), (*strides, 1)) for _ in range(2))
        k.copy_(heads(b, h, l, dh, 1))
        v.copy_(heads(b, h, l, dh, 2))
        for lq in (2, 130):
            q, table = heads(b, h, lq, dh, 3), table_of(32, h)
            assert same(step(q, k, v, table), step(q, k.contiguous(), v.contiguous(), table))
            assert same(step(k, k, v, table), step(k.contiguous(), k.contiguous(), v.contiguous(), table))
        del k, v


def test_other_streams():
    args = [inputs(2, 4, 2, 70, 3000, 64, seed=i) for i in range(4)]
    table = table_of(32, 4)
    want = [step(*a, table) for a in args]
    streams = [torch.cuda.Stream() for _ in args]
    torch.cuda.synchronize()
    got = []
    for a, s in zip(args, streams):  # at once, each with workspaces of its own
        with torch.cuda.stream(s):
            got.append(step(*a, table))
    torch.cuda.synchronize()
    assert all(same(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("lq", [1, 70])
def test_captured_and_replayed(lq):
    # Two graphs, replayed in turn with eager work between, on inputs that change; splits and lengths from memory.
    b, h, hk, lk, dh = 2, 4, 2, 3000, 64
    table, lengths = table_of(32, h), torch.tensor([lk, 1700], dtype=torch.int32).cuda()
    grad = torch.zeros(b, lq, h * dh, dtype=BF, device="cuda")
    sets = [inputs(b, h, hk, lq, lk, dh, seed=i) for i in (0, 10)]
    kw = dict(lengths=lengths, q_start=lengths, bidirectional=False)

    def work(q, k, v):
        out, lse = text_attention(q, k, v, table, return_lse=True, **kw)
        return out, lse, *text_attention_backward(grad, q, k, v, out, lse, table, **kw)

    graphs = []
    for x in sets:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            work(*x)
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = work(*x)
        graphs.append((g, got))
    for turn in range(4):
        grad.copy_(torch.randn(grad.shape, generator=seeded(turn)))
        lengths.copy_(torch.tensor([lk - 100 * turn, 1700 + turn]))
        for i, x in enumerate(sets):
            for j, t in enumerate(x):
                t.copy_(heads(*[t.shape[n] for n in (0, 1, 2, 3)], 100 * turn + 10 * i + j))
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for x, (_, got) in zip(sets, graphs):
            assert same(work(*x), got)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_an_encoders_layer_and_what_reads_its_states(dtype):
    # x -> qkv -> attention with the bias -> projection = the states; image tokens attend to them; the gradients go back
    # through both. Against the same chain in 64 bits, where each stage starts from the values that the kernels handed on.
    b, l, h, dh, li = 2, 77, 4, 64, 150
    d = h * dh
    x = torch.randn(b, l, d, generator=seeded(1)).to(dtype).cuda()
    wq = (torch.randn(3 * d, d, generator=seeded(2)) * d ** -0.5).to(dtype).cuda()
    wo = (torch.randn(d, d, generator=seeded(3)) * d ** -0.5).to(dtype).cuda()
    wkv = (torch.randn(2 * d, d, generator=seeded(4)) * d ** -0.5).to(dtype).cuda()
    table, lengths = table_of(32, h, dtype=dtype), torch.tensor([77, 31], dtype=torch.int32).cuda()
    qkv = raw_linear(x, wq).unflatten(-1, (3, h, dh)).permute(2, 0, 3, 1, 4)
    q, k, v = qkv
    kw = dict(lengths=lengths, scale=1.0)
    out, lse = text_attention(q, k, v, table, return_lse=True, **kw)
    first = Reference(q, k, v, table, **kw)
    within(out, first.out, first.out_bound)
    states = raw_linear(out, wo, residual=x)
    kc, vc = raw_linear(states, wkv).unflatten(-1, (2, h, dh)).permute(2, 0, 3, 1, 4)
    qi = heads(b, h, li, dh, 5, dtype)
    image, lse_i = cross_attention(qi, kc, vc, lengths=lengths, return_lse=True)
    second = Reference(qi, kc, vc, lengths=lengths)
    within(image, second.out, second.out_bound)
    grad = grad_of(qi)
    got = cross_attention_backward(grad, qi, kc, vc, image, lse_i, lengths=lengths)
    for y, want in zip(got, second.backward(grad)):
        within(y, *want)
    dkv = torch.stack(got[1:]).permute(1, 3, 0, 2, 4).reshape(b, l, 2 * d)  # columns of the kv linear's output
    dout = raw_linear(raw_linear(dkv, wkv.t().contiguous()), wo.t().contiguous())
    got = text_attention_backward(dout, q, k, v, out, lse, table, **kw)
    for y, want in zip(got, first.backward(dout)):
        within(y, *want)
    assert not got[1][1, :, 31:].any() and not got[2][1, :, 31:].any()


@pytest.mark.parametrize("lq,group", [(1, 1), (2, 4), (40, 2), (150, 1)])
@pytest.mark.parametrize("dh", [64, 128])
def test_a_cache_whose_later_keys_were_never_written(lq, group, dh):
    # No lengths: the causal mask alone says where the text ends, for each at a place of its own.
    b, hk, lk = 3, 2, 400
    q, k, v = inputs(b, hk * group, hk, lq, lk, dh, seed=lq)
    start = torch.tensor([0, 63, 217], dtype=torch.int32).cuda()
    table = table_of(32, hk * group)
    kw = dict(causal=True, q_start=start, bidirectional=False)
    want = step(q, k, v, table, **kw)
    later = (torch.arange(lk, device="cuda") >= start[:, None] + lq)[:, None, :, None]
    got = step(q, k.masked_fill(later, float("nan")), v.masked_fill(later, float("inf")), table, **kw)
    assert same(got, want) and not any(x.isnan().any() for x in got)
    assert not got[3].masked_select(later).any() and not got[4].masked_select(later).any()
