"""cross_attention and text_attention at the edges of what they take: axes of no and of one element, strides that say
nothing, weight on few of many keys, extreme entries of the bias table."""

from __future__ import annotations

import pytest
import torch

from selas_amd.text_attention import (cross_attention, cross_attention_backward, text_attention, text_attention_backward)

from .conftest import seeded
from .test_gpu_text_attention import BF, F32, FP, inputs, table_of
from .test_gpu_text_attention_backward import grad_of
from .text_attention_reference import Reference, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("dh", [64, 96, 128])
@pytest.mark.parametrize("lk", [1, 77, 3000])
def test_without_queries_the_gradients_are_zeros(dtype, dh, lk):
    q, k, v = inputs(2, 4, 2, 0, lk, dh, dtype=dtype)
    mask = torch.ones(2, lk, dtype=torch.bool).cuda()
    out, lse = cross_attention(q, k, v, return_lse=True)
    assert out.shape == (2, 0, 4 * dh) and lse.shape == (2, 4, 0)
    for kw in (dict(), dict(mask=mask), dict(lengths=torch.tensor([lk, 1]).cuda())):
        stale = [torch.full_like(t, float("nan")) for t in (k, v)]
        del stale  # what the allocator hands out next holds no zeros
        dq, dk, dv = cross_attention_backward(out, q, k, v, out, lse, **kw)
        assert (dq.shape, dk.shape, dv.shape) == (q.shape, k.shape, v.shape) and not dk.any() and not dv.any()
    for t in (dtype, F32):
        table = table_of(32, 4, dtype=t)
        out, lse = text_attention(q, k, v, table, causal=True, return_lse=True)
        dq, dk, dv, dtable = text_attention_backward(out, q, k, v, out, lse, table, causal=True)
        assert not dk.any() and not dv.any() and dtable.shape == table.shape and dtable.dtype == t and not dtable.any()


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("dh", [64, 72, 128])
@pytest.mark.parametrize("lk", [1, 40, 200, 2000])  # up to 2000: one range of keys, and several
@pytest.mark.parametrize("stride", [0, 8, 4096])
def test_the_row_stride_of_one_row_says_nothing(dtype, dh, lk, stride):
    # 16 query heads of one key head: the kernel of 32 rows, of which one exists.
    q, k, v = inputs(2, 16, 1, 1, lk, dh, seed=lk, dtype=dtype)
    want = cross_attention(q, k, v)
    n = 16 * dh
    for b in (1, 2):
        given = torch.full((2 * n + 8,), 7.0, dtype=dtype, device="cuda")
        out = given[4:].as_strided((b, 1, n), (n, stride, 1))
        assert torch.equal(cross_attention(q[:b], k[:b], v[:b], out=out), want[:b])
        assert bool((given[:4] == 7).all()) and bool((given[4 + b * n:] == 7).all())


@pytest.mark.parametrize("lq", [1, 3])
def test_strides_of_axes_of_one_element_are_not_looked_at(lq):
    q, k, v = inputs(1, 16, 1, lq, 100, 64, seed=lq)
    want, n = cross_attention(q, k, v), 16 * 64
    for sb, sl in ((0, n), (3, n), (1 << 40, n), (n, n if lq > 1 else 1), (n, n if lq > 1 else 1 << 30)):
        out = torch.empty(lq * n, dtype=BF, device="cuda").as_strided((1, lq, n), (sb, sl, 1))
        assert torch.equal(cross_attention(q, k, v, out=out), want)
        assert out.stride() == (sb, sl, 1)
    with pytest.raises(ValueError, match="out must be"):
        cross_attention(q.expand(2, -1, -1, -1), k.expand(2, -1, -1, -1), v.expand(2, -1, -1, -1),
                        out=torch.empty(2 * lq * n + 3, dtype=BF, device="cuda").as_strided((2, lq, n), (lq * n + 3, n, 1)))


@pytest.mark.parametrize("dtype", [BF, FP])
def test_gradients_of_one_query_and_one_key_at_any_stride(dtype):
    q, k, v = inputs(2, 16, 2, 1, 1, 64, dtype=dtype)
    q2, k2, v2 = inputs(2, 16, 2, 1, 90, 64, dtype=dtype)
    grad = torch.ones(2, 1, 1024, dtype=dtype, device="cuda")

    def folded(t, stride):  # the same elements, the row stride of the one row replaced
        t = t.contiguous()
        return t.as_strided(t.shape, (*t.stride()[:-2], stride, 1))

    for args in ((q, k, v), (q2, k2, v2)):
        out, lse = cross_attention(*args, return_lse=True)
        want = (out, lse, *cross_attention_backward(grad, *args, out, lse))
        for stride in (0, 8, 1 << 30):
            x = [folded(t, stride) if t.shape[2] == 1 else t for t in args]
            out, lse = cross_attention(*x, return_lse=True)
            got = (out, lse, *cross_attention_backward(folded(grad, stride), *x, folded(out, stride), lse))
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def roundings(q, k, v, *args, **kw):
    """Holds the gradients to what rounding dS and each result once costs these very inputs, in the 2-norm against 64 bits.

    Beyond that D may be off where it does not pay to mend it, by three quarters of half a step of what |dS| sums to in the row
    (`left`, spread evenly below it and over rows: 1 / sqrt(3) of it in the mean square): dS of key j is then off by p times
    that. A tenth is left for chance. p is rounded for dv, and the table's gradient is not made of rounded dS."""
    grad = grad_of(q)
    out, lse = text_attention(q, k, v, *args, return_lse=True, **kw)

    def run():
        return text_attention_backward(grad, q, k, v, out, lse, *args, **kw)

    got = run()
    assert all(torch.equal(x, y) for x, y in zip(got, run()) if x is not None)
    ref = Reference(q, k, v, *args, **kw)
    want, half, hk = ref.backward(grad), torch.finfo(q.dtype).eps / 2, k.shape[1]

    def rounded(x, like):
        return x.to(like.dtype).double()

    def shared(x):
        return x.unflatten(1, (hk, -1)).sum(2)

    g = grad.cpu().double().view(*out.shape[:2], q.shape[1], -1).transpose(1, 2)
    dp = g @ ref.v.mT
    ds = ref.p * (dp - (g * ref.o).sum(-1, keepdim=True))
    left = 0.75 / 3 ** 0.5 * half * ds.abs().sum(-1, keepdim=True)
    twice = [rounded(ref.scale * rounded(ds, q) @ ref.k, q), rounded(shared(ref.scale * rounded(ds, q).mT @ ref.q), q),
             rounded(shared(rounded(ref.p, q).mT @ g), q)]
    share = [ref.scale * left * (ref.p @ ref.k), shared((ref.scale * left * ref.p).mT.square() @ ref.q.square()).sqrt(), 0.0]
    if want[3] is not None:
        hot = torch.nn.functional.one_hot(ref.bucket, want[3][0].shape[0]).double()  # [b, lq, lk, buckets]
        twice.append(rounded(want[3][0], got[3]))
        share.append(torch.einsum("bhij,bijr->bhir", left * ref.p, hot).square().sum((0, 2)).sqrt().t())
    for name, y, (x, _), two, rest in zip(("dq", "dk", "dv", "dtable"), got, want, twice, share):
        error, least = (y.cpu().double() - x).norm(), (two - x).norm()
        rest = rest.norm() if torch.is_tensor(rest) else 0.0
        unit = half * x.norm()
        print(f"{name}: off by {error / unit:.3f}, rounded {least / unit:.3f}, of D {rest / unit:.3f}", flush=True)
        assert error <= 1.1 * (least ** 2 + rest ** 2) ** 0.5, name


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("l", [256, 257, 300, 600])
@pytest.mark.parametrize("raised", [6.0, 10.0])
@pytest.mark.parametrize("both,causal", [(False, True), (True, False)])
def test_weight_on_few_of_many_keys(l, raised, both, causal, dtype):
    # The learned bias draws the weight to the nearest keys; with 10, 0.9 and more of it to a row's own.
    q, k, v = inputs(2, 4, 2, l, l, 64, seed=l, dtype=dtype)
    table = table_of(32, 4, dtype=dtype)
    table[0] = raised
    roundings(q, k, v, table, causal=causal, bidirectional=both)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("dh", [40, 72, 128])
@pytest.mark.parametrize("h,lq,lk", [(8, 300, 600), (1, 40, 3000), (2, 2049, 700)])  # the second with its keys split
def test_scores_far_apart_and_values_of_one_mean(h, lq, lk, dh, dtype):
    q, k, v = inputs(1, h, h, lq, lk, dh, seed=dh, dtype=dtype)
    roundings(q * 3, k, v)
    mean = torch.randn(dh, generator=seeded(9)).to(dtype).cuda()
    for size in (1, 5):
        roundings(q, k, v + size * mean)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("h,l", [(8, 300), (1, 3000)])
def test_few_seen_keys_of_many(h, l, dtype):
    # Rows see 3 keys, which are all over the tiles.
    q, k, v = inputs(2, h, h, 130, l, 64, seed=l, dtype=dtype)
    mask = torch.zeros(2, l, dtype=torch.bool)
    mask[:, [0, l // 2, l - 1]] = True
    roundings(q, k, v, mask=mask.cuda())


@pytest.mark.parametrize("lq,lk", [(40, 3000), (300, 700)])  # keys split, and not
def test_a_captured_backward_pass_follows_its_inputs(lq, lk):
    # Values of one mean, whose rows begin again, and values of none, whose rows do not, replayed in turn.
    q, k, v = inputs(1, 2, 1, lq, lk, 64, seed=lq)
    plain, grad, mean = v.clone(), grad_of(q), torch.randn(64, generator=seeded(9)).to(BF).cuda()

    def work():
        out, lse = cross_attention(q, k, v, return_lse=True)
        return out, lse, *cross_attention_backward(grad, q, k, v, out, lse)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    for turn in range(5):
        v.copy_(plain + 5 * mean if turn % 2 else plain)
        want = work()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def checked(q, k, v, table, ref_table, ref_kw=None, **kw):
    """Forward and gradients of a call with `table` against the definition with `ref_table`."""
    grad = grad_of(q)
    out, lse = text_attention(q, k, v, table, return_lse=True, **kw)
    ref = Reference(q, k, v, ref_table, **kw, **(ref_kw or {}))
    within(out, ref.out, ref.out_bound)
    within(lse, ref.lse, ref.lse_bound)
    for name, y, want in zip(("dq", "dk", "dv", "dtable"), text_attention_backward(grad, q, k, v, out, lse, table, **kw),
                             ref.backward(grad)):
        print(name, flush=True)
        within(y, *want)
    return out, lse


LIMIT = 2.0 ** 17


@pytest.mark.parametrize("dtype,ttype,low", [(BF, F32, -torch.finfo(F32).max), (BF, BF, -torch.finfo(BF).max), (FP, F32, -1e9),
                                             (FP, FP, -torch.finfo(FP).max), (FP, F32, -torch.finfo(F32).max), (BF, F32, -1e30)])
@pytest.mark.parametrize("lq,scale", [(1, None), (2, 1.0), (40, None), (130, 1e-3)])
def test_lowest_entries_of_the_table(lq, scale, dtype, ttype, low):
    # Keys after the query have the lowest entry: no weight beside any other key, and weights by their products among
    # themselves, where the first row sees no other. Entries count as 2^17 beyond that.
    q, k, v = inputs(2, 8, 4, lq, 150, 64, seed=lq, dtype=dtype)
    table = table_of(32, 8, dtype=ttype)
    table[16:] = low
    mask = torch.ones(2, 150, dtype=torch.bool)
    mask[0, 0] = False
    checked(q, k, v, table, table.clamp(-LIMIT, LIMIT), mask=mask.cuda(), scale=scale)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lq", [1, 40, 130])
def test_largest_entries_of_the_table(lq, dtype):
    q, k, v = inputs(2, 8, 4, lq, 150, 64, seed=lq, dtype=dtype)
    table = table_of(32, 8, dtype=F32)
    table[0] = torch.finfo(F32).max
    out, _ = checked(q, k, v, table, table.clamp(-LIMIT, LIMIT))
    # Each row's own key alone. Its weight is 2^r, r what the maximum of the scores was rounded by; that is rounded to the type
    # for the product and not for the sum, and the result again: two halves of a step, the second of a value larger by the first.
    own, half = v[:, :, :lq].repeat_interleave(2, 1).double().cpu(), torch.finfo(dtype).eps / 2
    within(out.view(2, lq, 8, 64).transpose(1, 2), own, own.abs() * (2 * half + 2 * half ** 2))


@pytest.mark.parametrize("dtype,ttype", [(BF, F32), (BF, BF), (FP, FP)])
@pytest.mark.parametrize("lq", [1, 40, 130])
def test_entries_of_minus_infinity_hide_their_keys(lq, dtype, ttype):
    q, k, v = inputs(2, 8, 4, lq, 150, 64, seed=lq, dtype=dtype)
    table = table_of(32, 8, dtype=ttype)
    table[16:] = 0.0
    hiding = table.clone()
    hiding[16:] = -torch.inf
    mask = torch.ones(2, 150, dtype=torch.bool)
    mask[0, 0] = False
    out, lse = checked(q, k, v, hiding, table, ref_kw=dict(causal=True), mask=mask.cuda())
    assert not out[0, 0].any() and bool((lse[0, :, 0] == -torch.inf).all())  # a row that sees no key


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("dh,bias", [(64, True), (72, False), (128, True)])
@pytest.mark.parametrize("l", [1, 70, 300, 2000])
def test_what_queries_that_see_no_key_hold_does_not_matter(l, dh, bias, dtype):
    # Texts padded at their front under a causal mask: the padding is hidden as keys, by the mask or by negative positions,
    # and its queries see nothing.
    q, k, v = inputs(3, 4, 2, l, l, dh, seed=l, dtype=dtype)
    table, grad = table_of(32, 4) if bias else None, grad_of(q)
    pads = torch.tensor([0, l // 3, l]).cuda()
    dead = torch.arange(l, device="cuda") < pads[:, None]
    shifted = -pads.to(torch.int32)
    for kw in (dict(mask=~dead), dict(q_start=shifted), dict(mask=~dead, q_start=shifted // 2)):
        at = dead if "mask" in kw else torch.arange(l, device="cuda") < pads[:, None]
        out, lse = text_attention(q, k, v, table, causal=True, return_lse=True, **kw)
        assert not out[at].any() and bool((lse.transpose(1, 2)[at] == -torch.inf).all())
        want = text_attention_backward(grad, q, k, v, out, lse, table, causal=True, **kw)
        assert not want[0].transpose(1, 2)[at].any()
        q2, grad2 = q.masked_fill(at[:, None, :, None], float("nan")), grad.masked_fill(at[:, :, None], float("nan"))
        grad3 = grad.masked_fill(at[:, :, None], float("inf"))
        out, lse = text_attention(q2, k, v, table, causal=True, return_lse=True, **kw)
        assert not out[at].any()
        for g in (grad2, grad3):
            got = text_attention_backward(g, q2, k, v, out, lse, table, causal=True, **kw)
            assert all(torch.equal(x, y) for x, y in zip(got, want) if x is not None)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("both,distance", [(True, 200), (False, 33), (False, 128)])
@pytest.mark.parametrize("lq,lk,start", [(129, 128, -43), (31, 200, 170), (333, 128, 99), (300, 300, 0)])
def test_a_buckets_gradient_holds_no_rounding_of_anothers(lq, lk, start, both, distance, dtype):
    # The entries are far apart: some buckets' sums are 1e-8 of their neighbours', element by element within their own bounds
    # (but for weights below fp32's normal numbers).
    q, k, v = inputs(2, 48, 3, lq, lk, 64, seed=lq, dtype=dtype)
    table, kw = table_of(32, 48, dtype=F32, std=4.0), dict(bidirectional=both, max_distance=distance, causal=not both, q_start=start)
    out, lse = text_attention(q, k, v, table, return_lse=True, **kw)
    grad = grad_of(q)
    dtable = text_attention_backward(grad, q, k, v, out, lse, table, **kw)[3]
    want, bound = Reference(q, k, v, table, **kw).backward(grad)[3]
    within(dtable, want, bound + 2.0 ** -100)
