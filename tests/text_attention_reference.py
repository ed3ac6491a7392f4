"""Attention with shared key heads, masks and a bias by buckets in 64 bits on the CPU, its gradients, and how far a kernel
may be from them.

The bounds count roundings, element by element. With h half a step of the type (eps / 2) and u = 2^-24:
  scores   a dot product of Dh terms, the scaling and the bias: (Dh + 4) u sum|q k| scale + 4 u |bias|; the exponent's
           subtractions and the base-2 exponential: 8 u (1 + |score| + |largest score|). Their sum is `ds`.
  weights  relative 2 ds' (numerator and sum, ds' the row's largest) + (Lk + 8) u for the sum; rounded once: h.
  out      sum p |v| (h + that) + h |out|; fp16 weights below its normal numbers: 2^-32 of a row's largest each.
  lse      ds' + (Lk + 8) u + 2 u |lse|.
  D        sum |dO| err(out) + (Dh + 2) u sum |dO out|;  dP: (Dh + 2) u sum |dO v|.
  dS       p (err(dP) + err(D)) + err(p) |dP - D| + 4 u |dS|, then rounded: h; fp16: scaled so that 2^-40 max|dO| max|v|
           bounds what falls below its normal numbers.
  sums of n terms add n u of the sum of their magnitudes, and each result is rounded once. The table's sums run over trees
  and rows of at most 4 sqrt(n) additions in a chain: 4 sqrt(n) u."""

from __future__ import annotations

import torch

U = 2.0 ** -24


def side_of(n: int, max_distance: int) -> list[int]:
    """The bucket of each distance 0 .. max_distance, by whole numbers."""
    e, found, t = n // 2, [], 0
    for d in range(max_distance + 1):
        while t + 1 < n and (d >= t + 1 if t + 1 <= e else
                             d ** (n - e) * e ** (t + 1 - e) >= e ** (n - e) * max_distance ** (t + 1 - e)):
            t += 1
        found.append(t)
    return found


def bucket_map(rel: torch.Tensor, buckets: int, max_distance: int, bidirectional: bool) -> torch.Tensor:
    n = buckets // 2 if bidirectional else buckets
    side = torch.tensor(side_of(n, max_distance))
    a = rel.abs() if bidirectional else (-rel).clamp(min=0)
    r = side[a.clamp(max=max_distance)]
    return r + n * (rel > 0) if bidirectional else r


class Reference:
    """Forward pass of one call; `backward` its gradients. Every value has its bound beside it."""

    def __init__(self, q, k, v, table=None, max_distance=128, bidirectional=True, causal=False, q_start=0, lengths=None,
                 mask=None, scale=None, positions=True):
        self.dtype, self.table = q.dtype, table
        self.h = torch.finfo(q.dtype).eps / 2
        q, k, v = (t.detach().cpu().double() for t in (q, k, v))
        (b, h, lq, dh), (hk, lk) = q.shape, k.shape[1:3]
        self.scale = dh ** -0.5 if scale is None else scale
        seen = torch.ones(b, 1, lq, lk, dtype=torch.bool)
        if lengths is not None:
            seen &= (torch.arange(lk) < lengths.cpu().long()[:, None])[:, None, None]
        if mask is not None:
            seen &= mask.cpu()[:, None, None]
        start = q_start.cpu().long() if isinstance(q_start, torch.Tensor) else torch.full((b,), q_start)
        rel = torch.arange(lk) - (start[:, None] + torch.arange(lq))[:, :, None]
        if causal:
            seen = seen & (rel <= 0)[:, None]
        # What is not seen may be NaN: out of every product.
        key_seen = seen.any(2).any(1) if lq else torch.zeros(b, lk, dtype=torch.bool)
        k, v = (torch.where(key_seen[:, None, :, None], t, 0.0) for t in (k, v))
        group = h // hk if hk else 0
        self.q, self.k, self.v, self.group = q, k.repeat_interleave(group, 1), v.repeat_interleave(group, 1), group
        s = self.q @ self.k.mT * self.scale
        err = (dh + 4) * U * self.scale * (self.q.abs() @ self.k.abs().mT)
        self.bucket = None
        if table is not None:
            self.bucket = bucket_map(rel, table.shape[0], max_distance, bidirectional)
            bias = table.detach().cpu().double()[self.bucket].permute(0, 3, 1, 2)
            s, err = s + bias, err + 4 * U * bias.abs()
        self.seen = seen
        top = torch.where(seen, s, -1e300).amax(-1, keepdim=True) if lk else torch.zeros(b, h, lq, 1).double()
        none = ~seen.any(-1, keepdim=True)
        top = torch.where(none, 0.0, top)
        e = torch.where(seen, torch.exp(torch.where(seen, s - top, 0.0)), 0.0)
        total = e.sum(-1, keepdim=True)
        self.p = e / torch.where(none, 1.0, total)
        err = torch.where(seen, err + 8 * U * (1 + s.abs() + top.abs()), 0.0)
        worst = err.amax(-1, keepdim=True) if lk else torch.zeros_like(top)
        self.perr = 2 * worst + (lk + 8) * U  # relative, of the probabilities
        self.lse = torch.where(none, -torch.inf, top + torch.log(torch.where(none, 1.0, total)))[..., 0]
        self.lse_bound = (worst + (lk + 8) * U)[..., 0] + 2 * U * torch.where(none[..., 0], 0.0, self.lse.abs())
        o = self.p @ self.v
        tiny = lk * 2.0 ** -32 * (self.v.abs().amax() if self.v.numel() else 0.0) if self.dtype == torch.float16 else 0.0
        self.oerr = (self.p * (self.h + self.perr)) @ self.v.abs() + tiny
        self.oerr = self.oerr + self.h * (o.abs() + self.oerr) + torch.finfo(self.dtype).smallest_normal * 2 * self.h
        self.o = o
        self.out, self.out_bound = (t.transpose(1, 2).reshape(b, lq, h * dh) for t in (o, self.oerr))

    def backward(self, grad):
        """[(gradient, bound)] of q, k, v and the table (None without one)."""
        b, h, lq, dh = self.q.shape
        hk, lk, fp16 = h // max(self.group, 1), self.k.shape[2], self.dtype == torch.float16
        step, tiny = self.h, torch.finfo(self.dtype).smallest_normal * 2 * self.h
        g = grad.detach().cpu().double().view(b, lq, h, dh).transpose(1, 2)
        dp = g @ self.v.mT
        dot = (g * self.o).sum(-1, keepdim=True)
        dot_err = (g.abs() * self.oerr).sum(-1, keepdim=True) + (dh + 2) * U * (g * self.o).abs().sum(-1, keepdim=True)
        dp_err = (dh + 2) * U * (g.abs() @ self.v.abs().mT)
        ds = self.p * (dp - dot)
        ds_err = self.p * (dp_err + dot_err + (self.perr + 4 * U) * (dp - dot).abs())
        # What fp16 drops below its normal numbers, per element (the norms' product bounds |dP|).
        low = 0.0
        if fp16 and self.v.numel() and g.numel():
            low = torch.where(self.seen, 2.0 ** -37 * g.norm(dim=-1).amax() * self.v.norm(dim=-1).amax(), 0.0)
        s_err = ds_err + step * (ds.abs() + ds_err) + low
        p_err = self.p * (self.perr + step) + torch.where(self.seen, 2.0 ** -39 if fp16 else 0.0, 0.0)
        u_q, u_k = (lk + 8) * U, (lq * max(self.group, 1) + 8) * U

        def rounded(x, e):
            return x, e + step * (x.abs() + e) + tiny

        def heads(t):
            return t.view(b, hk, self.group, lk, dh).sum(2) if h else t.view(b, hk, lk, dh)

        dq = rounded(self.scale * ds @ self.k, self.scale * (s_err + u_q * ds.abs()) @ self.k.abs())
        dk = rounded(heads(self.scale * ds.mT @ self.q), heads(self.scale * (s_err + u_k * ds.abs()).mT @ self.q.abs()))
        dv = rounded(heads(self.p.mT @ g), heads((p_err + u_k * self.p).mT @ g.abs()))
        if self.table is None:
            return [dq, dk, dv, None]
        hot = torch.nn.functional.one_hot(self.bucket.expand(b, lq, lk).reshape(-1), self.table.shape[0]).double()
        flat = [x.transpose(0, 1).reshape(h, -1) @ hot for x in (ds, ds_err + (lq * lk + 64) ** 0.5 * 4 * U * ds.abs())]
        half = torch.finfo(self.table.dtype).eps / 2
        x, e = flat[0].t(), flat[1].t()
        return [dq, dk, dv, (x, e + half * (x.abs() + e) + torch.finfo(self.table.dtype).smallest_normal * 2 * half)]


def within(y: torch.Tensor, ref: torch.Tensor, bound: torch.Tensor) -> None:
    y = y.detach().cpu().double()
    assert y.shape == ref.shape
    same = (y == ref) | (y.isnan() & ref.isnan())
    d = torch.where(same, 0.0, (y - ref).abs() / bound.clamp(min=1e-300))
    assert bool((d <= 1).all()), f"worst {d.max().item():.3g} of the bound, {int((d > 1).sum())} of {d.numel()} past it"
