"""The attention of the text side, as cases that a timing program can prepare, run and check.

A case is a dict of plain values with an "op":

  cross  out = softmax(scale q k^T) v where the keys are an encoder's states, of another length than the queries, with
         shared key heads and images whose states end early or are masked: selas_amd.text_attention.cross_attention.
  text   the attention of a text encoder or decoder: a learned bias for each head by buckets of the distance between key
         and query, and a causal mask, each optional: selas_amd.text_attention.text_attention.

With "train" a case is a training step: the output and the gradients of q, k, v and the bias table, through
cross_attention_backward and text_attention_backward. Without it, it is the forward pass alone.

The plain forms below are elementary torch operations in 32 bits (64 for the buckets' borders), rounded once.
"""

from __future__ import annotations

import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
MAX_FLOPS = 4 * 24 * 20280 * 512 * 128  # the largest listed forward pass
MAX_SCORES = 24 * 20280 * 512  # scores that a plain form holds at once


# ---------------------------------------------------------------------------------------------- the cases


def _cross(name, b, heads, kv_heads, lq, lk, dh, keys="all", dtype="bf16", train=False):
    return dict(name=name, op="cross", train=train, b=b, heads=heads, kv_heads=kv_heads, lq=lq, lk=lk, dh=dh, keys=keys,
                dtype=dtype)


def _text(name, b, heads, lq, lk, dh, buckets=32, distance=128, both=True, causal=False, kv_heads=None, keys="all",
          dtype="bf16", train=False):
    """buckets 0: no bias. both: keys on either side of the query have buckets of their own. The queries are the last lq of
    each text's positions."""
    return dict(name=name, op="text", train=train, b=b, heads=heads, kv_heads=kv_heads or heads, lq=lq, lk=lk, dh=dh,
                buckets=buckets, distance=distance, both=both, causal=causal, keys=keys, dtype=dtype)


def listed():
    return [
        # One pooled query over a prompt's 512 states. The smallest call: latency.
        _cross("cross_one_query", 1, 24, 24, 1, 512, 128),
        # An image of 1024 x 1024 (4096 tokens) over the states of its prompt, two prompts of different lengths.
        _cross("cross_image_1024_batch2", 2, 24, 24, 4096, 512, 128, keys="lengths"),
        # 64 learned queries that sum up a clip's 20,280 tokens, with shared key heads: few rows, a long axis.
        _cross("cross_64_queries_clip", 1, 16, 4, 64, 20280, 96, dtype="fp16"),
        # A clip of 13 latent frames of 30 x 52 tokens over 512 states: the largest forward pass.
        _cross("cross_clip_20280", 1, 24, 24, 20280, 512, 128),
        # Training a cross attention at 1024 x 1024, with the mask of the tokenizer.
        _cross("cross_train_1024", 1, 24, 24, 4096, 512, 128, keys="mask", train=True),
        # Sizes that fill no tile, shared key heads and fp16, short texts: a model of another width.
        _cross("cross_train_odd_fp16", 3, 16, 4, 1031, 77, 72, keys="lengths", dtype="fp16", train=True),
        # The text encoder's layer for one prompt of 512 tokens.
        _text("encoder_512", 1, 64, 512, 512, 64),
        # The same for a batch of 16 prompts of different lengths.
        _text("encoder_512_batch16", 16, 64, 512, 512, 64, keys="lengths"),
        # The other text encoder: 77 tokens, causal, no bias.
        _text("causal_77_fp16_batch4", 4, 12, 77, 77, 64, buckets=0, causal=True, dtype="fp16"),
        # One more token of 16 texts that a decoder writes, over caches of up to 2048 keys.
        _text("decode_2048_batch16", 16, 32, 1, 2048, 64, both=False, causal=True, keys="lengths"),
        # Training the encoder's layer: q, k, v and the table.
        _text("encoder_train_512_batch4", 4, 64, 512, 512, 64, train=True),
        # Training a causal decoder's layer on an odd length, shared key heads, fp16, buckets of other sizes.
        _text("decoder_train_odd_fp16", 2, 16, 1491, 1491, 80, buckets=24, distance=200, both=False, causal=True, kv_heads=8,
              dtype="fp16", train=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    cross, train = rng.random() < 0.5, rng.random() < 0.4
    case = dict(op="cross" if cross else "text", train=train)
    dtype, dh = rng.choice(("bf16", "bf16", "fp16")), rng.choice((40, 64, 64, 72, 80, 96, 128, 128))
    keys = rng.choice(("all", "lengths", "mask"))
    while True:
        kv_heads = rng.choice((1, 2, 4, 8, 12, 16, 24, 32, 64))
        heads = kv_heads * rng.choice((1, 1, 1, 2, 4))
        b = rng.choice((1, 1, 2, 3, 4, 8, 16))
        if cross:
            lq = rng.randint(1, 64) if rng.random() < 0.25 else _log_int(rng, 65, 20280)
            lk = _log_int(rng, 1, 20280) if rng.random() < 0.3 else _log_int(rng, 1, 1024)
        else:
            lk = _log_int(rng, 1, 4096)
            lq = rng.randint(1, min(8, lk)) if not train and rng.random() < 0.3 else lk
        flops = (14 if train else 4) * b * heads * lq * lk * dh
        moved = b * dh * 2 * (2 * heads * lq + 2 * kv_heads * lk)
        if heads <= 64 and flops <= MAX_FLOPS and b * heads * lq * lk <= MAX_SCORES and moved <= 1 << 29:
            break
    case |= dict(b=b, heads=heads, kv_heads=kv_heads, lq=lq, lk=lk, dh=dh, keys=keys, dtype=dtype)
    if not cross:
        both = rng.random() < 0.5
        buckets = rng.choice((0, 32, 32, 2 * rng.randint(2, 32)))
        case |= dict(buckets=buckets, distance=rng.choice((128, 128, rng.randint(33, 512))), both=both,
                     causal=not both or rng.random() < 0.3)
    return case


# ---------------------------------------------------------------------------------------------- inputs


def _lengths(case):
    """The keys that each image or text has: from all of them down to a share of 1 / (b + 1)."""
    b, lk = case["b"], case["lk"]
    return [lk - lk * i // (b + 1) if case["keys"] == "lengths" else lk for i in range(b)]


def prepare(case, seed):
    g, dt = torch.Generator(device="cuda").manual_seed(seed), DT[case["dtype"]]
    b, h, hk, lq, lk, dh = (case[n] for n in ("b", "heads", "kv_heads", "lq", "lk", "dh"))

    def normal(*shape, std=1.0, dtype=dt):
        return torch.empty(shape, device="cuda").normal_(0.0, std, generator=g).to(dtype)

    # q, k and v are columns of linears' outputs, [b, tokens, heads, dh], seen as [b, heads, tokens, dh].
    q_std = 1.0 if case["op"] == "cross" else dh ** -0.5  # a text encoder's scale is in its weights
    if case["op"] == "text" and lq == lk:
        qkv = normal(b, lk, h + 2 * hk, dh).transpose(1, 2)
        q, k, v = qkv.split((h, hk, hk), dim=1)
        q.mul_(q_std)
    else:
        q = normal(b, lq, h, dh, std=q_std).transpose(1, 2)
        k, v = normal(b, lk, 2, hk, dh).permute(2, 0, 3, 1, 4)
    lengths = _lengths(case)
    state = dict(case=case, q=q, k=k, v=v, scale=dh ** -0.5 if case["op"] == "cross" else 1.0,
                 grad=normal(b, lq, h * dh) if case["train"] else None, table=None, mask=None, lengths=None, start=0)
    if case["keys"] == "lengths":
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    if case["keys"] == "mask":
        state["mask"] = torch.rand(b, lk, device="cuda", generator=g) < 0.85
    if case["op"] == "text":
        if case["buckets"]:
            state["table"] = normal(case["buckets"], h)
        if lq < lk:  # the position of the first query, for each text
            state["start"] = torch.tensor([max(n - lq, 0) for n in lengths], dtype=torch.int32, device="cuda")
    return state


# ---------------------------------------------------------------------------------------------- one pass


def run(state):
    return (_own if own else _plain)(state)


def _own(s):
    from selas_amd import text_attention as ta

    case = s["case"]
    q, k, v, keys = s["q"], s["k"], s["v"], dict(lengths=s["lengths"], mask=s["mask"], scale=s["scale"])
    if case["op"] == "text":
        keys |= dict(table=s["table"], max_distance=case["distance"], bidirectional=case["both"], causal=case["causal"],
                     q_start=s["start"])
    forward = ta.cross_attention if case["op"] == "cross" else ta.text_attention
    if not case["train"]:
        return forward(q, k, v, **keys)
    out, lse = forward(q, k, v, return_lse=True, **keys)
    backward = ta.cross_attention_backward if case["op"] == "cross" else ta.text_attention_backward
    return (out, *backward(s["grad"], q, k, v, out, lse, **keys))


def _offsets(s):
    """Key position minus query position, [b or 1, lq, lk]."""
    case = s["case"]
    start = s["start"] if torch.is_tensor(s["start"]) else torch.tensor([s["start"]], device="cuda")
    at = start[:, None].long() + torch.arange(case["lq"], device="cuda")
    return torch.arange(case["lk"], device="cuda")[None, None, :] - at[:, :, None]


def _buckets(case, rel):
    """The first half of a side's buckets are distances of their own, the rest grows by a constant factor up to `distance`."""
    n, first, side = case["buckets"], 0, -rel.clamp(max=0)
    if case["both"]:
        n, first, side = n // 2, (rel > 0).long() * (n // 2), rel.abs()
    e = n // 2
    far = torch.log(side.clamp(min=1).double() / e) / math.log(case["distance"] / e) * (n - e)
    far = e + torch.floor(far + 1e-9).long()  # a distance on a border belongs to the bucket that begins there
    return first + torch.where(side < e, side, far.clamp(max=n - 1))


def _plain(s):
    case = s["case"]
    b, h, hk, lq, lk, dh = (case[n] for n in ("b", "heads", "kv_heads", "lq", "lk", "dh"))
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if h > hk:
        k, v = (t.repeat_interleave(h // hk, 1) for t in (k, v))
    scores = q @ k.mT.contiguous() * s["scale"]
    seen = torch.ones(1, 1, 1, 1, dtype=torch.bool, device="cuda")
    if s["lengths"] is not None:
        seen = seen & (torch.arange(lk, device="cuda") < s["lengths"][:, None])[:, None, None]
    if s["mask"] is not None:
        seen = seen & s["mask"][:, None, None]
    bucket = None
    if case["op"] == "text":
        rel = _offsets(s)
        if case["buckets"]:
            bucket = _buckets(case, rel)
            scores += s["table"].float()[bucket].permute(0, 3, 1, 2)
        if case["causal"]:
            seen = seen & (rel <= 0)[:, None]
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total == 0, 1.0, total)  # a row that sees nothing: zeros
    del scores
    out = (p @ v).transpose(1, 2).reshape(b, lq, h * dh).to(s["q"].dtype)
    if not case["train"]:
        return out
    grad = s["grad"].float().view(b, lq, h, dh).transpose(1, 2).contiguous()
    dv = p.mT.contiguous() @ grad
    ds = grad @ v.mT.contiguous()
    ds -= (p * ds).sum(-1, keepdim=True)
    ds *= p
    dq = ds @ k * s["scale"]
    dk = ds.mT.contiguous() @ q * s["scale"]
    if h > hk:
        dk, dv = (t.view(b, hk, h // hk, lk, dh).sum(2) for t in (dk, dv))
    grads = [t.to(s["q"].dtype) for t in (dq, dk, dv)]
    if case["op"] == "text":
        grads.append(_plain_table(case, ds, bucket) if case["buckets"] else None)
    return (out, *grads)


def _plain_table(case, ds, bucket):
    """The sums of ds over each bucket: a product with the buckets as columns of ones and zeros."""
    hot = (bucket.view(-1, 1) == torch.arange(case["buckets"], device="cuda")).float()
    return (ds.sum(0).flatten(1) @ hot).t().to(DT[case["dtype"]])


# ---------------------------------------------------------------------------------------------- the definition in 64 bits


def _side_of(n, e, distance):
    """bucket of every distance up to `distance`, by whole numbers: bucket t begins where (d / e)^(n - e) >= (distance / e)^(t - e)."""
    found, t = [], 0
    for d in range(distance + 1):
        while t + 1 < n and (d >= t + 1 if t + 1 <= e else
                             d ** (n - e) * e ** (t + 1 - e) >= e ** (n - e) * distance ** (t + 1 - e)):
            t += 1
        found.append(t)
    return torch.tensor(found, device="cuda")


def exact(case, seed):
    """Image by image and head by head in 64 bits; the gradients by automatic differentiation of the definition."""
    s = prepare(case, seed)
    b, h, hk, lq, lk = (case[n] for n in ("b", "heads", "kv_heads", "lq", "lk"))
    if b * h * max(lq * lk, 1 << 16) * (4 if case["train"] else 1) > 1 << 31:
        return None
    rows, cols = torch.arange(lq, device="cuda"), torch.arange(lk, device="cuda")
    leaf = {n: s[n].detach().double().requires_grad_(case["train"]) for n in ("q", "k", "v")}
    table = None if s["table"] is None else s["table"].double().requires_grad_(case["train"])
    n = (case["buckets"] // 2 if case["both"] else case["buckets"]) if table is not None else 0
    side = _side_of(n, n // 2, case["distance"]) if n else None
    outs = []
    for i in range(b):
        hidden = torch.zeros(lq, lk, dtype=torch.bool, device="cuda")
        if s["lengths"] is not None:
            hidden |= cols >= s["lengths"][i]
        if s["mask"] is not None:
            hidden |= ~s["mask"][i]
        if case["op"] == "text":
            start = s["start"][i] if torch.is_tensor(s["start"]) else s["start"]
            ahead = cols - (rows + start)[:, None]
            if case["causal"]:
                hidden |= ahead > 0
            if n:
                which = side[(ahead.abs() if case["both"] else (-ahead).clamp(min=0)).clamp(max=case["distance"])]
                which = which + n * (ahead > 0) if case["both"] else which
        none = hidden.all(1, keepdim=True)
        image = []
        for j in range(h):
            kv = j * hk // h
            z = s["scale"] * torch.mm(leaf["q"][i, j], leaf["k"][i, kv].t())
            if n:
                z = z + table[:, j].index_select(0, which.flatten()).view(lq, lk)
            z = torch.where(hidden, -1e300, z)
            w = torch.where(none, 0.0, torch.exp(z - torch.logsumexp(z, 1, keepdim=True)))
            o = torch.mm(w, leaf["v"][i, kv])
            if case["train"]:
                dh = case["dh"]
                (o * s["grad"][i, :, j * dh:(j + 1) * dh].double()).sum().backward()
            image.append(o.detach())
        outs.append(torch.cat(image, 1))
    out = torch.stack(outs)
    if not case["train"]:
        return out
    grads = [leaf[t].grad for t in ("q", "k", "v")]
    if case["op"] == "text":
        grads.append(None if table is None else table.grad)
    return (out, *grads)


# ---------------------------------------------------------------------------------------------- what a pass needs


def work(case):
    b, h, hk, lq, lk, dh = (case[n] for n in ("b", "heads", "kv_heads", "lq", "lk", "dh"))
    lengths, causal = _lengths(case), case["op"] == "text" and case["causal"]
    pairs = 0
    for n in lengths:
        if causal:  # the queries are the last lq positions of the text (the first, where it has fewer)
            first = max(n - lq, 0) if lq < lk else 0
            full = max(0, min(lq, n - first))  # queries that see first + 1, first + 2, .. keys; the others see all n
            pairs += full * first + full * (full + 1) // 2 + (lq - full) * n
        else:
            pairs += lq * n
    by = 2 * dh * (2 * b * h * lq + 2 * hk * sum(lengths))
    if case["train"]:  # the gradient of the output as well, and dq, dk, dv
        by += 2 * dh * (2 * b * h * lq + 2 * b * hk * lk)
    by += b * lk if case["keys"] == "mask" else 0
    if case["op"] == "text" and case["buckets"]:
        by += 2 * case["buckets"] * h * (2 if case["train"] else 1)
    return {"bytes": by, "flops": (14 if case["train"] else 4) * dh * h * pairs}
