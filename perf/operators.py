"""Two operators of an unquantized transformer block, as cases that a timing program can prepare, run and check.

A case is a dict of plain values with an "op":

  linear  out = residual + gate * act(x W^T + bias) with a raw (bf16 or fp16) weight [n, k]: selas_amd.linear.raw_linear.
          x is [b, l, k]; act is "none", "gelu" (tanh approximation) or "silu"; a gate is one row per image; the output
          has the residual's dtype, or out's.
  rope    rotary positions with several axes (time, row, column) on q and k, taken from the positions themselves, after
          an optional RMS norm of the heads, with v laid out on the way: selas_amd.rope.rope_qk.

The plain forms below are elementary torch operations in 32 bits (64 for the angles of the positions), rounded once.
"""

from __future__ import annotations

import math

import torch

own = False

D, MLP = 3072, 12288  # FLUX-dev: width and MLP width (heads of 128)
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "int32": torch.int32}
MAX_MACS = 4608 * D * (D + MLP)  # the largest listed linear
MAX_ROPE = 2 * 20280 * (24 + 24) * 128  # elements of q and k in the largest listed rotation


# ---------------------------------------------------------------------------------------------- the cases


def _linear(name, b, l, n, k, act="none", bias=True, residual=False, dtype="bf16", out="bf16"):
    return dict(name=name, op="linear", b=b, l=l, n=n, k=k, act=act, bias=bias, residual=residual, dtype=dtype, out=out)


def _rope(name, b, text, t, h, w, heads, kv_heads, dh, axes, norm, with_v, pairs="interleaved", inverse=False,
          dtype="bf16", ids="fp32"):
    a0, a1, a2 = axes
    return dict(name=name, op="rope", b=b, text=text, t=t, h=h, w=w, heads=heads, kv_heads=kv_heads, dh=dh, axis_t=a0,
                axis_h=a1, axis_w=a2, norm=norm, with_v=with_v, pairs=pairs, inverse=inverse, dtype=dtype, ids=ids)


def listed():
    return [
        # The pooled text's embedding: one row, in_layer and its SiLU. The smallest call: latency.
        _linear("pooled_text_silu", 1, 1, D, 768, act="silu"),
        # One modulation linear for the 28 steps of an image: the weight is read once.
        _linear("modulation_28_steps", 1, 28, 6 * D, D),
        # The text stream's second MLP linear with its gated residual: few tiles, long K.
        _linear("text_mlp2_residual", 1, 512, D, MLP, residual=True, out="fp32"),
        # The image stream's first MLP linear at 1024 x 1024, GELU on the way out.
        _linear("mlp0_gelu_1024", 1, 4096, MLP, D, act="gelu"),
        # A single block's linear2 with its gated residual at 1024 x 1024: the largest product.
        _linear("linear2_residual_1024", 1, 4608, D, D + MLP, residual=True, out="fp32"),
        # img_in at 1024 x 1024, straight to the fp32 residual stream: the output's bytes.
        _linear("img_in_1024", 1, 4096, D, 64, out="fp32"),
        # The final layer of four 512 x 512 images: 64 columns.
        _linear("final_layer_512_batch4", 4, 1024, 64, D, out="fp32"),
        # Sizes that fill no tile and rows off every alignment, two images, in fp16: a model of another width.
        _linear("odd_fp16", 2, 693, 1431, 667, act="gelu", residual=True, dtype="fp16", out="fp16"),
        # One token's q and k: latency.
        _rope("one_token", 1, 1, 0, 1, 1, 24, 24, 128, (16, 56, 56), norm=True, with_v=True),
        # A FLUX block's attention input at 1024 x 1024 with 512 text tokens: norm, rotation, and v laid out.
        _rope("image_1024", 1, 512, 1, 64, 64, 24, 24, 128, (16, 56, 56), norm=True, with_v=True),
        # A clip of 13 latent frames of 30 x 52 tokens with whole-number positions, two at once, fp16, halves paired.
        _rope("video_13x30x52_batch2", 2, 0, 13, 30, 52, 24, 24, 128, (44, 42, 42), norm=False, with_v=False,
              pairs="halves", dtype="fp16", ids="int32"),
        # The gradient of a rotation (its inverse) in fp32: shared k heads, channels that are not rotated, odd length.
        _rope("inverse_fp32_shared_heads", 1, 77, 1, 37, 41, 16, 4, 96, (16, 32, 32), norm=False, with_v=False,
              inverse=True, dtype="fp32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    return _draw_linear(rng) if rng.random() < 0.6 else _draw_rope(rng)


def _draw_linear(rng):
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    residual = rng.random() < 0.5
    out = rng.choice((dtype, "fp32"))
    act = rng.choice(("none", "gelu", "silu"))
    bias = rng.random() < 0.8
    while True:
        if rng.random() < 0.7:  # widths of a model: whole chunks of 8 channels
            n, k = 8 * _log_int(rng, 8, 2688), 8 * _log_int(rng, 8, 1920)
        else:
            n, k = _log_int(rng, 33, 6000), _log_int(rng, 33, 6000)
        b = rng.choice((1, 1, 1, 2, 3))
        l = rng.randint(1, 64) if rng.random() < 0.4 else _log_int(rng, 65, 6144)
        if 1 << 22 <= b * l * n * k <= MAX_MACS and b * l * n <= 1 << 27:
            return dict(op="linear", b=b, l=l, n=n, k=k, act=act, bias=bias, residual=residual, dtype=dtype, out=out)


def _draw_rope(rng):
    dh = rng.choice((64, 80, 96, 128, 128, 128))
    dtype, norm = rng.choice(("bf16", "bf16", "fp16", "fp32")), rng.random() < 0.5
    kv_heads = rng.choice((1, 2, 4, 8, 12, 16, 24))
    heads = kv_heads * rng.choice((1, 1, 2, 4))
    half = rng.choice((dh, dh, dh // 4 * 3)) // 2  # rotated pairs of channels
    half -= half % 4
    at = 2 * rng.randint(1, half // 4)
    ah = (half - at // 2) // 2 * 2
    axes = (at, ah, 2 * half - at - ah)
    inverse = not norm and rng.random() < 0.3
    while True:
        if rng.random() < 0.2:
            t, h, w, text = 0, 1, 1, rng.randint(1, 64)
        else:
            t = rng.choice((1, 1, 1, _log_int(rng, 2, 21)))
            h, w = _log_int(rng, 8, 96), _log_int(rng, 8, 96)
            text = rng.choice((0, 0, 77, 256, 512))
        b = rng.choice((1, 1, 2, 3))
        if b * (text + t * h * w) * (heads + kv_heads) * dh * (2 if dtype == "fp32" else 1) <= MAX_ROPE:
            return dict(op="rope", b=b, text=text, t=t, h=h, w=w, heads=heads, kv_heads=kv_heads, dh=dh,
                        axis_t=axes[0], axis_h=axes[1], axis_w=axes[2], norm=norm,
                        with_v=not inverse and rng.random() < 0.5, pairs=rng.choice(("interleaved", "halves")),
                        inverse=inverse, dtype=dtype, ids=rng.choice(("fp32", "int32")))


# ---------------------------------------------------------------------------------------------- inputs


class _Inputs:
    """Seeded random tensors on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape, std=1.0, mean=0.0, dtype=torch.float32):
        return torch.empty(shape, device="cuda").normal_(mean, std, generator=self.g).to(dtype)


def prepare(case, seed):
    g, dt = _Inputs(seed), DT[case["dtype"]]
    if case["op"] == "linear":
        b, l, n, k = case["b"], case["l"], case["n"], case["k"]
        state = dict(case=case, x=g.normal(b, l, k, dtype=dt), weight=g.normal(n, k, std=k ** -0.5, dtype=dt),
                     bias=g.normal(n, std=0.1, dtype=dt) if case["bias"] else None, gate=None, residual=None)
        if case["residual"]:
            # The block's vectors are slices of one modulation row, as the modulation linears lay them out.
            state["gate"] = g.normal(b, 1, 3 * n, std=0.5)[..., 2 * n:]
            state["residual"] = g.normal(b, l, n, std=2.0, dtype=DT[case["out"]])
        return state
    b, dh, length = case["b"], case["dh"], _tokens(case)
    hq, hk = case["heads"], case["kv_heads"]
    # q, k and v are the columns of one linear's output, [b, tokens, (hq + 2 hk) dh], seen as [b, heads, tokens, dh].
    qkv = g.normal(b, length, hq + 2 * hk, dh, dtype=dt).transpose(1, 2)
    q, k, v = qkv.split((hq, hk, hk), dim=1)
    state = dict(case=case, q=q, k=k, v=v if case["with_v"] else None, ids=_positions(case, seed),
                 axes=(case["axis_t"], case["axis_h"], case["axis_w"]), q_scale=None, k_scale=None)
    if case["norm"]:
        state["q_scale"], state["k_scale"] = g.normal(dh, std=0.1, mean=1.0), g.normal(dh, std=0.1, mean=1.0)
    return state


def _tokens(case):
    return case["text"] + case["t"] * case["h"] * case["w"]


def _positions(case, seed):
    """(time, row, column) of every token, text at 0; each image of a batch is a window of a larger canvas."""
    b, text, t, h, w = case["b"], case["text"], case["t"], case["h"], case["w"]
    grid = torch.cartesian_prod(torch.arange(t), torch.arange(h), torch.arange(w)).view(-1, 3)
    shift = torch.tensor([[i * (1 + seed % 3), 7 * i + seed % 100, 11 * i + seed % 50] for i in range(b)])
    ids = torch.zeros(b, text + t * h * w, 3, dtype=torch.int64)
    ids[:, text:] = grid[None] + shift[:, None]
    return ids.to(DT[case["ids"]]).cuda()


# ---------------------------------------------------------------------------------------------- one pass


def run(state):
    case = state["case"]
    if case["op"] == "linear":
        return (_own_linear if own else _plain_linear)(state)
    return (_own_rope if own else _plain_rope)(state)


def _own_linear(s):
    from selas_amd.linear import raw_linear

    case = s["case"]
    act = None if case["act"] == "none" else case["act"]
    return raw_linear(s["x"], s["weight"], s["bias"], act=act, gate=s["gate"], residual=s["residual"],
                      out_dtype=DT[case["out"]])


def _own_rope(s):
    from selas_amd.rope import rope_qk

    case = s["case"]
    return rope_qk(s["q"], s["k"], s["ids"], s["axes"], 10000.0, v=s["v"], q_scale=s["q_scale"], k_scale=s["k_scale"],
                   pairs=case["pairs"], inverse=case["inverse"])


def _plain_linear(s):
    y = s["x"].float() @ s["weight"].float().t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["case"]["act"] == "gelu":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    elif s["case"]["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    if s["gate"] is not None:
        y = s["gate"].float() * y
    if s["residual"] is not None:
        y = s["residual"].float() + y
    return y.to(DT[s["case"]["out"]])


def _plain_rope(s):
    case, ids = s["case"], s["ids"]
    angles = []
    for i, d in enumerate(s["axes"]):
        omega = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device=ids.device) / d)
        angles.append(ids[..., i].double()[..., None] * omega)
    angle = torch.cat(angles, -1)[:, None]  # [b, 1, tokens, pairs]
    cos, sin = angle.cos().float(), angle.sin().float()
    if case["inverse"]:
        sin = -sin
    r = 2 * cos.shape[-1]

    def rotate(x, scale):
        y = x.float()
        if scale is not None:
            y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6) * scale
        z = y.clone()
        if case["pairs"] == "interleaved":
            a, b = y[..., 0:r:2], y[..., 1:r:2]
            z[..., 0:r:2], z[..., 1:r:2] = a * cos - b * sin, a * sin + b * cos
        else:
            a, b = y[..., :r // 2], y[..., r // 2:r]
            z[..., :r // 2], z[..., r // 2:r] = a * cos - b * sin, a * sin + b * cos
        return z.to(x.dtype)

    out = (rotate(s["q"], s["q_scale"]), rotate(s["k"], s["k_scale"]))
    return out if s["v"] is None else (*out, s["v"].contiguous())


# ---------------------------------------------------------------------------------------------- the definition in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        return _exact_linear(s)
    q, k = _exact_rope(s, s["q"], s["q_scale"]), _exact_rope(s, s["k"], s["k_scale"])
    return (q, k) if s["v"] is None else (q, k, s["v"].double())


def _exact_linear(s):
    case = s["case"]
    w, n = s["weight"].double(), case["n"]
    rows = []
    for i in range(case["b"]):
        z = torch.addmm(torch.zeros(n, dtype=torch.float64, device="cuda") if s["bias"] is None else s["bias"].double(),
                        s["x"][i].double(), w.mT)
        if case["act"] != "none":  # z / (1 + e^-u): SiLU with u = z, the tanh GELU with u = sqrt(8 / pi)(z + ...)
            u = z if case["act"] == "silu" else (z + 0.044715 * z ** 3) * (8 / math.pi) ** 0.5
            z = z * torch.sigmoid(u)
        if s["gate"] is not None:
            z = z * s["gate"][i].double()
        rows.append(z if s["residual"] is None else z + s["residual"][i].double())
    return torch.stack(rows)


def _exact_rope(s, x, scale):
    """Each pair as a complex number times e^(i angle)."""
    case = s["case"]
    pos = s["ids"].double()
    turn = torch.cat([torch.outer(pos[..., i].reshape(-1), torch.exp(torch.linspace(0, -1, d // 2 + 1, dtype=torch.float64,
                      device="cuda")[:-1] * math.log(10000.0))).view(*pos.shape[:2], -1) for i, d in enumerate(s["axes"])], -1)
    phase = torch.polar(torch.ones_like(turn), -turn if case["inverse"] else turn).unsqueeze(1)
    r = 2 * turn.shape[-1]
    outs = []
    for h in range(x.shape[1]):  # head by head: the 64-bit copies of a long clip are large
        y = x[:, h:h + 1].double()
        if scale is not None:
            y = y * scale.double() * (y.square().mean(-1, keepdim=True) + 1e-6) ** -0.5
        if case["pairs"] == "interleaved":
            z = torch.view_as_real(torch.view_as_complex(y[..., :r].unflatten(-1, (-1, 2)).contiguous()) * phase).flatten(-2)
        else:
            c = torch.complex(y[..., :r // 2].contiguous(), y[..., r // 2:r].contiguous()) * phase
            z = torch.cat((c.real, c.imag), -1)
        outs.append(torch.cat((z, y[..., r:]), -1))
    return torch.cat(outs, 1)


# ---------------------------------------------------------------------------------------------- what a pass needs


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4, "int32": 4}
    e = size[case["dtype"]]
    if case["op"] == "linear":
        m, n, k, eo = case["b"] * case["l"], case["n"], case["k"], size[case["out"]]
        by = e * (m * k + n * k) + eo * m * n + (e * n if case["bias"] else 0)
        if case["residual"]:
            by += eo * m * n + 4 * case["b"] * n
        per = {"none": 1, "gelu": 9, "silu": 5}[case["act"]] + (2 if case["residual"] else 0)
        return {"bytes": by, "flops": 2 * m * n * k + per * m * n}
    tokens = case["b"] * _tokens(case)
    rotated = tokens * (case["heads"] + case["kv_heads"]) * case["dh"]
    moved = rotated + (tokens * case["kv_heads"] * case["dh"] if case["with_v"] else 0)
    return {"bytes": 2 * e * moved + tokens * 12 + (8 * case["dh"] if case["norm"] else 0),
            "flops": rotated * (7 if case["norm"] else 3)}
