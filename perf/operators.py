"""Cases of the token-sequence operators: the root-mean-square norm of a residual sum (with a gradient, or with 8-bit outputs and
their scales), rotary positions, and attention over a sliding window with a few first tokens that stay visible.

A pass in plain form writes the formulas out in elementary torch operations in 32 bits; a pass with `own` makes the calls that a
user of the package makes. `exact` gives the same outputs from the definitions in 64 bits.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_E4M3_MAX = 448.0


def _ops():
    import __graft_entry__
    return __graft_entry__.load_package()


# ---- cases --------------------------------------------------------------------------------------------------------------------
def _norm(name, mode, rows, width, dtype, group=0):
    return {"name": name, "op": "norm", "mode": mode, "rows": rows, "width": width, "dtype": dtype, "group": group}


def _rotary(name, mode, batch, length, heads, kv_heads, dim, rotary, interleaved, axes, start, dtype):
    return {"name": name, "op": "rotary", "mode": mode, "batch": batch, "length": length, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "rotary": rotary, "interleaved": interleaved, "axes": axes, "start": start, "dtype": dtype}


def _attention(name, mode, batch, queries, keys, heads, kv_heads, dim, window, sinks, ragged, dtype):
    return {"name": name, "op": "attention", "mode": mode, "batch": batch, "queries": queries, "keys": keys, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "window": window, "sinks": sinks, "ragged": ragged, "dtype": dtype}


def listed():
    return [
        # the residual stream of one decoding step of a small batch: latency
        _norm("norm_step", "infer", 16, 4096, "bf16"),
        # a prompt's tokens on their way into an 8-bit product, one scale for each 128 values
        _norm("norm_quant_prompt", "quant", 8192, 5120, "bf16", 128),
        # image tokens of an encoder of odd width, one scale a token
        _norm("norm_quant_odd", "quant", 1031, 1144, "fp16", 0),
        # a training step's forward and backward
        _norm("norm_train", "train", 8192, 4096, "bf16"),
        # one new token of each sequence of a batch, far into a long context
        _rotary("rotary_step", "infer", 32, 1, 32, 8, 128, 128, False, 1, 120000, "bf16"),
        # a long prompt, positions on the first half of each head only, neighbouring pairs
        _rotary("rotary_prompt_part", "infer", 1, 16384, 32, 8, 128, 64, True, 1, 0, "bf16"),
        # image and text tokens with three position axes, head width of a vision encoder, forward and backward
        _rotary("rotary_train_axes", "train", 2, 4099, 16, 16, 80, 80, False, 3, 0, "fp16"),
        # decoding: one query a sequence over caches of different lengths
        _attention("attention_step", "infer", 32, 1, 8192, 32, 8, 128, 1024, 4, True, "bf16"),
        # a prompt
        _attention("attention_prompt", "infer", 1, 8192, 8192, 16, 4, 128, 1024, 4, False, "bf16"),
        # a chunk of new tokens behind caches of different lengths, head width of a vision encoder
        _attention("attention_chunk", "infer", 3, 301, 5000, 16, 16, 80, 700, 1, True, "fp16"),
        # training, forward and backward
        _attention("attention_train", "train", 2, 4096, 4096, 16, 4, 128, 1024, 4, False, "bf16"),
        # training in 32 bits, odd sizes and a padded batch
        _attention("attention_train_fp32", "train", 2, 777, 777, 6, 2, 72, 200, 3, True, "fp32"),
    ]


def _spread(rng, low, high):
    """A whole number spread evenly over the logarithm of the range."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    kind = rng.choice(["norm", "rotary", "attention"])
    if kind == "norm":
        mode = rng.choice(["infer", "quant", "train"])
        width = 8 * _spread(rng, 16, 1024) if rng.random() < 0.7 else _spread(rng, 100, 8191)
        return _drop(_norm("", mode, _spread(rng, 1, max(1, (1 << 25) // width)), width, dtype, rng.choice([0, 128]) if mode == "quant" else 0))
    dim = rng.choice([64, 80, 96, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4])
    if kind == "rotary":
        axes = rng.choice([1, 1, 2, 3])
        length = _spread(rng, 1, 16384)
        batch = rng.randint(1, max(1, min(8, 32768 // length)))
        rotary = rng.choice([dim, dim // 2])
        return _drop(_rotary("", rng.choice(["infer", "train"]), batch, length, heads, kv_heads, dim, rotary, rng.random() < 0.4, axes,
                             rng.choice([0, 5000, 1000000]), dtype))
    mode = rng.choice(["step", "prompt", "chunk", "train"])
    window, sinks = _spread(rng, 16, 2048), rng.choice([0, 1, 4, 64])
    if mode == "step":
        keys = _spread(rng, 100, 8192)
        return _drop(_attention("", "infer", rng.randint(1, 32), 1, keys, heads, kv_heads, dim, window, sinks, rng.random() < 0.7, dtype))
    top = 1500 if dtype == "fp32" else 4096
    if mode == "chunk":
        keys = _spread(rng, 600, top)
        return _drop(_attention("", "infer", rng.randint(1, 3), _spread(rng, 2, 512), keys, heads, kv_heads, dim, window, sinks, True, dtype))
    length = _spread(rng, 100, top)
    heads, kv_heads = min(heads, 16), min(kv_heads, 4) if heads <= 16 else 4
    return _drop(_attention("", "infer" if mode == "prompt" else "train", rng.randint(1, 2), length, length, heads, kv_heads, dim, window, sinks,
                            rng.random() < 0.5, dtype))


def _drop(case):
    return {k: v for k, v in case.items() if k != "name"}


# ---- inputs -------------------------------------------------------------------------------------------------------------------
def _lengths(case):
    """The sequences' lengths, in keys and in queries: the whole extent, or shorter ones. A decoding step or a chunk keeps all its
    queries; a padded batch of prompts has as many queries as keys."""
    b, q, k = case["batch"], case["queries"], case["keys"]
    if not case["ragged"]:
        return [k] * b, [q] * b
    kv = [k - (i * 613) % max(1, k // 2) for i in range(b)]
    return (kv, list(kv)) if q == k else ([max(n, q) for n in kv], [q] * b)


def _sections(case):
    """How many frequencies turn by each axis of the positions."""
    n, a = case["rotary"] // 2, case["axes"]
    return [n - (a - 1) * (n // a)] + [n // a] * (a - 1)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    t = _TYPES[case["dtype"]]

    def normal(*shape, spread=1.0):
        return (torch.randn(shape, generator=gen, device=dev) * spread).to(t)

    state = {"case": case}
    if case["op"] == "norm":
        shape = (case["rows"], case["width"])
        state |= {"x": normal(*shape), "residual": normal(*shape, spread=3.0), "weight": normal(case["width"], spread=0.2) + 1, "eps": 1e-6}
        if case["mode"] == "train":
            state |= {"grad_y": normal(*shape), "grad_sum": normal(*shape)}
    elif case["op"] == "rotary":
        b, n, h, hk, d, a = (case[k] for k in ("batch", "length", "heads", "kv_heads", "dim", "axes"))
        # queries, keys and values come out of one product: two views of its rows are turned
        qkv = normal(b, n, h + 2 * hk, d)
        state |= {"q": qkv[:, :, :h], "k": qkv[:, :, h:h + hk]}
        if a == 1:
            first = torch.randint(0, case["start"] // 8 + 16, (b, 1), generator=gen, device=dev) + case["start"]
            state["positions"] = first + torch.arange(n, device=dev)
            state["sections"] = None
        else:  # time, row and column of image patches
            side = max(1, int(math.isqrt(n)))
            i = torch.arange(n, device=dev) + torch.randint(0, 64, (1,), generator=gen, device=dev)
            axes = [i // (side * side) + case["start"], (i // side) % side, i % side]
            state["positions"] = torch.stack(axes[:a]).unsqueeze(1).expand(a, b, n).contiguous()
            state["sections"] = _sections(case)
        half = case["rotary"] // 2
        base = 500000.0 if case["start"] else 10000.0
        state["inv_freq"] = (base ** (-torch.arange(half, dtype=torch.float64, device=dev) / half)).float()
        state["scale"] = 1.0 + 0.1 * math.log(8.0) if case["start"] else 1.0
        if case["mode"] == "train":
            state |= {"grad_q": normal(b, n, h, d), "grad_k": normal(b, n, hk, d)}
    else:
        b, nq, nk, h, hk, d = (case[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
        state |= {"q": normal(b, nq, h, d), "k": normal(b, nk, hk, d), "v": normal(b, nk, hk, d), "kv_lengths": None, "q_lengths": None}
        if case["ragged"]:
            kv, qn = _lengths(case)
            state["kv_lengths"] = torch.tensor(kv, dtype=torch.int32, device=dev)
            if nq == nk:
                state["q_lengths"] = torch.tensor(qn, dtype=torch.int32, device=dev)
        if case["mode"] == "train":
            state["grad_out"] = normal(b, nq, h, d)
    return state


# ---- one pass -----------------------------------------------------------------------------------------------------------------
def run(state):
    return _RUN[state["case"]["op"]](state)


def _norm_run(s):
    mode, eps = s["case"]["mode"], s["eps"]
    if own:
        ops = _ops()
        if mode == "quant":
            return ops.residual_rms_norm_quant(s["x"], s["residual"], s["weight"], eps, group=s["case"]["group"])
        y, total, rstd = ops.residual_rms_norm(s["x"], s["residual"], s["weight"], eps)
        if mode == "infer":
            return y, total
        gx, gw = ops.residual_rms_norm_backward(s["grad_y"], total, rstd, s["weight"], s["grad_sum"])
        return y, total, gx, gw
    t = s["x"].dtype
    total = (s["x"].float() + s["residual"].float()).to(t)
    z, w = total.float(), s["weight"].float()
    rstd = torch.rsqrt(z.square().mean(-1, keepdim=True) + eps)
    unit = z * rstd
    y = unit * w
    if mode == "quant":
        rows, width = y.shape
        g = s["case"]["group"] or width
        n = -(-width // g)
        tiles = torch.zeros(rows, n * g, dtype=y.dtype, device=y.device)
        tiles[:, :width] = y
        tiles = tiles.view(rows, n, g)
        scale = tiles.abs().amax(-1) / _E4M3_MAX
        q = (tiles / torch.where(scale > 0, scale, 1).unsqueeze(-1)).clamp(-_E4M3_MAX, _E4M3_MAX)
        return q.view(rows, n * g)[:, :width].to(torch.float8_e4m3fn), scale, total
    if mode == "infer":
        return y.to(t), total
    gy = s["grad_y"].float()
    gu = gy * w
    gx = (gu - unit * (gu * unit).mean(-1, keepdim=True)) * rstd + s["grad_sum"].float()
    gw = (gy * unit).sum(0)
    return y.to(t), total, gx.to(t), gw.to(t)


def _angles(positions, inv_freq, sections, scale):
    """cos and sin of each token's angles, [..., 1, frequencies] (computed in 64 bits: far positions lose their angle in 32)."""
    f = inv_freq.double()
    if sections is None:
        angle = positions.double().unsqueeze(-1) * f
    else:
        axis = torch.repeat_interleave(torch.arange(len(sections), device=f.device), torch.tensor(sections, device=f.device), output_size=f.numel())
        angle = positions.double()[axis].movedim(0, -1) * f
    return (angle.cos() * scale).float().unsqueeze(-2), (angle.sin() * scale).float().unsqueeze(-2)


def _turn(x, cos, sin, rotary, interleaved):
    z = x[..., :rotary].float()
    a, b = (z[..., 0::2], z[..., 1::2]) if interleaved else (z[..., :rotary // 2], z[..., rotary // 2:])
    u, v = a * cos - b * sin, b * cos + a * sin
    z = torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)
    return torch.cat((z.to(x.dtype), x[..., rotary:]), -1)


def _rotary_run(s):
    c = s["case"]
    if own:
        ops = _ops()
        how = {"interleaved": c["interleaved"], "sections": s["sections"], "scale": s["scale"]}
        q, k = ops.rotary_embedding(s["q"], s["k"], s["positions"], s["inv_freq"], **how)
        if c["mode"] == "infer":
            return q, k
        return (q, k) + tuple(ops.rotary_embedding_backward(s["grad_q"], s["grad_k"], s["positions"], s["inv_freq"], **how))
    cos, sin = _angles(s["positions"], s["inv_freq"], s["sections"], s["scale"])
    out = [_turn(s[n], cos, sin, c["rotary"], c["interleaved"]) for n in ("q", "k")]
    if c["mode"] == "train":
        out += [_turn(s[n], cos, -sin, c["rotary"], c["interleaved"]) for n in ("grad_q", "grad_k")]
    return tuple(out)


def _visible(s):
    """[batch, queries, keys]: the last query of a sequence sits at its last key; a query sees itself, the window - 1 keys before it
    and the first `sinks` keys."""
    c = s["case"]
    dev = s["q"].device
    b, nq, nk = c["batch"], c["queries"], c["keys"]
    kv = s["kv_lengths"] if s["kv_lengths"] is not None else torch.full((b,), nk, dtype=torch.int32, device=dev)
    qn = s["q_lengths"] if s["q_lengths"] is not None else torch.full((b,), nq, dtype=torch.int32, device=dev)
    i = torch.arange(nq, device=dev)
    at = (kv - qn)[:, None, None] + i[None, :, None]
    j = torch.arange(nk, device=dev)[None, None, :]
    return (j <= at) & ((j > at - c["window"]) | (j < c["sinks"])) & (i[None, :, None] < qn[:, None, None]) & (j < kv[:, None, None])


def _attention_run(s):
    c = s["case"]
    scale = 1.0 / math.sqrt(c["dim"])
    if own:
        ops = _ops()
        how = {"q_lengths": s["q_lengths"], "kv_lengths": s["kv_lengths"]}
        out, lse = ops.window_attention(s["q"], s["k"], s["v"], c["window"], c["sinks"], **how)
        if c["mode"] == "infer":
            return out
        return (out,) + tuple(ops.window_attention_backward(s["grad_out"], s["q"], s["k"], s["v"], out, lse, c["window"], c["sinks"], **how))
    t = s["q"].dtype
    b, nq, h, d = s["q"].shape
    hk = s["k"].shape[2]
    # [batch, kv heads, group, queries, dim] against [batch, kv heads, 1, keys, dim]
    q = s["q"].float().view(b, nq, hk, h // hk, d).permute(0, 2, 3, 1, 4)
    k, v = (s[n].float().permute(0, 2, 1, 3).unsqueeze(2) for n in ("k", "v"))
    seen = _visible(s)[:, None, None]
    score = (q @ k.transpose(-1, -2)).mul_(scale).masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = (score - torch.where(top == -math.inf, 0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total == 0, 1, total)
    o = p @ v
    back = lambda z: z.permute(0, 3, 1, 2, 4).reshape(b, nq, h, d).to(t)  # noqa: E731
    if c["mode"] == "infer":
        return back(o)
    g = s["grad_out"].float().view(b, nq, hk, h // hk, d).permute(0, 2, 3, 1, 4)
    gv = (p.transpose(-1, -2) @ g).sum(2)
    gs = (g @ v.transpose(-1, -2)).sub_((g * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    gq = gs @ k
    gk = (gs.transpose(-1, -2) @ q).sum(2)
    return back(o), back(gq), gk.transpose(1, 2).to(t), gv.transpose(1, 2).to(t)


_RUN = {"norm": _norm_run, "rotary": _rotary_run, "attention": _attention_run}


# ---- what a pass cannot do without --------------------------------------------------------------------------------------------
def _pairs(case):
    """(pairs of a query and a key that it sees, keys that some query sees), summed over the batch, for one head."""
    pairs = keys = 0
    for kv, qn in zip(*_lengths(case)):
        at = np.arange(kv - qn, kv, dtype=np.int64)
        near = np.minimum(at + 1, case["window"])
        pairs += int(near.sum() + np.minimum(case["sinks"], at + 1 - near).sum())
        first = max(0, kv - qn - case["window"] + 1)
        keys += kv - first + min(case["sinks"], first)
    return pairs, keys


def work(case):
    size = _BYTES[case["dtype"]]
    if case["op"] == "norm":
        n, w = case["rows"] * case["width"], case["width"]
        if case["mode"] == "infer":
            return {"bytes": size * (4 * n + w), "flops": 5 * n}
        if case["mode"] == "quant":
            return {"bytes": size * (3 * n + w) + n + 4 * case["rows"] * -(-w // (case["group"] or w)), "flops": 8 * n}
        return {"bytes": size * (4 * n + w) + size * (3 * n + w), "flops": 16 * n}
    if case["op"] == "rotary":
        tokens = case["batch"] * case["length"]
        n = tokens * (case["heads"] + case["kv_heads"])
        passes = 2 if case["mode"] == "train" else 1
        return {"bytes": passes * 2 * size * n * case["dim"] + 8 * tokens * case["axes"] + 2 * case["rotary"], "flops": passes * 3 * n * case["rotary"]}
    pairs, keys = _pairs(case)
    rows = sum(_lengths(case)[1])
    q, kv = rows * case["heads"] * case["dim"], keys * case["kv_heads"] * case["dim"]
    if case["mode"] == "infer":
        return {"bytes": size * (2 * q + 2 * kv), "flops": 4 * pairs * case["dim"] * case["heads"]}
    return {"bytes": size * (4 * q + 4 * kv), "flops": 14 * pairs * case["dim"] * case["heads"]}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _EXACT[case["op"]](s)


def _norm_exact(s):
    mode, t = s["case"]["mode"], s["x"].dtype
    total = s["x"].double() + s["residual"].double()
    z, w = total.to(t).double(), s["weight"].double()  # the norm is that of the sum as it is stored
    inverse = 1 / (z.pow(2).sum(-1) / z.shape[-1] + s["eps"]).sqrt()
    y = z * inverse[:, None] * w[None, :]
    if mode == "infer":
        return y, total
    if mode == "quant":
        parts = torch.split(y, s["case"]["group"] or y.shape[-1], dim=-1)
        scales = [p.abs().max(-1).values / _E4M3_MAX for p in parts]
        return torch.cat([p / a[:, None].clamp_min(1e-300) for p, a in zip(parts, scales)], -1), torch.stack(scales, -1), total
    gy = s["grad_y"].double()
    dot = (gy * w * z).sum(-1) / z.shape[-1]
    gx = gy * w * inverse[:, None] - z * (dot * inverse ** 3)[:, None] + s["grad_sum"].double()
    return y, total, gx, torch.einsum("rc,rc,r->c", gy, z, inverse)


def _rotary_exact(s):
    c = s["case"]
    half, positions = c["rotary"] // 2, s["positions"].double()
    if s["sections"] is not None:
        parts = [p[..., None].expand(*p.shape, n) for p, n in zip(positions, s["sections"])]
        angle = torch.cat(parts, -1) * s["inv_freq"].double()
    else:
        angle = positions[..., None] * s["inv_freq"].double()
    turn = torch.polar(torch.full_like(angle, s["scale"]), angle)[:, :, None]

    def turned(x, by):
        x = x.double()
        z, rest = x[..., :c["rotary"]], x[..., c["rotary"]:]
        if c["interleaved"]:
            z = torch.view_as_real(torch.view_as_complex(z.unflatten(-1, (half, 2)).contiguous()) * by).flatten(-2)
        else:
            pair = torch.complex(z[..., :half].contiguous(), z[..., half:].contiguous()) * by
            z = torch.cat((pair.real, pair.imag), -1)
        return torch.cat((z, rest), -1)

    out = [turned(s["q"], turn), turned(s["k"], turn)]
    if c["mode"] == "train":
        out += [turned(s["grad_q"], turn.conj()), turned(s["grad_k"], turn.conj())]
    return tuple(out)


def _attention_exact(s):
    c = s["case"]
    b, nq, h, d = s["q"].shape
    hk, dev = s["k"].shape[2], s["q"].device
    train = c["mode"] == "train"
    out = torch.zeros(b, nq, h, d, dtype=torch.float64, device=dev)
    gq = torch.zeros_like(out)
    gk = torch.zeros(b, c["keys"], hk, d, dtype=torch.float64, device=dev)
    gv = torch.zeros_like(gk)
    kv, qn = _lengths(c)
    for i in range(b):
        n, m = qn[i], kv[i]
        row = torch.arange(m - n, m, device=dev)[:, None]
        col = torch.arange(m, device=dev)[None, :]
        hidden = (col > row) | ((row - col >= c["window"]) & (col >= c["sinks"]))
        for a in range(h):
            u = a * hk // h
            q, k, v = s["q"][i, :n, a].double(), s["k"][i, :m, u].double(), s["v"][i, :m, u].double()
            p = torch.softmax((q @ k.T / math.sqrt(d)).masked_fill(hidden, -math.inf), -1)
            o = p @ v
            out[i, :n, a] = o
            if train:
                g = s["grad_out"][i, :n, a].double()
                gv[i, :m, u] += p.T @ g
                gs = p * (g @ v.T - (g * o).sum(-1, keepdim=True)) / math.sqrt(d)
                gq[i, :n, a] = gs @ k
                gk[i, :m, u] += gs.T @ q
    return (out, gq, gk, gv) if train else out


_EXACT = {"norm": _norm_exact, "rotary": _rotary_exact, "attention": _attention_exact}
