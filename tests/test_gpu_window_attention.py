"""Attention over a sliding window with sinks against its formulas in 64 bits.

Tolerances. u is half a step of the storage type, 2^-24 for fp32 and at most 2^-11 (fp16) or 2^-8 (bf16); s = 2^-24.
A score is a sum of `dim` products in fp32: off by at most E = (dim + 4) s sum_d |scale q_d k_d|, which moves its weight by a factor
of exp(E), with the largest E of the call. A weight may be rounded to the storage type before its product (1 u; fp16 weights below
2^-14 by 2^-25 each), values add up in fp32 over at most `keys` terms, and the result is rounded once (1 u):
  |out - exact| <= u |out| + (u + 2 E + (keys + 16) s) sum_j p_j |v_j| + keys 2^-25 max|v| (fp16).
Backward: delta is formed from the rounded out (its error is u + 2E.. of sum_d |g_d| |o_d|), dP and the weights as above, ds is rounded
to the storage type once (fp16 scales it to its range first), so with A_j = p_j (sum_d |g_d v_jd| + sum_d |g_d| sum_j p_j |v_jd|) scale
  |gradQ - exact| <= u |gradQ| + (2 u + 4 E + (keys + dim + 32) s) sum_j A_j |k_j|,   the same for gradK with |q_i|, and
  |gradV - exact| <= u |gradV| + (u + 2 E + (queries + 16) s) sum_i p_ij |g_i|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
S = 2.0 ** -24


def normal(shape, t, seed, dev, spread=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * spread).to(t).to(dev)


def seen_by(b, lq, lk, window, sinks, qn, kn, dev):
    i, j = torch.arange(lq, device=dev)[None, :, None], torch.arange(lk, device=dev)[None, None, :]
    p = (kn - qn)[:, None, None] + i
    return (i < qn[:, None, None]) & (j < kn[:, None, None]) & (j <= p) & ((j > p - window) | (j < sinks))


class Reference:
    """out, lse, the gradients and the bounds of their errors. Masked keys do not enter, whatever they hold."""

    def __init__(self, q, k, v, window, sinks, scale=None, qn=None, kn=None, g=None):
        t, dev = q.dtype, q.device
        b, lq, h, d = q.shape
        lk, hk = k.shape[1:3]
        r = h // hk
        scale = 1 / math.sqrt(d) if scale is None else scale
        qn = torch.full((b,), lq, device=dev) if qn is None else qn.clamp(0, lq)
        kn = torch.full((b,), lk, device=dev) if kn is None else kn.clamp(0, lk)
        seen = seen_by(b, lq, lk, window, sinks, qn, kn, dev)[:, None]
        q, k, v = (x.double().transpose(1, 2) for x in (q, k, v))
        k, v = k.repeat_interleave(r, 1), v.repeat_interleave(r, 1)
        key_ok = seen.any(2)[:, 0][:, None, :, None]
        row_ok = seen.any(3)[:, 0][:, None, :, None]
        k, v, q = torch.where(key_ok, k, 0), torch.where(key_ok, v, 0), torch.where(row_ok, q, 0)
        score = (q @ k.transpose(-1, -2) * scale).masked_fill(~seen, -math.inf)
        self.lse = torch.logsumexp(score, -1)
        p = torch.exp(score - torch.where(self.lse == -math.inf, 0, self.lse)[..., None])
        o = p @ v
        u = torch.finfo(t).eps / 2
        tiny = torch.finfo(t).tiny
        size = (q.abs() @ k.abs().transpose(-1, -2) * abs(scale)).masked_fill(~seen, 0)
        e = (d + 4) * S * size.amax(-1).amax(-1)[..., None, None].clamp_min(1)
        flush = lk * 2.0 ** -25 * v.abs().amax((-1, -2))[..., None, None] if t == F16 else 0
        self.out = o.transpose(1, 2)
        self.out_bound = (u * o.abs() + (u + 2 * e + (lk + 16) * S) * (p @ v.abs()) + flush + tiny).transpose(1, 2)
        self.lse_bound = 2 * e[..., 0] + 4 * S * self.lse.abs().nan_to_num(0, 0, 0) + (lk + 16) * S
        if g is None:
            return
        g = torch.where(row_ok, g.double().transpose(1, 2), 0)
        dp = g @ v.transpose(-1, -2)
        ds = p * (dp - (g * o).sum(-1, keepdim=True)) * scale
        a = p * (g.abs() @ v.abs().transpose(-1, -2) + (g.abs() * (p @ v.abs())).sum(-1, keepdim=True)) * abs(scale)
        rel = 2 * u + 4 * e + (max(lq * r, lk) + d + 32) * S
        # what fp16 weights and scaled ds lose below its normal range
        low = 2.0 ** -25 if t == F16 else 0.0
        low_ds = low * a.amax((-1, -2), keepdim=True)

        def shared(x):
            return x.unflatten(1, (hk, r)).sum(2).transpose(1, 2)

        self.gq = (ds @ k).transpose(1, 2)
        self.gq_bound = u * self.gq.abs() + (rel * (a @ k.abs()) + low_ds * k.abs().sum(-2, keepdim=True) + tiny).transpose(1, 2)
        self.gk = shared(ds.transpose(-1, -2) @ q)
        self.gk_bound = u * self.gk.abs() + shared(rel * (a.transpose(-1, -2) @ q.abs()) + low_ds * q.abs().sum(-2, keepdim=True)) + tiny
        self.gv = shared(p.transpose(-1, -2) @ g)
        self.gv_bound = u * self.gv.abs() + shared(rel * (p.transpose(-1, -2) @ g.abs()) + low * g.abs().sum(-2, keepdim=True)) + tiny


def close(name, got, want, bound):
    assert got.shape == want.shape
    if got.numel() == 0:
        return
    got = got.double()
    assert torch.isfinite(got).all(), f"{name}: not finite at {(~torch.isfinite(got)).nonzero()[0].tolist()}"
    over = (got - want).abs() - bound
    worst = over.argmax().item()
    where = torch.unravel_index(torch.tensor(worst), over.shape)
    assert (over <= 0).all(), f"{name}: {over.max().item():.3g} over the bound at {[int(w) for w in where]}"


def close_lse(got, ref):
    assert torch.equal(got == -math.inf, ref.lse == -math.inf)
    fine = ref.lse > -math.inf
    assert ((got.double() - ref.lse).abs() <= ref.lse_bound)[fine].all()


def check(ops, q, k, v, window, sinks, scale=None, qn=None, kn=None, g=None):
    ref = Reference(q, k, v, window, sinks, scale, qn, kn, g)
    out, lse = ops.window_attention(q, k, v, window, sinks, scale, qn, kn)
    assert out.dtype == q.dtype and lse.dtype == F32
    close("out", out, ref.out, ref.out_bound)
    close_lse(lse, ref)
    again = ops.window_attention(q, k, v, window, sinks, scale, qn, kn)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    if g is not None:
        grads = ops.window_attention_backward(g, q, k, v, out, lse, window, sinks, scale, qn, kn)
        close("gradQ", grads[0], ref.gq, ref.gq_bound)
        close("gradK", grads[1], ref.gk, ref.gk_bound)
        close("gradV", grads[2], ref.gv, ref.gv_bound)
        again = ops.window_attention_backward(g, q, k, v, out, lse, window, sinks, scale, qn, kn)
        assert all(torch.equal(x, y) for x, y in zip(again, grads))
    return out, lse


CASES = [  # batch, queries, keys, heads, kv heads, dim, window, sinks
    (1, 1, 1, 1, 1, 1, 1, 0), (2, 1, 7, 4, 2, 8, 3, 1), (3, 1, 300, 8, 2, 64, 100, 4), (2, 1, 1000, 8, 8, 128, 2000, 0),
    (1, 1, 513, 16, 1, 128, 64, 70), (2, 2, 129, 4, 1, 80, 33, 2), (1, 5, 64, 6, 2, 96, 1, 0), (2, 7, 500, 3, 3, 40, 200, 9),
    (1, 16, 16, 2, 1, 64, 16, 0), (2, 33, 33, 4, 2, 72, 9, 3), (1, 128, 128, 2, 2, 64, 128, 0), (1, 129, 129, 2, 1, 128, 50, 1),
    (2, 200, 200, 4, 2, 128, 1, 0), (1, 257, 257, 2, 2, 80, 1000, 0), (1, 300, 300, 3, 1, 56, 64, 130), (2, 100, 400, 4, 4, 128, 150, 5),
    (1, 70, 1000, 2, 1, 64, 333, 200), (1, 640, 640, 4, 1, 128, 200, 4), (2, 513, 513, 2, 1, 64, 129, 1), (1, 40, 10, 2, 1, 64, 7, 2),
    (1, 300, 100, 2, 2, 128, 40, 0), (1, 90, 90, 2, 1, 33, 20, 1), (1, 60, 60, 1, 1, 160, 30, 2), (1, 50, 90, 2, 1, 256, 64, 3),
    (1, 1, 200, 4, 1, 256, 100, 1), (1, 1, 200, 5, 1, 3, 100, 1), (1, 1500, 1500, 1, 1, 64, 1100, 3),
]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("b,lq,lk,h,hk,d,window,sinks", CASES)
def test_against_64_bits(ops, dev, t, b, lq, lk, h, hk, d, window, sinks):
    q, k, v, g = normal((b, lq, h, d), t, 1, dev), normal((b, lk, hk, d), t, 2, dev), normal((b, lk, hk, d), t, 3, dev), normal(
        (b, lq, h, d), t, 4, dev)
    check(ops, q, k, v, window, sinks, g=g)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("b,lq,lk,h,hk,d,window,sinks", [
    (1, 2000, 2000, 2, 1, 64, 130, 200),   # several tiles of sinks, whose far queries go to blocks of their own
    (2, 900, 900, 4, 4, 72, 100, 70), (1, 1100, 1300, 3, 1, 128, 64, 1), (40, 70, 70, 8, 4, 32, 20, 2),  # many blocks, few blocks
    (1, 9, 2000, 4, 2, 64, 500, 3), (1, 600, 600, 2, 1, 200, 90, 40),
])
def test_more_shapes(ops, dev, t, b, lq, lk, h, hk, d, window, sinks):
    q, k, v, g = normal((b, lq, h, d), t, 41, dev), normal((b, lk, hk, d), t, 42, dev), normal((b, lk, hk, d), t, 43, dev), normal(
        (b, lq, h, d), t, 44, dev)
    check(ops, q, k, v, window, sinks, g=g)
    kn = torch.tensor([lk - 7 * i % lk for i in range(b)], device=dev)
    check(ops, q, k, v, window, sinks, kn=kn, g=g)


def test_two_streams(ops, dev):
    """Calls of different sizes that run side by side on two streams, each with a workspace of its own."""
    work = []
    for n, (lq, lk, d) in enumerate(((700, 700, 128), (1, 900, 64), (300, 600, 64))):
        q, k, v, g = normal((2, lq, 4, d), BF16, 50 + n, dev), normal((2, lk, 2, d), BF16, 60 + n, dev), normal(
            (2, lk, 2, d), BF16, 70 + n, dev), normal((2, lq, 4, d), BF16, 80 + n, dev)
        out, lse = ops.window_attention(q, k, v, 200, 3)
        work.append((q, k, v, g, out, lse) + tuple(ops.window_attention_backward(g, q, k, v, out, lse, 200, 3)))
    torch.cuda.synchronize(dev)
    streams = [torch.cuda.Stream(dev), torch.cuda.Stream(dev)]
    spaces = [ops.Workspace(dev), ops.Workspace(dev)]
    got = []
    for turn in range(6):
        for s, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                q, k, v, g, *want = work[(turn + s) % 3]
                out, lse = ops.window_attention(q, k, v, 200, 3, workspace=spaces[s])
                got.append(((out, lse) + tuple(ops.window_attention_backward(g, q, k, v, out, lse, 200, 3, workspace=spaces[s])), want))
    torch.cuda.synchronize(dev)
    for have, want in got:
        assert all(torch.equal(x, y) for x, y in zip(have, want))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("lq,lk,d", [(1, 300, 64), (5, 300, 128), (130, 130, 80), (300, 300, 128), (90, 400, 64)])
def test_lengths(ops, dev, t, lq, lk, d):
    """Sequences of all lengths, empty ones and ones with more queries than keys; what lies behind the lengths is NaN and infinity."""
    b, h, hk = 7, 4, 2
    q, k, v, g = normal((b, lq, h, d), t, 5, dev), normal((b, lk, hk, d), t, 6, dev), normal((b, lk, hk, d), t, 7, dev), normal(
        (b, lq, h, d), t, 8, dev)
    kn = torch.tensor([lk, 1, 0, lk // 2, lk - 1, 2 * lk, -3], device=dev)
    qn = torch.tensor([lq, lq, lq, lq // 2, 0, 2 * lq, -1], device=dev)
    for kv, qs in ((kn, None), (kn.int(), qn), (None, qn.int())):
        k1, v1, q1, g1 = k.clone(), v.clone(), q.clone(), g.clone()
        for i in range(b):
            if kv is not None:
                end = max(0, min(lk, int(kv[i])))
                k1[i, end:], v1[i, end:] = math.nan, math.inf
            if qs is not None:
                end = max(0, min(lq, int(qs[i])))
                q1[i, end:], g1[i, end:] = math.inf, math.nan
        out, lse = check(ops, q1, k1, v1, 70, 3, qn=qs, kn=kv, g=g1)
        if kv is not None:
            assert (out[2] == 0).all() and (lse[2] == -math.inf).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("lq,d", [(1, 64), (6, 128), (200, 64), (200, 128)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_masked_places(ops, dev, t, lq, d, bad):
    """A NaN or an infinity in a key reaches the queries that see it and no other; in a query, itself and the keys it sees."""
    lk, h, hk, window, sinks = 200, 4, 2, 50, 2
    q, k, v, g = normal((1, lq, h, d), t, 9, dev), normal((1, lk, hk, d), t, 10, dev), normal((1, lk, hk, d), t, 11, dev), normal(
        (1, lq, h, d), t, 12, dev)
    out, lse = ops.window_attention(q, k, v, window, sinks)
    grads = ops.window_attention_backward(g, q, k, v, out, lse, window, sinks)
    seen = seen_by(1, lq, lk, window, sinks, torch.tensor([lq], device=dev), torch.tensor([lk], device=dev), dev)[0]
    at = 150 if lq > 1 else 120  # not seen by some (by any of a single token's) queries
    ref = Reference(q, k, v, window, sinks, g=g)
    for where in ("k", "v"):
        k1, v1 = k.clone(), v.clone()
        (k1 if where == "k" else v1)[0, at, 1, d // 2] = bad
        out1, lse1 = ops.window_attention(q, k1, v1, window, sinks)
        rows = ~seen[:, at]
        close("out", out1[:, rows], ref.out[:, rows], ref.out_bound[:, rows])
        close("out of the other head", out1[:, :, :2], ref.out[:, :, :2], ref.out_bound[:, :, :2])
        if where == "v" and seen[:, at].any():
            assert not torch.isfinite(out1[0, seen[:, at], 2:, d // 2]).any()
        gq, gk, gv = ops.window_attention_backward(g, q, k1, v1, out1, lse1, window, sinks)
        close("gradQ", gq[:, rows], ref.gq[:, rows], ref.gq_bound[:, rows])
        apart = ~(seen[seen[:, at]].any(0))  # keys that share no query with it
        close("gradK", gk[:, apart], ref.gk[:, apart], ref.gk_bound[:, apart])
        close("gradV", gv[:, apart], ref.gv[:, apart], ref.gv_bound[:, apart])
    if lq == lk:
        q1 = q.clone()
        q1[0, at, 3, 0] = bad
        out1, lse1 = ops.window_attention(q1, k, v, window, sinks)
        gq, gk, gv = ops.window_attention_backward(g, q1, k, v, out1, lse1, window, sinks)
        rows = torch.arange(lq, device=dev) != at
        close("out", out1[:, rows], ref.out[:, rows], ref.out_bound[:, rows])
        close("gradQ", gq[:, rows], ref.gq[:, rows], ref.gq_bound[:, rows])
        close("gradK", gk[:, ~seen[at]], ref.gk[:, ~seen[at]], ref.gk_bound[:, ~seen[at]])
        close("gradV", gv[:, ~seen[at]], ref.gv[:, ~seen[at]], ref.gv_bound[:, ~seen[at]])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
@pytest.mark.parametrize("lq", [1, 150])
def test_scales(ops, dev, t, scale, lq):
    """No scale at all (equal weights), a negative one, and scores of +-100, where one key takes nearly all of the weight."""
    q, k, v, g = normal((1, lq, 2, 64), t, 13, dev), normal((1, 150, 1, 64), t, 14, dev), normal((1, 150, 1, 64), t, 15, dev), normal(
        (1, lq, 2, 64), t, 16, dev)
    check(ops, q, k, v, 70, 2, scale, g=g)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("d", [40, 128, 136])
@pytest.mark.parametrize("sinks,window", [(1, 5), (31, 33), (63, 64), (64, 65), (65, 1), (130, 100), (300, 7)])
def test_sinks_at_the_ends_of_steps(ops, dev, t, d, sinks, window):
    q, g = normal((1, 190, 4, d), t, 111, dev), normal((1, 190, 4, d), t, 114, dev)
    k, v = normal((1, 333, 2, d), t, 112, dev), normal((1, 333, 2, d), t, 113, dev)
    check(ops, q, k, v, window, sinks, g=g)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("lq,lk,h,hk,d,window,sinks", [
    (1, 9000, 4, 1, 128, 10 ** 6, 0), (1, 5000, 2, 2, 64, 4000, 5), (5, 3001, 6, 2, 80, 10 ** 6, 0), (8, 2500, 8, 1, 40, 2100, 70),
    (2, 700, 2, 1, 64, 600, 33), (16, 6000, 4, 1, 128, 10 ** 6, 0)])
def test_few_blocks(ops, dev, t, lq, lk, h, hk, d, window, sinks):
    """So few that they take twice the warps; the sequence ends inside a step, and what lies behind it says nothing."""
    q = normal((1, lq, h, d), t, 141, dev)
    k, v = normal((1, lk, hk, d), t, 142, dev), normal((1, lk, hk, d), t, 143, dev)
    check(ops, q, k, v, window, sinks)
    n = torch.tensor([lk - 61], device=dev)
    want = Reference(q, k, v, window, sinks, kn=n)
    k, v = k.clone(), v.clone()
    k[:, lk - 61:], v[:, lk - 61:] = math.nan, math.inf
    got, lse = ops.window_attention(q, k, v, window, sinks, kv_lengths=n)
    close("out", got, want.out, want.out_bound)
    close_lse(lse, want)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("lq,lk,h,hk,d,window,sinks", [
    (9, 1024, 4, 2, 64, 10 ** 6, 0), (17, 1500, 8, 1, 128, 2000, 3), (33, 3001, 6, 2, 80, 1100, 40), (100, 1111, 3, 3, 40, 990, 130),
    (150, 2500, 2, 1, 128, 1000, 0), (300, 2000, 2, 1, 96, 1500, 1700), (16, 1300, 4, 1, 200, 1290, 5), (70, 1800, 2, 2, 256, 5000, 0)])
def test_some_queries_over_many_keys(ops, dev, t, lq, lk, h, hk, d, window, sinks):
    b = 3
    q, g = normal((b, lq, h, d), t, 131, dev), normal((b, lq, h, d), t, 134, dev)
    k, v = normal((b, lk, hk, d), t, 132, dev), normal((b, lk, hk, d), t, 133, dev)
    check(ops, q, k, v, window, sinks, g=g)
    qn, kn = torch.tensor([lq, lq // 2, lq], device=dev), torch.tensor([lk, lk - 7, lq - 3], device=dev)
    check(ops, q, k, v, window, sinks, qn=qn, kn=kn, g=g)
    wide = torch.full((b, lk + 50, hk, d), math.nan, dtype=t, device=dev)  # keys behind the sequences hold anything
    wide_v = wide.clone()
    wide[:, :lk], wide_v[:, :lk] = k, v
    got = ops.window_attention(q, wide, wide_v, window, sinks, kv_lengths=torch.full((b,), lk, device=dev))[0]
    ref = Reference(q, k, v, window, sinks)
    close("out", got, ref.out, ref.out_bound)


@pytest.mark.parametrize("t,d", [(F32, 64), (BF16, 64), (F16, 40)])
@pytest.mark.parametrize("b,hk,lq,sinks", [(32, 4, 700, 700), (24, 4, 1300, 600), (2, 2, 1500, 10 ** 9)])
def test_sinks_of_many_tiles(ops, dev, t, d, b, hk, lq, sinks):
    q, g = normal((b, lq, hk, d), t, 121, dev), normal((b, lq, hk, d), t, 124, dev)
    k, v = normal((b, lq, hk, d), t, 122, dev), normal((b, lq, hk, d), t, 123, dev)
    check(ops, q, k, v, 40, sinks, g=g)


@pytest.mark.parametrize("lq", [1, 140])
def test_fp16_gradients_of_any_size(ops, dev, lq):
    """Gradients a million times smaller or a thousand times larger (and values of 1000) keep their precision in fp16."""
    q, k = normal((1, lq, 2, 64), F16, 17, dev), normal((1, 140, 1, 64), F16, 18, dev)
    for spread, values in ((2.0 ** -14, 1.0), (2.0 ** -10, 1000.0), (4.0, 1.0)):
        v, g = normal((1, 140, 1, 64), F16, 19, dev, values), normal((1, lq, 2, 64), F16, 20, dev, spread)
        check(ops, q, k, v, 60, 1, g=g)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("lq,d", [(1, 64), (4, 80), (140, 128), (140, 72)])
def test_views(ops, dev, t, lq, d):
    """Heads of a fused product, heads in front of tokens, odd offsets, steps in the last dimension, shared (broadcast) keys."""
    lk, h, hk = 140, 4, 2
    fused = normal((2, lk, h + 2 * hk, d), t, 21, dev)
    q, k, v = fused[:, lk - lq:, :h], fused[:, :, h:h + hk], fused[:, :, h + hk:]
    g = normal((2, h, lq, d), t, 22, dev).transpose(1, 2)
    check(ops, q, k, v, 60, 2, g=g)
    check(ops, q, k.transpose(1, 2).contiguous().transpose(1, 2), v, 60, 2, g=g)
    odd = torch.zeros(2 * lk * hk * d + 1, dtype=t, device=dev)[1:].view(2, lk, hk, d)
    odd.copy_(k)
    check(ops, q, odd, v, 60, 2, g=g)
    steps = torch.zeros(2, lk, hk, 2 * d, dtype=t, device=dev)[..., ::2]
    steps.copy_(v)
    check(ops, q, k, steps, 60, 2, g=g)
    check(ops, q, k[:1].expand(2, lk, hk, d), v[:, :1].expand(2, lk, hk, d), 60, 2, g=g)
    out = torch.zeros(2, h, lq, d, dtype=t, device=dev).transpose(1, 2)
    want, lse = ops.window_attention(q, k, v, 60, 2)
    ops.window_attention(q, k, v, 60, 2, out=out)
    assert torch.equal(out, want)
    gk = torch.zeros(2, lk, h + 2 * hk, d, dtype=t, device=dev)
    grads = ops.window_attention_backward(g, q, k, v, want, lse, 60, 2)
    ops.window_attention_backward(g, q, k, v, want, lse, 60, 2, grad_q=torch.zeros_like(q), grad_k=gk[:, :, h:h + hk],
                                  grad_v=gk[:, :, h + hk:])
    assert torch.equal(gk[:, :, h:h + hk], grads[1]) and torch.equal(gk[:, :, h + hk:], grads[2]) and (gk[:, :, :h] == 0).all()


def test_long_cache_past_32_bits(ops, dev):
    """Keys behind 2^31 elements of a cache, of which the window and the sinks are read."""
    lk, d = 2 ** 24 + 77, 128  # 2^31 + elements, 4.3 GB each
    k, v = torch.empty(1, lk, 1, d, dtype=BF16, device=dev), torch.empty(1, lk, 1, d, dtype=BF16, device=dev)
    window, sinks = 300, 4
    near, first = slice(lk - 400, lk), slice(0, sinks)
    for x, seed in ((k, 23), (v, 24)):
        x[:, near] = normal((1, 400, 1, d), BF16, seed, dev)
        x[:, first] = normal((1, sinks, 1, d), BF16, seed + 10, dev)
    for lq in (1, 40):
        q = normal((1, lq, 4, d), BF16, 25, dev)
        out, lse = ops.window_attention(q, k, v, window, sinks)
        k1, v1 = (torch.cat((x[:, first], x[:, near]), 1) for x in (k, v))
        ref = Reference(q, k1, v1, window, sinks)  # the same keys but for the gap, which no query sees
        close("out", out, ref.out, ref.out_bound)
        close_lse(lse, ref)


def test_backward_against_differences(ops, dev):
    q, k, v, g = (normal(shape, F32, seed, dev).double() for shape, seed in (((1, 6, 2, 8), 26), ((1, 9, 1, 8), 27), ((1, 9, 1, 8), 28),
                                                                           ((1, 6, 2, 8), 29)))

    def loss(q, k, v):
        return (Reference(q, k, v, 4, 2).out * g).sum().item()

    out, lse = ops.window_attention(q.float(), k.float(), v.float(), 4, 2)
    grads = ops.window_attention_backward(g.float(), q.float(), k.float(), v.float(), out, lse, 4, 2)
    h = 1e-5
    for n, x in enumerate((q, k, v)):
        for i in range(0, x.numel(), 7):
            d = torch.zeros(x.numel(), dtype=torch.float64, device=dev)
            d[i] = h
            up, down = [q, k, v], [q, k, v]
            up[n], down[n] = x + d.view_as(x), x - d.view_as(x)
            diff = (loss(*up) - loss(*down)) / (2 * h)
            assert abs(diff - grads[n].reshape(-1)[i].item()) < 2e-5 * max(1.0, abs(diff))


def test_empty(ops, dev):
    q, k = torch.randn(2, 3, 4, 16, device=dev), torch.randn(2, 0, 2, 16, device=dev)
    out, lse = ops.window_attention(q, k, k, 5, 1)
    assert (out == 0).all() and (lse == -math.inf).all()
    gq, gk, gv = ops.window_attention_backward(q, q, k, k, out, lse, 5, 1)
    assert (gq == 0).all() and gk.shape == k.shape
    k = torch.randn(2, 6, 2, 16, device=dev)
    out, lse = ops.window_attention(q[:, :0], k, k, 5, 1)
    assert out.shape == (2, 0, 4, 16)
    gq, gk, gv = ops.window_attention_backward(out, out, k, k, out, lse, 5, 1, grad_k=torch.ones_like(k))
    assert (gk == 0).all() and (gv == 0).all()


def test_without_lse(ops, dev):
    """The C entry point takes a null lse."""
    import ctypes
    for lq in (1, 200):
        q, k = normal((1, lq, 2, 64), BF16, 30, dev), normal((1, 200, 1, 64), BF16, 31, dev)
        want, _ = ops.window_attention(q, k, k, 50, 1)
        out = torch.zeros_like(q)
        tq, tk, to = (ops.acl_tensor(x, "ND") for x in (q, k, out))
        ops.lib().opscvVersion()
        ops.two_phase("aclnnWindowAttention", [tq.ptr, tk.ptr, tk.ptr, None, None, 50, 1, ctypes.c_double(0.125), to.ptr, None], q.device)
        assert torch.equal(out, want)


@pytest.mark.parametrize("lq", [1, 150])
def test_graph_and_stream(ops, dev, lq):
    q, k, v, g = normal((2, lq, 4, 64), BF16, 32, dev), normal((2, 150, 2, 64), BF16, 33, dev), normal((2, 150, 2, 64), BF16, 34, dev), normal(
        (2, lq, 4, 64), BF16, 35, dev)
    kn = torch.tensor([150, 150], device=dev)

    def step():
        out, lse = ops.window_attention(q, k, v, 60, 2, kv_lengths=kn)
        return (out, lse) + ops.window_attention_backward(g, q, k, v, out, lse, 60, 2, kv_lengths=kn)

    want = step()
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream(dev).wait_stream(side)
    torch.cuda.synchronize(dev)
    assert all(torch.equal(x, y) for x, y in zip(other, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed, lengths in ((40, (150, 20)), (50, (3, 100))):  # lengths are read when the graph runs
        for n, x in enumerate((q, k, v, g)):
            x.copy_(normal(x.shape, BF16, seed + n, dev))
        kn.copy_(torch.tensor(lengths))
        graph.replay()
        torch.cuda.synchronize(dev)
        assert all(torch.equal(x, y) for x, y in zip(got, step()))


def test_no_wait_ran_out(ops, dev):
    """After all of the above: the bounded waits inside the kernels have all ended by themselves."""
    q, k = normal((1, 700, 2, 64), BF16, 70, dev), normal((1, 700, 1, 64), BF16, 71, dev)
    out, lse = ops.window_attention(q, k, k, 100, 2)
    ops.window_attention_backward(q, q, k, k, out, lse, 100, 2)
    torch.cuda.synchronize(dev)
    assert ops.async_copy_timeouts() == 0


def test_block_of_a_model(ops, dev):
    """Norm, projections, rotary positions, attention and the way back, as a block of a model strings them together, against 64 bits."""
    b, n, h, hk, d, width, window, sinks = 2, 150, 4, 2, 64, 256, 40, 2
    x, r = normal((b, n, width), F32, 60, dev), normal((b, n, width), F32, 61, dev)
    w = normal((width,), F32, 62, dev, 0.1) + 1
    proj = normal(((h + 2 * hk) * d, width), F32, 63, dev, 0.05)
    f = ops.rotary_frequencies(d, device=dev)
    p = torch.arange(n, device=dev)
    g = normal((b, n, h, d), F32, 64, dev)

    y, total, rstd = ops.residual_rms_norm(x, r, w)
    qkv = (y @ proj.t()).view(b, n, h + 2 * hk, d)
    q, k = ops.rotary_embedding(qkv[:, :, :h], qkv[:, :, h:h + hk], p, f)
    v = qkv[:, :, h + hk:]
    out, lse = ops.window_attention(q, k, v, window, sinks)
    gq, gk, gv = ops.window_attention_backward(g, q, k, v, out, lse, window, sinks)
    gq, gk = ops.rotary_embedding_backward(gq, gk, p, f)
    g_qkv = torch.cat((gq, gk, gv), 2).view(b, n, -1)
    gx, gw = ops.residual_rms_norm_backward(g_qkv @ proj, total, rstd, w)

    with torch.enable_grad():
        x6, w6 = x.double().requires_grad_(), w.double().requires_grad_()
        z = x6 + r.double()
        y6 = z * torch.rsqrt(z.square().mean(-1, keepdim=True) + 1e-6) * w6
        qkv6 = (y6 @ proj.double().t()).view(b, n, h + 2 * hk, d)
        angle = (p.double()[:, None] * f.double())[None, :, None]

        def turn(a):
            a, c = a.chunk(2, -1)
            return torch.cat((a * angle.cos() - c * angle.sin(), c * angle.cos() + a * angle.sin()), -1)

        q6, k6, v6 = turn(qkv6[:, :, :h]), turn(qkv6[:, :, h:h + hk]), qkv6[:, :, h + hk:]
        k6, v6 = k6.repeat_interleave(h // hk, 2), v6.repeat_interleave(h // hk, 2)
        seen = seen_by(1, n, n, window, sinks, torch.tensor([n], device=dev), torch.tensor([n], device=dev), dev)
        s = torch.einsum("bihd,bjhd->bhij", q6, k6) / math.sqrt(d)
        o6 = torch.einsum("bhij,bjhd->bihd", torch.softmax(s.masked_fill(~seen, -math.inf), -1), v6)
        want_x, want_w = torch.autograd.grad((o6 * g.double()).sum(), (x6, w6))
    # a chain of fp32 steps with sums of at most 256 terms: 2^-12 of the largest value is 2^12 half steps of slack
    for got, want in ((out, o6.detach()), (gx, want_x), (gw, want_w)):
        assert (got.double() - want).abs().max() < 2.0 ** -12 * want.abs().max()


@pytest.mark.parametrize("t", [F16, BF16])
@pytest.mark.parametrize("d", [8, 16, 24, 32, 48, 64, 80, 88, 96, 104, 112, 120, 128])
def test_heads_of_every_number_of_steps(ops, dev, t, d):
    q, g = normal((2, 140, 4, d), t, 151, dev), normal((2, 140, 4, d), t, 154, dev)
    k, v = normal((2, 200, 2, d), t, 152, dev), normal((2, 200, 2, d), t, 153, dev)
    check(ops, q, k, v, 70, 3, g=g)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("lq,lk,h,hk,d,window,sinks", [
    (200, 300, 4, 2, 64, 150, 3), (300, 300, 4, 2, 128, 150, 3), (5, 300, 4, 2, 64, 150, 3), (130, 300, 4, 2, 80, 150, 0), (1, 700, 4, 1, 128, 600, 2),
    (400, 400, 2, 1, 128, 1000, 0), (257, 257, 6, 2, 96, 20, 200), (700, 700, 2, 2, 64, 40, 140), (64, 64, 2, 1, 40, 10, 1), (150, 150, 2, 1, 200, 70, 3)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_padding_costs_nothing(ops, dev, t, lq, lk, h, hk, d, window, sinks, bad):
    """What lies behind the sequences' lengths changes no bit of the results: no row is formed again on its account."""
    b = 5
    q, k, v, g = normal((b, lq, h, d), t, 161, dev), normal((b, lk, hk, d), t, 162, dev), normal((b, lk, hk, d), t, 163, dev), normal(
        (b, lq, h, d), t, 164, dev)
    kn = torch.tensor([lk, lk - 1, lk - lk // 3, max(1, lk - 129), 1], device=dev)
    qn = torch.tensor([lq, max(1, lq - 1), lq - lq // 3, max(1, lq - 129), 1], device=dev)
    same = torch.minimum(kn, qn)

    def padded(x, n, value):
        x = x.clone()
        for i in range(b):
            x[i, int(n[i]):] = value
        return x

    for qs, ks in ((qn, kn), (None, kn), (qn, None), (same, same)):
        results = []
        for value in (0.0, bad):
            q1, g1 = (padded(x, qs, value) if qs is not None else x for x in (q, g))
            k1, v1 = (padded(x, ks, value) if ks is not None else x for x in (k, v))
            out, lse = ops.window_attention(q1, k1, v1, window, sinks, q_lengths=qs, kv_lengths=ks)
            results.append((out, lse) + tuple(ops.window_attention_backward(g1, q1, k1, v1, out, lse, window, sinks, q_lengths=qs, kv_lengths=ks)))
        for name, x, y in zip(("out", "lse", "gradQ", "gradK", "gradV"), *results):
            assert torch.isfinite(y if name != "lse" else y.nan_to_num(neginf=0.0)).all() and torch.equal(x, y), name
