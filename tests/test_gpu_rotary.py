"""Rotary positions against the formula in 64 bits. A stored value is off by at most half a step of its type; before that, the fp32 turn
is off by the roundings of the reduced angle (2 pi 2^-26), of sine and cosine (2 steps), of scale, the products and their sum."""
import math
from fractions import Fraction

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def turn64(x, positions, f, interleaved, sections, scale, sign=1.0):
    half = f.numel()
    p = positions.double()
    if sections is not None:
        angle = torch.cat([p[i].unsqueeze(-1).expand(*p.shape[1:], n) for i, n in enumerate(sections)], -1) * f.double()
    else:
        angle = p.unsqueeze(-1) * f.double()
    c, s = angle.cos().unsqueeze(-2) * scale, sign * angle.sin().unsqueeze(-2) * scale
    x = x.double()
    z = x[..., :2 * half]
    a, b = (z[..., 0::2], z[..., 1::2]) if interleaved else (z[..., :half], z[..., half:])
    u, v, size = a * c - b * s, b * c + a * s, (a.abs() + b.abs()) * abs(scale)
    if interleaved:
        u, size = torch.stack((u, v), -1).flatten(-2), torch.stack((size, size), -1).flatten(-2)
    else:
        u, size = torch.cat((u, v), -1), torch.cat((size, size), -1)
    rest = x[..., 2 * half:]
    return torch.cat((u, rest), -1), torch.cat((size, torch.zeros_like(rest)), -1)


def check(got, x, *how):
    want, size = turn64(x, *how)
    assert got.shape == x.shape and got.dtype == x.dtype
    bound = torch.finfo(x.dtype).eps / 2 * want.abs() + (2 * math.pi * 2.0 ** -26 + 8 * 2.0 ** -24) * size + torch.finfo(x.dtype).tiny
    over = (got.double() - want).abs() - bound
    assert (over <= 0).all(), over.max().item()
    half = how[1].numel()
    assert torch.equal(got[..., 2 * half:], x[..., 2 * half:])


def frequencies(half, dev, t=torch.float32):
    return (10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)).to(t).to(dev)


def normal(shape, t, seed, dev):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(t).to(dev)


CASES = [  # batch, length, heads, kv heads, dim, half, interleaved
    (1, 1, 1, 1, 2, 1, False), (1, 1, 1, 1, 2, 1, True), (2, 1, 32, 8, 128, 64, False), (3, 37, 4, 2, 64, 32, True),
    (1, 300, 3, 1, 80, 40, False), (2, 19, 5, 5, 72, 36, True), (1, 50, 2, 1, 96, 24, False), (1, 50, 2, 1, 96, 24, True),
    (2, 13, 3, 2, 35, 5, False), (2, 13, 3, 2, 35, 5, True), (1, 7, 2, 1, 33, 16, True), (1, 2000, 8, 2, 128, 64, False),
    (1, 3, 1, 1, 4096, 2048, False), (1, 5, 130, 7, 256, 17, True),
]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("b,n,h,hk,d,half,interleaved", CASES)
def test_turns(ops, dev, t, b, n, h, hk, d, half, interleaved):
    q, k = normal((b, n, h, d), t, 1, dev), normal((b, n, hk, d), t, 2, dev)
    f = frequencies(half, dev)
    p = torch.randint(-50, 200000, (b, n), generator=torch.Generator().manual_seed(3)).to(dev)
    for scale in (1.0, 1.25):
        how = (p, f, interleaved, None, scale)
        q1, k1 = ops.rotary_embedding(q, k, p, f, interleaved, scale=scale)
        check(q1, q, *how)
        check(k1, k, *how)
        gq, gk = ops.rotary_embedding_backward(q, k, p, f, interleaved, scale=scale)
        check(gq, q, *how, -1.0)
        check(gk, k, *how, -1.0)
    alone, none = ops.rotary_embedding(q, None, p.int(), f.double(), interleaved, scale=1.25)
    assert none is None and torch.equal(alone, q1)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("sections", [(16,), (8, 8), (6, 5, 5), (0, 16, 0, 0), (1, 2, 3, 10)])
def test_axes(ops, dev, sections, interleaved):
    q, k = normal((2, 21, 3, 40), torch.float16, 4, dev), normal((2, 21, 1, 40), torch.float16, 5, dev)
    f = frequencies(16, dev)
    p = torch.randint(0, 5000, (len(sections), 2, 21), generator=torch.Generator().manual_seed(6)).to(dev)
    q1, k1 = ops.rotary_embedding(q, k, p, f, interleaved, sections)
    check(q1, q, p, f, interleaved, sections, 1.0)
    check(k1, k, p, f, interleaved, sections, 1.0)


def test_far_positions(ops, dev):
    """Angles keep their value at positions up to 10^12, where one double is off by 10^-4: held against exact rationals."""
    q = normal((1, 6, 2, 64), torch.float32, 7, dev)
    f = frequencies(32, dev)
    p = [0, 2 ** 24 + 1, 2 ** 31 - 1, 2 ** 31 + 7, 10 ** 12, -10 ** 12]
    two_pi = 2 * Fraction("3.14159265358979323846264338327950288419716939937510")
    exact = torch.tensor([[float(n * Fraction(v) % two_pi) for v in f.tolist()] for n in p], dtype=torch.float64, device=dev)
    got = ops.rotary_embedding(q, None, torch.tensor([p], device=dev), f)[0]
    for i in range(len(p)):  # the reduced angles as frequencies of position 1
        check(got[:, i:i + 1], q[:, i:i + 1], torch.ones(1, 1, device=dev), exact[i], False, None, 1.0)


def test_backward_is_the_gradient(ops, dev):
    """The turn is linear: <turn(x), g> = <x, back(g)> for all x and g."""
    q, g = normal((2, 9, 3, 24), torch.float32, 8, dev), normal((2, 9, 3, 24), torch.float32, 9, dev)
    f = frequencies(8, dev)
    p = torch.arange(9, device=dev) * 1000
    turned, _ = ops.rotary_embedding(q, None, p, f, scale=1.5)
    back, _ = ops.rotary_embedding_backward(g, None, p, f, scale=1.5)
    left, right = (turned.double() * g.double()).sum(), (q.double() * back.double()).sum()
    assert abs(left - right) < 16 * 2.0 ** -24 * 1.5 * (q.double().abs() * g.double().abs()).sum() * 2


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_views(ops, dev, t, interleaved):
    f = frequencies(16, dev)
    p = torch.arange(11, device=dev) + 77
    qkv = normal((3, 11, 8, 48), t, 10, dev)
    q, k = qkv[:, :, :5], qkv[:, :, 5:7]
    want = ops.rotary_embedding(q.contiguous(), k.contiguous(), p, f, interleaved)
    got = ops.rotary_embedding(q, k, p, f, interleaved)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # heads in front of tokens, as inputs and outputs
    out = torch.zeros(3, 5, 11, 48, dtype=t, device=dev).transpose(1, 2)
    ops.rotary_embedding(q.transpose(1, 2).contiguous().transpose(1, 2), k, p, f, interleaved, q_out=out)
    assert torch.equal(out, want[0])
    # an odd offset, a strided last dimension, positions in steps
    odd = torch.zeros(3 * 11 * 5 * 48 + 1, dtype=t, device=dev)[1:].view(3, 11, 5, 48)
    odd.copy_(q)
    assert torch.equal(ops.rotary_embedding(odd, None, p, f, interleaved)[0], want[0])
    spread = torch.zeros(3, 11, 5, 96, dtype=t, device=dev)[..., ::2]
    spread.copy_(q)
    assert torch.equal(ops.rotary_embedding(spread, None, torch.stack((p, p), -1)[:, 0], f, interleaved, q_out=spread)[0], want[0])
    # in place, the values around untouched
    whole = qkv.clone()
    ops.rotary_embedding(whole[:, :, :5], whole[:, :, 5:7], p, f, interleaved, q_out=whole[:, :, :5], k_out=whole[:, :, 5:7])
    assert torch.equal(whole[:, :, :5], want[0]) and torch.equal(whole[:, :, 5:7], want[1]) and torch.equal(whole[:, :, 7:], qkv[:, :, 7:])


def test_offsets_past_32_bits(ops, dev):
    far = torch.empty(2, 2 ** 31 + 64, dtype=torch.bfloat16, device=dev)
    q = far[:, :64].unsqueeze(1)
    q.copy_(normal((2, 1, 64), torch.bfloat16, 11, dev))
    f, p = frequencies(32, dev), torch.tensor([3, 90], device=dev)
    want, _ = ops.rotary_embedding(q.contiguous(), None, p, f)
    assert torch.equal(ops.rotary_embedding(q, None, p, f, q_out=q)[0], want)


def test_empty(ops, dev):
    f = frequencies(4, dev)
    q, k = torch.zeros(2, 0, 3, 8, device=dev), torch.zeros(2, 0, 1, 8, device=dev)
    assert ops.rotary_embedding(q, k, torch.zeros(2, 0, dtype=torch.int64, device=dev), f)[0].shape == q.shape
    q, k = torch.randn(2, 5, 0, 8, device=dev), torch.randn(2, 5, 1, 8, device=dev)
    p = torch.arange(5, device=dev)
    q1, k1 = ops.rotary_embedding(q, k, p, f)
    check(k1, k, p.expand(2, 5), f, False, None, 1.0)


def test_graph(ops, dev):
    q, k = normal((2, 30, 4, 64), torch.bfloat16, 12, dev), normal((2, 30, 2, 64), torch.bfloat16, 13, dev)
    f, p = frequencies(32, dev), torch.arange(30, device=dev).expand(2, 30).contiguous()
    ops.rotary_embedding(q, k, p, f)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.rotary_embedding(q, k, p, f)
    p += 1000
    q.copy_(normal((2, 30, 4, 64), torch.bfloat16, 14, dev))
    graph.replay()
    check(out[0], q, p, f, False, None, 1.0)
    check(out[1], k, p, f, False, None, 1.0)


def reference_frequencies(half, base, scaling, factor, length, low, high):
    if scaling == "base":
        base = base * factor ** (half / (half - 1))
    f = torch.tensor([base ** (-i / half) for i in range(half)], dtype=torch.float64)
    if scaling == "linear":
        return f / factor
    if scaling == "wavelength":
        times = length * f / (2 * math.pi)
        keep = ((times - low) / (high - low)).clamp(0, 1)
        return f * keep + f / factor * (1 - keep)
    if scaling == "ramp":
        a = max(0.0, math.floor(half * math.log(length / (high * 2 * math.pi)) / math.log(base)))
        b = min(2 * half - 1.0, math.ceil(half * math.log(length / (low * 2 * math.pi)) / math.log(base)))
        stretch = ((torch.arange(half, dtype=torch.float64) - a) / (max(b, a + 0.001) - a)).clamp(0, 1)
        return f * (1 - stretch) + f / factor * stretch
    return f


@pytest.mark.parametrize("scaling", [None, "linear", "base", "wavelength", "ramp"])
@pytest.mark.parametrize("half,base", [(64, 10000.0), (32, 500000.0), (20, 1000.0)])
def test_frequencies(ops, dev, scaling, half, base):
    how = dict(factor=8.0, original_length=8192.0, low=1.0, high=32.0 if scaling == "ramp" else 4.0)
    want = reference_frequencies(half, base, scaling, how["factor"], how["original_length"], how["low"], how["high"])
    got = ops.rotary_frequencies(2 * half, base, scaling, dtype=torch.float64, device=dev, **how).cpu()
    assert ((got - want).abs() <= 1e-14 * want).all()
    got = ops.rotary_frequencies(2 * half, base, scaling, device=dev, **how).cpu()
    assert ((got.double() - want).abs() <= (2.0 ** -24 + 1e-14) * want).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("d", [33, 40, 48, 56, 72, 100, 136])
@pytest.mark.parametrize("interleaved", [False, True])
def test_values_behind_the_pairs_are_copied(ops, dev, t, d, interleaved):
    q, k = normal((2, 19, 5, d), t, 21, dev), normal((2, 19, 2, d), t, 22, dev)
    f, p = frequencies(16, dev), torch.arange(19, device=dev) + 300
    whole = ops.rotary_embedding(q[..., :32].contiguous(), k[..., :32].contiguous(), p.expand(2, 19), f, interleaved)
    into = q.clone(), k.clone()
    for got in (ops.rotary_embedding(q, k, p.expand(2, 19), f, interleaved),
                ops.rotary_embedding(*into, p.expand(2, 19), f, interleaved, q_out=into[0], k_out=into[1])):
        for x, y, w in zip((q, k), got, whole):
            assert torch.equal(y[..., 32:], x[..., 32:]) and torch.equal(y[..., :32], w)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_positions_that_broadcast(ops, dev, t, kind):
    """Stride 0 along any of the leading dimensions, between others too, with and without axes; views of q that need copies as well."""
    q, k = normal((2, 3, 5, 4, 24), t, 23, dev), normal((2, 3, 5, 2, 24), t, 24, dev)
    f = frequencies(8, dev)
    whole = torch.randint(0, 9000, (3, 2, 3, 5), generator=torch.Generator().manual_seed(25)).to(kind).to(dev)
    for cut in ((0, 0, 0), (1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (1, 1, 0), (0, 1, 1), (1, 1, 1)):
        p = whole[(slice(None), *(slice(0, 1) if c else slice(None) for c in cut))].contiguous().expand(3, 2, 3, 5)
        full = p.contiguous()
        for at, flat, sections in ((p[0], full[0], None), (p, full, (3, 4, 1)), (p[:1], full[:1], (8,))):
            want = ops.rotary_embedding(q, k, flat, f, sections=sections)
            check(want[0], q, flat, f, False, sections, 1.0)
            got = ops.rotary_embedding(q, k, at, f, sections=sections)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
            apart = torch.zeros(2, 4, 3, 6, 4, 24, dtype=t, device=dev)[:, ::2, :, 1:].transpose(1, 2)[:, :, 0]
            apart.copy_(q)
            assert torch.equal(ops.rotary_embedding(apart, k, at, f, sections=sections, q_out=apart)[0], want[0])
            back = ops.rotary_embedding_backward(q, k, at, f, sections=sections)
            assert torch.equal(back[0], ops.rotary_embedding_backward(q, k, flat, f, sections=sections)[0])


def test_axes_of_a_table_for_all_sequences(ops, dev):
    q, k = normal((4, 9, 3, 40), torch.float16, 26, dev), normal((4, 9, 1, 40), torch.float16, 27, dev)
    f, sections = frequencies(16, dev), (6, 5, 5)
    p = torch.randint(0, 5000, (3, 9), generator=torch.Generator().manual_seed(28)).to(dev)
    full = p[:, None].expand(3, 4, 9).contiguous()
    want = ops.rotary_embedding(q, k, full, f, sections=sections)
    for at in (p, p[:, None]):
        got = ops.rotary_embedding(q, k, at, f, sections=sections)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    check(want[0], q, full, f, False, sections, 1.0)


@pytest.mark.parametrize("half", [4, 64])
def test_ramp_without_frequencies_between(ops, dev, half):
    """Contexts so short that every frequency turns far less than `low` times are divided throughout, so long that all turn more than `high`
    times are left as they are; where both bounds fall on one index, it stays."""
    plain = ops.rotary_frequencies(2 * half, 10000.0, dtype=torch.float64, device=dev)
    but_first = torch.cat((plain[:1], plain[1:] / 8))
    for length, low, high in ((2.0, 1.0, 32.0), (6.0, 1.0, 2.0), (0.5, 1.0, 4.0), (1e12, 1.0, 32.0)):
        last = math.ceil(half * math.log(length / (low * 2 * math.pi)) / math.log(10000.0))  # an index in (-1, 0) is rounded outwards to 0
        want = plain / 8 if last < 0 else but_first if last == 0 else plain
        got = ops.rotary_frequencies(2 * half, 10000.0, "ramp", 8.0, length, low, high, torch.float64, dev)
        assert ((got - want).abs() <= 1e-14 * want).all()
    got = ops.rotary_frequencies(2 * half, 10000.0, "ramp", 8.0, 2 * math.pi * 1.5, 1.5, 1.5 + 1e-13, torch.float64, dev)
    assert ((got[1:] - plain[1:] / 8).abs() <= 1e-14 * plain[1:]).all()


@pytest.mark.parametrize("axes", [1, 2, 4])
def test_positions_of_many_dimensions_that_broadcast(ops, dev, axes):
    """Strided dimensions with broadcast ones in front, between and behind, for each axis."""
    lead, f = (2, 3, 2, 5, 3), frequencies(8, dev)
    q, k = normal((*lead, 3, 20), torch.bfloat16, 31, dev), normal((*lead, 1, 20), torch.bfloat16, 32, dev)
    sections = (8,) if axes == 1 else (5, 3) if axes == 2 else (1, 2, 0, 5)
    for n, shape in enumerate(((2, 1, 2, 1, 3), (1, 3, 1, 5, 1), (2, 1, 2, 1, 1), (1, 1, 2, 1, 3), (2, 3, 1, 5, 3), (1, 3, 1, 1, 3), (2, 1, 1, 5, 1))):
        p = torch.randint(0, 9000, (axes, *shape), generator=torch.Generator().manual_seed(33 + n)).to(dev)
        full = p.expand(axes, *lead).contiguous()
        want = ops.rotary_embedding(q, k, full, f, sections=sections)
        if shape == (2, 1, 2, 1, 3):  # five that do not merge
            with pytest.raises(ops.AclnnError, match="positions"):
                ops.rotary_embedding(q, k, p, f, sections=sections)
            continue
        got = ops.rotary_embedding(q, k, p, f, sections=sections)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    check(want[0], q, full, f, False, sections, 1.0)
