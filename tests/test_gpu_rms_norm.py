"""The norm of a residual sum against its formulas in 64 bits. A stored value is off by at most half a step of its type; the fp32 sums
behind it add their terms in an order of at most 64 dependent additions (plus one a row for the weight's gradient), each off by
half a step of fp32."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
STEP32 = 2.0 ** -24
CHAIN = 64
# rows, width: one value, one vector, a warp's row, odd ones, rows of a block, rows of 512 and 1024 threads, rows too wide for them
SHAPES = [(1, 1), (3, 2), (5, 7), (1, 8), (17, 64), (9, 255), (4, 256), (33, 1000), (2, 1143), (6, 1152), (3, 4096), (2, 4097),
          (5, 5120), (2, 8190), (2, 8191), (3, 8192), (2, 16384), (2, 16388), (2, 32768), (2, 32776), (1, 70001),
          # many rows take fewer threads each
          (600, 4096), (601, 5120), (640, 8200)]


def inputs(shape, t, seed, dev, count=2):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(shape, generator=gen) * s).to(t).to(dev) for s in (1.0, 3.0, 1.0, 1.0)[:count]]


def weights(width, t, seed, dev):
    return (torch.randn(width, generator=torch.Generator().manual_seed(seed)) * 0.2 + 1).to(t).to(dev)


def half_step(t):
    return torch.finfo(t).eps / 2


def close(got, want, bound):
    got = got.double()
    assert torch.isfinite(got).all()
    over = (got - want).abs() - bound
    assert (over <= 0).all(), f"over the bound by {over.max().item():.3g} at {over.argmax().item()}"


def stored_sum(x, r):
    return (x.float() + r.float()).to(x.dtype)


def forward64(z, w, eps):
    z = z.double()
    rstd = 1 / (z.square().mean(-1, keepdim=True) + eps).sqrt()
    return z * rstd * (w.double() if w is not None else 1), rstd


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,width", SHAPES)
def test_forward(ops, dev, t, rows, width):
    x, r = inputs((rows, width), t, 1, dev)
    for residual, w, eps in ((r, weights(width, t, 2, dev), 1e-6), (None, weights(width, torch.float32, 3, dev), 1e-2), (r, None, 0.0)):
        y, z, rstd = ops.residual_rms_norm(x, residual, w, eps)
        assert torch.equal(z, stored_sum(x, residual) if residual is not None else x)
        want, want_rstd = forward64(z, w, eps)
        close(rstd.unsqueeze(-1), want_rstd, CHAIN * STEP32 * want_rstd)
        close(y, want, (half_step(t) + 2 * CHAIN * STEP32) * want.abs() + torch.finfo(t).tiny)
        again = ops.residual_rms_norm(x, residual, w, eps)
        assert torch.equal(again[0], y) and torch.equal(again[2], rstd)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,width", SHAPES + [(700, 768), (2000, 40), (601, 1025)])
def test_backward(ops, dev, t, rows, width):
    z, gy, gs, _ = inputs((rows, width), t, 4, dev, 4)
    for w, add in ((weights(width, t, 5, dev), gs), (weights(width, torch.float32, 6, dev), None), (None, gs)):
        want_y, rstd = forward64(z, w, 1e-6)
        gx, gw = ops.residual_rms_norm_backward(gy, z, rstd.float().squeeze(-1), w, add)
        u = z.double() * rstd
        g = gy.double() * (w.double() if w is not None else 1)
        mean, size = (g * u).mean(-1, keepdim=True), (g * u).abs().mean(-1, keepdim=True)
        a = add.double() if add is not None else torch.zeros_like(u)
        want = a + rstd * (g - u * mean)
        # the rounding of rstd to fp32 counts as one more step
        terms = a.abs() + rstd * (g.abs() + u.abs() * size)
        close(gx, want, half_step(t) * want.abs() + 2 * CHAIN * STEP32 * terms + torch.finfo(t).tiny)
        if w is None:
            assert gw is None
        else:
            want = (gy.double() * u).sum(0)
            bound = half_step(w.dtype) * want.abs() + (rows + CHAIN) * STEP32 * (gy.double() * u).abs().sum(0)
            close(gw, want, bound + torch.finfo(w.dtype).tiny)
            assert gw.dtype == w.dtype
        again = ops.residual_rms_norm_backward(gy, z, rstd.float().squeeze(-1), w, add)
        assert torch.equal(again[0], gx) and (w is None or torch.equal(again[1], gw))


def test_backward_against_differences(ops, dev):
    """The gradient of sum(y * a + sum * b) by central differences of the 64-bit forward."""
    x, r, a, b = (v.double() for v in inputs((2, 24), torch.float32, 7, dev, 4))
    w = weights(24, torch.float32, 8, dev).double()

    def loss(x, w):
        y, _ = forward64(x + r, w, 1e-5)
        return (y * a + (x + r) * b).sum().item()

    z = (x + r).float()
    _, rstd = forward64(z, w, 1e-5)
    gx, gw = ops.residual_rms_norm_backward(a.float(), z, rstd.float().squeeze(-1), w.float(), b.float())
    h = 1e-4
    for v, got in ((x, gx), (w, gw)):
        for i in range(0, v.numel(), 5):
            d = torch.zeros_like(v).view(-1)
            d[i] = h
            d = d.view_as(v)
            diff = (loss(x + d, w) - loss(x - d, w)) if v is x else (loss(x, w + d) - loss(x, w - d))
            assert abs(diff / (2 * h) - got.reshape(-1)[i].item()) < 2e-5 * max(1.0, abs(diff / (2 * h))) + 1e-5


def quant_bound(y, scale, dtype):
    """Half a step of the 8-bit type at y / scale, and the fp32 roundings of y, of the scale's inverse and of their product."""
    slack = 2 * (CHAIN + 4) * STEP32
    if dtype == torch.int8:
        return scale * (0.5 + 127 * slack)
    return torch.maximum(y.abs() * 2.0 ** -4, scale * 2.0 ** -10) + slack * y.abs() * (1 + 2.0 ** -3)


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,width", SHAPES)
@pytest.mark.parametrize("group", [0, 32, 128, 160])
def test_quant(ops, dev, t, rows, width, dtype, group):
    x, r = inputs((rows, width), t, 9, dev)
    x[0] *= 0.01
    w = weights(width, t, 10, dev)
    q, scales, z = ops.residual_rms_norm_quant(x, r, w, 1e-6, dtype, group)
    assert torch.equal(z, stored_sum(x, r)) and q.dtype == dtype
    y, _ = forward64(z, w, 1e-6)
    g = group if 0 < group < width else width
    parts = torch.split(y, g, -1)
    assert scales.shape == (rows, len(parts))
    range_ = 127.0 if dtype == torch.int8 else 448.0
    want = torch.stack([p.abs().amax(-1) for p in parts], -1) / range_
    close(scales, want, want * 2 * CHAIN * STEP32)
    wide = torch.repeat_interleave(scales.double(), g, -1)[:, :width]
    close(q.double() * wide, y, quant_bound(y, wide, dtype))
    no_sum = ops.residual_rms_norm_quant(z, None, w, 1e-6, dtype, group)
    assert torch.equal(no_sum[0].view(torch.uint8), q.view(torch.uint8)) and torch.equal(no_sum[1], scales)


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("group", [0, 128])
def test_quant_of_zeros_and_non_finite_rows(ops, dev, dtype, group):
    x = torch.randn(5, 256, generator=torch.Generator().manual_seed(11)).to(dev)
    x[0] = 0
    x[1, 7] = float("nan")
    x[2, 200] = float("inf")
    x[3, :128] = 0
    q, scales, _ = ops.residual_rms_norm_quant(x, dtype=dtype, group=group)
    assert (scales[0] == 0).all() and (q[0].float() == 0).all()
    assert scales[1].isnan().all()  # every value of the row is NaN: its norm is
    assert not scales[2].isfinite().any() or scales[2].isnan().any()
    if group:
        assert scales[3, 0] == 0 and (q[3, :128].float() == 0).all() and scales[3, 1] > 0
    assert scales[4].isfinite().all() and (scales[4] > 0).all()


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("group", [0, 32, 128])
def test_quant_of_tiny_rows(ops, dev, dtype, group):
    """Magnitudes whose scale has no finite inverse become zeros with scale 0."""
    x = torch.ones(2, 256, device=dev)
    q, scales, _ = ops.residual_rms_norm_quant(x, None, torch.full((256,), 1e-37, device=dev), dtype=dtype, group=group)
    assert (scales == 0).all() and (q.float() == 0).all()
    q, scales, _ = ops.residual_rms_norm_quant(x, None, torch.full((256,), 1e-33, device=dev), dtype=dtype, group=group)
    back = q.double() * scales.double().repeat_interleave(group or 256, -1)
    assert ((back - 1e-33).abs() < 1e-33 * 2.0 ** -4).all()


def test_non_finite_rows_stay_in_their_rows(ops, dev):
    x = torch.randn(9, 300, generator=torch.Generator().manual_seed(12)).to(dev)
    clean, _, _ = ops.residual_rms_norm(x)
    x[4, 2] = float("inf")
    x[6, 299] = float("nan")
    y, _, _ = ops.residual_rms_norm(x)
    rest = [i for i in range(9) if i not in (4, 6)]
    assert torch.equal(y[rest], clean[rest])
    assert y[6].isnan().all() and y[4, 2].isnan() and (y[4, :2] == 0).all()


@pytest.mark.parametrize("t", TYPES)
def test_views(ops, dev, t):
    """Heads of a fused product (rows in two levels), transposed and odd-offset views, as inputs and as outputs."""
    gen = torch.Generator().manual_seed(13)
    base = torch.randn(3, 11, 5 * 16 + 1, generator=gen).to(t).to(dev)
    heads = base[:, :, 1:].view(3, 11, 5, 16)[:, :, 1:4]
    w = weights(16, t, 14, dev)

    def holds(x, residual, got):
        # not the bits of a contiguous call: another vector width adds a row's squares in another order
        y, z, rstd = got
        assert torch.equal(z, stored_sum(x, residual) if residual is not None else x)
        want, want_rstd = forward64(z, w, 1e-6)
        close(rstd.unsqueeze(-1), want_rstd, CHAIN * STEP32 * want_rstd)
        close(y, want, (half_step(t) + 2 * CHAIN * STEP32) * want.abs() + torch.finfo(t).tiny)

    holds(heads, None, ops.residual_rms_norm(heads, None, w))
    turned = torch.randn(3, 16, 7, generator=gen).to(t).to(dev).transpose(1, 2)
    out = torch.zeros(3, 16, 7, dtype=t, device=dev).transpose(1, 2)
    got = ops.residual_rms_norm(turned, None, w, out=out)
    assert got[0].data_ptr() == out.data_ptr()
    holds(turned, None, got)
    deep = torch.randn(2, 6, 4, 10, 16, generator=gen).to(t).to(dev)[:, ::2, ::2, ::3]
    residual = torch.randn(2, 3, 2, 4, 16, generator=gen).to(t).to(dev)
    holds(deep, residual, ops.residual_rms_norm(deep, residual, w))
    one = torch.randn(1, 1, 16, generator=gen).to(t).to(dev).expand(3, 7, 16)
    want = ops.residual_rms_norm_backward(one.contiguous(), turned.contiguous(), want_rstd(turned), w)
    got = ops.residual_rms_norm_backward(one, turned, want_rstd(turned), w)  # both of contiguous copies, so the same bits
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def want_rstd(z):
    return forward64(z, None, 1e-6)[1].float().squeeze(-1).contiguous()


@pytest.mark.parametrize("width", [7, 512, 40000])
def test_in_place(ops, dev, width):
    x, r, g, _ = inputs((5, width), torch.bfloat16, 15, dev, 4)
    w = weights(width, torch.bfloat16, 16, dev)
    y, z, rstd = ops.residual_rms_norm(x, r, w)
    x1, r1 = x.clone(), r.clone()
    y1, z1, _ = ops.residual_rms_norm(x1, r1, w, out=x1, sum_out=r1)
    assert torch.equal(y1, y) and torch.equal(z1, z) and y1.data_ptr() == x1.data_ptr() and z1.data_ptr() == r1.data_ptr()
    gx, gw = ops.residual_rms_norm_backward(g, z, rstd, w, x)
    for over in range(3):
        args = [g.clone(), z.clone(), x.clone()]
        gx1, gw1 = ops.residual_rms_norm_backward(args[0], args[1], rstd, w, args[2], grad_x=args[over])
        assert torch.equal(gx1, gx) and torch.equal(gw1, gw)


def test_no_rows(ops, dev):
    x = torch.zeros(0, 12, device=dev)
    y, z, rstd = ops.residual_rms_norm(x, x, torch.ones(12, device=dev))
    assert y.shape == (0, 12) and rstd.shape == (0,)
    gw = torch.full((12,), 3.0, device=dev)
    ops.residual_rms_norm_backward(x, x, rstd, torch.ones(12, device=dev), grad_weight=gw)
    assert (gw == 0).all()


def test_rows_past_32_bits(ops, dev):
    """Two rows whose distance is above 2^31 elements."""
    far = torch.empty(2, 2 ** 31 + 8, dtype=torch.bfloat16, device=dev)
    x = far[:, :64]
    x.copy_(torch.randn(2, 64, generator=torch.Generator().manual_seed(17)))
    want = ops.residual_rms_norm(x.contiguous())[0]
    assert torch.equal(ops.residual_rms_norm(x)[0], want)
    ops.residual_rms_norm(x, out=far[:, 64:128])
    assert torch.equal(far[:, 64:128], want)


def test_graph_and_stream(ops, dev):
    x, r, g, _ = inputs((70, 384), torch.bfloat16, 18, dev, 4)
    w = weights(384, torch.bfloat16, 19, dev)

    def step():
        y, z, rstd = ops.residual_rms_norm(x, r, w)
        return (y, z) + ops.residual_rms_norm_backward(g, z, rstd, w, y)

    want = step()
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream(dev).wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (20, 21):
        fresh = inputs((70, 384), torch.bfloat16, seed, dev, 4)
        for a, b in zip((x, r, g), fresh):
            a.copy_(b)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,width,wide", [(2, 8194, 8194), (3, 10002, 10002), (3, 12290, 12290), (2, 16382, 16382), (300, 8198, 8198),
                                             (2, 12288, 12290), (2, 16384, 16386)])
def test_backward_of_wide_rows_in_pairs(ops, dev, t, rows, width, wide):
    """Rows of more than 8192 values that can only be read two at a time, by their width or by their distance."""
    z, gy, gs, _ = (x[:, :width] for x in inputs((rows, wide), t, 22, dev, 4))
    w = weights(width, t, 23, dev)
    y, rstd = forward64(z, w, 1e-6)
    got = ops.residual_rms_norm(z, None, w)[0]
    close(got, y, (half_step(t) + 2 * CHAIN * STEP32) * y.abs() + torch.finfo(t).tiny)
    gx, gw = ops.residual_rms_norm_backward(gy, z, rstd.float().squeeze(-1), w, gs)
    u, g = z.double() * rstd, gy.double() * w.double()
    want = gs.double() + rstd * (g - u * (g * u).mean(-1, keepdim=True))
    terms = gs.double().abs() + rstd * (g.abs() + u.abs() * (g * u).abs().mean(-1, keepdim=True))
    close(gx, want, half_step(t) * want.abs() + 2 * CHAIN * STEP32 * terms + torch.finfo(t).tiny)
    want = (gy.double() * u).sum(0)
    close(gw, want, half_step(t) * want.abs() + (rows + CHAIN) * STEP32 * (gy.double() * u).abs().sum(0) + torch.finfo(t).tiny)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("width", [40, 200, 1144, 5000])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_quant_of_a_weight_that_is_not_finite(ops, dev, t, width, bad):
    """It reaches the scale of its own group and no other, the shorter last one least of all."""
    x = inputs((3, width), t, 24, dev)[0]
    for w in (torch.ones(width, device=dev), torch.ones(width, dtype=t, device=dev)):
        clean = [ops.residual_rms_norm_quant(x, None, w, group=group)[1] for group in (32, 128)]
        w[0] = bad
        for group, want in zip((32, 128), clean):
            got = ops.residual_rms_norm_quant(x, None, w, group=group)[1]
            assert not got[:, 0].isfinite().any() and torch.equal(got[:, 1:], want[:, 1:])


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("rows,width", [(256, 4096), (64, 5120), (300, 96), (37, 1143), (9, 40000)])
@pytest.mark.parametrize("group", [0, 32, 128, 160])
def test_quant_divides_the_fp32_values(ops, dev, rows, width, dtype, group):
    """The 8-bit values are those of y / scale, divided in fp32 and rounded to nearest even (y of fp32 tensors comes out as it is)."""
    x = inputs((rows, width), torch.float32, 25, dev)[0]
    w = weights(width, torch.float32, 26, dev)
    y = ops.residual_rms_norm(x, None, w)[0]
    q, scales, _ = ops.residual_rms_norm_quant(x, None, w, dtype=dtype, group=group)
    range_ = 127.0 if dtype == torch.int8 else 448.0
    g = group if 0 < group < width else width
    tops = torch.stack([p.abs().amax(-1) for p in torch.split(y, g, -1)], -1)
    assert torch.equal(scales, tops / torch.full_like(tops, range_))  # by a tensor: torch takes a number's inverse
    want = y / torch.repeat_interleave(scales, g, -1)[:, :width]
    want = want.round() if dtype == torch.int8 else want.clamp(-448, 448).to(dtype).float()
    assert torch.equal(q.float(), want)


def test_backward_of_rows_of_16_million_values(ops, dev):
    """More columns than a grid's second dimension has blocks for."""
    width, t = 65535 * 256 + 4, torch.bfloat16
    z, gy = ((torch.randn(2, width, generator=torch.Generator(device=dev).manual_seed(s), device=dev)).to(t) for s in (27, 28))
    w = z[0].abs() + 0.5
    _, rstd = forward64(z, w, 1e-6)
    gx, gw = ops.residual_rms_norm_backward(gy, z, rstd.float().squeeze(-1), w)
    u, g = z.double() * rstd, gy.double() * w.double()
    want = (gy.double() * u).sum(0)
    close(gw, want, half_step(t) * want.abs() + CHAIN * STEP32 * (gy.double() * u).abs().sum(0) + torch.finfo(t).tiny)
    want = rstd * (g - u * (g * u).mean(-1, keepdim=True))
    terms = rstd * (g.abs() + u.abs() * (g * u).abs().mean(-1, keepdim=True))
    chain = width // 1024 + CHAIN  # a thread adds up its share of the row in turn
    close(gx, want, half_step(t) * want.abs() + 2 * chain * STEP32 * terms + torch.finfo(t).tiny)


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,width", [(5, 64), (9, 500), (33, 1000), (6, 1153), (700, 2050), (3, 5120), (2, 8196), (2, 40000)])
@pytest.mark.parametrize("group", [32, 64, 128, 256, 512])
def test_quant_by_groups_of_a_power_of_two(ops, dev, t, rows, width, dtype, group):
    """Groups that one to 32 lanes hold and wider ones, of rows that end inside one, read 8, 4, 2 and 1 values at a time."""
    x = inputs((rows, width), t, 29, dev)[0]
    w = weights(width, torch.float32, 30, dev)
    q, scales, _ = ops.residual_rms_norm_quant(x, None, w, dtype=dtype, group=group)
    y, _ = forward64(x, w, 1e-6)
    g = min(group, width)
    want = torch.stack([p.abs().amax(-1) for p in torch.split(y, g, -1)], -1) / (127.0 if dtype == torch.int8 else 448.0)
    assert scales.shape == want.shape
    close(scales, want, want * 2 * CHAIN * STEP32)
    wide = torch.repeat_interleave(scales.double(), g, -1)[:, :width]
    close(q.double() * wide, y, quant_bound(y, wide, dtype))
