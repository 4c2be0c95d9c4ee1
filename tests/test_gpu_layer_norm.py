"""kc_layer_norm and its backward pass against float64.

Tolerances. A float32 sum of C terms is made of chains: a thread adds at most 32 elements (of rows above 8,192 channels
C / 512), then lanes and warps join in 10 steps, so that with N = 42 + C / 512 additions it is off by N 2^-24 of the sum
of the sizes. The mean of the distances from the first mean is off by N 2^-24 of the mean distance, at most one
standard deviation: xh is off by N 2^-24 (1 + |xh|) with the reciprocal root's share (half of the squares' N 2^-24, and
4 roundings). With E = (N + 8) 2^-24: y is off by its rounding and E (1 + |xh|) |w| + 2^-23 |b|, dx by its rounding and
E times the sizes of its terms. dweight and dbias add at most 400 rows in a chain here: 2^-15 of the sum of the sizes."""

import pytest
import torch

import row_ops as r
import token_ops as t
from katago_cuda import api

pytestmark = pytest.mark.gpu

SUMS = 2.0**-15


def unit(channels):
    return (50 + channels / 512) * 2.0**-24


def make(n, points, channels, dtype, seed, masked, pad=0, shift=0.4):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rows(scale, at):
        wide = torch.empty(n, points, channels + pad, device="cuda").normal_(at, scale, generator=g).to(t.DTYPES[dtype])
        return wide[:, :, :channels]

    x, dy = rows(1.3, shift), rows(1.0, 0.0)
    w = torch.empty(channels, device="cuda").uniform_(0.5, 1.5, generator=g)
    b = torch.empty(channels, device="cuda").normal_(0, 0.3, generator=g)
    mask = (torch.rand(n, points, device="cuda", generator=g) < 0.7).float() if masked else None
    return x, dy, w, b, mask


def on_of(x, mask):
    return torch.ones(x.shape[:2], dtype=torch.bool, device=x.device) if mask is None else mask != 0


def check_forward(x, mask, w, b, kind, y, stats, eps=r.EPS):
    want, mean, rstd, xh = r.layer64(x, on_of(x, mask), w, b, kind, eps)
    half, tiny = t.half_step(x.dtype)
    e = unit(x.shape[2])
    wa = 1.0 if w is None else w.double().abs()
    ba = 0.0 if b is None else b.double().abs()
    on = on_of(x, mask)[:, :, None]
    t.within(y, want, torch.where(on, half * want.abs() + tiny + e * (1 + xh.abs()) * wa + 2.0**-23 * ba, 0.0))
    if stats is not None:
        std = torch.where(rstd > 0, 1 / rstd.clamp(min=1e-30), 0.0)
        t.within(stats[..., 0], mean, 2.0**-24 * mean.abs() + e * std)
        t.within(stats[..., 1], rstd, 2 * e * rstd)


def check_backward(x, mask, w, stats, dy, kind, dx, dw, db):
    want, ww, wb, size, sw, sb = r.layer_back64(x, on_of(x, mask), w, stats[..., 0], stats[..., 1], dy, kind)
    half, tiny = t.half_step(x.dtype)
    on = on_of(x, mask)[:, :, None]
    t.within(dx, want, torch.where(on, half * want.abs() + tiny + 2 * unit(x.shape[2]) * size, 0.0))
    if dw is not None:
        t.within(dw, ww, SUMS * sw)
        t.within(db, wb, SUMS * sb)


CASES = [
    # n, points, channels, pad
    (1, 1, 384, 0), (1, 1, 1, 0), (3, 361, 384, 0), (2, 361, 768, 0), (5, 137, 100, 4), (4, 81, 99, 0), (2, 33, 7, 3),
    (1, 1000, 8, 0), (7, 3, 256, 8), (2, 19, 1024, 0), (1, 50, 1000, 0), (3, 5, 2048, 0), (2, 9, 1030, 0),
    (1, 6, 4096, 0), (2, 2, 4099, 0), (1, 3, 8192, 8), (1, 3, 16384, 0), (1, 2, 40000, 0), (2, 1, 20003, 0),
    (300, 40, 16, 0), (1, 5, 130, 0), (2, 70, 640, 1), (1, 17, 192, 0), (3, 2, 513, 0),
    # rows that begin anywhere: whole and partial last vectors, as many vectors as a group of lanes holds
    (3, 40, 768, 3), (2, 50, 767, 0), (3, 31, 384, 5), (2, 90, 24, 1), (1, 77, 8, 1), (2, 33, 760, 2), (1, 9, 769, 1),
    (5, 60, 128, 7), (1, 300, 3, 0),
]


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,points,channels,pad", CASES)
def test_forward_and_backward(n, points, channels, pad, dtype, kind):
    for masked in (False, True):
        x, dy, w, b, mask = make(n, points, channels, dtype, channels + points, masked, pad)
        y, stats = r.layer_forward(x, mask, w, b, kind)
        check_forward(x, mask, w, b, kind, y, stats)
        dx, dw, db = r.layer_backward(x, mask, w, stats, dy, kind)
        check_backward(x, mask, w, stats, dy, kind, dx, dw, db)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 16, 17, 64, 255, 256, 257, 1023, 1024, 1025, 2047, 2048, 2049, 8192, 8193])
def test_ends_of_the_ways_to_add(rows, dtype):
    """Parameter gradients by clusters of 1 to 16 blocks and by a second launch, of 4 to 128 rows to a block at once."""
    for channels, pad in ((384, 0), (100, 3), (9, 0), (16, 0)):
        x, dy, w, b, mask = make(1, rows, channels, dtype, rows, rows % 2 == 0, pad)
        for kind in r.KINDS:
            y, stats = r.layer_forward(x, mask, w, b, kind)
            check_backward(x, mask, w, stats, dy, kind, *r.layer_backward(x, mask, w, stats, dy, kind))


@pytest.mark.parametrize("channels,blocks", [(2000, 592), (4096, 296), (1500, 740), (1030, 296), (8192, 148)])
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_blocks_whose_rows_are_on_in_turn(kind, channels, blocks):
    """Every other row of a block is off, so that the sums of those that are on follow each other without what a row
    between them would wait for: the bits of the rows that are on by themselves."""
    rows = 9 * blocks
    x, dy, w, b, _ = make(1, rows, channels, "bf16", 31, False)
    mask = (torch.arange(rows, device="cuda") // blocks % 2 == 0).float()[None]
    on = mask[0] != 0
    y, stats = r.layer_forward(x, mask, w, b, kind)
    alone, own = r.layer_forward(x[:, on].contiguous(), None, w, b, kind)
    assert torch.equal(y[:, on], alone) and torch.equal(stats[:, on], own) and y[:, ~on].eq(0).all()
    for _ in range(5):
        dx, dw, db = r.layer_backward(x, mask, w, stats, dy, kind)
        check_backward(x, mask, w, stats, dy, kind, dx, dw, db)
        single = r.layer_backward(x[:, on].contiguous(), None, w, own, dy[:, on].contiguous(), kind)[0]
        assert torch.equal(dx[:, on], single)


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_many_rows(kind):
    """A block goes over many rows: 92,416 x 96 over at most 296 blocks of 16 rows or more, chains of 20."""
    x, dy, w, b, mask = make(256, 361, 96, "bf16", 5, True)
    y, stats = r.layer_forward(x, mask, w, b, kind)
    check_forward(x, mask, w, b, kind, y, stats)
    check_backward(x, mask, w, stats, dy, kind, *r.layer_backward(x, mask, w, stats, dy, kind))


@pytest.mark.parametrize("channels", [384, 2000, 24000])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_optional_tensors(dtype, channels):
    x, dy, w, b, mask = make(2, 30, channels, dtype, 11, True)
    for weight, bias in ((None, None), (w, None), (None, b)):
        for kind in r.KINDS:
            y, stats = r.layer_forward(x, mask, weight, bias, kind)
            check_forward(x, mask, weight, bias, kind, y, stats)
            again, _ = r.layer_forward(x, mask, weight, bias, kind, want_stats=False)
            assert torch.equal(again, y)
            dx, dw, db = r.layer_backward(x, mask, weight, stats, dy, kind)
            check_backward(x, mask, weight, stats, dy, kind, dx, dw, db)
            alone, _, _ = r.layer_backward(x, mask, weight, stats, dy, kind, want=False)
            assert torch.equal(alone, dx)
    # one of the parameter gradients alone
    desc = r.layer_desc(x, dy, "layer", mask=mask)
    size = api.layer_norm_backward_workspace(desc)
    y, stats = r.layer_forward(x, mask, w, b, "layer")
    want = r.layer_backward(x, mask, w, stats, dy, "layer")
    for k in (1, 2):
        one = torch.full((channels,), float("nan"), device="cuda")
        dx = torch.empty_like(x)
        ws = t.workspace(size, "cuda")
        api.layer_norm_backward(desc, x.data_ptr(), mask.data_ptr(), w.data_ptr(), stats.data_ptr(), dy.data_ptr(),
                                dx.data_ptr(), one.data_ptr() if k == 1 else 0, one.data_ptr() if k == 2 else 0,
                                ws.data_ptr(), size, t.stream())
        assert torch.equal(one, want[k]) and torch.equal(dx, want[0])


@pytest.mark.parametrize("channels", [100, 384, 1500, 24000])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_masked_rows_have_no_effect(dtype, channels):
    """NaN, infinities and the type's ends at tokens that are off; all tokens off; masks of NaN count as on."""
    x, dy, w, b, mask = make(3, 20, channels, dtype, 13, True)
    mask[1] = 0
    junk = torch.tensor([float("nan"), float("inf"), float("-inf"), torch.finfo(x.dtype).min], device="cuda")
    off = (mask == 0)[:, :, None]
    fill = junk.repeat(channels // 4 + 1)[:channels].to(x.dtype)
    bad_x, bad_dy = torch.where(off, fill, x), torch.where(off, fill, dy)
    for kind in r.KINDS:
        y, stats = r.layer_forward(x, mask, w, b, kind)
        y2, stats2 = r.layer_forward(bad_x, mask, w, b, kind)
        assert torch.equal(y, y2) and torch.equal(stats, stats2)
        a = r.layer_backward(x, mask, w, stats, dy, kind)
        stats2[mask == 0] = float("nan")
        c = r.layer_backward(bad_x, mask, w, stats2, bad_dy, kind)
        assert all(torch.equal(u, v) for u, v in zip(a, c))
        assert y[mask == 0].eq(0).all() and a[0][mask == 0].eq(0).all() and stats[mask == 0].eq(0).all()
        none = torch.zeros_like(mask)
        y, stats = r.layer_forward(bad_x, none, w, b, kind)
        dx, dw, db = r.layer_backward(bad_x, none, w, stats, bad_dy, kind)
        assert all(v.eq(0).all() for v in (y, stats, dx, dw, db))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("channels", [64, 384, 1200, 20000])
def test_strides_offsets_guards_and_in_place(dtype, channels):
    n, points = 3, 17
    x, dy, w, b, mask = make(n, points, channels, dtype, 17, True)
    for kind in r.KINDS:
        y, stats = r.layer_forward(x, mask, w, b, kind)
        grads = r.layer_backward(x, mask, w, stats, dy, kind)
        # rows of a longer sequence and of a wider buffer; what is around them stays
        for off in (0, 8, 3):
            buf = torch.full((n, points + 5, channels + 24), 5.0, device="cuda").to(x.dtype)
            out = buf[:, 2:2 + points, off:off + channels]
            xs = torch.zeros(n, points + 1, channels + 16, device="cuda").to(x.dtype)[:, 1:, off:off + channels]
            xs.copy_(x)
            big = torch.zeros(n, points + 9, device="cuda")
            big[:, :points] = mask
            got, st = r.layer_forward(xs, big[:, :points], w, b, kind, y=out)
            check_forward(xs, mask, w, b, kind, got, st)
            keep = torch.ones_like(buf, dtype=torch.bool)
            keep[:, 2:2 + points, off:off + channels] = False
            assert buf[keep].eq(5).all()
            d2 = buf.clone()[:, 2:2 + points, off:off + channels]
            d2.copy_(dy)
            wide = torch.full((n, points + 1, channels + 16), 7.0, device="cuda").to(x.dtype)
            dxs = wide[:, 1:, off:off + channels]
            check_backward(xs, mask, w, st, d2, kind, *r.layer_backward(xs, mask, w, st, d2, kind, dx=dxs))
            keep = torch.ones_like(wide, dtype=torch.bool)
            keep[:, 1:, off:off + channels] = False
            assert wide[keep].eq(7).all()
        # boards inside out: rows of all boards side by side
        inner = x.transpose(0, 1).contiguous().transpose(0, 1)
        got, st = r.layer_forward(inner, mask, w, b, kind)
        assert torch.equal(got, y) and torch.equal(st, stats)
        # in place
        z = x.clone()
        r.layer_forward(z, mask, w, b, kind, y=z)
        assert torch.equal(z, y)
        for z, args in ((x.clone(), "x"), (dy.clone(), "dy")):
            xi, di = (z, dy) if args == "x" else (x, z)
            got = r.layer_backward(xi, mask, w, stats, di, kind, dx=z)
            assert all(torch.equal(u, v) for u, v in zip(got, grads))
        # parameters that are aligned to a float only
        w1, b1 = torch.zeros(2, channels + 1, device="cuda")[:, 1:]
        w1.copy_(w), b1.copy_(b)
        assert torch.equal(r.layer_forward(x, mask, w1, b1, kind)[0], y)


def test_large_means_and_small_spreads():
    """The variance and x - mean keep their digits under a mean 10^4 times the spread."""
    for channels in (384, 1500, 20000):
        x, dy, w, b, _ = make(2, 10, channels, "f32", 19, False, shift=13000.0)
        y, stats = r.layer_forward(x, None, w, b, "layer")
        check_forward(x, None, w, b, "layer", y, stats)


def test_ends_of_the_range():
    """Squares beyond float32's range give NaN in that row alone; a row of equal values gives the bias."""
    for channels in (384, 1500, 20000):
        x = torch.randn(1, 4, channels, device="cuda")
        x[0, 1] *= 1e20
        x[0, 2] = 2.5
        b = torch.randn(channels, device="cuda")
        for kind in r.KINDS:
            y, stats = r.layer_forward(x, None, None, b, kind)
            assert y[0, 1].isnan().all() and stats[0, 1, 1].isnan()
            assert y[0, [0, 2, 3]].isfinite().all()
        y, stats = r.layer_forward(x, None, None, b, "layer")
        assert torch.equal(y[0, 2], b)
        x[0, 3, 5] = float("nan")
        y, _ = r.layer_forward(x, None, None, b, "layer")
        assert y[0, 3].isnan().all() and y[0, 0].isfinite().all()


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("channels", [48, 1600])
def test_gradient_is_the_difference_quotient(kind, channels):
    """sum(dy y) along random directions, in float64: the quotient's error is h^2 of third derivatives of order 1."""
    x, dy, w, b, mask = make(2, 15, channels, "f32", 23, True)
    y, stats = r.layer_forward(x, mask, w, b, kind)
    dx, dw, db = r.layer_backward(x, mask, w, stats, dy, kind)
    on = on_of(x, mask)
    v, vw, vb = (torch.randn(s.shape, device="cuda").double() for s in (x, w, b))

    def loss(h):
        return (r.layer64(x.double() + h * v, on, w.double() + h * vw, b.double() + h * vb, kind)[0] * dy.double()).sum()

    h = 1e-4
    slope = (loss(h) - loss(-h)) / (2 * h)
    got = (dx.double() * v).sum() + (dw.double() * vw).sum() + (db.double() * vb).sum()
    scale = (dx.double() * v).abs().sum() + (dw.double() * vw).abs().sum() + (db.double() * vb).abs().sum()
    assert abs(got - slope) <= 1e-5 * scale


def test_same_bits_alone_in_batches_on_streams_and_in_graphs():
    x, dy, w, b, mask = make(40, 361, 384, "bf16", 29, True)
    y, stats = r.layer_forward(x, mask, w, b, "rms")
    # a token alone gives its bits in the batch
    for i, p in ((0, 0), (7, 100), (39, 360)):
        one, st = r.layer_forward(x[i:i + 1, p:p + 1], mask[i:i + 1, p:p + 1], w, b, "rms")
        assert torch.equal(one[0, 0], y[i, p]) and torch.equal(st[0, 0], stats[i, p])

    def both():
        yy, ss = r.layer_forward(x, mask, w, b, "layer")
        return (yy, ss) + r.layer_backward(x, mask, w, ss, dy, "layer")

    want = both()
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(3)]:
        with torch.cuda.stream(s):
            got.append(both())
    torch.cuda.synchronize()
    for a in got:
        assert all(torch.equal(u, v) for u, v in zip(a, want))
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = both()
        graphs.append((gr, out))
    for gr, out in graphs:
        for _ in range(2):
            for v in out:
                v.fill_(9)
            gr.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(u, v) for u, v in zip(out, want))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("channels", [1, 7, 100, 384, 767, 1000, 1031, 4096, 20000, 40000])
def test_rows_of_equal_values_without_eps(dtype, channels):
    """NaN with eps 0, whatever the first mean's rounding leaves; the other rows as ever. With an eps, the bias."""
    values = torch.tensor([1.7, 0.1, -3e4, 1e-3, 0.0, 1.0, -7.3, 0.30001], device="cuda").to(t.DTYPES[dtype])
    x, _, w, b, _ = make(1, 16, channels, dtype, channels, False)
    x[0, ::2] = values[:, None]
    for bias in (None, b):
        y, stats = r.layer_forward(x, None, w, bias, "layer", eps=0.0)
        assert y[0, ::2].isnan().all() and stats[0, ::2, 1].isnan().all()
        if channels > 1:
            check_forward(x[:, 1::2], None, w, bias, "layer", y[:, 1::2], stats[:, 1::2], eps=0.0)
        y, stats = r.layer_forward(x, None, w, bias, "rms", eps=0.0)
        assert y[0, 8].isnan().all() and stats[0, 8, 1].isnan()
        keep = torch.arange(16, device="cuda") != 8
        check_forward(x[:, keep], None, w, bias, "rms", y[:, keep], stats[:, keep], eps=0.0)
        # with an eps: the first mean is off by E of the value, what is left of the distance from it by E of that
        y, stats = r.layer_forward(x[:, ::2], None, w, bias, "layer")
        want, mean, rstd, _ = r.layer64(x[:, ::2], on_of(x[:, ::2], None), w, bias, "layer")
        left = unit(channels) ** 2 * mean.abs()
        half, tiny = t.half_step(x.dtype)
        add = 0.0 if bias is None else 2.0**-23 * b.double().abs()
        t.within(y, want, half * want.abs() + tiny + (left * rstd)[:, :, None] * w.double() * 1.01 + add)
        t.within(stats[..., 0], mean, 2.0**-24 * mean.abs() + left)
        t.within(stats[..., 1], rstd, 2 * unit(channels) * rstd)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("channels", [1, 7, 99, 100, 383, 769, 1031, 4099, 384])
def test_means_whose_quotient_by_the_spread_passes_float32(dtype, channels):
    """mean x rstd beyond float32's range, where x - mean is 0: dx = rstd (g - mean of g), whatever stands beside the
    row's last element in its vector."""
    x, dy, w, _, _ = make(2, 5, channels, dtype, channels, False)
    x.fill_(2.0**119)
    stats = torch.tensor([2.0**119, 2.0**10], device="cuda").expand(2, 5, 2).contiguous()
    check_backward(x, None, w, stats, dy, "layer", *r.layer_backward(x, None, w, stats, dy, "layer"))


@pytest.mark.parametrize("channels", [384, 767, 1500, 20000])
def test_gradients_under_large_means(channels):
    """Against float64 from float64 statistics. The saved mean is a float32, off by 2^-24 of itself: xh is off by
    h = |mean| rstd 2^-24 in the whole row, besides what check_backward allows and rstd's own error."""
    x, dy, w, b, _ = make(2, 10, channels, "f32", 19, False, shift=13000.0)
    on = on_of(x, None)
    _, stats = r.layer_forward(x, None, w, b, "layer")
    _, mean, rstd, xh = r.layer64(x, on, w, b, "layer")
    dx, dw, db = r.layer_backward(x, None, w, stats, dy, "layer")
    want, ww, wb, size, sw, sb = r.layer_back64(x, on, w, mean, rstd, dy, "layer")
    e = unit(channels)
    h = (mean.abs() * rstd * 2.0**-24 + e)[:, :, None]
    g = dy.double() * w.double()
    c1, c2 = g.mean(2, keepdim=True).abs(), (g * xh).mean(2, keepdim=True).abs()
    t.within(dx, want, 2.0**-24 * want.abs() + 2 * e * size + 6 * e * size
             + rstd[:, :, None] * (h * c2 + xh.abs() * h * c1 + h * h * c1) * 1.01)
    t.within(dw, ww, SUMS * sw + 2 * e * sw + (dy.double().abs() * h).sum((0, 1)))
    t.within(db, wb, SUMS * sb)
