"""kc_group_norm_act and its backward pass against float64.

Tolerances. A result of type t is off by one rounding, half_step(t), plus what the float32 evaluation leaves. Every
float32 sum here is a tree whose longest chain is below 64 additions, and the remaining operations of an element (two
statistics, subtraction, product, sum, activation with a fast exponential and divide) are below 64 roundings in all:
each error is then at most K = 128 half steps of float32 (2^-24) of the size of the terms that enter. mish and silu
have slopes below 1.1, so that the error of z passes on with that factor.
Statistics: mean and variance are sums of that kind, (x - mean)^2 is off by 2 (x - mean) d(mean)."""

import pytest
import torch

import token_ops as t
from katago_cuda import api

pytestmark = pytest.mark.gpu

K24 = 128 * 2.0**-24


def make(n, points, channels, dtype, seed, pad=0, scale=1.3, shift=0.4):
    g = torch.Generator(device="cuda").manual_seed(seed)
    wide = torch.empty(n, points, channels + pad, device="cuda").normal_(0, scale, generator=g).add_(shift)
    wide = wide.to(t.DTYPES[dtype])
    w = torch.empty(channels, device="cuda").uniform_(0.5, 1.5, generator=g)
    b = torch.empty(channels, device="cuda").normal_(0, 0.5, generator=g)
    return wide, wide[:, :, :channels], w, b, g


def masks(kind, n, points, g):
    """float32 [n][points], or None."""
    if kind == "none":
        return None
    p = torch.arange(points, device="cuda")
    side = torch.tensor([(19, 13, 9)[i % 3] for i in range(n)], device="cuda")[:, None]
    m = ((p % 19 < side) & (p // 19 % 19 < side)).float()
    if kind == "random":
        m = (torch.rand(n, points, device="cuda", generator=g) < 0.5).float()
    if kind == "empty":      # every second board without a point
        m[::2] = 0
    if kind == "one":        # one point a board
        m = torch.zeros(n, points, device="cuda")
        m[:, points // 2] = 1
    if kind == "values":     # any value but 0 is on
        m = m * torch.where(p % 2 == 0, -3.0, 1e-30)
    return m


def check_forward(x, mask, w, b, groups, act, y, stats, eps=t.EPS):
    on = torch.ones(x.shape[:2], dtype=torch.bool, device="cuda") if mask is None else mask != 0
    wd = torch.ones(x.shape[2], device="cuda") if w is None else w
    bd = torch.zeros(x.shape[2], device="cuda") if b is None else b
    want, mean, rstd, xh, z = t.norm64(x, on, wd, bd, groups, act, eps)
    half, tiny = t.half_step(x.dtype)
    xon = torch.where(on[:, :, None], x.double(), 0.0)
    top = xon.abs().reshape(*x.shape[:2], groups, -1).amax((1, 3))       # largest |x| of a group
    if stats is not None:
        t.within(stats[:, :, 0], mean, K24 * top)
        # d(var) / var from the sum itself and from the mean, halved by the square root, plus roundings
        t.within(stats[:, :, 1], rstd, rstd * (K24 + (K24 * top * rstd) ** 2))
    cg = x.shape[2] // groups
    zsize = (xh.abs() + (top * rstd).repeat_interleave(cg, 1)[:, None, :]) * wd.double().abs() + bd.double().abs()
    far = (K24 * top * rstd).repeat_interleave(cg, 1)[:, None, :] ** 2 * xh.abs() * wd.double().abs()
    tol = half * want.abs() + tiny + 1.1 * (K24 * zsize + far)
    tol = torch.where(on[:, :, None], tol, 0.0)                          # off the board: exactly 0
    t.within(y, want, tol)


CASES = [
    # n, points, channels, groups, pad
    (1, 361, 384, 32, 0), (3, 361, 384, 32, 0), (2, 361, 768, 1, 0), (5, 37, 100, 20, 4), (2, 169, 33, 3, 0),
    (2, 169, 33, 11, 2), (4, 400, 96, 96, 0), (2, 5776, 256, 32, 0), (1, 6000, 768, 1, 0), (2, 9000, 40, 5, 0),
    (1, 1, 1, 1, 0), (3, 1, 8, 2, 0), (2, 2, 6, 3, 0), (9, 81, 24, 2, 8), (40, 19, 48, 4, 0), (2, 361, 200, 8, 0),
    (1, 20000, 16, 2, 0), (3, 50, 2056, 2, 0), (300, 5, 64, 8, 0), (2, 130, 90, 6, 0), (1, 3, 5000, 1, 0),
    (2, 700, 56, 8, 0), (6, 361, 128, 16, 0), (1, 70000, 5, 1, 0),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,points,channels,groups,pad", CASES)
def test_forward(n, points, channels, groups, pad, dtype):
    for i, (act, kind) in enumerate([("mish", "boards"), ("relu", "none"), ("silu", "random"), ("identity", "empty")]):
        wide, x, w, b, g = make(n, points, channels, dtype, 17 * i + n, pad)
        mask = masks(kind, n, points, g)
        y, stats = t.norm_forward(x, mask, w, b, groups, act)
        check_forward(x, mask, w, b, groups, act, y, stats)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("points,channels,groups", [(361, 384, 32), (90, 33, 3), (6000, 64, 1), (9000, 24, 3)])
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), float("-inf"), 3e38])
def test_masked_places_have_no_effect(points, channels, groups, dtype, junk):
    for kind in ("boards", "empty", "one", "values"):
        wide, x, w, b, g = make(3, points, channels, dtype, 5)
        mask = masks(kind, 3, points, g)
        clean, s0 = t.norm_forward(x, mask, w, b, groups, "mish")
        dy = torch.randn(x.shape, device="cuda", generator=g).to(x.dtype)
        back0 = t.norm_backward(x, mask, w, b, s0, dy, groups, "mish")
        off = (mask == 0)[:, :, None]
        x2 = torch.where(off, torch.full_like(x, junk), x)
        dy2 = torch.where(off, torch.full_like(x, junk), dy)
        got, s1 = t.norm_forward(x2, mask, w, b, groups, "mish")
        assert torch.equal(got, clean) and torch.equal(s0, s1)
        assert got[off.expand_as(got)].eq(0).all()
        for a, c in zip(t.norm_backward(x2, mask, w, b, s1, dy2, groups, "mish"), back0):
            assert torch.isfinite(a).all() and torch.equal(a, c)
        if kind == "empty":
            assert s1[::2].eq(0).all()


@pytest.mark.parametrize("points,channels", [(361, 64), (30, 30), (7000, 64)])
def test_optional_tensors(points, channels):
    wide, x, w, b, g = make(2, points, channels, "f16", 3)
    y, stats = t.norm_forward(x, None, None, None, 2, "silu", want_stats=False)
    assert stats is None
    check_forward(x, None, None, None, 2, "silu", y, None)
    _, stats = t.norm_forward(x, None, w, None, 2, "silu")
    dy = torch.randn(x.shape, device="cuda", generator=g).half()
    dx, dw, db = t.norm_backward(x, None, w, None, stats, dy, 2, "silu")
    only, none_w, none_b = t.norm_backward(x, None, w, None, stats, dy, 2, "silu", want=False)
    assert none_w is None and none_b is None and torch.equal(dx, only)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("points,channels,groups", [(361, 384, 32), (5000, 96, 1), (50, 33, 3), (9000, 64, 2)])
def test_strides_and_what_lies_between(points, channels, groups, dtype):
    """Channel slices of wider rows, points-major boards, a mask shared by all boards, in place; nothing else is
    written."""
    n = 3
    wide, x, w, b, g = make(n, points, channels, dtype, 11, pad=8)
    mask = masks("boards", 1, points, g).expand(n, points)   # board stride 0
    want, s0 = t.norm_forward(x.contiguous(), mask.contiguous(), w, b, groups, "mish")
    out = torch.full((n, points, channels + 24), 7.0, device="cuda").to(x.dtype)
    y, s1 = t.norm_forward(x, mask, w, b, groups, "mish", y=out[:, :, 8:8 + channels])
    assert torch.equal(y, want) and torch.equal(s0, s1)
    assert out[:, :, :8].eq(7).all() and out[:, :, 8 + channels:].eq(7).all()
    # points-major: board b's row r at (r * n + b)
    pm = torch.full((points, n, channels), 7.0, device="cuda").to(x.dtype)
    y, _ = t.norm_forward(x, mask, w, b, groups, "mish", y=pm.transpose(0, 1))
    assert torch.equal(y, want)
    # slices of one buffer, side by side
    both = torch.cat([x, torch.zeros_like(x)], 2)
    y, _ = t.norm_forward(both[:, :, :channels], mask, w, b, groups, "mish", y=both[:, :, channels:])
    assert torch.equal(y, want) and torch.equal(both[:, :, :channels], x)
    # backward into a slice, dy in a slice
    dy = torch.randn((n, points, channels + 8), device="cuda", generator=g).to(x.dtype)[:, :, :channels]
    want = t.norm_backward(x.contiguous(), mask.contiguous(), w, b, s0, dy.contiguous(), groups, "mish")
    rest = wide[:, :, channels:].clone()
    out = wide.clone()
    got = t.norm_backward(x, mask, w, b, s0, dy, groups, "mish", dx=out[:, :, :channels])
    assert all(torch.equal(a, c) for a, c in zip(got, want)) and torch.equal(out[:, :, channels:], rest)
    # in place: forward over x, backward over dy and over x
    dyc = dy.contiguous()
    xc = x.contiguous()
    got = t.norm_backward(xc, mask, w, b, s0, dyc, groups, "mish", dx=dyc)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    xb = xc.clone()
    got = t.norm_backward(xb, mask, w, b, s0, dy.contiguous(), groups, "mish", dx=xb)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    y0, _ = t.norm_forward(xc, mask, w, b, groups, "mish")
    y, _ = t.norm_forward(xc, mask, w, b, groups, "mish", y=xc)
    assert torch.equal(y, y0)


def test_off_alignment():
    """Tensors whose first element lies 2, 4, 6 .. bytes off a vector boundary."""
    n, points, channels, groups = 2, 100, 64, 8
    _, x, w, b, g = make(n, points, channels, "bf16", 2)
    want, _ = t.norm_forward(x, None, w, b, groups, "silu")
    for off in (1, 2, 3, 4, 5):
        buf = torch.full((x.numel() + 16,), 5.0, device="cuda").bfloat16()
        xo = buf[off:off + x.numel()].view_as(x)
        xo.copy_(x)
        out = torch.full((x.numel() + 16,), 5.0, device="cuda").bfloat16()
        y = out[off:off + x.numel()].view_as(x)
        t.norm_forward(xo, None, w, b, groups, "silu", y=y)
        on = torch.ones(n, points, dtype=torch.bool, device="cuda")
        check_forward(xo, None, w, b, groups, "silu", y, None)
        assert on.all() and out[:off].eq(5).all() and out[off + x.numel():].eq(5).all()
        assert (y.double() - want.double()).abs().max() < 0.05


@pytest.mark.parametrize("points,channels,groups", [(361, 64, 8), (9000, 64, 8)])
def test_large_mean_keeps_the_variance(points, channels, groups):
    """A mean 1000 times the spread: the variance is taken around the mean, so it keeps its digits."""
    _, x, w, b, _ = make(2, points, channels, "f32", 8, scale=1.0, shift=1000.0)
    y, stats = t.norm_forward(x, None, w, b, groups, "identity")
    check_forward(x, None, w, b, groups, "identity", y, stats)


def test_huge_values_and_zero_eps():
    _, x, w, b, _ = make(2, 90, 16, "f32", 9)
    for big in (1e15, 1e-15):
        y, stats = t.norm_forward(x * big, None, w, b, 2, "identity", eps=0.0)
        check_forward(x * big, None, w, b, 2, "identity", y, stats, eps=0.0)


def test_nan_on_the_board_stays_in_its_group():
    for points in (361, 9000):
        _, x, w, b, _ = make(2, points, 64, "f32", 4)
        x[1, 5, 17] = float("nan")  # group 2 of 8
        for act in t.ACTS:
            y, stats = t.norm_forward(x, None, w, b, 8, act)
            bad = torch.isnan(y)
            assert bad[1, :, 16:24].all() and not bad[0].any() and not bad[1, :, :16].any() and not bad[1, :, 24:].any()
            assert torch.isnan(stats[1, 2]).all()


def check_backward(x, mask, w, b, stats, dy, groups, act, got):
    on = torch.ones(x.shape[:2], dtype=torch.bool, device="cuda") if mask is None else mask != 0
    dx, dw, db, size, wsize, bsize = t.norm_back64(x, on, w, b, stats[:, :, 0], stats[:, :, 1], dy, groups, act)
    half, tiny = t.half_step(x.dtype)
    # the slope's own error: |slope''| < 1 for mish and silu, so an error of z, 4 half steps of its terms, enters dy
    cg = x.shape[2] // groups
    r = stats[:, :, 1].double().repeat_interleave(cg, 1)[:, None, :]
    m = stats[:, :, 0].double().repeat_interleave(cg, 1)[:, None, :]
    xh = torch.where(on[:, :, None], (x.double() - m).abs() * r, 0.0)
    dyd = torch.where(on[:, :, None], dy.double().abs(), 0.0)
    dz = (xh * w.double().abs() + b.double().abs()) * dyd if act in ("mish", "silu") else torch.zeros_like(dyd)
    wd = w.double().abs()
    count = (on.sum(1) * cg).double().clamp(min=1)[:, None]

    def share(v):
        s = (v.sum(1) * wd).reshape(x.shape[0], groups, cg).sum(2) / count
        return s.repeat_interleave(cg, 1)[:, None]

    more = r * (dz * wd + share(dz) + xh * share(dz * xh))
    t.within(got[0], dx, torch.where(on[:, :, None], half * dx.abs() + tiny + K24 * (size + more + r * dyd * wd), 0.0))
    t.within(got[1], dw, K24 * (wsize + (dz * xh).sum((0, 1)) + (dyd * xh).sum((0, 1))))
    t.within(got[2], db, K24 * (bsize + dz.sum((0, 1)) + dyd.sum((0, 1))))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,points,channels,groups,pad", CASES)
def test_backward(n, points, channels, groups, pad, dtype):
    for i, (act, kind) in enumerate([("mish", "boards"), ("relu", "none"), ("silu", "random"), ("identity", "empty")]):
        wide, x, w, b, g = make(n, points, channels, dtype, 19 * i + n, pad)
        mask = masks(kind, n, points, g)
        _, stats = t.norm_forward(x, mask, w, b, groups, act)
        dy = torch.empty(n, points, channels, device="cuda").normal_(generator=g).to(x.dtype)
        got = t.norm_backward(x, mask, w, b, stats, dy, groups, act)
        check_backward(x, mask, w, b, stats, dy, groups, act, got)


@pytest.mark.parametrize("act", ["mish", "silu", "identity", "relu"])
@pytest.mark.parametrize("points,channels,groups", [(50, 24, 4), (50, 21, 3), (9000, 8, 1)])
def test_gradient_is_the_difference_quotient(points, channels, groups, act):
    """Along a random direction of x, weight and bias the gradients add up to the slope of sum(dy * y) in float64.
    The quotient's own error is h^2 / 6 of a third derivative (below 1e-6 of the terms' size for h = 1e-4, apart from
    relu, where it is exact but for the points within h of 0: each at most h of its term); the gradients' float32
    errors are at most K24 of the terms' size."""
    _, x, w, b, g = make(3, points, channels, "f32", 21)
    mask = masks("random", 3, points, g)
    dy = torch.randn(x.shape, device="cuda", generator=g)
    _, stats = t.norm_forward(x, mask, w, b, groups, act)
    dx, dw, db = t.norm_backward(x, mask, w, b, stats, dy, groups, act)
    vx, vw, vb = (torch.randn(v.shape, device="cuda", generator=g).double() for v in (x, w, b))
    on = mask != 0

    def loss(h):
        y = t.norm64(x.double() + h * vx, on, w.double() + h * vw, b.double() + h * vb, groups, act)[0]
        return (y * dy.double()).sum().item()

    h = 1e-4
    slope = (loss(h) - loss(-h)) / (2 * h)
    got = ((dx.double() * vx).sum() + (dw.double() * vw).sum() + (db.double() * vb).sum()).item()
    size = ((dx.double() * vx).abs().sum() + (dw.double() * vw).abs().sum() + (db.double() * vb).abs().sum()).item()
    assert abs(got - slope) <= (1e-4 if act == "relu" else 1e-6 + K24) * size


def test_relu_next_to_its_corner():
    """z = 0 up to float32's rounding at every element: the side is the sign in float64, as the formula has it."""
    n, points, channels = 2, 200, 32
    _, x, w, b, g = make(n, points, channels, "f32", 31)
    _, stats = t.norm_forward(x, None, w, b, 4, "relu")
    one = x[0, 0].double()
    m, r = (stats[0, :, i].double().repeat_interleave(8) for i in (0, 1))
    b = (-(one - m) * r * w.double()).float()                     # z of that row is 0 but for b's rounding
    x = x[:1, :1].expand(n, points, channels).contiguous()
    stats = stats[:1].expand(n, 4, 2).contiguous()
    z = (x.double() - m) * r * w.double() + b.double()
    assert 0.2 < (z > 0).double().mean() < 0.8
    dy = torch.randn(x.shape, device="cuda", generator=g)
    got = t.norm_backward(x, None, w, b, stats, dy, 4, "relu")
    check_backward(x, None, w, b, stats, dy, 4, "relu", got)


@pytest.mark.parametrize("n,points,channels,groups", [(64, 361, 96, 8), (2, 9000, 64, 4), (3, 50, 33, 3)])
def test_same_bits_again_on_other_streams_and_in_graphs(n, points, channels, groups):
    _, x, w, b, g = make(n, points, channels, "bf16", 41)
    mask = masks("boards", n, points, g)
    dy = torch.randn(x.shape, device="cuda", generator=g).bfloat16()
    y0, s0 = t.norm_forward(x, mask, w, b, groups, "mish")
    back0 = t.norm_backward(x, mask, w, b, s0, dy, groups, "mish")
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                y, st = t.norm_forward(x, mask, w, b, groups, "mish")
                got.append((y, st) + t.norm_backward(x, mask, w, b, st, dy, groups, "mish"))
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(a, c) for a, c in zip(r, (y0, s0) + back0))
    # two captured graphs with a workspace each, replayed on two streams at once on new inputs
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        xi = torch.zeros_like(x)
        with torch.cuda.graph(gr):
            y, st = t.norm_forward(xi, mask, w, b, groups, "mish")
            r = (y, st) + t.norm_backward(xi, mask, w, b, st, dy, groups, "mish")
        graphs.append((gr, xi, r))
    for _ in range(3):
        for gr, xi, r in graphs:
            xi.copy_(x)
            for v in r:
                v.fill_(9)
        torch.cuda.synchronize()
        for s, (gr, xi, r) in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        for gr, xi, r in graphs:
            assert all(torch.equal(a, c) for a, c in zip(r, (y0, s0) + back0))


def test_offsets_past_32_bits():
    """Boards 2^31 + 64 elements apart (4 GB of f16), rows 2^30 apart."""
    far = (1 << 31) + 64
    _, x, w, b, g = make(2, 40, 64, "f16", 51)
    want, s0 = t.norm_forward(x, None, w, b, 8, "mish")
    dy = torch.randn(x.shape, device="cuda", generator=g).half()
    back0 = t.norm_backward(x, None, w, b, s0, dy, 8, "mish")
    buf = torch.empty(far + 40 * 64, dtype=torch.float16, device="cuda")
    xf = buf.as_strided((2, 40, 64), (far, 64, 1))
    xf.copy_(x)
    y, _ = t.norm_forward(xf, None, w, b, 8, "mish")
    assert torch.equal(y, want)
    got = t.norm_backward(xf, None, w, b, s0, dy, 8, "mish", dx=xf)
    assert all(torch.equal(a, c) for a, c in zip(got, back0))
    rows = buf.as_strided((1, 3, 64), (64, 1 << 30, 1))
    rows.copy_(x[:1, :3])
    y, _ = t.norm_forward(rows, None, w, b, 8, "mish")
    assert torch.equal(y, t.norm_forward(x[:1, :3].contiguous(), None, w, b, 8, "mish")[0])


def test_boards_without_points():
    d = api.GroupNormDesc(api.PRECISION_F32, api.ACT_MISH, 3, 0, 16, 2, 1e-5)
    stats, dw, db = (torch.full((s,), 5.0, device="cuda") for s in (12, 16, 16))
    api.group_norm_act(d, 0, 0, 0, 0, 0, stats.data_ptr(), 0, 0, t.stream())
    api.group_norm_act_backward(d, 0, 0, 0, 0, 0, 0, 0, dw.data_ptr(), db.data_ptr(), 0, 0, t.stream())
    assert all(v.eq(0).all() for v in (stats, dw, db))


def test_host_memory_is_refused():
    x = torch.zeros(1, 4, 8)
    y = torch.zeros(1, 4, 8, device="cuda")
    d = api.GroupNormDesc(api.PRECISION_F32, api.ACT_MISH, 1, 4, 8, 2, 1e-5)
    ws = torch.zeros(max(1, api.group_norm_act_workspace(d, False)), dtype=torch.uint8, device="cuda")
    for xi in (x, x.pin_memory()):
        with pytest.raises(api.KcError) as e:
            api.group_norm_act(d, xi.data_ptr(), 0, 0, 0, y.data_ptr(), 0, ws.data_ptr(), ws.numel(), t.stream())
        assert e.value.status == api.KC_ERR_INVALID and "device memory" in str(e.value)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,points,channels,groups", [
    (900, 361, 48, 4),      # many boards to a block
    (300, 169, 200, 25),    # a narrower last chunk, blocks that change chunks
    (70, 5776, 64, 8),      # clusters that go over several boards, more rows than the early mask loads
    (45, 361, 768, 1),      # one group over a cluster of 16
    (333, 20, 21, 3),       # single channels
])
def test_blocks_that_take_several_boards(n, points, channels, groups, dtype):
    for act, kind in (("mish", "boards"), ("relu", "random"), ("silu", "none"), ("identity", "empty")):
        _, x, w, b, g = make(n, points, channels, dtype, n)
        mask = masks(kind, n, points, g)
        y, stats = t.norm_forward(x, mask, w, b, groups, act)
        check_forward(x, mask, w, b, groups, act, y, stats)
        dy = torch.randn(x.shape, device="cuda", generator=g).to(x.dtype)
        got = t.norm_backward(x, mask, w, b, stats, dy, groups, act)
        check_backward(x, mask, w, b, stats, dy, groups, act, got)
        z, _ = t.norm_forward(x, mask, w, b, groups, act, y=x)   # in place
        assert torch.equal(z, y)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("n,points,channels,groups", [(2, 30000, 256, 1), (1, 90000, 24, 3), (3, 4000, 1000, 5)])
def test_boards_beyond_a_cluster(n, points, channels, groups, dtype):
    for act, kind in (("mish", "boards"), ("relu", "none"), ("silu", "empty")):
        _, x, w, b, g = make(n, points, channels, dtype, n)
        mask = masks(kind, n, points, g)
        y, stats = t.norm_forward(x, mask, w, b, groups, act)
        check_forward(x, mask, w, b, groups, act, y, stats)
        dy = torch.randn(x.shape, device="cuda", generator=g).to(x.dtype)
        check_backward(x, mask, w, b, stats, dy, groups, act, t.norm_backward(x, mask, w, b, stats, dy, groups, act))


def test_large_activations():
    """z far outside the range of exp: mish and silu go to z and to 0, their slopes to 1 and 0."""
    x = torch.linspace(-1, 1, 64, device="cuda").reshape(1, 64, 1).repeat(1, 1, 8)
    on = torch.ones(1, 64, dtype=torch.bool, device="cuda")
    b = torch.zeros(8, device="cuda")
    for dtype in t.DTYPES.values():
        for scale in (30.0, 200.0, 3e4):
            w = torch.full((8,), scale, device="cuda")
            for act in ("mish", "silu"):
                xt = x.to(dtype)
                y, stats = t.norm_forward(xt, None, w, b, 1, act)
                want, _, _, xh, z = t.norm64(xt, on, w, b, 1, act)
                half, tiny = t.half_step(dtype)
                t.within(y, want, half * want.abs() + tiny + 1.1 * K24 * 3 * scale)
                dy = torch.ones_like(xt)
                got = t.norm_backward(xt, None, w, b, stats, dy, 1, act)
                check_backward(xt, None, w, b, stats, dy, 1, act, got)


def test_first_call_inside_a_capture():
    """A fresh process whose first call of each operator is captured into a graph."""
    import os
    import subprocess
    import sys
    code = """
import sys, torch
sys.path[:0] = [%r, %r]
import token_ops as t
x = torch.randn(4, 361, 64, device="cuda").bfloat16()
w, b = torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")
q = torch.randn(5000, 2, 64, device="cuda").bfloat16()
pos = torch.zeros(5000, 2, dtype=torch.int32, device="cuda")
freqs = torch.ones(1, 32, 2, device="cuda")
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y, st = t.norm_forward(x, None, w, b, 8, "mish")
    back = t.norm_backward(x, None, w, b, st, x, 8, "mish")
    qo, _ = t.rope_forward(q, None, pos, freqs, 64, "halves")
    dq = t.rope_backward(q, None, q, None, pos, freqs, 64, "halves")
g.replay()
torch.cuda.synchronize()
y2, st2 = t.norm_forward(x, None, w, b, 8, "mish")
assert torch.equal(y, y2) and torch.equal(st, st2) and torch.equal(qo, q)
assert all(torch.equal(a, c) for a, c in zip(back, t.norm_backward(x, None, w, b, st, x, 8, "mish")))
print("captured")
"""
    here = os.path.dirname(os.path.abspath(__file__))
    code = code % (here, os.path.join(os.path.dirname(here), "katago-rs_b200", "python"))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout + r.stderr


def test_many_shapes():
    """Random sizes, groups, strides, masks, types and directions."""
    import random
    rng = random.Random(12)
    for i in range(120):
        groups = rng.choice([1, 2, 3, 4, 8, 16, 32])
        channels = groups * rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16, 24, 40])
        points = rng.choice([1, 2, 7, 31, 64, 81, 169, 361, 400, 1000, 3001])
        n = rng.randint(1, 6)
        dtype, act = rng.choice(list(t.DTYPES)), rng.choice(list(t.ACTS))
        wide, x, w, b, g = make(n, points, channels, dtype, i, rng.choice([0, 0, 1, 4, 8]))
        mask = masks(rng.choice(["none", "boards", "random", "empty", "one"]), n, points, g)
        y, stats = t.norm_forward(x, mask, w, b, groups, act)
        check_forward(x, mask, w, b, groups, act, y, stats)
        dy = torch.randn(x.shape, device="cuda", generator=g).to(x.dtype)
        got = t.norm_backward(x, mask, w, b, stats, dy, groups, act)
        check_backward(x, mask, w, b, stats, dy, groups, act, got)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,points,channels,groups", [(3, 361, 64, 8), (2, 361, 21, 7), (2, 9000, 64, 8),
                                                      (2, 60000, 24, 8), (2, 20000, 512, 2), (3, 6, 64, 8)])
def test_squares_beyond_float32(n, points, channels, groups, dtype):
    """Where a group's sum of squares passes float32's range its results are not numbers, never those of another
    variance; other groups and boards, and values whose squares stay within it, are as ever."""
    cg = channels // groups
    _, x, w, b, g = make(n, points, channels, dtype, 61, scale=1.0, shift=0.0)
    mask = masks("boards", n, points, g)
    on = (mask != 0)[:, :, None]
    x[1, :, cg:2 * cg] = (x[1, :, cg:2 * cg].float() * 4e19).to(x.dtype)
    for act in t.ACTS:
        y, stats = t.norm_forward(x, mask, w, b, groups, act)
        hit = torch.zeros_like(y, dtype=torch.bool)
        hit[1, :, cg:2 * cg] = True
        assert torch.isnan(y[hit & on]).all() and torch.isfinite(y[~hit | ~on]).all()
        assert y[~on.expand_as(y)].eq(0).all()
        assert torch.isnan(stats[1, 1, 1]) and torch.isnan(stats).sum() <= 2
        dx, _, _ = t.norm_backward(x, mask, w, b, stats, torch.ones_like(x), groups, act)
        assert torch.isnan(dx[hit & on]).all() and torch.isfinite(dx[~hit | ~on]).all()
    x[1, :, cg:2 * cg] = (torch.randn(points, cg, device="cuda", generator=g) * 1e16).to(x.dtype)
    y, stats = t.norm_forward(x, mask, w, b, groups, "identity")
    check_forward(x, mask, w, b, groups, "identity", y, stats)


@pytest.mark.parametrize("act", ["mish", "silu"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("points,channels", [(64, 8), (361, 384), (9000, 64), (9000, 384)])
def test_tails_keep_their_digits(points, channels, dtype, act):
    """z from -12.4 to 8.4. Below -5 |y'(z) / y| is at most 1, so that an error of z, K24 of its terms, is a relative
    error of y; exponential, products and quotient add less than another K24 of y: the type's rounding is what is
    left in the 2-byte types."""
    x = torch.linspace(-1, 1, points, device="cuda")[None, :, None].repeat(2, 1, channels).to(t.DTYPES[dtype])
    w, b = torch.full((channels,), 6.0, device="cuda"), torch.full((channels,), -2.0, device="cuda")
    on = torch.ones(2, points, dtype=torch.bool, device="cuda")
    y, stats = t.norm_forward(x, None, w, b, 1, act)
    want, mean, rstd, xh, z = t.norm64(x, on, w, b, 1, act)
    half, tiny = t.half_step(x.dtype)
    zsize = (xh.abs() + rstd.max()) * 6 + 2
    tail = z < -5
    assert z.min() < -12 and tail.any()
    tol = want.abs() * (half + K24 * (1 + zsize)) * 1.01 + tiny
    t.within(y[tail], want[tail], tol[tail])


def test_row_strides_of_boards_of_one_point():
    _, x, w, b, g = make(70, 1, 96, "bf16", 71)
    mask = masks("empty", 70, 1, g)
    want = t.norm_forward(x, mask, w, b, 8, "mish")
    back = t.norm_backward(x, mask, w, b, want[1], x, 8, "mish")
    d = api.GroupNormDesc(api.PRECISION_BF16, api.ACT_MISH, 70, 1, 96, 8, t.EPS, x_strides=(96, 1 << 62),
                          y_strides=(96, (1 << 63) - 1))
    y, dx = torch.zeros_like(x), torch.zeros_like(x)
    stats, dw, db = torch.zeros_like(want[1]), torch.zeros_like(w), torch.zeros_like(b)
    for backward in (False, True):
        size = api.group_norm_act_workspace(d, backward)
        ws = t.workspace(size, x.device)
        if not backward:
            api.group_norm_act(d, x.data_ptr(), mask.data_ptr(), w.data_ptr(), b.data_ptr(), y.data_ptr(),
                               stats.data_ptr(), t.ptr(ws), size, t.stream())
        else:
            api.group_norm_act_backward(d, x.data_ptr(), mask.data_ptr(), w.data_ptr(), b.data_ptr(), stats.data_ptr(),
                                        x.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(), t.ptr(ws), size,
                                        t.stream())
    assert torch.equal(y, want[0]) and torch.equal(stats, want[1])
    assert all(torch.equal(a, c) for a, c in zip((dx, dw, db), back))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("points", [361, 400, 420, 421, 460])
@pytest.mark.parametrize("channels,groups", [(96, 8), (30, 6), (21, 3)])
def test_boards_around_what_one_block_holds(points, channels, groups, dtype):
    n = 40
    for act, kind in (("mish", "boards"), ("silu", "none")):
        _, x, w, b, g = make(n, points, channels, dtype, points)
        mask = masks(kind, n, points, g)
        y, stats = t.norm_forward(x, mask, w, b, groups, act)
        check_forward(x, mask, w, b, groups, act, y, stats)
        dy = torch.randn(x.shape, device="cuda", generator=g).to(x.dtype)
        check_backward(x, mask, w, b, stats, dy, groups, act, t.norm_backward(x, mask, w, b, stats, dy, groups, act))
