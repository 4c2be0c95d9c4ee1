"""kc_distill_top and its backward pass against float64.

Tolerances. An exponential is off by 2^-21 (the hardware's 2^-22 and its argument's rounding, which weighs x e^-x < 0.4 of
2^-23), and the sum of a row's n is made of chains of n / (a row's threads) float32 additions and 10 merges of 3
roundings: E = (n / threads + 40) 2^-24 + 2^-21 of the sum, so that the loss, whose terms are differences of logarithms
in 64 bits, is off by T^2 P E and its rounding. Gradient, from the saved pair: g P q with an exponential whose argument
x is rounded to 2^-23 |x|, and at an entry's class g p rounded to float32; exponentials below 2^-126 are 0."""

import pytest
import torch

import row_ops as r
import token_ops as t

pytestmark = pytest.mark.gpu
NEG = float("-inf")


def unit(classes, threads):
    return (classes / threads + 40) * 2.0**-24 + 2.0**-21


def make(rows, classes, k, dtype, seed, absent=True, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = torch.empty(rows, classes, device="cuda").normal_(0, spread, generator=g).to(t.DTYPES[dtype])
    ids = torch.randint(0, classes, (rows, k), device="cuda", generator=g, dtype=torch.int32)
    if k <= classes <= 5000:
        ids = torch.rand(rows, classes, device="cuda", generator=g).argsort(1)[:, :k].int().contiguous()
    top = torch.empty(rows, k, device="cuda").normal_(0, 2, generator=g)
    if absent:
        n = torch.arange(rows, device="cuda")[:, None] % 4
        j = torch.arange(k, device="cuda")[None]
        ids = torch.where((n == 1) & (j >= (k + 1) // 2), -1, ids)
        ids = torch.where((n == 2) & (j % 3 == 1), classes, ids)
        top = torch.where((n == 2) & (j % 5 == 2), NEG, top)
        ids = torch.where((n == 3) & (rows > 4), torch.where(j % 2 == 0, -1, 2**31 - 1), ids).int()
    dloss = torch.empty(rows, device="cuda").uniform_(-1, 1, generator=g)
    return z, ids, top, dloss


def check_forward(z, ids, top, whole, temp, loss, stats):
    want, m, s = r.distill64(z, ids, top, whole, temp)
    _, _, p, _ = r.teacher64(ids, top, whole, z.shape[1], temp)
    e = unit(z.shape[1], 32 if z.shape[1] <= 2048 else 256)
    t.within(loss, want, temp**2 * p.sum(1) * e + 2.0**-23 * want.abs())
    if stats is not None:
        assert torch.equal(stats[:, 0].double(), m)
        t.within(stats[:, 1], s, e * s)


def check_backward(z, ids, top, whole, temp, stats, dloss, dz):
    want, gq, gp = r.distill_back64(z, ids, top, whole, temp, stats, dloss)
    half, tiny = t.half_step(z.dtype)
    x = ((z.double() - stats[:, :1].double()) / temp).abs()
    x = torch.where(gq > 0, x, 0.0)
    t.within(dz, want, half * want.abs() + tiny + gq * (2.0**-20 + x * 2.0**-22) + gp * 2.0**-22 + 2.0**-120)


CASES = [
    # rows, classes, entries, temperature
    (1, 362, 32, 1.0), (9, 362, 64, 1.0), (40, 362, 362, 2.0), (5, 1, 1, 1.0), (6, 2, 7, 0.5), (300, 361, 5, 1.0),
    (33, 2048, 128, 1.0), (17, 2047, 129, 4.0), (8, 2049, 16, 1.0), (5, 5001, 1024, 0.7), (3, 40000, 100, 1.0),
    (1, 131071, 64, 2.0), (12, 65537, 33, 1.0), (2, 300007, 1000, 1.0), (1500, 4100, 8, 1.0), (7, 33, 3, 20.0),
    (1, 8192, 1, 0.1), (1300, 2100, 150, 1.0), (4, 4096, 70, 1.0),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,classes,k,temp", CASES)
def test_forward_and_backward(rows, classes, k, temp, dtype):
    z, ids, top, dloss = make(rows, classes, k, dtype, rows + classes)
    for whole in (None, torch.logsumexp(top.double().clamp(min=-50) / temp, 1).float() + 0.3):
        loss, stats = r.distill_forward(z, ids, top, whole, temp)
        check_forward(z, ids, top, whole, temp, loss, stats)
        again, _ = r.distill_forward(z, ids, top, whole, temp, want_stats=False)
        assert torch.equal(again, loss)
        for dl in (dloss, None):
            dz = r.distill_backward(z, ids, top, stats, whole, temp, dl)
            check_backward(z, ids, top, whole, temp, stats, dl, dz)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("classes", [362, 1999, 3001, 20011])
def test_masked_logits(dtype, classes):
    """Illegal classes at -inf or at the type's lowest value have probability 0 and no gradient."""
    z, ids, top, dloss = make(20, classes, 20, dtype, 5, absent=False)
    ids = ids % (classes // 2)  # the teacher's moves are legal
    for fill in (NEG, torch.finfo(z.dtype).min):
        zz = z.clone()
        zz[:, classes // 2:] = fill
        zz[3, 30:] = fill
        ids[3] = ids[3] % 30
        zz[4, :] = fill
        zz[4, 5] = -3.0
        ids[4] = 5
        for temp in (1.0, 0.25, 3.0):
            loss, stats = r.distill_forward(zz, ids, top, None, temp)
            check_forward(zz, ids, top, None, temp, loss, stats)
            dz = r.distill_backward(zz, ids, top, stats, None, temp, dloss)
            check_backward(zz, ids, top, None, temp, stats, dloss, dz)
            assert dz[:, classes // 2:].eq(0).all()
    # every class at the lowest value: equal probabilities
    zz[:] = torch.finfo(z.dtype).min
    loss, stats = r.distill_forward(zz, ids, top)
    check_forward(zz, ids, top, None, 1.0, loss, stats)
    check_backward(zz, ids, top, None, 1.0, stats, dloss, r.distill_backward(zz, ids, top, stats, None, 1.0, dloss))


@pytest.mark.parametrize("classes", [362, 3001, 30011])
def test_entries_of_one_class_add_up(classes):
    for k in (2, 40, 130, 1024):
        z, ids, top, dloss = make(6, classes, k, "f32", 7, absent=False)
        ids[0] = 17
        ids[1] = ids[1] % 5
        ids[2, k // 2:] = ids[2, :k - k // 2]
        ids[3] = torch.where(torch.arange(k, device="cuda") % 2 == 0, -1, 3)
        ids[4, -1] = ids[4, 0]
        loss, stats = r.distill_forward(z, ids, top)
        check_forward(z, ids, top, None, 1.0, loss, stats)
        dz = r.distill_backward(z, ids, top, stats, None, 1.0, dloss)
        want, gq, gp = r.distill_back64(z, ids, top, None, 1.0, stats, dloss)
        # the entries of a class are added in float32, at most k of them
        t.within(dz, want, 2.0**-24 * want.abs() + gq * 2.0**-18 + gp * ((k + 4) * 2.0**-24) + 2.0**-140)
        again = r.distill_backward(z, ids, top, stats, None, 1.0, dloss)
        assert torch.equal(dz, again)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("classes", [362, 4001, 70001])
def test_rows_without_entries_are_not_read(dtype, classes):
    z, ids, top, dloss = make(9, classes, 30, dtype, 9, absent=False)
    ids[2], ids[5], top[7] = -1, classes, NEG
    want = r.distill_forward(z, ids, top)
    back = r.distill_backward(z, ids, top, want[1], None, 1.0, dloss)
    for i in (2, 5, 7):
        z[i] = float("nan")
    got = r.distill_forward(z, ids, top)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    bad = want[1].clone()
    for i in (2, 5, 7):
        bad[i] = float("nan")
        dloss[i] = float("nan")
    dz = r.distill_backward(z, ids, top, bad, None, 1.0, dloss)
    assert torch.equal(dz, back) and dz[[2, 5, 7]].eq(0).all() and want[0][[2, 5, 7]].eq(0).all()


def test_not_finite():
    """Each in its row alone: NaN among the logits, +inf, nothing but -inf; an entry at a class of probability 0."""
    for classes in (362, 20000):
        z, ids, top, dloss = make(8, classes, 10, "f32", 11, absent=False)
        z[1, 100], z[2, 7], z[3] = float("nan"), float("inf"), NEG
        z[4, int(ids[4, 0])] = NEG
        loss, stats = r.distill_forward(z, ids, top)
        assert loss[[1, 2, 3]].isnan().all() and loss[4] == float("inf") and loss[[0, 5, 6, 7]].isfinite().all()
        dz = r.distill_backward(z, ids, top, stats)
        assert dz[1].isnan().any() and dz[2].isnan().any() and dz[3].isnan().any()
        assert dz[[0, 4, 5, 6, 7]].isfinite().all()
        # an entry without weight may have any class
        top[4, 0] = -1e5
        loss, _ = r.distill_forward(z, ids, top)
        assert loss[4].isfinite()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("classes,k", [(362, 20), (362, 200), (3001, 50), (50001, 50)])
def test_strides_guards_and_in_place(dtype, classes, k):
    rows = 11
    z, ids, top, dloss = make(rows, classes, k, dtype, 13)
    loss, stats = r.distill_forward(z, ids, top)
    want = r.distill_backward(z, ids, top, stats, None, 1.0, dloss)
    wide_i, wide_t = (torch.full((rows, k + 3), 2.0, device="cuda").to(v.dtype)[:, 1:1 + k] for v in (ids, top))
    wide_i.copy_(ids), wide_t.copy_(top)
    for off in (0, 1, 3, 8):
        buf = torch.full((rows + 2, classes + 13), 5.0, device="cuda").to(z.dtype)
        zs = buf[1:1 + rows, off:off + classes]
        zs.copy_(z)
        got, st = r.distill_forward(zs, wide_i, wide_t)
        check_forward(z, ids, top, None, 1.0, got, st)
        out = torch.full((rows + 2, classes + 19), 7.0, device="cuda").to(z.dtype)
        dz = out[1:1 + rows, 2:2 + classes]
        r.distill_backward(zs, wide_i, wide_t, stats, None, 1.0, dloss, dz=dz)
        assert torch.equal(dz, want)
        keep = torch.ones_like(out, dtype=torch.bool)
        keep[1:1 + rows, 2:2 + classes] = False
        assert out[keep].eq(7).all()
        r.distill_backward(zs, wide_i, wide_t, stats, None, 1.0, dloss, dz=zs)  # in place
        assert torch.equal(zs, want)
        keep = torch.ones_like(buf, dtype=torch.bool)
        keep[1:1 + rows, off:off + classes] = False
        assert buf[keep].eq(5).all()


@pytest.mark.parametrize("classes", [300, 9000])
def test_gradient_is_the_difference_quotient(classes):
    """Along a random direction in float64: the quotient's error is h^2 of third derivatives of order 1 / T^3."""
    z, ids, top, dloss = make(6, classes, 12, "f32", 17)
    temp = 1.5
    loss, stats = r.distill_forward(z, ids, top, None, temp)
    dz = r.distill_backward(z, ids, top, stats, None, temp, dloss)
    v = torch.randn(z.shape, device="cuda").double()
    f = lambda h: (r.distill64(z.double() + h * v, ids, top, None, temp)[0] * dloss.double()).sum()  # noqa: E731
    h = 1e-4
    slope = (f(h) - f(-h)) / (2 * h)
    assert abs((dz.double() * v).sum() - slope) <= 1e-5 * (dz.double() * v).abs().sum()
    # a row's gradient adds up to 0: q and p both add up to 1
    g = dloss.double().abs() * temp
    assert (dz.double().sum(1).abs() <= g * 2.0**-17).all()


def test_same_bits_alone_on_streams_and_in_graphs():
    for rows, classes in ((200, 362), (3, 100003)):
        z, ids, top, dloss = make(rows, classes, 64, "bf16", 19)

        def both():
            loss, stats = r.distill_forward(z, ids, top, None, 2.0)
            return loss, stats, r.distill_backward(z, ids, top, stats, None, 2.0, dloss)

        want = both()
        torch.cuda.synchronize()
        got = []
        for s in [torch.cuda.Stream() for _ in range(3)]:
            with torch.cuda.stream(s):
                got += [both(), both()]
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
            for v in out:
                v.fill_(9)
            gr.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(u, v) for u, v in zip(out, want))


NEAR = [(64, 362, 362), (64, 100, 100), (16, 1024, 1024), (200, 362, 120)]


@pytest.mark.parametrize("temp", [1.0, 4.0, 20.0, 32.0])
@pytest.mark.parametrize("rows,classes,k", NEAR)
def test_student_near_its_teacher(rows, classes, k, temp):
    """The loss is a small difference, about half the noise's variance at any temperature, and its error's bound T^2 P E
    grows with T, to 1024 x 2^-18 = 4e-3 at the highest: 0.8% of a loss of 0.5. The gradient is a difference too, of g q
    and g p, about g q / T: E of g q is T E = 1.3e-4 of it at the highest temperature."""
    z, _, _, dloss = make(rows, classes, 1, "f32", 3, absent=False)
    g = torch.Generator(device="cuda").manual_seed(41)
    ids = torch.rand(z.shape, device="cuda", generator=g).argsort(1)[:, :k].int().contiguous()
    top = z.gather(1, ids.long()) + torch.randn(rows, k, device="cuda", generator=g)
    whole = None if k == classes else torch.logsumexp(torch.scatter(z, 1, ids.long(), top).double() / temp, 1).float()
    loss, stats = r.distill_forward(z, ids, top, whole, temp)
    want, _, _ = r.distill64(z, ids, top, whole, temp)
    _, _, p, _ = r.teacher64(ids, top, whole, classes, temp)
    bound = temp**2 * p.sum(1) * unit(classes, 32 if classes <= 2048 and k <= 128 else 128) + 2.0**-23 * want.abs()
    t.within(loss, want, bound)
    dz = r.distill_backward(z, ids, top, stats, whole, temp, dloss)
    check_backward(z, ids, top, whole, temp, stats, dloss, dz)
    if k == classes:
        assert (bound / want).max() < 0.04 and loss.min() > 0
        assert (bound / want).mean() < 0.011
        exact = torch.stack(r.distill64(z, ids, top, None, temp)[1:], 1)
        full = r.distill_back64(z, ids, top, None, temp, exact, dloss)[0]
        assert (dz.double() - full).norm() <= 2e-4 * full.norm()


@pytest.mark.parametrize("temp", [2.0**-20, 32.0])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,classes,k", [(40, 362, 30), (10, 362, 300), (6, 9001, 64)])
def test_ends_of_the_temperature(rows, classes, k, dtype, temp):
    """Weights are off by 2^-22 (expf) and a rounding: 2^-21 of the terms' sizes, twice with the division by the sum."""
    z, ids, top, dloss = make(rows, classes, k, dtype, 29)
    for scale in (1.0, temp):  # scaled by T: probabilities as at T = 1
        zs, ts = (z.float() * scale).to(z.dtype), top * scale
        loss, stats = r.distill_forward(zs, ids, ts, None, temp)
        want, m, s = r.distill64(zs, ids, ts, None, temp)
        there, _, p, _ = r.teacher64(ids, ts, None, classes, temp)
        at = torch.where(there, ids, 0).long()
        best = torch.where(there, ts.double(), NEG).amax(1, keepdim=True)
        x = ((ts.double() - best) - (zs.double().gather(1, at) - m[:, None])) / temp
        size = torch.where(p > 0, p * x.abs(), 0.0).sum(1)
        e = unit(classes, 32 if classes <= 2048 else 128)
        t.within(loss, want, temp**2 * (p.sum(1) * e + 2.0**-20 * size) + 2.0**-23 * want.abs())
        assert torch.equal(stats[:, 0].double(), m)
        t.within(stats[:, 1], s, e * s)
        dz = r.distill_backward(zs, ids, ts, stats, None, temp, dloss)
        check_backward(zs, ids, ts, None, temp, stats, dloss, dz)


@pytest.mark.parametrize("classes,k", [(362, 20), (362, 200), (9001, 40)])
@pytest.mark.parametrize("given", [False, True])
def test_teachers_that_are_not_finite(classes, k, given):
    """NaN among a row's top logits, or +inf, or NaN as its log sum: loss and gradient of that row are NaN."""
    z, ids, top, dloss = make(6, classes, k, "f32", 37, absent=False)
    whole = torch.logsumexp(top.double(), 1).float() + 0.1 if given else None
    want = r.distill_forward(z, ids, top, whole)
    back = r.distill_backward(z, ids, top, want[1], whole, 1.0, dloss)
    top[1, k // 2] = float("nan")
    ids[2, 1] = ids[2, 0]  # that meet
    top[2, 0] = float("nan")
    top[3, 0] = float("inf")
    if given:
        whole[4] = float("nan")
    else:
        top[4] = float("nan")
    loss, stats = r.distill_forward(z, ids, top, whole)
    dz = r.distill_backward(z, ids, top, stats, whole, 1.0, dloss)
    ok, bad = [0, 5], [1, 2, 3, 4]
    assert loss[bad].isnan().all() and dz[bad].isnan().all()
    assert torch.equal(loss[ok], want[0][ok]) and torch.equal(dz[ok], back[ok])


@pytest.mark.parametrize("classes,k", [(362, 20), (362, 200), (20011, 40)])
@pytest.mark.parametrize("given", [False, True])
def test_light_entries_at_classes_without_probability(classes, k, given):
    """An entry at a logit of -inf makes the loss infinite as long as 64 bits hold its weight, float32 or not."""
    z, ids, top, dloss = make(8, classes, k, "f32", 31, absent=False)
    g = torch.Generator(device="cuda").manual_seed(43)
    ids = torch.rand(8, classes, device="cuda", generator=g).argsort(1)[:, :k].int().contiguous()
    temp = 0.1
    top[:, 0] = top.amax(1) + 1.0
    for i, below in enumerate((0.0, 5.0, 10.0, 10.5, 20.0, 60.0, 100.0)):  # T = 0.1: e^0 to e^-1000
        top[i, 1] = top[i, 0] - below
        z[i, ids[i, 1].long()] = NEG
    whole = torch.logsumexp(top.double() / temp, 1).float() if given else None
    loss, stats = r.distill_forward(z, ids, top, whole, temp)
    assert loss[:6].eq(float("inf")).all() and loss[6:].isfinite().all()
    want = r.distill64(z, ids, top, whole, temp)[0]
    assert torch.equal(loss.isinf(), want.isinf())
    dz = r.distill_backward(z, ids, top, stats, whole, temp, dloss)
    assert dz.isfinite().all()
    check_backward(z, ids, top, whole, temp, stats, dloss, dz)
