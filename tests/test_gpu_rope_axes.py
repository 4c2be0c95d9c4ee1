"""kc_rope_axes and its backward pass against float64.

Tolerances. y = x1 cos - x2 sin: one rounding to the type, and in float32 the sine and cosine are off by at most
2^-21 (angle reduced in 64 bits to half a turn, rounded to 24 bits: 2 pi 2^-26; 2 half steps of 2^-24 more from the
function; sine and cosine of 2-byte types may come from the fast functions, off by 2^-21 more), two products and a sum
by 2 half steps: S = 2^-20 of |x1| + |x2| covers both. The angle itself is a float64 sum: off by 2^-51 of its size.
The frequencies' gradient adds terms pos * d angle, each off by 2 S of its size, over chains of below 128 float32
additions (128 * 2^-24 = 2^-17)."""

import pytest
import torch

import token_ops as t
from katago_cuda import api

pytestmark = pytest.mark.gpu

S = 2.0**-20


def make(tokens, hq, hk, hd, rd, axes, tables, dtype, seed, far=361):
    g = torch.Generator(device="cuda").manual_seed(seed)
    wide = torch.empty(tokens, hq + 2 * hk, hd, device="cuda").normal_(generator=g).to(t.DTYPES[dtype])
    q, k = wide[:, :hq], wide[:, hq:hq + hk] if hk else None
    pos = torch.randint(-far, far, (tokens, axes), device="cuda", generator=g, dtype=torch.int32)
    freqs = torch.empty(tables, rd // 2, axes, device="cuda").normal_(0, 0.5, generator=g)
    return wide, q, k, pos, freqs, g


def check(got, x, pos, freqs, rd, layout, back=False):
    want, size = t.turn64(x, pos, freqs, rd, layout, back)
    half, tiny = t.half_step(x.dtype)
    angle = torch.einsum("ta,hja->thj", pos.double().abs(), freqs.double().abs()).amax()
    t.within(got, want, half * want.abs() + torch.where(size > 0, tiny, 0.0) + (S + angle * 2.0**-51) * size)
    assert torch.equal(got[..., rd:], x[..., rd:])


CASES = [
    # tokens, q heads, k heads, head dim, rotary dim, axes, tables
    (1, 6, 6, 64, 64, 2, 1), (1, 1, 0, 2, 2, 1, 1), (722, 6, 2, 64, 64, 2, 2), (361, 12, 12, 64, 32, 3, 12),
    (100, 16, 4, 128, 96, 3, 1), (33, 4, 4, 102, 102, 2, 4), (50, 3, 1, 30, 10, 4, 1), (17, 8, 2, 16, 16, 1, 2),
    (4099, 2, 1, 64, 48, 3, 1), (9, 2, 2, 1024, 1024, 2, 1), (65, 36, 12, 32, 32, 3, 12), (5, 7, 7, 18, 18, 2, 7),
    (3000, 1, 1, 8, 6, 2, 1), (40, 64, 8, 128, 128, 3, 1),
    (20000, 6, 6, 64, 64, 2, 6), (30011, 8, 2, 64, 48, 4, 2),  # tiles of tokens
    (300, 64, 64, 128, 128, 2, 64),                           # tables beyond shared memory
    (9001, 3, 1, 34, 34, 1, 1), (7000, 5, 5, 20, 12, 3, 5),   # narrower vectors
]


@pytest.mark.parametrize("layout", ["halves", "pairs"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens,hq,hk,hd,rd,axes,tables", CASES)
def test_forward_and_backward(tokens, hq, hk, hd, rd, axes, tables, dtype, layout):
    wide, q, k, pos, freqs, g = make(tokens, hq, hk, hd, rd, axes, tables, dtype, tokens)
    q_out, k_out = t.rope_forward(q, k, pos, freqs, rd, layout)
    check(q_out, q, pos, freqs, rd, layout)
    dq_out = torch.randn(q.shape, device="cuda", generator=g).to(q.dtype)
    dk_out = None
    if k is not None:
        check(k_out, k, pos, freqs, rd, layout)
        dk_out = torch.randn(k.shape, device="cuda", generator=g).to(q.dtype)
    for learned in (True, False):
        grads = torch.full_like(wide, 3.0)
        dq, dk, df = t.rope_backward(dq_out, dk_out, q, k, pos, freqs, rd, layout, dq=grads[:, :hq],
                                     dk=None if k is None else grads[:, hq:hq + hk], learned=learned)
        check(dq, dq_out, pos, freqs, rd, layout, back=True)
        if k is not None:
            check(dk, dk_out, pos, freqs, rd, layout, back=True)
            assert grads[:, hq + hk:].eq(3).all()
        if learned:
            want, size = t.freqs_back64(dq_out, q, dk_out, k, pos, freqs, rd, layout)
            t.within(df, want, (2 * S + 2.0**-17) * size)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("layout", ["halves", "pairs"])
def test_strides_in_place_and_one_buffer(dtype, layout):
    tokens, hq, hk, hd, rd = 77, 6, 2, 64, 48
    wide, q, k, pos, freqs, g = make(tokens, hq, hk, hd, rd, 2, 2, dtype, 3)
    want = t.rope_forward(q, k, pos, freqs, rd, layout)
    # head-major outputs
    qo, ko = (torch.full((h, tokens, hd), 5.0, device="cuda").to(q.dtype).transpose(0, 1) for h in (hq, hk))
    t.rope_forward(q, k, pos, freqs, rd, layout, qo, ko)
    assert torch.equal(qo, want[0]) and torch.equal(ko, want[1])
    # outputs side by side in one buffer with a guard behind each head
    buf = torch.full((tokens, hq + hk, hd + 8), 5.0, device="cuda").to(q.dtype)
    t.rope_forward(q, k, pos, freqs, rd, layout, buf[:, :hq, :hd], buf[:, hq:, :hd])
    assert torch.equal(buf[:, :hq, :hd], want[0]) and torch.equal(buf[:, hq:, :hd], want[1])
    assert buf[:, :, hd:].eq(5).all()
    # rows behind the last token stay as they were
    buf = torch.full((tokens + 3, hq + hk, hd), 5.0, device="cuda").to(q.dtype)
    t.rope_forward(q, k, pos, freqs, rd, layout, buf[:tokens, :hq], buf[:tokens, hq:])
    assert buf[tokens:].eq(5).all()
    # an odd element offset
    flat = torch.zeros(wide.numel() + 8, device="cuda").to(q.dtype)
    off = flat[3:3 + wide.numel()].view_as(wide)
    off.copy_(wide)
    got = t.rope_forward(off[:, :hq], off[:, hq:hq + hk], pos, freqs, rd, layout)
    check(got[0], q, pos, freqs, rd, layout)
    check(got[1], k, pos, freqs, rd, layout)
    # in place, V columns untouched; and the gradient in place
    v = wide[:, hq + hk:].clone()
    dq_out, dk_out = want[0].clone(), want[1].clone()
    q0, k0 = q.clone(), k.clone()
    back = t.rope_backward(dq_out, dk_out, q0, k0, pos, freqs, rd, layout)
    t.rope_forward(q, k, pos, freqs, rd, layout, q, k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(wide[:, hq + hk:], v)
    got = t.rope_backward(dq_out, dk_out, q0, k0, pos, freqs, rd, layout, dq=dq_out, dk=dk_out)
    assert all(torch.equal(a, b) for a, b in zip(got, back))


@pytest.mark.parametrize("tokens", [64, 60000])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_far_positions(dtype, tokens):
    """Positions up to the ends of int32 keep the resolution of one step."""
    wide, q, k, pos, freqs, g = make(tokens, 2, 2, 64, 64, 2, 1, dtype, 7, far=2**31 - 1)
    pos[0] = -2**31
    pos[1] = 2**31 - 1
    q_out, k_out = t.rope_forward(q, k, pos, freqs, 64, "halves")
    check(q_out, q, pos, freqs, 64, "halves")
    check(k_out, k, pos, freqs, 64, "halves")
    # one axis with a frequency of 1: a step at 10^6 turns by what a step at 0 does
    near = torch.arange(8, device="cuda", dtype=torch.int32)[:, None]
    one = torch.ones(1, 1, 1, device="cuda")
    x = torch.ones(8, 1, 2, device="cuda")
    a, _ = t.rope_forward(x, None, near + 1000000, one, 2, "pairs")
    check(a, x, near + 1000000, one, 2, "pairs")


def test_same_as_the_engine_on_a_board():
    """Two axes with the reference's fixed table on a 19x19 board, halves layout: the rotation of the engine's float32
    tier (tables rounded to float32 from float32 angles: 18 * 2^-24 + 2^-24 off)."""
    pos = torch.stack([torch.arange(361) // 19, torch.arange(361) % 19], 1).int().cuda()
    freqs = torch.from_numpy(api.rope_axes_freqs([16, 16], 100.0, 64)).cuda()[None]
    q = torch.randn(361, 6, 64, device="cuda")
    got, _ = t.rope_forward(q, None, pos, freqs, 64, "halves")
    angle = (pos.float()[:, None, :] * freqs).sum(2)[:, None, :]
    c, s = torch.cos(angle), torch.sin(angle)
    want = torch.cat([q[..., :32] * c - q[..., 32:] * s, q[..., :32] * s + q[..., 32:] * c], 2)
    assert (got - want).abs().max() <= 2 * (19 * 2.0**-24 + S) * q.abs().max()


def test_gradient_of_frequencies_is_the_difference_quotient():
    """sum(g * y) along a random direction of the frequencies, in float64: the quotient's error is h^2 / 6 of a third
    derivative, |pos|^2 h^2 / 6 (below 1e-7 at |pos| <= 20, h = 3e-5) of the terms' size."""
    for layout in t.LAYOUTS:
        wide, q, k, pos, freqs, g = make(300, 4, 2, 32, 24, 3, 2, "f32", 13, far=20)
        dq_out, dk_out = (torch.randn(v.shape, device="cuda", generator=g) for v in (q, k))
        _, _, df = t.rope_backward(dq_out, dk_out, q, k, pos, freqs, 24, layout)
        v = torch.randn(freqs.shape, device="cuda", generator=g).double()

        def loss(h):
            f = freqs.double() + h * v
            turned = [t.turn64(x, pos, f, 24, layout)[0] for x in (q, k)]
            return sum((y * o.double()).sum().item() for y, o in zip(turned, (dq_out, dk_out)))

        h = 3e-5
        slope = (loss(h) - loss(-h)) / (2 * h)
        _, size = t.freqs_back64(dq_out, q, dk_out, k, pos, freqs, 24, layout)
        assert abs((df.double() * v).sum().item() - slope) <= (2 * S + 2.0**-17 + 1e-6) * (size * v.abs()).sum().item()


def test_turned_back_is_the_input():
    """The backward pass undoes the rotation: two roundings and 2 S of |x1| + |x2|."""
    wide, q, k, pos, freqs, g = make(500, 6, 6, 64, 64, 2, 6, "f32", 23)
    q_out, k_out = t.rope_forward(q, k, pos, freqs, 64, "halves")
    dq, dk, _ = t.rope_backward(q_out, k_out, q, k, pos, freqs, 64, "halves", learned=False)
    assert (dq - q).abs().max() <= 8 * S * q.abs().max() and (dk - k).abs().max() <= 8 * S * k.abs().max()


def test_same_bits_again_on_other_streams_and_in_graphs():
    wide, q, k, pos, freqs, g = make(2000, 6, 2, 64, 64, 2, 2, "bf16", 29)
    dq_out, dk_out = (torch.randn(v.shape, device="cuda", generator=g).bfloat16() for v in (q, k))

    def both():
        return t.rope_forward(q, k, pos, freqs, 64, "halves") + t.rope_backward(dq_out, dk_out, q, k, pos, freqs, 64,
                                                                                "halves")

    want = both()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(both())
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(a, b) for a, b in zip(r, want))
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            r = both()
        graphs.append((gr, r))
    for _ in range(3):
        for gr, r in graphs:
            for v in r:
                v.fill_(9)
        torch.cuda.synchronize()
        for s, (gr, r) in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        for gr, r in graphs:
            assert all(torch.equal(a, b) for a, b in zip(r, want))


def test_offsets_past_32_bits():
    far = (1 << 31) + 64
    wide, q, k, pos, freqs, g = make(3, 2, 1, 64, 64, 2, 1, "f16", 31)
    want = t.rope_forward(q, k, pos, freqs, 64, "pairs")
    buf = torch.empty(2 * far + 256, dtype=torch.float16, device="cuda")
    qf, kf = buf.as_strided((3, 2, 64), (far, 64, 1)), buf[128:].as_strided((3, 1, 64), (far, 64, 1))
    qf.copy_(q)
    kf.copy_(k)
    dq_out, dk_out = (torch.randn(v.shape, device="cuda", generator=g).half() for v in (q, k))
    dq, dk, df = t.rope_backward(dq_out, dk_out, q, k, pos, freqs, 64, "pairs")
    check(dq, dq_out, pos, freqs, 64, "pairs", back=True)
    wantf, size = t.freqs_back64(dq_out, q, dk_out, k, pos, freqs, 64, "pairs")
    far_grads = torch.empty(2 * far + 256, dtype=torch.float16, device="cuda")
    gq, gk = far_grads.as_strided((3, 2, 64), (far, 64, 1)), far_grads[128:].as_strided((3, 1, 64), (far, 64, 1))
    _, _, df = t.rope_backward(dq_out, dk_out, qf, kf, pos, freqs, 64, "pairs", dq=gq, dk=gk)
    assert torch.equal(gq, dq) and torch.equal(gk, dk)
    t.within(df, wantf, (2 * S + 2.0**-17) * size)
    t.rope_forward(qf, kf, pos, freqs, 64, "pairs", qf, kf)
    assert torch.equal(qf, want[0]) and torch.equal(kf, want[1])


@pytest.mark.parametrize("tokens", [50, 40000])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_frequencies_that_are_not_finite(tokens, bad):
    """They make their own pairs NaN and nothing else."""
    wide, q, k, pos, freqs, g = make(tokens, 4, 2, 32, 32, 2, 2, "bf16", 41)
    want = t.rope_forward(q, k, pos, freqs, 32, "halves")
    freqs[1, 5, 0] = bad
    got = t.rope_forward(q, k, pos, freqs, 32, "halves")
    for a, w, per in zip(got, want, (2, 1)):
        hit = torch.zeros(w.shape[1:], dtype=torch.bool, device="cuda")
        hit[per:, 5] = hit[per:, 21] = True
        assert torch.isnan(a[:, hit]).all() and torch.equal(a[:, ~hit], w[:, ~hit])
    dq, dk, df = t.rope_backward(want[0], want[1], q, k, pos, freqs, 32, "halves")
    assert torch.isnan(df[1, 5]).all() and torch.isfinite(df[0]).all() and torch.isfinite(df[1, 6:]).all()


def test_no_tokens():
    d = api.RopeDesc(api.PRECISION_F16, api.ROPE_HALVES, 2, 0, 6, 2, 64, 64, 2)
    df = torch.full((2, 32, 2), 5.0, device="cuda")
    api.rope_axes_backward(d, 0, 0, 0, 0, 0, 0, 0, 0, df.data_ptr(), 0, 0, t.stream())
    assert df.eq(0).all()


def test_host_memory_is_refused():
    wide, q, k, pos, freqs, g = make(4, 2, 2, 16, 16, 2, 1, "f32", 37)
    d = t.rope_desc(q, k, q, k, 16, "halves", 2, 1)
    with pytest.raises(api.KcError) as e:
        api.rope_axes(d, q.data_ptr(), k.data_ptr(), pos.cpu().data_ptr(), freqs.data_ptr(), q.data_ptr(), k.data_ptr(),
                      t.stream())
    assert e.value.status == api.KC_ERR_INVALID and "device memory" in str(e.value)


def learned_backward(tokens, hq, hk, hd, axes, tables, dtype):
    """One backward pass with the frequencies' gradient, against float64."""
    wide, q, k, pos, freqs, g = make(tokens, hq, hk, hd, hd, axes, tables, dtype, 43)
    dq_out, dk_out = (torch.randn(v.shape, device="cuda", generator=g).to(q.dtype) for v in (q, k))
    dq, dk, df = t.rope_backward(dq_out, dk_out, q, k, pos, freqs, hd, "halves")
    check(dq, dq_out, pos, freqs, hd, "halves", back=True)
    check(dk, dk_out, pos, freqs, hd, "halves", back=True)
    want, size = t.freqs_back64(dq_out, q, dk_out, k, pos, freqs, hd, "halves")
    t.within(df, want, (2 * S + 2.0**-17) * size)


@pytest.mark.parametrize("tokens,hq,hk,hd,axes,tables,dtype", [
    (4440, 12, 12, 64, 4, 12, "bf16"), (13804, 12, 12, 96, 2, 12, "bf16"), (20000, 12, 12, 64, 4, 12, "f16")])
def test_first_call_with_tiles_near_48_kb(tokens, hq, hk, hd, axes, tables, dtype):
    """The tiles alone stay below the 48 KB that a block gets unasked, with the kernel's own shared memory they pass
    it. A fresh process each: an earlier call of the same kernel may have raised its limit."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    code = "import sys; sys.path[:0] = %r; import test_gpu_rope_axes as m; m.learned_backward%r" % (
        [here, os.path.join(os.path.dirname(here), "katago-rs_b200", "python")],
        (tokens, hq, hk, hd, axes, tables, dtype))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("tokens", [64, 60000])
def test_far_positions_with_small_frequencies(tokens, sign):
    """Frequencies of either sign keep their digits at the far end of int32. The rotated (1, 0) is (cos, sin): the
    angle is off by the rounding of half a turn to 24 bits, pi 2^-25, and 3e-9 of the fraction and the float64
    reference; the function by 2^-24, the result's rounding by 2^-24 and the sum's by another: below 2^-21 in all."""
    g = torch.Generator(device="cuda").manual_seed(47)
    pos = torch.randint(2**30, 2**31 - 1, (tokens, 1), device="cuda", generator=g, dtype=torch.int32)
    freqs = sign * torch.empty(1, 32, 1, device="cuda").uniform_(1e-4, 1e-2, generator=g)
    x = torch.cat([torch.ones(tokens, 2, 32, device="cuda"), torch.zeros(tokens, 2, 32, device="cuda")], 2)
    q_out, _ = t.rope_forward(x, None, pos, freqs, 64, "halves")
    want, _ = t.turn64(x, pos, freqs, 64, "halves")
    t.within(q_out, want, 2.0**-21)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,tables,hd", [(1, 1, 1024), (2, 2, 256), (64, 64, 128)])  # (64: beyond shared memory)
def test_gradient_of_frequencies_has_float32_sines(heads, tables, hd, dtype):
    """It is float32 whatever the heads' type. One token at position 1 with x = (1, 0): the gradient is cos for
    g = (0, 1) and sin for g = (-1, 0), every product and sum of it exact. The angle is off by pi 2^-25 (half a turn
    in 24 bits) and 2^-52 more, sine and cosine by 2^-24: below 2^-22."""
    g = torch.Generator(device="cuda").manual_seed(53)
    freqs = torch.empty(tables, hd // 2, 1, device="cuda").uniform_(-3.1, 3.1, generator=g)
    pos = torch.ones(1, 1, dtype=torch.int32, device="cuda")
    x = torch.cat([torch.ones(1, heads, hd // 2, device="cuda"), torch.zeros(1, heads, hd // 2, device="cuda")], 2)
    x = x.to(t.DTYPES[dtype])
    for dy, want in ((x.roll(hd // 2, 2), torch.cos(freqs.double())), (-x, torch.sin(freqs.double()))):
        _, _, df = t.rope_backward(dy, None, x, None, pos, freqs, hd, "halves")
        t.within(df, want, 2.0**-22)


def test_strides_that_no_address_needs():
    """One token, one head, no k: the strides between tokens, heads and k heads may be any."""
    for tokens, hq in ((1, 4), (5000, 1)):
        wide, q, _, pos, freqs, g = make(tokens, hq, 0, 64, 64, 2, 1, "bf16", 67)
        q = q.contiguous()
        dq_out = torch.randn(q.shape, device="cuda", generator=g).bfloat16()
        want = t.rope_forward(q, None, pos, freqs, 64, "halves")
        back = t.rope_backward(dq_out, None, q, None, pos, freqs, 64, "halves")
        st = (hq * 64 if tokens > 1 else 1 << 62, 64 if hq > 1 else (1 << 63) - 1)
        d = api.RopeDesc(api.PRECISION_BF16, api.ROPE_HALVES, 2, tokens, hq, 0, 64, 64, 1, q_strides=st,
                         k_strides=(1 << 62, -1), q_out_strides=st, k_out_strides=(-1, 1 << 62))
        y, dq, df = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(freqs)
        api.rope_axes(d, q.data_ptr(), 0, pos.data_ptr(), freqs.data_ptr(), y.data_ptr(), 0, t.stream())
        size = api.rope_axes_backward_workspace(d)
        ws = t.workspace(size, q.device)
        api.rope_axes_backward(d, dq_out.data_ptr(), 0, q.data_ptr(), 0, pos.data_ptr(), freqs.data_ptr(),
                               dq.data_ptr(), 0, df.data_ptr(), t.ptr(ws), size, t.stream())
        assert torch.equal(y, want[0]) and torch.equal(dq, back[0]) and torch.equal(df, back[2])
