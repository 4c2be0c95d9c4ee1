"""The operators in a row, as a block uses them: masked group norm with activation of a trunk of several positions of
a game, the Q | K | V linear, rotary positions (move, row, column) on Q and K in place in the linear's output, and
attention over the tokens; forward and backward, against the same chain in float64."""

import pytest
import torch

import token_ops as t
from katago_cuda import api

pytestmark = pytest.mark.gpu


def positions(moves, points):
    p = torch.arange(moves * points, device="cuda")
    return torch.stack([p // points, p % points // 19, p % points % 19], 1).int()


def attend(q, k, v, on):
    """softmax(q k^T / sqrt(d)) v over the tokens that are on; q [boards][tokens][heads][d], shared K heads."""
    group = q.shape[2] // k.shape[2]
    k, v = k.repeat_interleave(group, 2), v.repeat_interleave(group, 2)
    s = torch.einsum("bthd,bshd->bhts", q, k) / q.shape[3] ** 0.5
    s = s.masked_fill(~on[:, None, None, :], float("-inf"))
    return torch.einsum("bhts,bshd->bthd", torch.softmax(s, 3), v)


@pytest.mark.parametrize("act", ["mish", "silu"])
def test_block(act):
    """float32 throughout (matmuls without reduced-precision products): each operator is within 2^-17 of its terms, and
    the chain's linear and softmax pass relative errors on with factors of about 10: 1e-3 of the largest value is far
    above that and far below any wrong angle, mask or statistic."""
    n, moves, channels, groups, hq, hk, hd = 3, 2, 96, 8, 4, 2, 32
    points = moves * 361
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x, w, b = r(n, points, channels), 1 + 0.2 * r(channels), 0.2 * r(channels)
    wqkv = r(channels, (hq + 2 * hk) * hd) / channels**0.5
    side = torch.tensor([19, 13, 9], device="cuda")[:, None]
    p = torch.arange(points, device="cuda") % 361
    mask = ((p % 19 < side) & (p // 19 < side)).float()
    on = mask != 0
    pos = positions(moves, 361).repeat(n, 1)
    freqs = torch.from_numpy(api.rope_axes_freqs([4, 6, 6], 100.0, hd)).cuda()[None].repeat(hk, 1, 1)
    do = r(n, points, hq, hd) * mask[:, :, None, None]

    # the framework's operators around torch's products
    y, stats = t.norm_forward(x, mask, w, b, groups, act)
    qkv = (y.reshape(-1, channels) @ wqkv).view(n * points, hq + 2 * hk, hd)
    before = qkv.clone()
    q, k = qkv[:, :hq], qkv[:, hq:hq + hk]
    t.rope_forward(q, k, pos, freqs, hd, "halves", q, k)
    leaf = qkv.detach().view(n, points, -1, hd).clone().requires_grad_()
    out = attend(leaf[:, :, :hq], leaf[:, :, hq:hq + hk], leaf[:, :, hq + hk:], on)
    (dqkv,) = torch.autograd.grad(out, leaf, do)
    dqkv = dqkv.reshape(n * points, -1, hd).contiguous()
    dq, dk = dqkv[:, :hq], dqkv[:, hq:hq + hk]
    _, _, dfreqs = t.rope_backward(dq, dk, before[:, :hq], before[:, hq:hq + hk], pos, freqs, hd, "halves", dq=dq,
                                   dk=dk)
    dy = (dqkv.reshape(n * points, -1) @ wqkv.T).view(n, points, channels)
    dx, dw, db = t.norm_backward(x, mask, w, b, stats, dy, groups, act)

    # float64
    leaves = [v.double().requires_grad_() for v in (x, w, b, freqs)]
    xd, wd, bd, fd = leaves
    yd = t.norm64(xd, on, wd, bd, groups, act)[0]
    qd = (yd.reshape(-1, channels) @ wqkv.double()).view(n * points, -1, hd)
    turned = [t.turn64(v, pos, fd, hd, "halves")[0] for v in (qd[:, :hq], qd[:, hq:hq + hk])]
    od = attend(*(v.reshape(n, points, -1, hd) for v in (*turned, qd[:, hq + hk:])), on)
    want = torch.autograd.grad(od, leaves, do.double())
    keep = on[:, :, None, None]
    for got, ref in ((torch.where(keep, out, 0.0), torch.where(keep, od, 0.0)), (dx, want[0]), (dw, want[1]),
                     (db, want[2]), (dfreqs, want[3])):
        assert (got.double() - ref).abs().max() <= 1e-3 * ref.abs().max()
    assert dx[~on].eq(0).all() and y[~on].eq(0).all()


def test_single_token_serving():
    """One token at a time (n = 1, points = 1) gives what the whole sequence gives where statistics do not mix tokens
    (rotary positions), bit for bit."""
    tokens, hq, hk, hd = 12, 6, 2, 64
    q, k = (torch.randn(tokens, h, hd, device="cuda").bfloat16() for h in (hq, hk))
    pos = positions(1, 361)[:tokens].contiguous()
    freqs = torch.randn(hk, hd // 2, 3, device="cuda")
    want = t.rope_forward(q, k, pos, freqs, hd, "pairs")
    for i in range(tokens):
        got = t.rope_forward(q[i:i + 1], k[i:i + 1], pos[i:i + 1], freqs, hd, "pairs")
        assert torch.equal(got[0][0], want[0][i]) and torch.equal(got[1][0], want[1][i])


def test_host_threads_on_streams_of_their_own():
    """Four host threads, each on its own stream, while the others call too: the same bits as alone."""
    import threading

    def work(seed, out):
        g = torch.Generator(device="cuda").manual_seed(seed)
        x = torch.randn(20, 361, 48 + 24 * seed, device="cuda", generator=g).bfloat16()
        w, b = torch.ones(x.shape[2], device="cuda"), torch.zeros(x.shape[2], device="cuda")
        q = torch.randn(4000, 4, 64, device="cuda", generator=g).bfloat16()
        pos = torch.randint(0, 361, (4000, 2), device="cuda", generator=g, dtype=torch.int32)
        freqs = torch.randn(2, 32, 2, device="cuda", generator=g)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            for _ in range(20):
                y, stats = t.norm_forward(x, None, w, b, 6, "mish")
                r = (y, stats) + t.norm_backward(x, None, w, b, stats, x, 6, "mish")
                r += t.rope_forward(q, q, pos, freqs, 64, "halves")
                r += t.rope_backward(q, q, q, q, pos, freqs, 64, "halves")
        stream.synchronize()
        out[seed] = r

    alone, together = {}, {}
    for seed in range(4):
        work(seed, alone)
    threads = [threading.Thread(target=work, args=(seed, together)) for seed in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    for seed in range(4):
        assert all(torch.equal(a, c) for a, c in zip(alone[seed], together[seed]))


@pytest.mark.parametrize("layout", ["halves", "pairs"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_single_token_is_the_long_sequence(dtype, layout):
    """One token at a time gives the bits of a sequence long enough for the kernel that goes over tiles of tokens."""
    tokens, hq, hk, hd = 20000, 6, 2, 64
    g = torch.Generator(device="cuda").manual_seed(59)
    q, k = (torch.randn(tokens, h, hd, device="cuda", generator=g).to(t.DTYPES[dtype]) for h in (hq, hk))
    pos = torch.randint(-400, 400, (tokens, 3), device="cuda", generator=g, dtype=torch.int32)
    freqs = torch.randn(hk, hd // 2, 3, device="cuda", generator=g)
    want = t.rope_forward(q, k, pos, freqs, hd, layout)
    for i in range(0, tokens, 397):
        got = t.rope_forward(q[i:i + 1], k[i:i + 1], pos[i:i + 1], freqs, hd, layout)
        assert torch.equal(got[0][0], want[0][i]) and torch.equal(got[1][0], want[1][i])
    few = t.rope_forward(q[:40], k[:40], pos[:40], freqs, hd, layout)
    assert torch.equal(few[0], want[0][:40]) and torch.equal(few[1], want[1][:40])
