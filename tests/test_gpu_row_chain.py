"""The operators in a row, as a distillation step of a small token net uses them: rows of moves and of points looked up and
added, RMS norm, a linear, layer norm, a policy linear, the loss against a teacher's top logits; backward through all of
it, against the same chain in float64."""

import threading

import pytest
import torch

import row_ops as r
import token_ops as t

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def full_products():
    before = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    yield
    torch.backends.cuda.matmul.allow_tf32 = before


def test_distillation_step():
    """float32 throughout: each operator is within 2^-17 of its terms, and the linears and norms pass relative errors on
    with factors of about 10: 1e-3 of the largest value is far above that and far below any wrong row, mask or weight."""
    n, points, channels, classes, k, temp = 6, 361, 96, 362, 24, 2.0
    g = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    moves, places = rand(classes + 1, channels) * 0.3, rand(points, channels) * 0.3
    w1, w2, b2 = 1 + 0.2 * rand(channels), 1 + 0.2 * rand(channels), 0.2 * rand(channels)
    lin, head = rand(channels, channels) / channels**0.5, rand(channels, classes) / channels**0.5 * 3
    tokens = n * points
    move_ids = torch.randint(-1, classes + 1, (tokens,), device="cuda", generator=g, dtype=torch.int32)
    place_ids = (torch.arange(tokens, device="cuda") % points).int()
    side = torch.tensor([19, 13, 9, 19, 13, 9], device="cuda")[:, None]
    p = torch.arange(points, device="cuda")
    mask = ((p % 19 < side) & (p // 19 < side)).float()
    on = mask != 0
    ids = rand(n, classes).argsort(1)[:, :k].int().contiguous()
    ids[2] = -1
    top, dloss = 2 * rand(n, k), rand(n).abs()

    # the library's operators around torch's products
    x0 = r.embed_forward(move_ids, moves, None, 2.0)
    x0 = r.embed_forward(place_ids, places, x0, 1.0, y=x0).view(n, points, channels)
    y1, st1 = r.layer_forward(x0, mask, w1, None, "rms")
    h = (y1.view(-1, channels) @ lin).view(n, points, channels)
    y2, st2 = r.layer_forward(h, mask, w2, b2, "layer")
    pooled = y2.sum(1) / on.sum(1, keepdim=True)
    logits = pooled @ head
    loss, stats = r.distill_forward(logits, ids, top, None, temp)
    dlogits = r.distill_backward(logits, ids, top, stats, None, temp, dloss)
    dpooled = dlogits @ head.T / on.sum(1, keepdim=True)
    dy2 = dpooled[:, None, :].expand(n, points, channels).contiguous()
    dh, dw2, db2 = r.layer_backward(h, mask, w2, st2, dy2, "layer")
    dy1 = (dh.view(-1, channels) @ lin.T).view(n, points, channels)
    dx0, dw1, _ = r.layer_backward(x0, mask, w1, st1, dy1, "rms")
    dx0 = dx0.view(tokens, channels)
    dmoves, dplaces = r.embed_backward(move_ids, dx0, classes + 1, 2.0), r.embed_backward(place_ids, dx0, points)

    # float64
    leaves = [v.double().requires_grad_() for v in (moves, places, w1, w2, b2)]
    md, pd, w1d, w2d, b2d = leaves
    there = (move_ids >= 0)[:, None]
    x = torch.where(there, md[move_ids.clamp(min=0).long()] * 2.0, 0.0) + pd[place_ids.long()]
    y = r.layer64(x.view(n, points, channels), on, w1d, None, "rms")[0]
    y = r.layer64((y.view(-1, channels) @ lin.double()).view(n, points, channels), on, w2d, b2d, "layer")[0]
    z = (y.sum(1) / on.sum(1, keepdim=True)) @ head.double()
    some = (ids >= 0).any(1)
    tt = torch.where(some[:, None], top.double() / temp, 0.0)
    lp = torch.log_softmax(tt, 1)
    lq = torch.log_softmax(z / temp, 1).gather(1, ids.clamp(min=0).long())
    want = torch.where(some, temp**2 * (lp.exp() * (lp - lq)).sum(1), 0.0)
    grads = torch.autograd.grad((want * dloss.double()).sum(), leaves)
    for got, ref in ((loss, want.detach()), (dmoves, grads[0]), (dplaces, grads[1]), (dw1, grads[2]), (dw2, grads[3]),
                     (db2, grads[4])):
        assert (got.double() - ref).abs().max() <= 1e-3 * ref.abs().max()
    assert loss[2] == 0 and dlogits[2].eq(0).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_one_token_at_a_time(dtype):
    """A token alone gives the bits that it has in a sequence, through the lookup and the norms."""
    tokens, channels, rows = 700, 384, 362
    g = torch.Generator(device="cuda").manual_seed(5)
    table = torch.randn(rows, channels, device="cuda", generator=g).to(t.DTYPES[dtype])
    ids = torch.randint(-1, rows, (tokens,), device="cuda", generator=g, dtype=torch.int32)
    w = torch.rand(channels, device="cuda", generator=g) + 0.5

    def run(ids):
        x = r.embed_forward(ids, table, None, 1.5)
        y, _ = r.layer_forward(x[None], None, w, None, "rms")
        return r.layer_forward(y, None, w, w, "layer")[0][0]

    want = run(ids)
    for i in range(0, tokens, 97):
        assert torch.equal(run(ids[i:i + 1])[0], want[i])


def test_host_threads_on_streams_of_their_own():
    """Four host threads, each on its own stream, while the others call too: the same bits as alone."""

    def work(seed, out):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        x = rand(4, 361, 96 + 40 * seed).bfloat16()
        w = rand(x.shape[2])
        ids = torch.randint(0, 50, (4 * 361 * (1 + 2 * seed),), device="cuda", generator=g, dtype=torch.int32)
        dy = rand(ids.shape[0], 64).half()
        z, top = rand(30, 900 * (1 + 2 * seed)), rand(30, 20)
        tid = torch.randint(0, 900, (30, 20), device="cuda", generator=g, dtype=torch.int32)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            for _ in range(20):
                y, st = r.layer_forward(x, None, w, w, "layer")
                res = (y, st) + r.layer_backward(x, None, w, st, x, "layer")
                res += (r.embed_backward(ids, dy, 50),)
                loss, stats = r.distill_forward(z, tid, top)
                res += (loss, stats, r.distill_backward(z, tid, top, stats))
        stream.synchronize()
        out[seed] = res

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


def test_first_calls_in_a_capture():
    """A fresh process whose first call of each kernel is captured into a graph."""
    import os
    import subprocess
    import sys
    code = """
import sys, torch
sys.path[:0] = [%r, %r]
import row_ops as r
x = [torch.randn(40, 50, c, device="cuda").bfloat16() for c in (96, 2000, 20000)] + [
    torch.randn(40, 50, 99, device="cuda")[:, :, 1:98]]
w = [torch.ones(v.shape[2], device="cuda") for v in x]
ids = [torch.arange(n, device="cuda").int() %% 300 for n in (500, 30000, 200000)]
dy = [torch.randn(i.shape[0], 16, device="cuda") for i in ids]
z = [torch.randn(n, c, device="cuda").half() for n, c in ((500, 362), (1300, 5000), (2, 90000))]
tid = [torch.zeros(v.shape[0], 40, device="cuda").int() for v in z]
top = [torch.zeros(v.shape[0], 40, device="cuda") for v in z]


def everything():
    out = []
    for v, u in zip(x, w):
        y, st = r.layer_forward(v, None, u, u, "layer")
        out += [y, st, *r.layer_backward(v, None, u, st, y, "layer")]
        y, st = r.layer_forward(v, None, u, None, "rms")
        out += [y, st, *r.layer_backward(v, None, u, st, y, "rms")]
    for i, d in zip(ids, dy):
        out += [r.embed_forward(i, d[:300], d), r.embed_backward(i, d, 300)]
    for v, i, t in zip(z, tid, top):
        loss, st = r.distill_forward(v, i, t)
        out += [loss, st, r.distill_backward(v, i, t, st)]
    return out


g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = everything()
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, everything()))
print("captured")
"""
    here = os.path.dirname(os.path.abspath(__file__))
    code = code % (here, os.path.join(os.path.dirname(here), "katago-rs_b200", "python"))
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured" in done.stdout, done.stdout + done.stderr


def test_offsets_beyond_32_bits():
    """Boards, table rows and logit rows 2^31 elements apart (and an odd number more). Lookups and losses have the bits of
    single rows; norms are within 2^-10 of the value (half a step of f16 is 2^-11) and 2^-12 of a standard deviation."""
    buf = torch.zeros(2**31 + 70000, device="cuda", dtype=torch.float16)
    out = torch.zeros(2**31 + 70000, device="cuda", dtype=torch.float16)
    for far in (2**31, 2**31 + 7):
        g = torch.Generator(device="cuda").manual_seed(7)
        v = torch.randn(2, 5, 384, device="cuda", generator=g).half()
        w = torch.rand(384, device="cuda", generator=g)
        x, y = (b.as_strided((2, 5, 384), (far, 384, 1)) for b in (buf, out))
        x.copy_(v)
        got = r.layer_forward(x, None, w, w, "layer", y=y)
        on = torch.ones(2, 5, dtype=torch.bool, device="cuda")
        want = r.layer64(v, on, w, w, "layer")[0]
        assert ((y.double() - want).abs() <= 2.0**-10 * want.abs() + 2.0**-12).all()
        dx = r.layer_backward(x, None, w, got[1], y, "layer", dx=buf.as_strided((2, 5, 384), (far, 384, 1)))[0]
        want = r.layer_back64(v, on, w, got[1][..., 0], got[1][..., 1], y, "layer")[0]
        assert ((dx.double() - want).abs() <= 2.0**-10 * want.abs() + 2.0**-12).all()

        table, rows = (b.as_strided((2, 384), (far, 1)) for b in (buf, out))
        table.copy_(v[:, 0])
        ids = torch.tensor([1, 0], device="cuda", dtype=torch.int32)
        r.embed_forward(ids, table, table, 1.0, y=rows)
        assert torch.equal(rows, (v[:, 0].float().flip(0) + v[:, 0].float()).half())
        grad = r.embed_backward(ids, rows, 2)
        assert torch.equal(grad, rows.float().flip(0))

        for classes in (362, 30000):
            z = buf.as_strided((2, classes), (far, 1))
            z.copy_(torch.randn(2, classes, device="cuda", generator=g))
            tid = torch.randint(0, classes, (2, 9), device="cuda", generator=g, dtype=torch.int32)
            top = torch.randn(2, 9, device="cuda", generator=g)
            loss, st = r.distill_forward(z, tid, top)
            dz = r.distill_backward(z, tid, top, st, dz=out.as_strided((2, classes), (far, 1)))
            for i in range(2):
                l1, s1 = r.distill_forward(z[i:i + 1], tid[i:i + 1], top[i:i + 1])
                assert torch.equal(loss[i:i + 1], l1) and torch.equal(st[i:i + 1], s1)
                assert torch.equal(dz[i:i + 1], r.distill_backward(z[i:i + 1], tid[i:i + 1], top[i:i + 1], s1))
