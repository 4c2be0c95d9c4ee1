"""kc_embed_rows and its backward pass against float64.

Tolerances. Forward: one fused product and sum in float32 and the rounding to the type. Backward: a row's sum is at most
its count of float32 additions, and no chain of them is longer than a piece (256), two runs of each of a block's pieces
(256), an eighth of the blocks and 8 (below 150 at these sizes): N = min(count, 700) roundings of the sum of the sizes,
and one of the scale."""

import pytest
import torch

import row_ops as r
import token_ops as t
from katago_cuda import api

pytestmark = pytest.mark.gpu


def make(tokens, channels, rows, dtype, seed, kind="even", pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    wide = lambda n: torch.empty(n, channels + pad, device="cuda").normal_(generator=g).to(t.DTYPES[dtype])  # noqa: E731
    u = torch.rand(tokens, device="cuda", generator=g)
    if kind == "skewed":
        u = u**8
    ids = (u * rows).int().clamp(max=rows - 1)
    if kind == "one":
        ids.fill_(rows // 2)
    if kind == "points":
        ids = (torch.arange(tokens, device="cuda") % rows).int()
    if kind == "padded":  # ids outside the table, the ends of int32 among them
        out = torch.tensor([-1, rows, -2**31, 2**31 - 1], device="cuda", dtype=torch.int32)
        ids = torch.where(torch.rand(tokens, device="cuda", generator=g) < 0.3,
                          out[torch.arange(tokens, device="cuda") % 4], ids)
    return ids, wide(rows)[:, :channels], wide(tokens)[:, :channels], g


def check_forward(got, ids, table, x, scale):
    want = r.embed64(ids, table, x, scale)
    half, tiny = t.half_step(table.dtype)
    t.within(got, want, (half + 2.0**-24) * want.abs() + tiny)


def check_backward(got, ids, dy, rows, scale):
    want, size, count = r.embed_back64(ids, dy, rows, scale)
    t.within(got, want, 2.0**-24 * (count.clamp(max=700)[:, None] * size + want.abs()))
    assert got[count == 0].eq(0).all()


CASES = [
    # tokens, channels, table rows, ids, pad
    (1, 384, 362, "even", 0), (1, 1, 1, "even", 0), (361, 384, 362, "points", 0), (361, 768, 5776, "even", 0),
    (1000, 100, 3, "even", 4), (777, 99, 50, "skewed", 0), (5000, 64, 1, "one", 0), (2048, 16, 513, "padded", 3),
    (2049, 8, 511, "padded", 0), (30000, 96, 362, "skewed", 0), (20000, 48, 70000, "even", 0),
    (9000, 33, 100000, "padded", 0), (40000, 40, 7, "skewed", 8), (60000, 24, 300, "one", 0), (3, 20000, 5, "even", 0),
    (4100, 2, 1 << 18, "skewed", 0), (100, 7, 1, "padded", 0), (6000, 260, 1 << 9, "points", 0), (17, 512, 2, "one", 0),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens,channels,rows,kind,pad", CASES)
def test_forward_and_backward(tokens, channels, rows, kind, pad, dtype):
    ids, table, x, g = make(tokens, channels, rows, dtype, tokens + channels, kind, pad)
    scale = channels**0.5
    check_forward(r.embed_forward(ids, table, None, scale), ids, table, None, scale)
    check_forward(r.embed_forward(ids, table, x, scale), ids, table, x, scale)
    check_backward(r.embed_backward(ids, x, rows, scale), ids, x, rows, scale)


@pytest.mark.parametrize("kind", ["skewed", "one", "even"])
def test_many_tokens(kind):
    """Pieces of their largest size, sorts of many tiles, runs over hundreds of blocks."""
    ids, _, dy, _ = make(1500000, 8, 1000, "bf16", 3, kind)
    check_backward(r.embed_backward(ids, dy, 1000), ids, dy, 1000, 1.0)
    ids, _, dy, _ = make(300000, 32, 3000000 // 32, "f32", 5, kind)
    check_backward(r.embed_backward(ids, dy, 3000000 // 32, -0.5), ids, dy, 3000000 // 32, -0.5)


@pytest.mark.parametrize("tokens", [1, 31, 32, 33, 255, 256, 511, 1024, 2047, 2048, 2049, 16383, 16384, 16385, 131072,
                                    131073])
@pytest.mark.parametrize("kind", ["skewed", "one", "padded"])
def test_ends_of_the_ways_to_sort(tokens, kind):
    """In a block's shared memory, by clusters of 1 to 16 blocks, by launches; digits of 1, 9 and 2 x 6 bits."""
    for channels, rows, dtype in ((8, 1, "f32"), (16, 500, "bf16"), (4, 4000, "f16")):
        ids, _, dy, _ = make(tokens, channels, rows, dtype, tokens, kind)
        check_backward(r.embed_backward(ids, dy, rows, 1.5), ids, dy, rows, 1.5)


def test_three_digits():
    ids, table, dy, _ = make(10000, 4, 1 << 20, "f32", 7, "padded")
    check_backward(r.embed_backward(ids, dy, 1 << 20), ids, dy, 1 << 20, 1.0)
    ids, table, dy, _ = make(1000, 1, (1 << 27) + 3, "f16", 7, "padded")
    got = r.embed_backward(ids, dy, (1 << 27) + 3)
    there = (ids >= 0) & (ids <= 1 << 27)
    assert int((got != 0).sum()) <= int(there.sum())
    at = ids[there].long()
    want = torch.zeros_like(got).index_add_(0, at, dy[there].float())
    t.within(got[at], want[at].double(), 2.0**-22 * want[at].double().abs() + 2.0**-20)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("channels", [64, 100, 33, 1, 1001, 2000])
def test_strides_guards_and_in_place(dtype, channels):
    tokens, rows = 500, 40
    ids, table, x, g = make(tokens, channels, rows, dtype, 11)
    want, back = r.embed_forward(ids, table, x, 0.5), r.embed_backward(ids, x, rows, 0.5)
    for off in (0, 8, 1):
        buf = torch.full((tokens + 2, channels + 24), 5.0, device="cuda").to(x.dtype)
        out = buf[1:1 + tokens, off:off + channels]
        tb, xb = (torch.zeros(v.shape[0], channels + 16, device="cuda").to(x.dtype)[:, off:off + channels]
                  for v in (table, x))
        tb.copy_(table), xb.copy_(x)
        r.embed_forward(ids, tb, xb, 0.5, y=out)
        assert torch.equal(out, want)
        keep = torch.ones_like(buf, dtype=torch.bool)
        keep[1:1 + tokens, off:off + channels] = False
        assert buf[keep].eq(5).all()
        r.embed_forward(ids, tb, xb, 0.5, y=xb)  # in place
        assert torch.equal(xb, want)
        xb.copy_(x)
        check_backward(r.embed_backward(ids, xb, rows, 0.5), ids, x, rows, 0.5)
        guard = torch.full((rows + 2, channels), 5.0, device="cuda")
        flat = torch.full((rows * channels + 8,), 5.0, device="cuda")
        odd = flat[3:3 + rows * channels].view(rows, channels)
        r.embed_backward(ids, x, rows, 0.5, dtable=guard[1:1 + rows])
        r.embed_backward(ids, x, rows, 0.5, dtable=odd)
        assert torch.equal(guard[1:1 + rows], back) and torch.equal(odd, back)
        assert guard[0].eq(5).all() and guard[-1].eq(5).all() and flat[:3].eq(5).all() and flat[-5:].eq(5).all()
    # one token's gradient for all: rows at stride 0
    one = x[:1].expand(tokens, channels)
    check_backward(r.embed_backward(ids, one, rows), ids, one, rows, 1.0)


def test_padding_has_no_effect():
    """NaN in dy at ids outside the table; a table row that no token has may hold anything."""
    ids, table, x, g = make(3000, 96, 50, "bf16", 13, "padded")
    out = (ids < 0) | (ids >= 50)
    want = r.embed_backward(ids, x, 50)
    bad = torch.where(out[:, None], float("nan"), x.float()).to(x.dtype)
    assert torch.equal(r.embed_backward(ids, bad, 50), want) and want.isfinite().all()
    assert torch.equal(r.embed_forward(ids, table, x)[out], x[out])
    assert r.embed_forward(ids, table)[out].eq(0).all()
    none = torch.full_like(ids, -1)
    assert r.embed_backward(none, bad, 50).eq(0).all()
    ids = torch.where(ids == 7, 8, ids)
    table[7] = float("nan")
    assert r.embed_forward(ids, table).isfinite().all()
    # NaN at one token: its row alone
    bad = x.clone()
    ids[:] = ids % 7
    bad[5, 3] = float("inf")
    got = r.embed_backward(ids, bad, 50)
    hit = int(ids[5]) if 0 <= int(ids[5]) < 50 else None
    assert torch.equal(got.isfinite().all(1), torch.tensor([i != hit for i in range(50)], device="cuda"))


def test_of_no_tokens():
    got = torch.full((5, 8), float("nan"), device="cuda")
    d = api.EmbedDesc(api.PRECISION_F16, 0, 8, 5)
    api.embed_rows_backward(d, 0, 0, got.data_ptr(), 0, 0, t.stream())
    assert got.eq(0).all()


def test_gradient_is_the_transpose_of_the_lookup():
    """sum(dy y(v)) = sum(dtable v) for any table v: both sums in float64, the gradient within its tolerance."""
    ids, table, dy, g = make(4000, 40, 300, "f32", 17, "padded")
    got = r.embed_backward(ids, dy, 300, 3.0)
    _, size, count = r.embed_back64(ids, dy, 300, 3.0)
    left = (dy.double() * r.embed64(ids, table, None, 3.0)).sum()
    tol = (2.0**-24 * (count.clamp(max=700)[:, None] + 1) * size * table.double().abs()).sum()
    assert abs(left - (got.double() * table.double()).sum()) <= tol


def test_same_bits_again_on_streams_and_in_graphs():
    ids, table, x, g = make(50000, 72, 362, "bf16", 19, "skewed")
    both = lambda: (r.embed_forward(ids, table, x, 2.0), r.embed_backward(ids, x, 362, 2.0))  # noqa: E731
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
        for _ in range(2):
            for v in out:
                v.fill_(9)
            gr.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(u, v) for u, v in zip(out, want))
    # other ids in the captured call's tensor
    ids.copy_(ids.flip(0))
    want = both()
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(graphs[0][1], want))
