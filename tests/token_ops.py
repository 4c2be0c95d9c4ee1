"""Plain float64 implementations of the standalone operators on board tokens and the calls of the library they are
compared with (tests/test_gpu_group_norm.py, tests/test_gpu_rope_axes.py, tests/test_gpu_token_ops.py)."""

import torch

from katago_cuda import api

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
PRECISION = {"f32": api.PRECISION_F32, "f16": api.PRECISION_F16, "bf16": api.PRECISION_BF16}
ACTS = {"identity": api.ACT_IDENTITY, "relu": api.ACT_RELU, "mish": api.ACT_MISH, "silu": api.ACT_SILU}
LAYOUTS = {"halves": api.ROPE_HALVES, "pairs": api.ROPE_PAIRS}
NAMES = {v: k for k, v in DTYPES.items()}
EPS = 1e-5


def half_step(t):
    """Largest relative error of one rounding to t, and its largest absolute error below the normal numbers."""
    return torch.finfo(t).eps / 2, float(torch.finfo(t).smallest_normal) * torch.finfo(t).eps / 2


def ptr(t):
    return 0 if t is None else t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


# ---- group norm -------------------------------------------------------------------------------------------------
def act64(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "mish":
        return z * torch.tanh(torch.nn.functional.softplus(z, threshold=1e9))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def slope64(z, act):
    if act == "relu":
        return (z > 0).double()
    if act == "mish":
        t = torch.tanh(torch.nn.functional.softplus(z, threshold=1e9))
        return t + z * torch.sigmoid(z) * (1 - t * t)
    if act == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def norm64(x, on, weight, bias, groups, act, eps=EPS):
    """y, mean, rstd [n][groups] in float64; x [n][points][channels], on [n][points] bool."""
    n, points, channels = x.shape
    cg = channels // groups
    xd = torch.where(on[:, :, None], x.double(), torch.zeros((), dtype=torch.float64, device=x.device))
    count = (on.sum(1) * cg).double()[:, None]
    some = count > 0
    xg = xd.reshape(n, points, groups, cg)
    mean = torch.where(some, xg.sum((1, 3)) / count.clamp(min=1), 0.0)
    d = torch.where(on[:, :, None, None], xg - mean[:, None, :, None], 0.0)
    rstd = torch.where(some, ((d * d).sum((1, 3)) / count.clamp(min=1) + eps) ** -0.5, 0.0)
    xh = (d * rstd[:, None, :, None]).reshape(n, points, channels)
    z = xh * weight.double() + bias.double()
    return torch.where(on[:, :, None], act64(z, act), 0.0), mean, rstd, xh, z


def norm_back64(x, on, weight, bias, mean, rstd, dy, groups, act):
    """dx, dweight, dbias by the formula in float64 from given statistics, the sums of the terms' sizes behind
    dweight and dbias, and for dx the size of the terms of each element."""
    n, points, channels = x.shape
    cg = channels // groups
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    sel = on[:, :, None]
    m = mean.double().repeat_interleave(cg, 1)[:, None, :]
    r = rstd.double().repeat_interleave(cg, 1)[:, None, :]
    w, b = weight.double(), bias.double()
    xh = torch.where(sel, (x.double() - m) * r, zero)
    z = xh * w + b
    gz = torch.where(sel, dy.double() * slope64(z, act), zero)
    s1, s2 = gz.sum(1), (gz * xh).sum(1)
    count = (on.sum(1) * cg).double().clamp(min=1)[:, None]

    def share(s):
        return ((s * w).reshape(n, groups, cg).sum(2) / count).repeat_interleave(cg, 1)[:, None, :]

    c1, c2 = share(s1), share(s2)
    dx = torch.where(sel, r * (gz * w - c1 - xh * c2), zero)

    # what the rounding of the sums is relative to
    a1, a2 = gz.abs().sum(1), (gz * xh).abs().sum(1)
    absw = w.abs()
    t1 = ((a1 * absw).reshape(n, groups, cg).sum(2) / count).repeat_interleave(cg, 1)[:, None, :]
    t2 = ((a2 * absw).reshape(n, groups, cg).sum(2) / count).repeat_interleave(cg, 1)[:, None, :]
    size = r * ((gz * w).abs() + t1 + xh.abs() * t2)
    return dx, s2.sum(0), s1.sum(0), size, a2.sum(0), a1.sum(0)


def norm_desc(x, y, groups, act, eps=EPS, mask=None):
    n, points, channels = x.shape
    return api.GroupNormDesc(PRECISION[NAMES[x.dtype]], ACTS[act], n, points, channels, groups, eps,
                             x_strides=(x.stride(0), x.stride(1)), y_strides=(y.stride(0), y.stride(1)),
                             mask_stride=None if mask is None else mask.stride(0))


def workspace(size, device):
    """A workspace of exactly `size` bytes with junk (NaN patterns) in it."""
    return torch.full((max(size, 1),), 0xFF, dtype=torch.uint8, device=device) if size else None


def norm_forward(x, mask, weight, bias, groups, act, y=None, want_stats=True, eps=EPS):
    y = torch.empty_like(x, memory_format=torch.contiguous_format) if y is None else y
    desc = norm_desc(x, y, groups, act, eps, mask)
    size = api.group_norm_act_workspace(desc, False)
    ws = workspace(size, x.device)
    stats = torch.full((x.shape[0], groups, 2), float("nan"), device=x.device) if want_stats else None
    api.group_norm_act(desc, x.data_ptr(), ptr(mask), ptr(weight), ptr(bias), y.data_ptr(), ptr(stats), ptr(ws), size,
                       stream())
    return y, stats


def norm_backward(x, mask, weight, bias, stats, dy, groups, act, dx=None, want=True):
    dx = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device=x.device) if dx is None else dx
    desc = norm_desc(x, dy, groups, act, EPS, mask)
    size = api.group_norm_act_workspace(desc, True)
    ws = workspace(size, x.device)
    dw, db = (torch.full((x.shape[2],), float("nan"), device=x.device) if want else None for _ in range(2))
    api.group_norm_act_backward(desc, x.data_ptr(), ptr(mask), ptr(weight), ptr(bias), stats.data_ptr(), dy.data_ptr(),
                                dx.data_ptr(), ptr(dw), ptr(db), ptr(ws), size, stream())
    return dx, dw, db


# ---- rotary positions -------------------------------------------------------------------------------------------
def split64(x, rotary_dim, layout):
    x = x[..., :rotary_dim].double()
    return (x[..., :rotary_dim // 2], x[..., rotary_dim // 2:]) if layout == "halves" else (x[..., 0::2], x[..., 1::2])


def join64(a, b, x, rotary_dim, layout):
    r = torch.cat([a, b], -1) if layout == "halves" else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([r, x[..., rotary_dim:].double()], -1)


def turn64(x, pos, freqs, rotary_dim, layout, back=False):
    """x [tokens][heads][head_dim] turned in float64; also the sizes |x1| + |x2| behind each element's rounding (0 for
    the unrotated rest)."""
    angle = torch.einsum("ta,hja->thj", pos.double(), freqs.double())
    if back:
        angle = -angle
    angle = angle.repeat_interleave(x.shape[1] // freqs.shape[0], 1)
    a, b = split64(x, rotary_dim, layout)
    c, s = torch.cos(angle), torch.sin(angle)
    size = a.abs() + b.abs()
    zero = torch.zeros_like(x)
    return join64(a * c - b * s, a * s + b * c, x, rotary_dim, layout), join64(size, size, zero, rotary_dim, layout)


def freqs_back64(dq_out, q, dk_out, k, pos, freqs, rotary_dim, layout):
    """The frequencies' gradient, and the sum of its terms' sizes."""
    tables = freqs.shape[0]
    total, size = 0.0, 0.0
    for g, x in ((dq_out, q), (dk_out, k)):
        if g is None:
            continue
        dx, _ = turn64(g, pos, freqs, rotary_dim, layout, back=True)
        da, db = split64(dx, rotary_dim, layout)
        a, b = split64(x, rotary_dim, layout)
        per = x.shape[1] // tables
        turn = (db * a - da * b).unflatten(1, (tables, per)).sum(2)
        sz = ((da.abs() + db.abs()) * (a.abs() + b.abs())).unflatten(1, (tables, per)).sum(2)
        total = total + torch.einsum("thj,ta->hja", turn, pos.double())
        size = size + torch.einsum("thj,ta->hja", sz, pos.double().abs())
    return total, size


def rope_desc(q, k, q_out, k_out, rotary_dim, layout, axes, tables):
    none = (0, 0)
    st = lambda t: none if t is None else (t.stride(0), t.stride(1))  # noqa: E731
    return api.RopeDesc(PRECISION[NAMES[q.dtype]], LAYOUTS[layout], axes, q.shape[0],
                        q.shape[1], 0 if k is None else k.shape[1], q.shape[2], rotary_dim, tables, q_strides=st(q),
                        k_strides=st(k), q_out_strides=st(q_out), k_out_strides=st(k_out))


def rope_forward(q, k, pos, freqs, rotary_dim, layout, q_out=None, k_out=None):
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if q_out is None else q_out
    if k is not None and k_out is None:
        k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    desc = rope_desc(q, k, q_out, k_out, rotary_dim, layout, pos.shape[1], freqs.shape[0])
    api.rope_axes(desc, q.data_ptr(), ptr(k), pos.data_ptr(), freqs.data_ptr(), q_out.data_ptr(), ptr(k_out), stream())
    return q_out, k_out


def rope_backward(dq_out, dk_out, q, k, pos, freqs, rotary_dim, layout, dq=None, dk=None, learned=True):
    dq = torch.empty_strided(q.shape, q.stride(), dtype=q.dtype, device=q.device) if dq is None else dq
    if k is not None and dk is None:
        dk = torch.empty_strided(k.shape, k.stride(), dtype=k.dtype, device=k.device)
    desc = rope_desc(q, k, dq_out, dk_out, rotary_dim, layout, pos.shape[1], freqs.shape[0])
    size = api.rope_axes_backward_workspace(desc) if learned else 0
    ws = workspace(size, q.device)
    df = torch.full_like(freqs, float("nan")) if learned else None
    api.rope_axes_backward(desc, dq_out.data_ptr(), ptr(dk_out), ptr(q) if learned else 0, ptr(k) if learned else 0,
                           pos.data_ptr(), freqs.data_ptr(), dq.data_ptr(), ptr(dk), ptr(df), ptr(ws), size, stream())
    return dq, dk, df


def within(got, want, tol):
    """got within the elementwise tolerance; what is furthest off is named."""
    got = got.double()
    assert torch.isfinite(got).all(), "not finite"
    over = (got - want).abs() - tol
    worst = int(over.flatten().argmax())
    assert over.max() <= 0, (f"element {worst}: got {got.flatten()[worst].item()}, want {want.flatten()[worst].item()}, "
                             f"tolerance {(tol + torch.zeros_like(want)).flatten()[worst].item()}")
