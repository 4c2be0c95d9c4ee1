"""Plain float64 implementations of the operators on rows (layer and RMS norm, looked-up rows, the loss against a
teacher's top logits) and the calls of the library they are compared with."""

import torch

import token_ops as t
from katago_cuda import api

KINDS = {"layer": api.NORM_LAYER, "rms": api.NORM_RMS}
EPS = 1e-6


def f32(v):
    """A descriptor's float32 field."""
    return float(torch.tensor(v, dtype=torch.float32))


# ---- norm of a token's row --------------------------------------------------------------------------------------
def layer64(x, on, weight, bias, kind, eps=EPS):
    """y, mean, rstd, xh in float64; x [n][points][channels], on [n][points] bool."""
    sel = on[:, :, None]
    xd = torch.where(sel, x.double(), 0.0)
    mean = xd.mean(2, keepdim=True) if kind == "layer" else torch.zeros_like(xd[:, :, :1])
    rstd = torch.where(sel, ((xd - mean).square().mean(2, keepdim=True) + eps) ** -0.5, 0.0)
    xh = (xd - mean) * rstd
    y = xh if weight is None else xh * weight.double()
    y = y if bias is None else y + bias.double()
    return torch.where(sel, y, 0.0), mean[:, :, 0], rstd[:, :, 0], xh


def layer_back64(x, on, weight, mean, rstd, dy, kind):
    """dx, dweight, dbias by the formula from given statistics; the sizes of dx's terms, and the sums of the sizes
    behind dweight and dbias."""
    sel = on[:, :, None]
    channels = x.shape[2]
    r = rstd.double()[:, :, None]
    xh = torch.where(sel, (x.double() - mean.double()[:, :, None]) * r, 0.0)
    dyd = torch.where(sel, dy.double(), 0.0)
    g = dyd if weight is None else dyd * weight.double()
    c1 = g.sum(2, keepdim=True) / channels if kind == "layer" else 0.0
    c2 = (g * xh).sum(2, keepdim=True) / channels
    dx = torch.where(sel, r * (g - c1 - xh * c2), 0.0)
    size = r * (g.abs() + g.abs().mean(2, keepdim=True) + xh.abs() * (g * xh).abs().mean(2, keepdim=True))
    size = torch.where(sel, size, 0.0)
    return dx, (dyd * xh).sum((0, 1)), dyd.sum((0, 1)), size, (dyd * xh).abs().sum((0, 1)), dyd.abs().sum((0, 1))


def layer_desc(x, y, kind, eps=EPS, mask=None):
    n, points, channels = x.shape
    return api.LayerNormDesc(t.PRECISION[t.NAMES[x.dtype]], KINDS[kind], n, points, channels, eps,
                             x_strides=(x.stride(0), x.stride(1)), y_strides=(y.stride(0), y.stride(1)),
                             mask_stride=None if mask is None else mask.stride(0))


def layer_forward(x, mask, weight, bias, kind, y=None, want_stats=True, eps=EPS):
    y = torch.empty_like(x, memory_format=torch.contiguous_format) if y is None else y
    stats = torch.full((*x.shape[:2], 2), float("nan"), device=x.device) if want_stats else None
    api.layer_norm(layer_desc(x, y, kind, eps, mask), x.data_ptr(), t.ptr(mask), t.ptr(weight), t.ptr(bias),
                   y.data_ptr(), t.ptr(stats), t.stream())
    return y, stats


def layer_backward(x, mask, weight, stats, dy, kind, dx=None, want=True):
    dx = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device=x.device) if dx is None else dx
    desc = layer_desc(x, dy, kind, EPS, mask)
    size = api.layer_norm_backward_workspace(desc) if want else 0
    ws = t.workspace(size, x.device)
    dw, db = (torch.full((x.shape[2],), float("nan"), device=x.device) if want else None for _ in range(2))
    api.layer_norm_backward(desc, x.data_ptr(), t.ptr(mask), t.ptr(weight), stats.data_ptr(), dy.data_ptr(),
                            dx.data_ptr(), t.ptr(dw), t.ptr(db), t.ptr(ws), size, t.stream())
    return dx, dw, db


# ---- looked-up rows ---------------------------------------------------------------------------------------------
def embed64(ids, table, x, scale):
    there = (ids >= 0) & (ids < table.shape[0])
    rows = table.double()[torch.where(there, ids, 0).long()] * f32(scale)
    y = torch.where(there[:, None], rows, 0.0)
    return y if x is None else y + x.double()


def embed_back64(ids, dy, table_rows, scale):
    """The table's gradient, the sum of its terms' sizes, and how many tokens have each row."""
    there = (ids >= 0) & (ids < table_rows)
    at = torch.where(there, ids, table_rows).long()
    s = f32(scale)
    total = torch.zeros(table_rows + 1, dy.shape[1], dtype=torch.float64, device=dy.device)
    size = total.clone().index_add_(0, at, dy.double().abs())[:-1] * abs(s)
    total = total.index_add_(0, at, dy.double())[:-1] * s
    return total, size, torch.bincount(at, minlength=table_rows + 1)[:-1]


def embed_forward(ids, table, x=None, scale=1.0, y=None):
    if y is None:
        y = torch.empty(ids.shape[0], table.shape[1], dtype=table.dtype, device=table.device)
    desc = api.EmbedDesc(t.PRECISION[t.NAMES[table.dtype]], ids.shape[0], table.shape[1], table.shape[0], scale,
                         table.stride(0), None if x is None else x.stride(0), y.stride(0))
    api.embed_rows(desc, ids.data_ptr(), table.data_ptr(), t.ptr(x), y.data_ptr(), t.stream())
    return y


def embed_backward(ids, dy, table_rows, scale=1.0, dtable=None):
    if dtable is None:
        dtable = torch.full((table_rows, dy.shape[1]), float("nan"), device=dy.device)
    desc = api.EmbedDesc(t.PRECISION[t.NAMES[dy.dtype]], ids.shape[0], dy.shape[1], table_rows, scale,
                         y_stride=dy.stride(0))
    size = api.embed_rows_backward_workspace(desc)
    ws = t.workspace(size, dy.device)
    api.embed_rows_backward(desc, ids.data_ptr(), dy.data_ptr(), dtable.data_ptr(), t.ptr(ws), size, t.stream())
    return dtable


# ---- loss against a teacher's top logits ------------------------------------------------------------------------
def teacher64(ids, top, whole, classes, temperature):
    """Which entries there are, p and log p (0 where absent)."""
    temperature = f32(temperature)
    there = (ids >= 0) & (ids < classes) & (top != float("-inf"))
    tt = torch.where(there, top.double() / temperature, float("-inf"))
    some = there.any(1)
    if whole is None:
        lse = torch.logsumexp(torch.where(some[:, None], tt, 0.0), 1)
    else:
        lse = whole.double()
    log_p = torch.where(there, tt - lse[:, None], 0.0)
    return there, some, torch.where(there, log_p.exp(), 0.0), log_p


def distill64(z, ids, top, whole, temperature):
    """loss, (largest, sum of exponentials), all 0 for rows without entries."""
    temperature = f32(temperature)
    there, some, p, log_p = teacher64(ids, top, whole, z.shape[1], temperature)
    log_q = torch.log_softmax(z.double() / temperature, 1).gather(1, torch.where(there, ids, 0).long())
    loss = temperature**2 * torch.where(p > 0, p * (log_p - log_q), 0.0).sum(1)
    m = z.double().amax(1)
    s = torch.exp((z.double() - m[:, None]) / temperature).sum(1)
    keep = lambda v: torch.where(some, v, 0.0)  # noqa: E731
    return keep(loss), keep(m), keep(s)


def distill_back64(z, ids, top, whole, temperature, stats, dloss):
    """The gradient; the sizes g P q and g p of its two terms."""
    temperature = f32(temperature)
    there, some, p, _ = teacher64(ids, top, whole, z.shape[1], temperature)
    m, s = stats.double().unbind(1)
    g = (torch.ones_like(m) if dloss is None else dloss.double()) * temperature
    base = torch.where(m == float("-inf"), 0.0, m)
    q = torch.exp((z.double() - base[:, None]) / temperature) / s[:, None] * p.sum(1, keepdim=True)
    dense = torch.zeros_like(q).scatter_add_(1, torch.where(there, ids, 0).long(), p)
    keep = lambda v: torch.where(some[:, None], v, 0.0)  # noqa: E731
    return keep(g[:, None] * (q - dense)), keep(g.abs()[:, None] * q), keep(g.abs()[:, None] * dense)


def distill_desc(z, dz, ids, temperature):
    return api.DistillDesc(t.PRECISION[t.NAMES[z.dtype]], z.shape[0], z.shape[1], ids.shape[1], temperature,
                           z.stride(0), z.shape[1] if dz is None else dz.stride(0), ids.stride(0))


def distill_forward(z, ids, top, whole=None, temperature=1.0, want_stats=True):
    assert ids.stride(0) == top.stride(0)
    loss = torch.full((z.shape[0],), float("nan"), device=z.device)
    stats = torch.full((z.shape[0], 2), float("nan"), device=z.device) if want_stats else None
    api.distill_top(distill_desc(z, None, ids, temperature), z.data_ptr(), ids.data_ptr(), top.data_ptr(),
                    t.ptr(whole), loss.data_ptr(), t.ptr(stats), t.stream())
    return loss, stats


def distill_backward(z, ids, top, stats, whole=None, temperature=1.0, dloss=None, dz=None):
    dz = torch.full_like(z, float("nan"), memory_format=torch.contiguous_format) if dz is None else dz
    api.distill_top_backward(distill_desc(z, dz, ids, temperature), z.data_ptr(), ids.data_ptr(), top.data_ptr(),
                             t.ptr(whole), stats.data_ptr(), t.ptr(dloss), dz.data_ptr(), t.stream())
    return dz
