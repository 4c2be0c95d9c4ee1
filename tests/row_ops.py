"""Plain float64 implementations of the operators on rows (layer and RMS norm, looked-up rows, the loss against a
teacher's top logits) and the calls of the library they are compared with."""

import torch

import token_ops as t
from katago_cuda import api

KINDS = {"layer": api.NORM_LAYER, "rms": api.NORM_RMS}
EPS = 1e-6


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
