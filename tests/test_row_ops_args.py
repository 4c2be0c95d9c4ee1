"""The arguments that the operators on rows refuse. Every refusal is decided before any CUDA call, so these run without
a GPU (addresses are made up and never read)."""

import pytest

from katago_cuda import api

A = 1 << 40  # made-up, 256-byte aligned addresses 1 GiB apart
X, Y, DY, DX, MASK, W, B, ST, DW, DB, WS = (A + (i << 30) for i in range(11))


def refused(f, *args, **kw):
    with pytest.raises(api.KcError) as e:
        f(*args, **kw)
    assert e.value.status == api.KC_ERR_INVALID, str(e.value)
    assert any(op in str(e.value) for op in ("layer norm", "looked-up rows", "top logits"))
    return str(e.value)


def ldesc(**kw):
    a = dict(dtype=api.PRECISION_F16, kind=api.NORM_LAYER, n=2, points=361, channels=384, eps=1e-5)
    strides = {k: kw.pop(k) for k in list(kw) if k.endswith("strides") or k == "mask_stride"}
    a.update(kw)
    return api.LayerNormDesc(*a.values(), **strides)


def lforward(d, x=X, mask=MASK, w=W, b=B, y=Y, st=ST):
    api.layer_norm(d, x, mask, w, b, y, st, 0)


def lbackward(d, x=X, mask=MASK, w=W, st=ST, dy=DY, dx=DX, dw=DW, db=DB, ws=WS, size=1 << 30):
    api.layer_norm_backward(d, x, mask, w, st, dy, dx, dw, db, ws, size, 0)


@pytest.mark.parametrize("kw", [
    dict(dtype=3), dict(dtype=-1), dict(kind=2), dict(kind=-1), dict(n=-1), dict(points=-1), dict(n=(1 << 30) + 1),
    dict(points=(1 << 30) + 1), dict(channels=0), dict(channels=(1 << 30) + 1), dict(eps=-1.0), dict(eps=float("nan")),
    dict(eps=float("inf")), dict(x_strides=(-384, 384)), dict(x_strides=(361 * 384, -1)),
    dict(y_strides=(1 << 50, 384)), dict(mask_stride=-1), dict(mask_stride=1 << 62)])
def test_layer_norm_refuses(kw):
    refused(lforward, ldesc(**kw))
    refused(lbackward, ldesc(**kw))
    refused(api.layer_norm_backward_workspace, ldesc(**kw))


@pytest.mark.parametrize("strides", [(361 * 384, 383), (0, 384), (361 * 384 - 1, 384)])
def test_layer_norm_refuses_outputs_on_themselves(strides):
    refused(lforward, ldesc(y_strides=strides))
    refused(lbackward, ldesc(x_strides=strides))


def test_layer_norm_refuses_tensors():
    d = ldesc()
    for name in ("x", "y"):
        assert "null" in refused(lforward, d, **{name: 0})
    for name, at in (("x", X + 1), ("y", Y + 1), ("mask", MASK + 2), ("w", W + 1), ("b", B + 2), ("st", ST + 4)):
        refused(lforward, d, **{name: at})
    refused(lforward, None)
    for name in ("x", "dy", "dx", "st"):
        refused(lbackward, d, **{name: 0})
    refused(lbackward, d, ws=WS + 4)
    refused(lbackward, d, dw=DW + 1)
    refused(lbackward, d, size=api.layer_norm_backward_workspace(d) - 1)
    assert "workspace" in refused(lbackward, d, ws=0)
    assert api.lib().kc_layer_norm_backward_workspace(ldesc(), None) == api.KC_ERR_INVALID


def test_layer_norm_refuses_overlaps():
    d = ldesc()
    refused(lforward, d, y=X + 768)
    refused(lforward, ldesc(y_strides=(361 * 400, 400)), y=X)
    for kw in (dict(mask=Y), dict(w=Y + 4), dict(b=Y), dict(st=X), dict(st=W), dict(st=Y), dict(st=MASK)):
        refused(lforward, d, **kw)
    for kw in (dict(dw=DB), dict(dw=W), dict(db=DX), dict(dx=DY + 768), dict(dx=ST), dict(ws=DW), dict(ws=DX),
               dict(ws=X), dict(dw=ST), dict(dx=MASK), dict(dx=W)):
        refused(lbackward, d, **kw)
    wide = dict(x_strides=(361 * 800, 800), y_strides=(361 * 800, 800))
    refused(lforward, ldesc(**wide), y=X + 2 * 383)


@pytest.mark.parametrize("n,points", [(0, 361), (0, 0), (3, 0)])
def test_layer_norm_of_nothing(n, points):
    d = ldesc(n=n, points=points)
    assert api.layer_norm_backward_workspace(d) == 0
    lforward(d, x=0, y=0, mask=0, st=0)
    lbackward(d, x=0, dy=0, dx=0, st=0, mask=0, dw=0, db=0, ws=0, size=0)
