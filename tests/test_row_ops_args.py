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
    dict(points=(1 << 30) + 1), dict(n=1 << 30, points=1 << 30, x_strides=(0, 0), y_strides=(0, 0), mask_stride=0),
    dict(channels=0), dict(channels=(1 << 30) + 1), dict(eps=-1.0), dict(eps=float("nan")),
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


IDS, TABLE, DT = (A + (i << 32) for i in range(20, 23))


def edesc(**kw):
    a = dict(dtype=api.PRECISION_BF16, tokens=722, channels=384, table_rows=362, scale=2.0)
    strides = {k: kw.pop(k) for k in list(kw) if k.endswith("stride")}
    a.update(kw)
    return api.EmbedDesc(*a.values(), **strides)


def look_up(d, ids=IDS, table=TABLE, x=X, y=Y):
    api.embed_rows(d, ids, table, x, y, 0)


def look_up_back(d, ids=IDS, dy=DY, dt=DT, ws=WS, size=1 << 30):
    api.embed_rows_backward(d, ids, dy, dt, ws, size, 0)


@pytest.mark.parametrize("kw", [
    dict(dtype=3), dict(dtype=-1), dict(tokens=-1), dict(tokens=(1 << 30) + 1), dict(channels=0),
    dict(channels=(1 << 20) + 1), dict(table_rows=0), dict(table_rows=(1 << 30) + 1), dict(scale=float("inf")),
    dict(scale=float("nan")), dict(y_stride=-1), dict(y_stride=1 << 50)])
def test_looked_up_rows_refuses(kw):
    refused(look_up, edesc(**kw))
    refused(look_up_back, edesc(**kw))
    if not any(k.endswith("stride") for k in kw):
        refused(api.embed_rows_backward_workspace, edesc(**kw))


def test_looked_up_rows_refuses_tensors_and_overlaps():
    d = edesc()
    for kw in (dict(ids=0), dict(table=0), dict(y=0), dict(ids=IDS + 1), dict(table=TABLE + 1), dict(x=X + 1),
               dict(y=Y + 1), dict(y=TABLE), dict(y=IDS), dict(y=X + 768), dict(y=TABLE + 361 * 768)):
        refused(look_up, d, **kw)
    refused(look_up, None)
    for kw in (dict(table_stride=-1), dict(x_stride=-1), dict(y_stride=383), dict(y_stride=0)):
        refused(look_up, edesc(**kw))
    refused(look_up, edesc(x_stride=400), y=X)
    look_up(edesc(tokens=0), 0, 0, 0, 0)
    for kw in (dict(ids=0), dict(dy=0), dict(dt=0), dict(ids=IDS + 2), dict(dy=DY + 1), dict(dt=DT + 2), dict(ws=0),
               dict(ws=WS + 8), dict(dt=DY), dict(dt=IDS), dict(ws=DT), dict(ws=DY), dict(ws=IDS),
               dict(size=api.embed_rows_backward_workspace(d) - 1)):
        refused(look_up_back, d, **kw)
    assert api.embed_rows_backward_workspace(edesc(tokens=0)) == 0
    assert api.lib().kc_embed_rows_backward_workspace(d, None) == api.KC_ERR_INVALID


LOG, TOP, WHOLE, LOSS, DL, DLOG = (A + (i << 33) for i in range(20, 26))


def ddesc(**kw):
    a = dict(dtype=api.PRECISION_F16, rows=256, classes=362, top=32, temperature=1.0)
    strides = {k: kw.pop(k) for k in list(kw) if k.endswith("stride")}
    a.update(kw)
    return api.DistillDesc(*a.values(), **strides)


def distill(d, z=LOG, ids=IDS, top=TOP, whole=WHOLE, loss=LOSS, st=ST):
    api.distill_top(d, z, ids, top, whole, loss, st, 0)


def distill_back(d, z=LOG, ids=IDS, top=TOP, whole=WHOLE, st=ST, dl=DL, dz=DLOG):
    api.distill_top_backward(d, z, ids, top, whole, st, dl, dz, 0)


@pytest.mark.parametrize("kw", [
    dict(dtype=3), dict(rows=-1), dict(rows=(1 << 30) + 1), dict(classes=0), dict(classes=(1 << 30) + 1), dict(top=0),
    dict(top=1025), dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("nan")),
    dict(temperature=float("inf")), dict(temperature=1e-7), dict(logits_stride=-1), dict(logits_stride=1 << 50),
    dict(top_stride=-1)])
def test_top_logits_refuses(kw):
    refused(distill, ddesc(**kw))
    refused(distill_back, ddesc(**kw))


def test_top_logits_refuses_tensors_and_overlaps():
    d = ddesc()
    for kw in (dict(z=0), dict(ids=0), dict(top=0), dict(loss=0), dict(z=LOG + 1), dict(ids=IDS + 2), dict(top=TOP + 1),
               dict(whole=WHOLE + 2), dict(loss=LOSS + 1), dict(st=ST + 4), dict(loss=LOG), dict(loss=ST), dict(st=TOP),
               dict(st=IDS), dict(loss=WHOLE)):
        refused(distill, d, **kw)
    refused(distill, None)
    for kw in (dict(z=0), dict(ids=0), dict(top=0), dict(st=0), dict(dz=0), dict(dz=DLOG + 1), dict(st=ST + 4),
               dict(dl=DL + 1), dict(dz=LOG + 724), dict(dz=IDS), dict(dz=TOP), dict(dz=ST), dict(dz=DL),
               dict(dz=WHOLE)):
        refused(distill_back, d, **kw)
    refused(distill_back, None)
    for kw in (dict(dlogits_stride=361), dict(dlogits_stride=-1), dict(dlogits_stride=0)):
        refused(distill_back, ddesc(**kw))
    refused(distill_back, ddesc(dlogits_stride=400), dz=LOG)
    distill(ddesc(rows=0), 0, 0, 0, 0, 0, 0)
    distill_back(ddesc(rows=0), 0, 0, 0, 0, 0, 0, 0)


@pytest.mark.parametrize("temperature", [32.00001, 64.0, 1024.0, 2.0**20, 2.0**-20 * (1 - 2.0**-24)])
def test_top_logits_refuses_temperatures(temperature):
    """Beyond 32 the loss of a student near its teacher would be lost in the error of its float32 sums."""
    assert "temperature" in refused(distill, ddesc(temperature=temperature))
    assert "temperature" in refused(distill_back, ddesc(temperature=temperature))
