"""The arguments that the standalone operators on board tokens refuse, and their host-side helpers. Every refusal is
decided before any CUDA call, so these run without a GPU (addresses are made up and never read)."""

import numpy as np
import pytest

from katago_cuda import api

A = 1 << 40  # made-up, 256-byte aligned addresses 1 GiB apart
X, Y, DY, DX, MASK, W, B, ST, DW, DB, WS = (A + (i << 30) for i in range(11))


def desc(**kw):
    a = dict(dtype=api.PRECISION_F16, act=api.ACT_MISH, n=2, points=361, channels=384, groups=32, eps=1e-5)
    strides = {k: kw.pop(k) for k in list(kw) if k.endswith("strides") or k == "mask_stride"}
    a.update(kw)
    return api.GroupNormDesc(*a.values(), **strides)


def forward(d, x=X, mask=MASK, w=W, b=B, y=Y, st=ST, ws=WS, size=1 << 30):
    api.group_norm_act(d, x, mask, w, b, y, st, ws, size, 0)


def backward(d, x=X, mask=MASK, w=W, b=B, st=ST, dy=DY, dx=DX, dw=DW, db=DB, ws=WS, size=1 << 30):
    api.group_norm_act_backward(d, x, mask, w, b, st, dy, dx, dw, db, ws, size, 0)


def refused(f, *args, **kw):
    with pytest.raises(api.KcError) as e:
        f(*args, **kw)
    assert e.value.status == api.KC_ERR_INVALID, str(e.value)
    assert "group norm" in str(e.value) or "rotary positions" in str(e.value)
    return str(e.value)


@pytest.mark.parametrize("kw", [
    dict(dtype=3), dict(dtype=-1), dict(act=4), dict(act=-1), dict(n=-1), dict(points=-1), dict(n=(1 << 30) + 1),
    dict(points=(1 << 30) + 1), dict(channels=0),
    dict(groups=0), dict(groups=7), dict(groups=385), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")),
    dict(x_strides=(-384, 384)), dict(x_strides=(361 * 384, -1)), dict(y_strides=(361 * 384, 383)),
    dict(y_strides=(0, 384)), dict(y_strides=(361 * 384 - 1, 384)), dict(y_strides=(1 << 50, 384)),
    dict(mask_stride=-1), dict(mask_stride=1 << 62)])
def test_group_norm_refuses(kw):
    refused(forward, desc(**kw))


def test_group_norm_refuses_tensors():
    d = desc()
    assert "null" in refused(forward, d, x=0)
    refused(forward, d, y=0)
    refused(forward, d, x=X + 1)
    refused(forward, d, y=Y + 1)
    refused(forward, d, mask=MASK + 2)
    refused(forward, d, w=W + 1)
    refused(forward, d, st=ST + 4)
    refused(forward, None)
    refused(backward, d, dy=0)
    refused(backward, d, dx=0)
    refused(backward, d, st=0)
    refused(backward, d, ws=WS + 4)
    refused(backward, d, size=api.group_norm_act_workspace(d, True) - 1)
    assert "workspace" in refused(backward, d, ws=0)


def test_group_norm_refuses_overlaps():
    d = desc()
    refused(forward, d, y=X + 768)                                   # neither in place nor apart
    refused(forward, desc(y_strides=(361 * 400, 400)), y=X)          # same address, other strides
    refused(forward, d, mask=Y)
    refused(forward, d, w=Y + 4)
    refused(forward, d, st=X)
    refused(forward, d, st=W)
    refused(backward, d, dw=DB)
    refused(backward, d, dw=W)
    refused(backward, d, db=DX)
    refused(backward, d, dx=DY + 768)
    refused(backward, d, ws=DW)
    # slices of one wider buffer that share elements: channels [0, 384) and [383, 767) of rows of 800
    wide = dict(x_strides=(361 * 800, 800), y_strides=(361 * 800, 800))
    refused(forward, desc(**wide), y=X + 2 * 383)
    refused(forward, desc(**wide), y=X + 2 * (800 * 7 + 417))  # wraps into the next row


@pytest.mark.parametrize("n,points", [(0, 361), (0, 0)])
def test_group_norm_of_nothing(n, points):
    d = desc(n=n, points=points)
    assert api.group_norm_act_workspace(d, False) == 0 and api.group_norm_act_workspace(d, True) == 0
    forward(d, x=0, y=0, mask=0, st=0, ws=0, size=0)
    backward(d, x=0, dy=0, dx=0, st=0, mask=0, dw=0, db=0, ws=0, size=0)


@pytest.mark.parametrize("kw", [
    dict(dtype=3), dict(act=4), dict(n=-1), dict(points=(1 << 30) + 1), dict(channels=0), dict(groups=7),
    dict(eps=-1.0), dict(x_strides=(-384, 384)), dict(x_strides=(361 * 384, -1)), dict(y_strides=(361 * 384, -384)),
    dict(y_strides=(1 << 50, 384)), dict(x_strides=(361 * 384, 1 << 62)), dict(y_strides=((1 << 63) - 1, 384)),
    dict(channels=(1 << 30) + 32), dict(channels=(1 << 31) - 1, groups=1), dict(n=1 << 30, points=0, channels=1 << 20)])
@pytest.mark.parametrize("backward", [False, True])
def test_workspace_query_refuses_what_the_calls_refuse(kw, backward):
    d = desc(**kw)
    refused(api.group_norm_act_workspace, d, backward)
    refused(forward, d)


def test_more_groups_than_a_launch():
    """Refused before anything is launched: boards of more channels than a cluster's tables hold, a group a channel."""
    d = desc(n=8192, points=1, channels=(1 << 18) + 8, groups=(1 << 18) + 8)
    assert "n * groups" in refused(api.group_norm_act_workspace, d, False)
    far = [(1 << 42) + (i << 38) for i in range(8)]
    assert "n * groups" in refused(forward, d, *far[:6], 1 << 45, 1 << 44)


@pytest.mark.parametrize("backward", [False, True])
def test_strides_of_one_row_play_no_part(backward):
    """Boards of one point: whatever the row stride says, the call is the one of contiguous rows."""
    want = api.group_norm_act_workspace(desc(points=1), backward)
    for far in (1 << 34, 1 << 62, (1 << 63) - 1):
        d = desc(points=1, x_strides=(384, far), y_strides=(384, far))
        assert api.group_norm_act_workspace(d, backward) == want


def test_workspace_null_result():
    assert api.lib().kc_group_norm_act_workspace(desc(), 0, None) == api.KC_ERR_INVALID
    assert api.lib().kc_rope_axes_backward_workspace(rdesc(), None) == api.KC_ERR_INVALID


Q, K, QO, KO, POS, FR, DF = (A + (i << 32) for i in range(20, 27))


def rdesc(**kw):
    a = dict(dtype=api.PRECISION_BF16, layout=api.ROPE_HALVES, axes=2, tokens=722, q_heads=6, k_heads=2, head_dim=64,
             rotary_dim=64, tables=1)
    strides = {k: kw.pop(k) for k in list(kw) if k.endswith("strides")}
    a.update(kw)
    return api.RopeDesc(*a.values(), **strides)


def rotate(d, q=Q, k=K, pos=POS, fr=FR, qo=QO, ko=KO):
    api.rope_axes(d, q, k, pos, fr, qo, ko, 0)


def rotate_back(d, dqo=QO, dko=KO, q=Q, k=K, pos=POS, fr=FR, dq=DX, dk=DY, df=DF, ws=WS, size=1 << 30):
    api.rope_axes_backward(d, dqo, dko, q, k, pos, fr, dq, dk, df, ws, size, 0)


@pytest.mark.parametrize("kw", [
    dict(dtype=3), dict(layout=2), dict(axes=0), dict(axes=5), dict(tokens=-1), dict(q_heads=0), dict(k_heads=-1),
    dict(q_heads=4098), dict(k_heads=4098),
    dict(head_dim=1), dict(head_dim=1026, rotary_dim=2), dict(rotary_dim=0), dict(rotary_dim=3), dict(rotary_dim=66),
    dict(tables=0), dict(tables=3), dict(tables=6), dict(q_strides=(-1, 64)), dict(k_strides=(64, -64)),
    dict(q_out_strides=(383, 64)), dict(q_out_strides=(0, 64)), dict(k_out_strides=(128, 63)),
    dict(q_strides=(1 << 50, 64))])
def test_rotary_refuses(kw):
    refused(rotate, rdesc(**kw))


def test_rotary_refuses_tensors():
    d = rdesc()
    for name in ("q", "k", "pos", "fr", "qo", "ko"):
        refused(rotate, d, **{name: 0})
    for name in ("q", "k", "qo", "ko"):
        refused(rotate, d, **{name: A + (40 << 32) + 1})
    refused(rotate, d, pos=POS + 2)
    refused(rotate, d, fr=FR + 1)
    refused(rotate, None)
    for name in ("dqo", "dko", "dq", "dk", "q", "k", "ws"):
        refused(rotate_back, d, **{name: 0})
    refused(rotate_back, d, df=DF + 1)
    refused(rotate_back, d, ws=WS + 8)
    refused(rotate_back, d, size=api.rope_axes_backward_workspace(d) - 1)


def test_rotary_refuses_overlaps():
    d = rdesc()
    refused(rotate, d, qo=Q + 2)
    refused(rotate, d, qo=K)
    refused(rotate, d, ko=Q)
    refused(rotate, d, ko=QO)
    refused(rotate, d, qo=POS)
    refused(rotate, d, ko=FR)
    refused(rotate, rdesc(q_out_strides=(400, 64)), qo=Q)
    refused(rotate_back, d, dq=Q)       # the inputs are still read for the frequencies' gradient
    refused(rotate_back, d, df=FR)
    refused(rotate_back, d, ws=DF)
    refused(rotate_back, d, df=DX)
    # heads of Q and K in one buffer that share elements
    wide = dict(q_strides=(1024, 64), k_strides=(1024, 64), q_out_strides=(1024, 64), k_out_strides=(1024, 64))
    refused(rotate, rdesc(**wide), qo=QO, ko=QO + 2 * 383)


def test_rotary_of_nothing():
    d = rdesc(tokens=0)
    assert api.rope_axes_backward_workspace(d) == 0
    rotate(d, 0, 0, 0, 0, 0, 0)
    rotate_back(d, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)


def test_rotary_workspace_query_refuses_what_the_calls_refuse():
    for kw in (dict(tokens=(1 << 46) + 1), dict(tokens=(1 << 63) - 1), dict(axes=5), dict(tables=3)):
        refused(api.rope_axes_backward_workspace, rdesc(**kw))
        refused(rotate, rdesc(**kw))


def test_rotary_strides_of_absent_heads_play_no_part():
    d = rdesc(tokens=0, k_heads=0, k_strides=(-1, 1 << 62), k_out_strides=(1 << 62, -64))
    rotate(d, 0, 0, 0, 0, 0, 0)
    rotate_back(d, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)


def test_rotary_frequencies():
    f = api.rope_axes_freqs([8, 12, 12], 100.0, 64)
    want = np.zeros((32, 3))
    want[:8, 0] = 100.0 ** -(np.arange(8) / 8)
    want[8:20, 1] = 100.0 ** -(np.arange(12) / 12)
    want[20:, 2] = 100.0 ** -(np.arange(12) / 12)
    # one rounding of a float64 power
    assert f.shape == (32, 3) and np.all(np.abs(f - want) <= want * 2.0**-24 * 1.001)
    assert np.array_equal(api.rope_axes_freqs([0, 1], 10.0, 2), np.array([[0, 1]], np.float32))
    for args in (([8, 12], 100.0, 64), ([32], 0.0, 64), ([32], float("inf"), 64), ([32], float("nan"), 64),
                 ([-1, 33], 2.0, 64), ([], 2.0, 2), ([1] * 5, 2.0, 10), ([1], 2.0, 3), ([0], 2.0, 0)):
        refused(api.rope_axes_freqs, *args)


def test_board_frequencies_match_the_engine_tables():
    """Two axes (row, column) with equal sections give the reference's fixed 2D table frequencies (theta 100, head dim
    64: pairs 0..15 turn by rows, 16..31 by columns, 1 / theta^(2 i / 32))."""
    f = api.rope_axes_freqs([16, 16], 100.0, 64)
    for p in range(32):
        i = p % 16
        want = np.float32(1.0) / np.float32(100.0 ** float(np.float32(2 * i) / np.float32(32)))
        assert abs(f[p, p // 16] - want) <= 2 * np.spacing(want) and f[p, 1 - p // 16] == 0
