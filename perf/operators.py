"""Workloads of the standalone operators on board tokens: the masked group norm with an activation (forward and
backward) and the rotary positions with several axes (forward, and backward with the gradient of learned
frequencies).

Channels 128 / 384 / 768, head dim 64 and 6 or 12 heads are those of the b10c128, b18c384nbt, b10c384h6 and
tf3-b11c768 nets; 361 points are a 19x19 board and multiples of it the positions of a game in a row. Where `own` is
false, `run` computes the operators in elementary torch operations; where it is true, it calls the library.
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5


def _norm(name, backward, n, points, channels, groups, act, dtype, masked, pad=0):
    return {"name": name, "op": "norm", "backward": backward, "n": n, "points": points, "channels": channels,
            "groups": groups, "act": act, "dtype": dtype, "masked": masked, "pad": pad}


def _rope(name, backward, tokens, q_heads, k_heads, head_dim, rotary_dim, axes, learned, layout, dtype):
    return {"name": name, "op": "rope", "backward": backward, "tokens": tokens, "q_heads": q_heads,
            "k_heads": k_heads, "head_dim": head_dim, "rotary_dim": rotary_dim, "axes": axes, "learned": learned,
            "layout": layout, "dtype": dtype}


def listed():
    return [
        # one position of a search: latency
        _norm("norm_1_board", False, 1, 361, 384, 32, "mish", "f16", True),
        # the benchmark batch, mixed board sizes
        _norm("norm_256_boards", False, 256, 361, 384, 32, "mish", "bf16", True),
        # one group per board, as the spatial norm of a transformer net's trunk tip
        _norm("norm_whole_board", False, 64, 361, 768, 1, "silu", "f32", True),
        # channel slice of a wider tensor, ragged sizes
        _norm("norm_ragged", False, 53, 137, 100, 20, "relu", "f16", True, 4),
        # 16 positions of a game as one sequence of points
        _norm("norm_game", False, 32, 5776, 256, 32, "silu", "bf16", False),
        # fine-tuning: a small float32 step and a full batch
        _norm("norm_back_8_boards", True, 8, 361, 128, 16, "relu", "f32", True),
        _norm("norm_back_512_boards", True, 512, 361, 384, 32, "mish", "bf16", True),
        # one token of a sequence: latency
        _rope("rotate_1_token", False, 1, 6, 6, 64, 64, 2, False, "halves", "bf16"),
        # Q and K of the benchmark batch with a learned table per key head
        _rope("rotate_256_boards", False, 256 * 361, 6, 6, 64, 64, 2, True, "halves", "f16"),
        # (move, row, column) positions of long games, grouped heads, part of each head rotated
        _rope("rotate_games", False, 160 * 361 + 7, 16, 4, 128, 96, 3, False, "pairs", "bf16"),
        # training: learned frequencies with grouped heads, and a fixed table in float32
        _rope("rotate_back_learned", True, 96 * 361, 12, 4, 64, 64, 2, True, "halves", "bf16"),
        _rope("rotate_back_fixed", True, 4099, 12, 12, 64, 64, 3, False, "pairs", "f32"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    dtype = rng.choice(["f32", "f16", "bf16"])
    backward = rng.random() < 0.45
    if rng.random() < 0.55:
        points = rng.choice([81, 169, 361, 400, _log_int(rng, 1, 6000), _log_int(rng, 20, 1000)])
        groups = rng.choice([1, 2, 4, 8, 16, 32, rng.randint(1, 40)])
        per = _log_int(rng, 1, max(1, 768 // groups))
        if rng.random() < 0.7:  # widths that vectors divide, as trunks have
            per = -(-per * groups // 8) * 8 // groups or 1
            per = max(per, 8 // math.gcd(8, groups))
            per -= per % (8 // math.gcd(8, groups))
        most = 40_000_000 // (points * per * groups)
        n = _log_int(rng, 1, max(1, min(512, most)))
        case = _norm("", backward, n, points, per * groups, groups, rng.choice(["identity", "relu", "mish", "silu"]),
                     dtype, rng.random() < 0.7, rng.choice([0, 0, 0, 8, 3]))
    else:
        axes = rng.randint(1, 4)
        head_dim = rng.choice([16, 32, 64, 64, 64, 96, 128, 2 * rng.randint(4, 60)])
        rotary_dim = head_dim if rng.random() < 0.7 else 2 * rng.randint(1, head_dim // 2)
        k_heads = rng.choice([1, 2, 4, 6, 8, 12])
        q_heads = k_heads * rng.choice([1, 1, 2, 3, 4])
        tokens = _log_int(rng, 1, max(1, min(100_000, 45_000_000 // ((q_heads + k_heads) * head_dim))))
        case = _rope("", backward, tokens, q_heads, k_heads, head_dim, rotary_dim, axes, rng.random() < 0.5,
                     rng.choice(["halves", "pairs"]), dtype)
    del case["name"]
    return case


def _board_side(i):
    return (19, 19, 13, 9)[i % 4]


def _on_points(points, i):
    """Points of board i that are on the board: the top-left corner of rows of 19 points."""
    side = _board_side(i)
    return sum(1 for p in range(points) if p % 19 < side and p // 19 % 19 < side)


def _on_total(case):
    if not case["masked"]:
        return case["n"] * case["points"]
    return sum((case["n"] + 3 - k) // 4 * _on_points(case["points"], k) for k in range(4))


def _norm_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, n, points, channels = DTYPES[case["dtype"]], case["n"], case["points"], case["channels"]

    def rows(scale, shift):
        wide = torch.empty(n, points, channels + case["pad"], dtype=dtype, device="cuda")
        wide.normal_(0.0, scale, generator=g).add_(shift)
        return wide[:, :, :channels]

    x = rows(1.3, 0.4)
    s = {"case": case, "x": x,
         "weight": torch.empty(channels, device="cuda").uniform_(0.8, 1.2, generator=g),
         "bias": torch.empty(channels, device="cuda").normal_(0.0, 0.2, generator=g), "mask": None}
    if case["masked"]:
        p = torch.arange(points, device="cuda")
        side = torch.tensor([_board_side(i) for i in range(n)], device="cuda")[:, None]
        s["mask"] = ((p % 19 < side) & (p // 19 % 19 < side)).float()
    if case["backward"]:
        s["dy"] = rows(1.0, 0.0)
        s["stats"] = _norm_stats(x.float(), s["mask"], case["groups"])  # saved by the forward pass
    return s


def _rope_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, tokens, axes, pairs = DTYPES[case["dtype"]], case["tokens"], case["axes"], case["rotary_dim"] // 2
    hq, hk, d = case["q_heads"], case["k_heads"], case["head_dim"]

    def qkv():  # Q | K | V columns of one linear's output, as its users see them
        wide = torch.empty(tokens, hq + 2 * hk, d, dtype=dtype, device="cuda").normal_(generator=g)
        return wide[:, :hq], wide[:, hq:hq + hk]

    t = torch.arange(tokens, device="cuda") + int(torch.randint(0, 361, (1,), generator=g, device="cuda"))
    pos = torch.stack([t % 361 % 19, t % 361 // 19, t // 361, t // 361 % 8][:axes], 1).to(torch.int32).contiguous()
    s = {"case": case, "pos": pos}
    s["q"], s["k"] = qkv()
    if case["learned"]:
        s["freqs"] = torch.empty(hk, pairs, axes, device="cuda").normal_(0.0, 0.3, generator=g)
    else:  # each axis its share of the pairs, frequencies theta^(-i / share) within it
        share = [(pairs + axes - 1 - a) // axes for a in range(axes)]
        freqs = torch.zeros(1, pairs, axes, dtype=torch.float64)
        at = 0
        for a in range(axes):
            if share[a]:
                freqs[0, at:at + share[a], a] = 100.0 ** -(torch.arange(share[a], dtype=torch.float64) / share[a])
            at += share[a]
        s["freqs"] = freqs.float().cuda()
    if case["backward"]:
        s["dq_out"] = torch.empty(tokens, hq, d, dtype=dtype, device="cuda").normal_(generator=g)
        s["dk_out"] = torch.empty(tokens, hk, d, dtype=dtype, device="cuda").normal_(generator=g)
    return s


def prepare(case, seed):
    return (_norm_inputs if case["op"] == "norm" else _rope_inputs)(case, seed)


# ---- plain forms: 32 bits (angles and the sums over all tokens in 64), rounded once at the end ----


def _norm_stats(xf, mask, groups):
    n, points, channels = xf.shape
    xg = xf.reshape(n, points, groups, -1)
    if mask is None:
        count = points * xg.shape[3]
        mean = xg.sum((1, 3)) / count
        d = xg - mean[:, None, :, None]
    else:
        on = (mask != 0)[:, :, None, None]
        count = (on.sum((1, 2, 3)) * xg.shape[3]).clamp(min=1).float()[:, None]
        mean = torch.where(on, xg, 0.0).sum((1, 3)) / count
        d = torch.where(on, xg - mean[:, None, :, None], 0.0)
    var = (d * d).sum((1, 3)) / count
    return torch.stack([mean, 1.0 / torch.sqrt(var + EPS)], 2)


def _sigmoid(z):
    e = torch.exp(-z.abs())
    return torch.where(z >= 0, 1.0, e) / (1.0 + e)


def _mish_gate(z):
    """tanh(softplus(z)) = n / (n + 2) with n = e^2 + 2 e, e = exp(z) (1 in 32 bits above 20)."""
    e = torch.exp(z.clamp(max=20.0))
    n = e * (e + 2.0)
    return n / (n + 2.0)


def _act(z, act):
    if act == "relu":
        return z.clamp(min=0.0)
    if act == "mish":
        return z * _mish_gate(z)
    if act == "silu":
        return z * _sigmoid(z)
    return z


def _relu_slope(x, stats, weight, bias):
    """1 where z > 0, in 64 bits from the saved statistics: 32 bits put values next to 0 on either side."""
    mean, rstd = stats.double()[:, None, :, None, 0], stats.double()[:, None, :, None, 1]
    z = ((x.double().unflatten(2, (stats.shape[1], -1)) - mean) * rstd).flatten(2) * weight.double() + bias.double()
    return (z > 0).float()


def _act_slope(z, act):
    if act == "mish":
        t = _mish_gate(z)
        return t + z * _sigmoid(z) * (1.0 - t * t)
    if act == "silu":
        s = _sigmoid(z)
        return s * (1.0 + z * (1.0 - s))
    return torch.ones_like(z)


def _plain_norm(s):
    case, mask = s["case"], s["mask"]
    n, points, channels, groups = case["n"], case["points"], case["channels"], case["groups"]
    xf = s["x"].float()
    stats = s["stats"] if case["backward"] else _norm_stats(xf, mask, groups)
    mean, rstd = stats[:, None, :, None, 0], stats[:, None, :, None, 1]
    xh = (xf.reshape(n, points, groups, -1) - mean) * rstd
    z = xh.reshape(n, points, channels) * s["weight"] + s["bias"]
    on = None if mask is None else (mask != 0)[:, :, None]
    if not case["backward"]:
        y = _act(z, case["act"])
        y = y if on is None else torch.where(on, y, 0.0)
        return {"y": y.to(s["x"].dtype), "stats": stats}
    slope = _relu_slope(s["x"], stats, s["weight"], s["bias"]) if case["act"] == "relu" else _act_slope(z, case["act"])
    gz = s["dy"].float() * slope
    gz = gz if on is None else torch.where(on, gz, 0.0)
    count = (torch.full((n, 1), float(points), device=gz.device) if on is None
             else on.sum((1, 2)).clamp(min=1).float()[:, None]) * (channels // groups)
    xh = xh.reshape(n, points, channels)
    s1, s2 = gz.sum(1), (gz * (xh if on is None else torch.where(on, xh, 0.0))).sum(1)
    c1 = (s1 * s["weight"]).reshape(n, groups, -1).sum(2) / count
    c2 = (s2 * s["weight"]).reshape(n, groups, -1).sum(2) / count
    dx = (gz * s["weight"]).reshape(n, points, groups, -1) - c1[:, None, :, None]
    dx = (dx - xh.reshape(n, points, groups, -1) * c2[:, None, :, None]) * rstd
    dx = dx.reshape(n, points, channels)
    dx = dx if on is None else torch.where(on, dx, 0.0)
    return {"dx": dx.to(s["x"].dtype), "dweight": s2.sum(0), "dbias": s1.sum(0)}


def _split(x, rotary_dim, layout):
    xf = x[..., :rotary_dim].float()
    if layout == "halves":
        return xf[..., :rotary_dim // 2], xf[..., rotary_dim // 2:]
    return xf[..., 0::2], xf[..., 1::2]


def _join(a, b, x, rotary_dim, layout):
    r = torch.cat([a, b], -1) if layout == "halves" else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([r.to(x.dtype), x[..., rotary_dim:]], -1)


def _plain_rope(s):
    case = s["case"]
    rd, layout, hk = case["rotary_dim"], case["layout"], case["k_heads"]
    angle = (s["pos"].double()[:, None, None, :] * s["freqs"].double()).sum(3)  # [tokens][tables][pairs]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    group = case["q_heads"] // hk
    if not case["learned"]:
        per_q, per_k = (cos, sin), (cos, sin)
    else:
        per_q, per_k = (cos.repeat_interleave(group, 1), sin.repeat_interleave(group, 1)), (cos, sin)

    def turned(x, table, back):
        a, b = _split(x, rd, layout)
        c, sn = table[0], -table[1] if back else table[1]
        return a * c - b * sn, a * sn + b * c

    if not case["backward"]:
        return {"q": _join(*turned(s["q"], per_q, False), s["q"], rd, layout),
                "k": _join(*turned(s["k"], per_k, False), s["k"], rd, layout)}
    dq, dk = turned(s["dq_out"], per_q, True), turned(s["dk_out"], per_k, True)
    out = {"dq": _join(*dq, s["dq_out"], rd, layout), "dk": _join(*dk, s["dk_out"], rd, layout)}
    if case["learned"]:
        qa, qb = _split(s["q"], rd, layout)
        ka, kb = _split(s["k"], rd, layout)
        turn = (dq[1] * qa - dq[0] * qb).reshape(case["tokens"], hk, group, rd // 2).sum(2) + (dk[1] * ka - dk[0] * kb)
        out["dfreqs"] = (turn.double()[..., None] * s["pos"].double()[:, None, None, :]).sum(0).float()
    return out


# ---- the library's calls ----


def _api():
    at = os.path.join(os.getcwd(), "katago-rs_b200", "python")
    if at not in sys.path:
        sys.path.insert(0, at)
    from katago_cuda import api
    return api


def _code(api, kind, name):
    return getattr(api, "%s_%s" % (kind, name.upper()))


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _own_norm(s):
    api, case, x, mask = _api(), s["case"], s["x"], s["mask"]
    stream = torch.cuda.current_stream().cuda_stream
    n, points, channels, groups = case["n"], case["points"], case["channels"], case["groups"]
    other = s["dy"] if case["backward"] else torch.empty(n, points, channels, dtype=x.dtype, device=x.device)
    desc = api.GroupNormDesc(_code(api, "PRECISION", case["dtype"]), _code(api, "ACT", case["act"]), n, points,
                             channels, groups, EPS, x_strides=(x.stride(0), x.stride(1)),
                             y_strides=(other.stride(0), other.stride(1)))
    size = api.group_norm_act_workspace(desc, case["backward"])
    work = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
    if not case["backward"]:
        stats = torch.empty(n, groups, 2, device=x.device)
        api.group_norm_act(desc, x.data_ptr(), _ptr(mask), s["weight"].data_ptr(), s["bias"].data_ptr(),
                           other.data_ptr(), stats.data_ptr(), _ptr(work), size, stream)
        return {"y": other, "stats": stats}
    dx = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device=x.device)
    dweight, dbias = torch.empty(channels, device=x.device), torch.empty(channels, device=x.device)
    api.group_norm_act_backward(desc, x.data_ptr(), _ptr(mask), s["weight"].data_ptr(), s["bias"].data_ptr(),
                                s["stats"].data_ptr(), other.data_ptr(), dx.data_ptr(), dweight.data_ptr(),
                                dbias.data_ptr(), _ptr(work), size, stream)
    return {"dx": dx, "dweight": dweight, "dbias": dbias}


def _own_rope(s):
    api, case, q, k = _api(), s["case"], s["q"], s["k"]
    stream = torch.cuda.current_stream().cuda_stream
    tokens, hq, hk, d = case["tokens"], case["q_heads"], case["k_heads"], case["head_dim"]
    desc = api.RopeDesc(_code(api, "PRECISION", case["dtype"]), _code(api, "ROPE", case["layout"]), case["axes"],
                        tokens, hq, hk, d, case["rotary_dim"], s["freqs"].shape[0],
                        q_strides=(q.stride(0), q.stride(1)), k_strides=(k.stride(0), k.stride(1)),
                        q_out_strides=(hq * d, d), k_out_strides=(hk * d, d))
    if not case["backward"]:
        q_out, k_out = torch.empty_like(q, memory_format=torch.contiguous_format), torch.empty_like(
            k, memory_format=torch.contiguous_format)
        api.rope_axes(desc, q.data_ptr(), k.data_ptr(), s["pos"].data_ptr(), s["freqs"].data_ptr(), q_out.data_ptr(),
                      k_out.data_ptr(), stream)
        return {"q": q_out, "k": k_out}
    wide = torch.empty(tokens, hq + 2 * hk, d, dtype=q.dtype, device=q.device)  # laid out as Q | K | V
    dq, dk = wide[:, :hq], wide[:, hq:hq + hk]
    out = {"dq": dq, "dk": dk}
    dfreqs, work, size = None, None, 0
    if case["learned"]:
        dfreqs = torch.empty_like(s["freqs"])
        size = api.rope_axes_backward_workspace(desc)
        work = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
        out["dfreqs"] = dfreqs
    api.rope_axes_backward(desc, s["dq_out"].data_ptr(), s["dk_out"].data_ptr(), q.data_ptr() if case["learned"] else 0,
                           k.data_ptr() if case["learned"] else 0, s["pos"].data_ptr(), s["freqs"].data_ptr(),
                           dq.data_ptr(), dk.data_ptr(), _ptr(dfreqs), _ptr(work), size, stream)
    return out


def run(state):
    norm = state["case"]["op"] == "norm"
    if own:
        return _own_norm(state) if norm else _own_rope(state)
    return _plain_norm(state) if norm else _plain_rope(state)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "norm":
        # rows off the board are written as zeros and need not be read
        on, rows, channels = _on_total(case), case["n"] * case["points"], case["channels"]
        mask = 4 * rows if case["masked"] else 0
        small = 4 * 2 * channels + 8 * case["n"] * case["groups"]
        if case["backward"]:
            moved = size * channels * (2 * on + rows) + mask + small + 8 * channels
            return {"bytes": moved, "flops": 30 * on * channels}
        return {"bytes": size * channels * (on + rows) + mask + small, "flops": 14 * on * channels}
    heads, tokens, d, rd = case["q_heads"] + case["k_heads"], case["tokens"], case["head_dim"], case["rotary_dim"]
    tables = case["k_heads"] if case["learned"] else 1
    freqs = 4 * tables * rd // 2 * case["axes"]
    moved = 2 * size * tokens * heads * d + 4 * tokens * case["axes"] + freqs
    flops = 3 * tokens * heads * rd + tokens * tables * rd // 2 * (2 * case["axes"] + 20)
    if case["backward"] and case["learned"]:
        moved += size * tokens * heads * rd + freqs
        flops += tokens * heads * rd * 2 + 2 * tokens * tables * rd // 2 * case["axes"]
    return {"bytes": moved, "flops": flops}


# ---- the definitions in 64 bits, by other means than the plain forms ----


def _exact_norm_part(x, mask, weight, bias, groups, act, saved=None):
    """act(weight * (x - mean) / sqrt(var + eps) + bias) of some boards, with the moments as E[x], E[(x - E[x])^2]
    over the points that are on; x [boards][points][channels] float64. A backward pass takes relu's side of 0 from
    the saved statistics, which are its inputs."""
    boards, points, channels = x.shape
    on = torch.ones(boards, points, dtype=torch.float64, device=x.device) if mask is None else (mask != 0).double()
    share = on / on.sum(1, keepdim=True).clamp(min=1.0) * groups / channels
    xg = (x * on[:, :, None]).unflatten(2, (groups, channels // groups))
    mean = torch.einsum("bpgc,bp->bg", xg, share)
    var = torch.einsum("bpgc,bp->bg", (xg - mean[:, None, :, None]) ** 2, share)
    rstd = (var + EPS) ** -0.5
    z = ((xg - mean[:, None, :, None]) * rstd[:, None, :, None]).flatten(2) * weight + bias
    if act == "relu":
        m, r = (mean, rstd) if saved is None else (saved[:, :, 0], saved[:, :, 1])
        side = ((xg - m[:, None, :, None]) * r[:, None, :, None]).flatten(2) * weight + bias
        z = z * (side > 0).detach()
    elif act == "mish":
        z = z * torch.tanh(torch.logaddexp(z, torch.zeros((), dtype=torch.float64, device=z.device)))
    elif act == "silu":
        z = z / (1.0 + torch.exp(-z))
    return z * on[:, :, None], torch.stack([mean, rstd], 2)


def _exact_norm(case, seed):
    s = _norm_inputs(case, seed)
    n, points, channels = case["n"], case["points"], case["channels"]
    weight, bias = s["weight"].double().requires_grad_(), s["bias"].double().requires_grad_()
    step = max(1, 30_000_000 // (points * channels))
    parts = []
    for i in range(0, n, step):
        x = s["x"][i:i + step].double()
        mask = None if s["mask"] is None else s["mask"][i:i + step]
        if not case["backward"]:
            with torch.no_grad():
                parts.append(_exact_norm_part(x, mask, weight, bias, case["groups"], case["act"]))
            continue
        x.requires_grad_()
        y, _ = _exact_norm_part(x, mask, weight, bias, case["groups"], case["act"], s["stats"][i:i + step].double())
        parts.append(torch.autograd.grad(y, [x, weight, bias], s["dy"][i:i + step].double()))
        del y, x
    if not case["backward"]:
        return {"y": torch.cat([p[0] for p in parts]), "stats": torch.cat([p[1] for p in parts])}
    return {"dx": torch.cat([p[0] for p in parts]), "dweight": sum(p[1] for p in parts),
            "dbias": sum(p[2] for p in parts)}


def _exact_rope(case, seed):
    """Each pair as a complex number, turned by exp(i angle)."""
    s = _rope_inputs(case, seed)
    rd, group = case["rotary_dim"], case["q_heads"] // case["k_heads"]
    angle = torch.einsum("ta,hja->thj", s["pos"].double(), s["freqs"].double())
    unit = torch.polar(torch.ones_like(angle), angle)

    def pairs(x):
        x = x[..., :rd].double()
        if case["layout"] == "halves":
            x = x.unflatten(-1, (2, rd // 2)).transpose(-1, -2).flatten(-2)
        return torch.view_as_complex(x.unflatten(-1, (rd // 2, 2)).contiguous())

    def rows(z, x):
        r = torch.view_as_real(z)
        r = r.flatten(-2) if case["layout"] == "pairs" else r.transpose(-1, -2).flatten(-2)
        return torch.cat([r, x[..., rd:].double()], -1)

    uq = unit if not case["learned"] else unit[:, torch.arange(case["q_heads"], device=unit.device) // group]
    if not case["backward"]:
        return {"q": rows(pairs(s["q"]) * uq, s["q"]), "k": rows(pairs(s["k"]) * unit, s["k"])}
    out = {"dq": rows(pairs(s["dq_out"]) * uq.conj(), s["dq_out"]),
           "dk": rows(pairs(s["dk_out"]) * unit.conj(), s["dk_out"])}
    if case["learned"]:
        # the loss is Re(conj(g) x exp(i angle)): its derivative by the angle is -Im(conj(g) x exp(i angle))
        dq = -(pairs(s["dq_out"]).conj() * pairs(s["q"]) * uq).imag.unflatten(1, (case["k_heads"], group)).sum(2)
        dk = -(pairs(s["dk_out"]).conj() * pairs(s["k"]) * unit).imag
        out["dfreqs"] = torch.einsum("thj,ta->hja", dq + dk, s["pos"].double())
    return out


def exact(case, seed):
    return (_exact_norm if case["op"] == "norm" else _exact_rope)(case, seed)
