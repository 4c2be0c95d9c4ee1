"""Workloads of the operators around a token net's blocks in training and serving: the norm of each token (layer and
RMS norm, forward and backward), learned rows looked up by token (forward and the gradient of the table), and the loss
against a teacher's top logits (forward and the gradient of the logits).

Channels 384 / 768 are those of the b18c384nbt, b10c384h6 and tf3-b11c768 nets, 361 points a 19x19 board, 362 the moves
of a policy row. Where `own` is false, `run` computes the operators in elementary torch operations; where it is true, it
calls the library.
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def _norm(name, backward, n, points, channels, kind, dtype, masked, pad=0):
    return {"name": name, "op": "norm", "backward": backward, "n": n, "points": points, "channels": channels,
            "kind": kind, "dtype": dtype, "masked": masked, "pad": pad}


def _embed(name, backward, tokens, channels, table_rows, ids, dtype, add=False, pad=0):
    return {"name": name, "op": "embed", "backward": backward, "tokens": tokens, "channels": channels,
            "table_rows": table_rows, "ids": ids, "dtype": dtype, "add": add, "pad": pad}


def _distill(name, backward, rows, classes, top, temperature, dtype, illegal, whole=False):
    return {"name": name, "op": "distill", "backward": backward, "rows": rows, "classes": classes, "top": top,
            "temperature": temperature, "dtype": dtype, "illegal": illegal, "whole": whole}


def listed():
    return [
        # one position of a search, the norm of the transformer nets: latency
        _norm("norm_1_board", False, 1, 361, 384, "rms", "f16", True),
        # the benchmark batch, mixed board sizes
        _norm("norm_256_boards", False, 256, 361, 384, "layer", "bf16", True),
        # channel slice of a wider tensor, ragged sizes
        _norm("norm_back_ragged", True, 53, 137, 100, "layer", "f16", True, 4),
        # fine-tuning step of the widest net
        _norm("norm_back_128_boards", True, 128, 361, 768, "rms", "bf16", False),
        # one board's points through a table of point rows: latency
        _embed("embed_1_board", False, 361, 384, 362, "points", "f16"),
        # learned positions of 16 moves x 361 points added to the tokens of many games
        _embed("embed_games", False, 160 * 361 + 7, 768, 16 * 361, "points", "bf16", True),
        # gradient of a table of moves, some far more frequent than others
        _embed("embed_back_moves", True, 256 * 361, 384, 362, "skewed", "bf16"),
        # gradient of a large table of which few rows are met, with padding
        _embed("embed_back_vocabulary", True, 20011, 512, 50000, "skewed", "f32"),
        # policy rows of a training batch, illegal points at -inf
        _distill("distill_policy", False, 256, 362, 32, 1.0, "f32", True),
        # few long rows, odd length
        _distill("distill_few_rows", False, 12, 131071, 64, 2.0, "f16", False),
        # gradient of the policy rows of 16,384 positions, their search's whole distribution known
        _distill("distill_back_policy", True, 16384, 362, 64, 1.0, "bf16", True, True),
        # gradient over a large vocabulary
        _distill("distill_back_vocabulary", True, 4096, 32000, 128, 1.5, "bf16", False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    dtype = rng.choice(["f32", "f16", "bf16"])
    backward = rng.random() < 0.5
    op = rng.choice(["norm", "embed", "distill"])
    if op == "norm":
        channels = rng.choice([128, 256, 384, 768, _log_int(rng, 1, 8192), 8 * _log_int(rng, 1, 1024)])
        points = rng.choice([1, 81, 169, 361, _log_int(rng, 1, 6000)])
        n = _log_int(rng, 1, max(1, min(512, 40_000_000 // (points * channels))))
        case = _norm("", backward, n, points, channels, rng.choice(["layer", "rms"]), dtype, rng.random() < 0.5,
                     rng.choice([0, 0, 0, 8, 3]))
    elif op == "embed":
        channels = rng.choice([128, 256, 384, 768, _log_int(rng, 1, 4096), 8 * _log_int(rng, 1, 512)])
        table_rows = rng.choice([2, 362, 5776, _log_int(rng, 1, max(1, min(200_000, 40_000_000 // channels)))])
        table_rows = min(table_rows, max(1, 40_000_000 // channels))
        tokens = _log_int(rng, 1, max(1, min(400_000, 40_000_000 // channels)))
        case = _embed("", backward, tokens, channels, table_rows, rng.choice(["points", "skewed", "even"]), dtype,
                      rng.random() < 0.5 and not backward, rng.choice([0, 0, 0, 8, 3]))
    else:
        illegal = rng.random() < 0.5
        classes = 362 if illegal else rng.choice([362, _log_int(rng, 2, 150_000), 64 * _log_int(rng, 1, 2000)])
        rows = _log_int(rng, 1, max(1, min(60_000, 80_000_000 // classes)))
        top = min(_log_int(rng, 1, 256), max(1, classes // 5))
        case = _distill("", backward, rows, classes, top, rng.choice([1.0, 1.0, 0.5, 2.0, 4.0]), dtype, illegal,
                        rng.random() < 0.3)
    del case["name"]
    return case


# ---- inputs ----


def _board_side(i):
    return (19, 19, 13, 9)[i % 4]


def _on_total(case):
    if not case["masked"]:
        return case["n"] * case["points"]
    on = [sum(1 for p in range(case["points"]) if p % 19 < s and p // 19 % 19 < s) for s in (19, 19, 13, 9)]
    return sum((case["n"] + 3 - k) // 4 * on[k] for k in range(4))


def _norm_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, n, points, channels = DTYPES[case["dtype"]], case["n"], case["points"], case["channels"]

    def rows(scale, shift):
        wide = torch.empty(n, points, channels + case["pad"], dtype=dtype, device="cuda")
        wide.normal_(0.0, scale, generator=g).add_(shift)
        return wide[:, :, :channels]

    s = {"case": case, "x": rows(1.3, 0.4), "mask": None,
         "weight": torch.empty(channels, device="cuda").uniform_(0.8, 1.2, generator=g),
         "bias": torch.empty(channels, device="cuda").normal_(0.0, 0.2, generator=g)}
    if case["kind"] == "rms":  # as the nets' blocks: a weight alone
        s["bias"] = None
    if case["masked"]:
        p = torch.arange(points, device="cuda")
        side = torch.tensor([_board_side(i) for i in range(n)], device="cuda")[:, None]
        s["mask"] = ((p % 19 < side) & (p // 19 % 19 < side)).float()
    if case["backward"]:
        s["dy"] = rows(1.0, 0.0)
        s["stats"] = _norm_stats(s["x"].float(), s["mask"], case["kind"])  # saved by the forward pass
    return s


def _embed_ids(case, g):
    tokens, rows = case["tokens"], case["table_rows"]
    if case["ids"] == "points":  # board after board, move after move
        start = torch.randint(0, rows, (1,), generator=g, device="cuda")
        ids = (torch.arange(tokens, device="cuda") + start) % rows
    else:
        u = torch.rand(tokens, generator=g, device="cuda", dtype=torch.float64)
        if case["ids"] == "skewed":  # a few rows most of the time
            order = torch.randperm(rows, generator=g, device="cuda")
            ids = order[((rows + 1.0) ** u - 1.0).long().clamp(max=rows - 1)]
        else:
            ids = (u * rows).long().clamp(max=rows - 1)
        pad = torch.rand(tokens, generator=g, device="cuda") < 0.03
        ids = torch.where(pad, -1, ids)
    return ids.to(torch.int32)


def _embed_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, tokens, channels = DTYPES[case["dtype"]], case["tokens"], case["channels"]

    def rows(count, scale):
        wide = torch.empty(count, channels + case["pad"], dtype=dtype, device="cuda").normal_(0.0, scale, generator=g)
        return wide[:, :channels]

    s = {"case": case, "ids": _embed_ids(case, g), "scale": channels ** 0.5}
    if case["backward"]:
        s["dy"] = rows(tokens, 1.0)
    else:
        s["table"] = rows(case["table_rows"], channels ** -0.5)
        s["x"] = rows(tokens, 1.0) if case["add"] else None
    return s


def _distill_inputs(case, seed):
    """A student near its teacher: the teacher's logits are the student's, scaled, with noise; its `top` best classes
    are known. Some rows have fewer entries (id -1 behind them) and some none."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, classes, top = case["rows"], case["classes"], case["top"]
    z = torch.empty(rows, classes, dtype=DTYPES[case["dtype"]], device="cuda").normal_(0.0, 2.0, generator=g)
    r = torch.arange(rows, device="cuda")
    if case["illegal"]:
        c = torch.arange(classes, device="cuda")
        side = torch.tensor([_board_side(i) for i in range(4)], device="cuda")[r % 4][:, None]
        off = (c < 361) & ((c % 19 >= side) | (c // 19 >= side))
        z.masked_fill_(off, float("-inf"))
    teacher = torch.empty_like(z).normal_(0.0, 1.0, generator=g).add_(z)
    best = teacher.float().topk(top, 1)
    whole = torch.logsumexp(teacher.double() / case["temperature"], 1).float() if case["whole"] else None
    del teacher
    count = torch.where(r % 3 == 1, (top + 1) // 2, top)
    count = torch.where(r % 17 == 5, 0, count)[:, None]
    ids = torch.where(torch.arange(top, device="cuda") < count, best.indices, -1).to(torch.int32)
    s = {"case": case, "logits": z, "ids": ids, "top_logits": best.values.contiguous(), "whole": whole}
    if case["backward"]:
        s["dloss"] = torch.empty(rows, device="cuda").uniform_(0.5, 1.5, generator=g) / rows
        m, total = _largest_and_sum(z, case["temperature"])
        some = ids.ge(0).any(1)
        s["stats"] = torch.stack([torch.where(some, m, 0.0), torch.where(some, total, 0.0)], 1)
    return s


_INPUTS = {"norm": _norm_inputs, "embed": _embed_inputs, "distill": _distill_inputs}


def prepare(case, seed):
    return _INPUTS[case["op"]](case, seed)


# ---- plain forms: 32 bits (sums over all tokens and differences of logarithms in 64), rounded once at the end ----


def _norm_stats(xf, mask, kind):
    mean = xf.sum(2) / xf.shape[2] if kind == "layer" else torch.zeros(xf.shape[:2], device=xf.device)
    d = xf - mean[:, :, None]
    stats = torch.stack([mean, 1.0 / torch.sqrt((d * d).sum(2) / xf.shape[2] + EPS)], 2)
    return stats if mask is None else torch.where((mask != 0)[:, :, None], stats, 0.0)


def _plain_norm(s):
    case, xf = s["case"], s["x"].float()
    on = None if s["mask"] is None else (s["mask"] != 0)[:, :, None]
    stats = s["stats"] if case["backward"] else _norm_stats(xf, s["mask"], case["kind"])
    mean, rstd = stats[:, :, 0:1], stats[:, :, 1:2]
    xh = (xf - mean) * rstd
    if not case["backward"]:
        y = xh * s["weight"]
        y = y if s["bias"] is None else y + s["bias"]
        y = y if on is None else torch.where(on, y, 0.0)
        return {"y": y.to(s["x"].dtype), "stats": stats}
    dy = s["dy"].float()
    if on is not None:
        xh, dy = torch.where(on, xh, 0.0), torch.where(on, dy, 0.0)
    g = dy * s["weight"]
    dx = g - xh * ((g * xh).sum(2, keepdim=True) / case["channels"])
    if case["kind"] == "layer":
        dx = dx - g.sum(2, keepdim=True) / case["channels"]
    out = {"dx": (dx * rstd).to(s["x"].dtype), "dweight": (dy * xh).sum((0, 1), dtype=torch.float64).float()}
    if s["bias"] is not None:
        out["dbias"] = dy.sum((0, 1), dtype=torch.float64).float()
    return out


def _plain_embed(s):
    case, ids = s["case"], s["ids"].long()
    there = ids >= 0
    if not case["backward"]:
        y = s["table"][ids.clamp(min=0)].float() * s["scale"]
        y = torch.where(there[:, None], y, 0.0)
        y = y if s["x"] is None else y + s["x"].float()
        return {"y": y.to(s["table"].dtype)}
    total = torch.zeros(case["table_rows"] + 1, case["channels"], dtype=torch.float64, device=ids.device)
    total.index_add_(0, torch.where(there, ids, case["table_rows"]), s["dy"].double())
    return {"dtable": (total[:-1] * s["scale"]).float()}


def _largest_and_sum(z, temperature):
    zf = z.float()
    m = zf.amax(1)
    return m, torch.exp((zf - m[:, None]) / temperature).sum(1)


def _teacher(s):
    """p and log p of the entries, 0 where there is none; in 64 bits, since the loss is a difference of logarithms."""
    there = s["ids"] >= 0
    t = s["top_logits"].double() / s["case"]["temperature"]
    if s["whole"] is None:
        m = torch.where(there, t, float("-inf")).amax(1, keepdim=True)
        m = torch.where(there.any(1, keepdim=True), m, 0.0)
        lse = m + torch.log(torch.where(there, torch.exp(t - m), 0.0).sum(1, keepdim=True))
    else:
        lse = s["whole"].double()[:, None]
    log_p = torch.where(there, t - lse, 0.0)
    return there, torch.where(there, torch.exp(log_p), 0.0), log_p


def _plain_distill(s):
    case, z, temperature = s["case"], s["logits"], s["case"]["temperature"]
    there, p, log_p = _teacher(s)
    ids = s["ids"].long().clamp(min=0)
    some = there.any(1)
    if not case["backward"]:
        m, total = _largest_and_sum(z, temperature)
        log_q = (z.gather(1, ids).double() - m.double()[:, None]) / temperature - torch.log(total.double())[:, None]
        loss = temperature ** 2 * torch.where(p > 0, p * (log_p - log_q), 0.0).sum(1)
        stats = torch.where(some[:, None], torch.stack([m, total], 1), 0.0)
        return {"loss": loss.float(), "stats": stats}
    m, total = s["stats"][:, 0:1], s["stats"][:, 1:2]
    p = p.float()
    dz = torch.exp((z.float() - m) / temperature) * (p.sum(1, keepdim=True) / total)
    dz.scatter_add_(1, ids, -p)
    dz = dz * (s["dloss"] * temperature)[:, None]
    return {"dlogits": torch.where(some[:, None], dz, 0.0).to(z.dtype)}


# ---- the library's calls ----


def _api():
    at = os.path.join(os.getcwd(), "katago-rs_b200", "python")
    if at not in sys.path:
        sys.path.insert(0, at)
    from katago_cuda import api
    return api


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _space(size, device):
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


def _own_norm(s):
    api, case, x = _api(), s["case"], s["x"]
    stream = torch.cuda.current_stream().cuda_stream
    n, points, channels = case["n"], case["points"], case["channels"]
    other = s["dy"] if case["backward"] else torch.empty(n, points, channels, dtype=x.dtype, device=x.device)
    desc = api.LayerNormDesc(getattr(api, "PRECISION_" + case["dtype"].upper()),
                             getattr(api, "NORM_" + case["kind"].upper()), n, points, channels, EPS,
                             x_strides=(x.stride(0), x.stride(1)), y_strides=(other.stride(0), other.stride(1)))
    if not case["backward"]:
        stats = torch.empty(n, points, 2, device=x.device)
        api.layer_norm(desc, x.data_ptr(), _ptr(s["mask"]), s["weight"].data_ptr(), _ptr(s["bias"]), other.data_ptr(),
                       stats.data_ptr(), stream)
        return {"y": other, "stats": stats}
    dx = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device=x.device)
    out = {"dx": dx, "dweight": torch.empty(channels, device=x.device)}
    if s["bias"] is not None:
        out["dbias"] = torch.empty(channels, device=x.device)
    size = api.layer_norm_backward_workspace(desc)
    work_space = _space(size, x.device)
    api.layer_norm_backward(desc, x.data_ptr(), _ptr(s["mask"]), s["weight"].data_ptr(), s["stats"].data_ptr(),
                            other.data_ptr(), dx.data_ptr(), out["dweight"].data_ptr(), _ptr(out.get("dbias")),
                            _ptr(work_space), size, stream)
    return out


def _own_embed(s):
    api, case, ids = _api(), s["case"], s["ids"]
    stream = torch.cuda.current_stream().cuda_stream
    tokens, channels, rows = case["tokens"], case["channels"], case["table_rows"]
    dtype = getattr(api, "PRECISION_" + case["dtype"].upper())
    if not case["backward"]:
        table, x = s["table"], s["x"]
        y = torch.empty(tokens, channels, dtype=table.dtype, device=table.device)
        desc = api.EmbedDesc(dtype, tokens, channels, rows, s["scale"], table_stride=table.stride(0),
                             x_stride=None if x is None else x.stride(0))
        api.embed_rows(desc, ids.data_ptr(), table.data_ptr(), _ptr(x), y.data_ptr(), stream)
        return {"y": y}
    dy = s["dy"]
    dtable = torch.empty(rows, channels, device=dy.device)
    desc = api.EmbedDesc(dtype, tokens, channels, rows, s["scale"], y_stride=dy.stride(0))
    size = api.embed_rows_backward_workspace(desc)
    work_space = _space(size, dy.device)
    api.embed_rows_backward(desc, ids.data_ptr(), dy.data_ptr(), dtable.data_ptr(), _ptr(work_space), size, stream)
    return {"dtable": dtable}


def _own_distill(s):
    api, case, z = _api(), s["case"], s["logits"]
    stream = torch.cuda.current_stream().cuda_stream
    rows = case["rows"]
    desc = api.DistillDesc(getattr(api, "PRECISION_" + case["dtype"].upper()), rows, case["classes"], case["top"],
                           case["temperature"])
    if not case["backward"]:
        loss, stats = torch.empty(rows, device=z.device), torch.empty(rows, 2, device=z.device)
        api.distill_top(desc, z.data_ptr(), s["ids"].data_ptr(), s["top_logits"].data_ptr(), _ptr(s["whole"]),
                        loss.data_ptr(), stats.data_ptr(), stream)
        return {"loss": loss, "stats": stats}
    dlogits = torch.empty_like(z)
    api.distill_top_backward(desc, z.data_ptr(), s["ids"].data_ptr(), s["top_logits"].data_ptr(), _ptr(s["whole"]),
                             s["stats"].data_ptr(), s["dloss"].data_ptr(), dlogits.data_ptr(), stream)
    return {"dlogits": dlogits}


_OWN = {"norm": _own_norm, "embed": _own_embed, "distill": _own_distill}
_PLAIN = {"norm": _plain_norm, "embed": _plain_embed, "distill": _plain_distill}


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "norm":
        # rows that are off are written as zeros and need not be read
        on, rows, channels = _on_total(case), case["n"] * case["points"], case["channels"]
        small = (4 * rows if case["masked"] else 0) + 8 * rows + 8 * channels
        if case["backward"]:
            return {"bytes": size * channels * (2 * on + rows) + small + 8 * channels, "flops": 14 * on * channels}
        return {"bytes": size * channels * (on + rows) + small, "flops": 8 * on * channels}
    if case["op"] == "embed":
        tokens, channels, rows = case["tokens"], case["channels"], case["table_rows"]
        if case["backward"]:
            return {"bytes": tokens * (4 + size * channels) + 4 * rows * channels, "flops": tokens * channels}
        met = min(tokens, rows)  # at most: a row is read once
        return {"bytes": 4 * tokens + size * channels * (met + tokens * (2 if case["add"] else 1)),
                "flops": (2 if case["add"] else 1) * tokens * channels}
    rows, classes, top = case["rows"], case["classes"], case["top"]
    some = rows - (rows + 11) // 17  # rows without entries are not read
    small = rows * (8 * top + 12 + (4 if case["whole"] else 0))
    if case["backward"]:
        return {"bytes": size * classes * (some + rows) + small, "flops": 5 * some * classes}
    return {"bytes": size * classes * some + small, "flops": 5 * some * classes}


# ---- the definitions in 64 bits, by other means than the plain forms ----


def _exact_norm(case, seed):
    s = _norm_inputs(case, seed)
    channels = case["channels"]
    x = s["x"].double().reshape(-1, channels)
    on = (torch.ones(x.shape[0], 1, device=x.device) if s["mask"] is None else s["mask"].reshape(-1, 1)) != 0
    w = s["weight"].double()
    b = torch.zeros_like(w) if s["bias"] is None else s["bias"].double()
    if not case["backward"]:
        mean = x.mean(1, keepdim=True) * (case["kind"] == "layer")
        rstd = ((x * x).mean(1, keepdim=True) - mean * mean + EPS) ** -0.5
        y = torch.addcmul(b, (x - mean) * rstd, w) * on
        shape = s["x"].shape
        return {"y": y.reshape(shape), "stats": (torch.cat([mean, rstd], 1) * on).reshape(*shape[:2], 2)}
    # by the statistics that are the call's inputs: the Jacobian's product with dy w
    mean, rstd = s["stats"].double().reshape(-1, 2).unbind(1)
    dy = s["dy"].double().reshape(-1, channels) * on
    xh = torch.einsum("rc,r->rc", x - mean[:, None], rstd) * on
    g = dy * w
    dx = g - torch.einsum("rc,r->rc", xh, torch.einsum("rc,rc->r", g, xh) / channels)
    if case["kind"] == "layer":
        dx -= g.mean(1, keepdim=True)
    out = {"dx": torch.einsum("rc,r->rc", dx, rstd).reshape(s["x"].shape), "dweight": torch.einsum("rc,rc->c", dy, xh)}
    if s["bias"] is not None:
        out["dbias"] = torch.einsum("rc->c", dy)
    return out


def _exact_embed(case, seed):
    s = _embed_inputs(case, seed)
    rows = case["table_rows"]
    if not case["backward"]:
        with_zero = torch.cat([s["table"].double(), s["table"].new_zeros(1, case["channels"], dtype=torch.float64)])
        y = s["scale"] * torch.nn.functional.embedding(s["ids"].long() % (rows + 1), with_zero)
        return {"y": y if s["x"] is None else y + s["x"].double()}
    # running sums over the tokens in the order of their ids, and their differences at each row's ends; in parts of
    # the channels
    order = torch.sort(s["ids"].long(), stable=True)
    ends = torch.searchsorted(order.values, torch.arange(-1, rows, device=order.values.device), right=True)
    out = torch.empty(rows, case["channels"], dtype=torch.float64, device=ends.device)
    for c in range(0, case["channels"], 64):
        dy = s["dy"][:, c:c + 64].double()[order.indices]
        sums = torch.cat([dy.new_zeros(1, dy.shape[1]), dy.cumsum(0)])
        out[:, c:c + 64] = (sums[ends[1:]] - sums[ends[:-1]]) * s["scale"]
    return {"dtable": out}


def _exact_distill(case, seed):
    s = _distill_inputs(case, seed)
    temperature, rows = case["temperature"], case["rows"]
    step = max(1, 30_000_000 // case["classes"])
    parts = []
    for i in range(0, rows, step):
        cut = slice(i, i + step)
        z, ids, t = s["logits"][cut].double(), s["ids"][cut].long(), s["top_logits"][cut].double() / temperature
        t = torch.where(ids >= 0, t, float("-inf"))
        some = (ids >= 0).any(1)
        t[~some] = 0.0
        lse = torch.logsumexp(t, 1) if s["whole"] is None else s["whole"][cut].double()
        log_p = t - lse[:, None]
        log_q = torch.log_softmax(z / temperature, 1)
        if case["backward"]:
            p = torch.exp(log_p)
            q = torch.exp(z / temperature - s["stats"][cut, :1].double() / temperature) / s["stats"][cut, 1:].double()
            dense = torch.zeros_like(z).scatter_add_(1, ids.clamp(min=0), p)
            dz = temperature * s["dloss"][cut, None].double() * (q * p.sum(1, keepdim=True) - dense)
            parts.append({"dlogits": torch.where(some[:, None], dz, 0.0)})
            continue
        term = torch.exp(log_p) * (log_p - log_q.gather(1, ids.clamp(min=0)))
        loss = temperature ** 2 * torch.where(ids >= 0, term, 0.0).sum(1)
        m = z.amax(1)
        total = torch.exp(torch.logsumexp(z / temperature, 1) - m / temperature)
        parts.append({"loss": loss, "stats": torch.where(some[:, None], torch.stack([m, total], 1), 0.0)})
    return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}


_EXACT = {"norm": _exact_norm, "embed": _exact_embed, "distill": _exact_distill}


def exact(case, seed):
    return _EXACT[case["op"]](case, seed)
