"""The 8-bit operators of gazenerf_amd, as cases that can be timed and compared.

Three operators around the network's feature maps [B, C, P] (P pixels, channels first) and the 1x1 convolutions on them
(a 1x1 convolution is a linear layer whose rows are the pixels):

  cache    write_featmaps + read_featmaps: maps go into the slots of a cache as 8-bit rows (one row a pixel, one scale a
           row) and are read back as values
  linear   int8_linear on floating rows or maps: quantise each row, multiply with 8-bit weights (one scale a channel)
  mapped   int8_linear on the rows of a cache, named by their slots

    row:      a = max(max_k |x_k|, 2^-100),  scale = a / 127,  q_k = round_half_even(f(x_k * f(127 / a)))
              f: rounding to 32 bits.  It belongs to the definition, so that a value on the border between two steps has ONE
              answer (a step is 1/127 of the row's largest value)
    product:  y_no = act((sum_k q_nk w_ok) * scale_n * wscale_o + bias_o),  act = identity or LeakyReLU(0.2)

Rows of 8-bit values stand on a pitch of a multiple of 16 bytes.  With ``own`` false the operators are computed in their
plain form.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}


def listed():
    return [
        # one 64 x 64 feature map of the default network is kept and shown again: the smallest step of an interactive viewer
        {"name": "cache one map", "op": "cache", "batch": 1, "reads": 2, "slots": 16, "channels": 258, "pixels": 4096, "type": "float32"},
        # a sweep of 32 views is kept at once, 64 views are read back for the merge / the upsampler
        {"name": "cache sweep", "op": "cache", "batch": 32, "reads": 64, "slots": 96, "channels": 258, "pixels": 4096, "type": "float32"},
        # a ragged map: half the channels, a 37 x 37 crop, narrow type
        {"name": "cache crop", "op": "cache", "batch": 5, "reads": 9, "slots": 12, "channels": 129, "pixels": 1369, "type": "bfloat16"},
        # the widest maps the upsampler takes (1024 channels)
        {"name": "cache wide", "op": "cache", "batch": 8, "reads": 16, "slots": 24, "channels": 1024, "pixels": 4096, "type": "float16"},
        # block 0, layer_1 of the default upsampler on one map: 258 -> 516 over 64 x 64 pixels
        {"name": "linear block 0", "op": "linear", "rows": 4096, "k": 258, "o": 516, "leaky": True, "bias": True, "maps": False, "type": "float32"},
        # block 0, layer_2 on the seven stacked maps of a two-image step: 516 -> 1032
        {"name": "linear block 0 stacked", "op": "linear", "rows": 28672, "k": 516, "o": 1032, "leaky": True, "bias": True, "maps": False, "type": "bfloat16"},
        # the last feat layer on one 512 x 512 image, channels first: 64 -> 32, all of it memory traffic
        {"name": "linear last map", "op": "linear", "rows": 262144, "k": 64, "o": 32, "leaky": True, "bias": True, "maps": True, "type": "float32"},
        # layer_2 of the widest block on four 64 x 64 maps: all of it arithmetic
        {"name": "linear wide", "op": "linear", "rows": 16384, "k": 2048, "o": 4096, "leaky": False, "bias": True, "maps": False, "type": "bfloat16"},
        # a single row through the widest layer: the time to read the weights
        {"name": "linear one row", "op": "linear", "rows": 1, "k": 2048, "o": 4096, "leaky": False, "bias": True, "maps": False, "type": "bfloat16"},
        # a handful of rows, every size odd
        {"name": "linear few rows", "op": "linear", "rows": 7, "k": 517, "o": 259, "leaky": True, "bias": False, "maps": False, "type": "float16"},
        # four cached views into the first layer of the upsampler, channels first
        {"name": "mapped four views", "op": "mapped", "reads": 4, "slots": 64, "channels": 258, "pixels": 4096, "o": 516, "leaky": True, "bias": True, "maps": True, "type": "float32"},
        # three cached crops, rows as the next quantiser reads them
        {"name": "mapped crops", "op": "mapped", "reads": 3, "slots": 12, "channels": 129, "pixels": 1369, "o": 387, "leaky": False, "bias": False, "maps": False, "type": "bfloat16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["cache", "linear", "linear", "mapped"])
    typ = rng.choice(list(TYPES))
    if op == "linear":
        case = {"op": op, "rows": _log(rng, 1, 262144), "k": _log(rng, 16, 2048), "o": _log(rng, 16, 4096), "leaky": rng.random() < 0.5,
                "bias": rng.random() < 0.7, "maps": rng.random() < 0.4, "type": typ}
        shrink = "rows"
    else:
        reads = _log(rng, 1, 64)
        case = {"op": op, "reads": reads, "slots": reads + _log(rng, 1, 64), "channels": _log(rng, 16, 1024), "pixels": _log(rng, 1, 16384), "type": typ}
        shrink = "pixels"
        if op == "cache":
            case["batch"] = rng.randint(1, reads)
        else:
            case.update(o=_log(rng, 16, 2048), leaky=rng.random() < 0.5, bias=rng.random() < 0.7, maps=rng.random() < 0.5)
    top = [work(c) for c in listed()]
    most = {k: max(w[k] for w in top) for k in ("bytes", "flops")}
    while any(work(case)[k] > most[k] for k in most) or case.get("slots", 0) * case.get("pixels", 0) * case.get("channels", 0) > 96 * 4096 * 1024:
        case[shrink] = max(1, case[shrink] * 2 // 3)
    return case


def _pitch(k):
    return -(-k // 16) * 16


def _features(gen, shape, axis):
    """Values as the network's maps hold them: channels of different size, some of them mostly positive, and pixels outside the head that are all zero."""
    x = torch.randn(shape, generator=gen, device=DEV)
    view = [1] * len(shape)
    view[axis] = shape[axis]
    size = torch.exp(torch.randn(shape[axis], generator=gen, device=DEV) * 0.7).view(view)
    x = torch.where(torch.rand(shape[axis], generator=gen, device=DEV).view(view) < 0.4, x.abs(), x) * size
    view = list(shape)
    view[axis] = 1
    return x * (torch.rand(view, generator=gen, device=DEV) > 0.02)


def _rows_of(values):
    """8-bit rows on the pitch and their scales, of the last axis."""
    q, s = _quantise(values)
    store = torch.zeros(*values.shape[:-1], _pitch(values.shape[-1]), dtype=torch.int8, device=DEV)
    rows = store[..., :values.shape[-1]]
    rows.copy_(q)
    return rows, s


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    t = TYPES[case["type"]]
    state = {"op": case["op"], "type": t}
    if case["op"] != "linear":
        n, c, p, r = case["slots"], case["channels"], case["pixels"], case["reads"]
        store = torch.zeros(n, p, _pitch(c), dtype=torch.int8, device=DEV)
        state["q"], state["scale"] = store[..., :c], torch.empty(n, p, device=DEV)
        state["q"].copy_(torch.randint(-127, 128, (n, p, c), generator=gen, device=DEV, dtype=torch.int8))
        state["scale"].copy_(torch.rand(n, p, generator=gen, device=DEV) * 0.05 + 0.005)
        order = torch.randperm(n, generator=gen, device=DEV)
        state["read"] = order[torch.randperm(r, generator=gen, device=DEV)]
        if case["op"] == "cache":
            state["write"] = order[:case["batch"]]
            state["maps"] = _features(gen, (case["batch"], c, p), 1).to(t)
            return state
        k = c
    else:
        k = case["k"]
        shape = (1, k, case["rows"]) if case["maps"] else (case["rows"], k)
        state["x"] = _features(gen, shape, 1).to(t)
    o = case["o"]
    w = torch.randn(o, k, generator=gen, device=DEV) * math.sqrt(2.0 / (k + o))
    state["wq"], state["wscale"] = _rows_of(w)
    state["bias"] = torch.randn(o, generator=gen, device=DEV) * 0.1 if case["bias"] else None
    state["leaky"], state["maps_out"] = case["leaky"], case["maps"]
    return state


def _quantise(x, axis=-1):
    x = x.float()
    a = x.abs().amax(dim=axis, keepdim=True).clamp_min(2.0 ** -100)
    most = torch.full_like(a, 127.0)          # a number in its place makes torch multiply with a rounded reciprocal
    return torch.round(x * (most / a)), (a / most).squeeze(axis)


def _product(q, scale, s, channels_first):
    """q [..., rows, k] of whole numbers in 32 bits, scale [..., rows]."""
    y = torch.matmul(q, s["wq"].float().t()) * scale.unsqueeze(-1) * s["wscale"]
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["leaky"]:
        y = torch.where(y > 0, y, y * 0.2)
    if channels_first:
        y = y.transpose(-1, -2).contiguous()
    return y.to(s["type"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    import gazenerf_amd as G
    if s["op"] == "cache":
        G.write_featmaps(s["q"], s["scale"], s["write"], s["maps"])
        return {"maps": G.read_featmaps(s["q"], s["scale"], s["read"], s["type"]), "scale": s["scale"]}
    if s["op"] == "mapped":
        return G.int8_linear(s["q"], s["wq"], s["wscale"], s["bias"], x_scale=s["scale"], slots=s["read"], leaky=s["leaky"],
                             channels_first=s["maps_out"], out_dtype=s["type"])
    return G.int8_linear(s["x"], s["wq"], s["wscale"], s["bias"], leaky=s["leaky"], channels_first=s["maps_out"], out_dtype=s["type"])


def _run_plain(s):
    if s["op"] == "cache":
        q, scale = _quantise(s["maps"], 1)
        s["q"][s["write"]] = q.transpose(1, 2).to(torch.int8)
        s["scale"][s["write"]] = scale
        back = s["q"][s["read"]].float() * s["scale"][s["read"]].unsqueeze(-1)
        return {"maps": back.transpose(1, 2).contiguous().to(s["type"]), "scale": s["scale"]}
    if s["op"] == "mapped":
        return _product(s["q"][s["read"]].float(), s["scale"][s["read"]], s, s["maps_out"])
    q, scale = _quantise(s["x"], 1)
    return _product(q.transpose(1, 2) if s["maps_out"] else q, scale, s, s["maps_out"])


def _steps(x, axis):
    """(whole steps, size of a step) along `axis` in 64 bits.  A quotient or product of two 32-bit numbers that is formed in 64 bits and then
    rounded to 32 is the rounded exact one (53 >= 2 * 24 + 2)."""
    a = torch.maximum(x.abs().amax(axis, keepdim=True), torch.full((), 2.0 ** -100, dtype=torch.float64, device=DEV))
    per = (127 / a).float().double()
    return torch.round((x * per).float().double()), a / 127


def exact(case, seed):
    """From the definition, in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "cache":
        values = s["q"].double() * s["scale"].double()[:, :, None]
        scales = s["scale"].double()
        whole, step = _steps(s["maps"].double(), 1)
        values.index_copy_(0, s["write"], (whole * step).permute(0, 2, 1))
        scales.index_copy_(0, s["write"], step[:, 0])
        return {"maps": values.index_select(0, s["read"]).permute(0, 2, 1).contiguous(), "scale": scales}
    w = s["wq"].double() * s["wscale"].double()[:, None]
    if case["op"] == "mapped":
        rows = s["q"].index_select(0, s["read"]).double() * s["scale"].index_select(0, s["read"]).double()[:, :, None]
        rows = rows.reshape(-1, rows.shape[-1])
    else:
        x = s["x"].double()
        whole, step = _steps(x[0].t() if case["maps"] else x, 1)
        rows = whole * step
    y = rows.mm(w.t())
    if s["bias"] is not None:
        y += s["bias"].double()
    if case["leaky"]:
        y = torch.maximum(y, y / 5)
    if case["op"] == "mapped":
        y = y.view(case["reads"], case["pixels"], -1)
    elif case["maps"]:
        y = y[None]
    return y.transpose(1, 2).contiguous() if case["maps"] else y


def work(case):
    e = SIZE[case["type"]]
    if case["op"] == "cache":
        c, p, b, r = case["channels"], case["pixels"], case["batch"], case["reads"]
        return {"bytes": b * p * (c * e + c + 4) + r * p * (c + 4 + c * e) + 8 * (b + r), "flops": 4 * b * p * c + r * p * c}
    o = case["o"]
    if case["op"] == "mapped":
        n, k, x = case["reads"] * case["pixels"], case["channels"], 1
    else:
        n, k, x = case["rows"], case["k"], e
    return {"bytes": n * k * x + (4 * n if x == 1 else 0) + o * k + 4 * o * (2 if case["bias"] else 1) + n * o * e, "flops": 2 * n * k * o}
