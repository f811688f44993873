"""Attention over sequences of Gaussians (`htgs_b200.sequence`) as measurable cases: rotary positions with several axes, attention over
packed sequences with grouped heads, and one more row of it over a cache.

Rows are Gaussians in the order of a space-filling curve.  Whole scenes (10^5 to 10^6 rows) attend within a window along the curve, single
objects (10^2 to 10^4 rows) to all of their rows, and a model that extends a scene Gaussian by Gaussian to the rows before.
"""
import math

import torch

own = False

DEVICE = "cuda"
BASE = 10000.0         # of the rotary frequencies
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _rotary(kind, rows, heads, key_heads, dim, axes=3, type="bf16", interleaved=False):
    return {"kind": kind, "rows": rows, "heads": heads, "key_heads": key_heads, "dim": dim, "axes": axes, "type": type, "interleaved": interleaved}


def _attention(kind, rows, heads, key_heads, dim, type="bf16", sequences=1, causal=False, window=-1):
    return {"kind": kind, "rows": rows, "heads": heads, "key_heads": key_heads, "dim": dim, "type": type, "sequences": sequences, "causal": causal, "window": window}


def _step(batch, capacity, heads, key_heads, dim, type="bf16", window=-1):
    return {"kind": "step", "batch": batch, "capacity": capacity, "heads": heads, "key_heads": key_heads, "dim": dim, "type": type, "window": window}


def listed():
    return [
        # One Gaussian is appended to a scene: its queries and keys are turned, latency is all there is.
        dict(_rotary("rotary", 1, 8, 2, 64, axes=1), name="rotary_token"),
        # Inference over a scene of 100 k Gaussians, turned by their places in space.
        dict(_rotary("rotary", 100_000, 8, 2, 64), name="rotary_scene"),
        # A training step in 32 bits, forward and backward, an odd number of rows and heads and sections that differ.
        dict(_rotary("rotary_train", 65_537, 3, 3, 40, type="fp32", interleaved=True), name="rotary_train"),
        # A small object on its own: latency counts.
        dict(_attention("attention", 200, 4, 4, 64), name="attention_object"),
        # Packed objects of very different sizes, empty ones among them, all rows of an object to all of its rows.
        dict(_attention("attention", 20_011, 8, 2, 64, type="fp16", sequences=33), name="attention_packed"),
        # A scene of a quarter of a million Gaussians: each attends to 512 neighbours on either side along the curve.
        dict(_attention("attention", 262_144, 4, 4, 64, window=512), name="attention_scene"),
        # A model that writes a scene Gaussian by Gaussian reads a long beginning.
        dict(_attention("attention", 32_768, 8, 2, 128, causal=True), name="attention_causal"),
        # A training step over packed scenes within windows, narrow heads: forward and backward.
        dict(_attention("attention_train", 100_003, 8, 8, 32, sequences=7, window=256), name="attention_train_scenes"),
        # A training step of the model that writes scenes.
        dict(_attention("attention_train", 16_384, 8, 4, 128, causal=True), name="attention_train_causal"),
        # One more Gaussian for one short scene: latency.
        dict(_step(1, 4096, 8, 2, 64), name="step_token"),
        # One more Gaussian for each of 32 scenes of different sizes.
        dict(_step(32, 8192, 8, 2, 128), name="step_scenes"),
        # One more Gaussian for one scene of about a million.
        dict(_step(1, 1_048_576, 8, 2, 64, type="fp16"), name="step_long"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "rotary_train", "attention", "attention", "attention_train", "attention_train", "step", "step"])
    key_heads, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 4, 8])
    heads = key_heads * group
    if kind.startswith("rotary"):
        dim, type = 2 * _log_uniform(rng, 8, 64), rng.choice(list(TYPES))
        rows = _log_uniform(rng, 1, min(200_000, 120_000_000 // (BYTES[type] * (heads + key_heads) * dim)))
        return _rotary(kind, rows, heads, key_heads, dim, rng.choice([1, 2, 3, 4]), type, rng.choice([False, True]))
    dim, type = 8 * _log_uniform(rng, 2, 16), rng.choice(["bf16", "fp16"])
    window = rng.choice([-1, _log_uniform(rng, 16, 1024)])
    if kind == "step":
        batch = _log_uniform(rng, 1, 256)
        return _step(batch, _log_uniform(rng, 64, min(1_048_576, 260_000_000 // (4 * batch * key_heads * dim))), heads, key_heads, dim, type, window)
    sequences, causal = rng.choice([1, 1, 2, 7, 33]), rng.choice([False, True])
    flops = 250_000_000_000 if kind == "attention" else 120_000_000_000       # of a forward pass: at most those of the largest listed
    most = math.isqrt(flops // (4 * heads * dim)) if window < 0 else flops // (4 * heads * dim * (2 * window + 1))
    return _attention(kind, _log_uniform(rng, 16, min(most, 262_144, 130_000_000 // (2 * heads * dim))), heads, key_heads, dim, type, sequences, causal, window)


# ---- inputs -----------------------------------------------------------------------------------------------------------------


def _sections(case):
    """Pairs turned by each axis: evenly, and one more for the first ones where they do not come out even."""
    pairs, axes = case["dim"] // 2, case["axes"]
    return [pairs // axes + (a < pairs % axes) for a in range(axes)]


def _ends(case):
    """Rows at which the packed sequences begin, and the last one's end: cuts that go by the case alone, so lengths differ widely; the
    second cut falls on the first, so that one of three or more sequences is empty."""
    g = torch.Generator().manual_seed(case["rows"] * 64 + case["sequences"])
    cuts = torch.sort((torch.rand(case["sequences"] - 1, generator=g, dtype=torch.float64) ** 2 * case["rows"]).long()).values
    if cuts.numel() > 1:
        cuts[1] = cuts[0]
    return [0, *cuts.tolist(), case["rows"]]


def _lengths(case):
    """Rows in each cache before the step, by the case alone: from a quarter of the capacity to all but the one row that the step fills."""
    g = torch.Generator().manual_seed(case["capacity"] * 64 + case["batch"])
    low = case["capacity"] // 4
    return (low + (torch.rand(case["batch"], generator=g, dtype=torch.float64) * (case["capacity"] - low)).long()).tolist()


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    type, kind = TYPES[case["type"]], case["kind"]
    heads, key_heads, dim = case["heads"], case["key_heads"], case["dim"]

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device=DEVICE) * scale).to(type)

    if kind == "step":
        batch, capacity = case["batch"], case["capacity"]
        s = {"case": case, "q": normal(batch, heads, dim, scale=2.0), "k": normal(batch, key_heads, dim), "v": normal(batch, key_heads, dim)}
        for name in ("keys", "values"):
            s[name] = torch.empty((batch, capacity, key_heads, dim), dtype=type, device=DEVICE).normal_(generator=g)
        s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=DEVICE)
        return s
    # queries, keys and values lie side by side, as one projection writes them
    rows = case["rows"]
    both = normal(rows, (heads + 2 * key_heads) * dim, scale=1.5)
    q, k, v = (part.unflatten(1, (-1, dim)) for part in both.split([heads * dim, key_heads * dim, key_heads * dim], dim=1))
    s = {"case": case, "q": q, "k": k}
    if kind.startswith("rotary"):
        if case["axes"] == 1:      # the row's number in a long sequence
            s["positions"] = torch.randint(0, 1_000_000, (rows, 1), generator=g, device=DEVICE, dtype=torch.int32)
        else:                      # places in a box 1024 cells wide
            s["positions"] = torch.rand((rows, case["axes"]), generator=g, device=DEVICE) * 1024.0
        grads = ("q", "k")
    else:
        s["v"] = v
        ends = _ends(case)
        s["offsets"] = torch.tensor(ends, dtype=torch.int32, device=DEVICE) if case["sequences"] > 1 else None
        s["ends"] = ends           # what the program that packed the sequences knows of them
        grads = ("q", "k", "v")
    if kind.endswith("_train"):
        s["grad_q" if kind == "rotary_train" else "grad"] = normal(rows, heads, dim)
        if kind == "rotary_train":
            s["grad_k"] = normal(rows, key_heads, dim)
        for name in grads:
            s[name] = s[name].detach().requires_grad_(True)
    return s


# ---- the framework's operators ------------------------------------------------------------------------------------------------


def _run_own(s):
    from htgs_b200 import sequence as seq
    case = s["case"]
    kind = case["kind"]
    if kind.startswith("rotary"):
        q, k = seq.rotary(s["q"], s["k"], s["positions"], base=BASE, interleaved=case["interleaved"])
        if kind == "rotary":
            return {"q": q, "k": k}
        gq, gk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["grad_q"], s["grad_k"]))
        return {"q": q, "k": k, "gq": gq, "gk": gk}
    window = case["window"] if case["window"] >= 0 else None
    if kind == "step":
        out = seq.attention_step(s["q"], s["k"], s["v"], s["keys"], s["values"], s["lengths"], window=window)
        return {"out": out, "keys": s["keys"], "values": s["values"]}
    out = seq.attention(s["q"], s["k"], s["v"], offsets=s["offsets"], causal=case["causal"], window=window)
    if kind == "attention":
        return out
    gq, gk, gv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["grad"])
    return {"out": out, "gq": gq, "gk": gk, "gv": gv}


# ---- the plain forms ------------------------------------------------------------------------------------------------------------


def _turned(x, cos, sin, interleaved):
    """Each pair of x turned by its angle; a pair is two neighbours, or a value of the first half and the one at its place in the second."""
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2)
    a, b = x.chunk(2, dim=-1)
    return torch.cat((a * cos - b * sin, a * sin + b * cos), dim=-1)


def _plain_rotary(s):
    case = s["case"]
    type = TYPES[case["type"]]
    angles = []
    for axis, pairs in enumerate(_sections(case)):
        frequencies = BASE ** (-torch.arange(pairs, dtype=torch.float64, device=DEVICE) / max(pairs, 1))
        angles.append(s["positions"][:, axis, None].double() * frequencies)       # far positions lose their angle in 32 bits
    angle = torch.cat(angles, dim=1)
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    out = {name: _turned(s[name].float(), cos, sin, case["interleaved"]).to(type) for name in ("q", "k")}
    if case["kind"] == "rotary_train":
        out.update({"g" + name: _turned(s["grad_" + name].float(), cos, -sin, case["interleaved"]).to(type) for name in ("q", "k")})
    return out


def _pieces(case, ends):
    """(first row, last row + 1, first key, last key + 1) of pieces of the sequences whose scores take about a gigabyte at most."""
    window = case["window"]
    for begin, end in zip(ends, ends[1:]):
        at = begin
        while at < end:
            span = end - begin if window < 0 else min(end - begin, 4 * window + 512)
            to = min(end, at + max(16, min(4 * window + 512 if window >= 0 else 4096, 250_000_000 // (span * case["heads"]))))
            low = begin if window < 0 else max(begin, at - window)
            high = min(end, to if case["causal"] else end if window < 0 else to + window)
            yield at, to, low, high
            at = to


def _visible(case, at, to, low, high):
    i, j = torch.arange(at, to, device=DEVICE)[:, None], torch.arange(low, high, device=DEVICE)[None]
    seen = torch.ones((to - at, high - low), dtype=torch.bool, device=DEVICE)
    if case["causal"]:
        seen &= j <= i
    if case["window"] >= 0:
        seen &= (i - j).abs() <= case["window"]
    return seen


def _plain_attention(s):
    case = s["case"]
    type, group, scale = TYPES[case["type"]], case["heads"] // case["key_heads"], case["dim"] ** -0.5
    train = case["kind"] == "attention_train"
    # heads first; a key head serves a group of query heads
    q = s["q"].float().transpose(0, 1).unflatten(0, (case["key_heads"], group))
    k, v = s["k"].float().transpose(0, 1)[:, None], s["v"].float().transpose(0, 1)[:, None]
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if train:
        grad = s["grad"].float().transpose(0, 1).unflatten(0, (case["key_heads"], group))
        gq, gk, gv = torch.empty_like(out), torch.zeros_like(k), torch.zeros_like(v)
    for at, to, low, high in _pieces(case, s["ends"]):
        qp, kp, vp = q[:, :, at:to], k[:, :, low:high], v[:, :, low:high]
        scores = (qp @ kp.transpose(-1, -2)).mul_(scale).masked_fill_(~_visible(case, at, to, low, high), float("-inf"))
        weights = scores.sub_(scores.amax(dim=-1, keepdim=True)).exp_()
        weights /= weights.sum(dim=-1, keepdim=True)
        out[:, :, at:to] = weights @ vp
        if train:
            gp = grad[:, :, at:to]
            change = gp @ vp.transpose(-1, -2)
            change = change.sub_((gp * out[:, :, at:to]).sum(dim=-1, keepdim=True)).mul_(weights).mul_(scale)
            gq[:, :, at:to] = change @ kp
            gk[:, 0, low:high] += (change.transpose(-1, -2) @ qp).sum(dim=1)
            gv[:, 0, low:high] += (weights.transpose(-1, -2) @ gp).sum(dim=1)
    rows_first = lambda t: t.flatten(0, 1).transpose(0, 1).to(type)  # noqa: E731
    if not train:
        return rows_first(out)
    return {"out": rows_first(out), "gq": rows_first(gq), "gk": rows_first(gk), "gv": rows_first(gv)}


def _plain_step(s):
    case = s["case"]
    group, scale = case["heads"] // case["key_heads"], case["dim"] ** -0.5
    each, lengths = torch.arange(case["batch"], device=DEVICE), s["lengths"].long()
    s["keys"][each, lengths] = s["k"]
    s["values"][each, lengths] = s["v"]
    row = torch.arange(case["capacity"], device=DEVICE)
    seen = row <= lengths[:, None]
    if case["window"] >= 0:
        seen &= row >= lengths[:, None] - case["window"]
    q = s["q"].float().unflatten(1, (case["key_heads"], group))
    scores = q @ s["keys"].float().permute(0, 2, 3, 1) * scale
    scores = scores.masked_fill(~seen[:, None, None], float("-inf"))
    weights = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
    weights = weights / weights.sum(dim=-1, keepdim=True)
    out = (weights @ s["values"].float().transpose(1, 2)).flatten(1, 2).to(TYPES[case["type"]])
    return {"out": out, "keys": s["keys"], "values": s["values"]}


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        kind = state["case"]["kind"]
        return _plain_step(state) if kind == "step" else _plain_rotary(state) if kind.startswith("rotary") else _plain_attention(state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------------


def _pairs(case):
    """Pairs of a row and a row that it attends to."""
    total = 0
    for begin, end in zip(ends := _ends(case), ends[1:]):
        n = end - begin
        w = n if case["window"] < 0 else min(case["window"], max(n - 1, 0))
        before = n * (n - 1) // 2 if w >= n else w * (w + 1) // 2 + (n - 1 - w) * w       # rows before a row, summed
        total += n + before * (1 if case["causal"] else 2)
    return total


def work(case):
    kind, heads, key_heads, dim, b = case["kind"], case["heads"], case["key_heads"], case["dim"], BYTES[case["type"]]
    if kind == "step":            # reads the rows that count of both caches, and the new row; writes it and the output
        rows = sum(min(n, case["window"]) if case["window"] >= 0 else n for n in _lengths(case))
        one = case["batch"] * dim * b
        return {"bytes": 2 * rows * key_heads * dim * b + one * (2 * heads + 4 * key_heads), "flops": 4 * rows * heads * dim}
    row = case["rows"] * dim * b
    if kind.startswith("rotary"):  # reads and writes q and k (and their gradients); reads the positions
        passes = 2 if kind == "rotary_train" else 1
        return {"bytes": passes * 2 * row * (heads + key_heads) + case["rows"] * case["axes"] * 4, "flops": passes * 3 * case["rows"] * (heads + key_heads) * dim}
    flops = 4 * _pairs(case) * heads * dim
    if kind == "attention":       # two products
        return {"bytes": row * (2 * heads + 2 * key_heads), "flops": flops}
    return {"bytes": row * (4 * heads + 4 * key_heads), "flops": flops * 7 // 2}       # and five for the gradients


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------------


def _exact_turn(x, angle, interleaved):
    """As a product of complex numbers."""
    z = torch.view_as_complex(x.unflatten(-1, (-1, 2)).contiguous() if interleaved else torch.stack(x.chunk(2, dim=-1), dim=-1).contiguous())
    z = torch.view_as_real(z * torch.polar(torch.ones_like(angle), angle)[:, None])
    return z.flatten(-2) if interleaved else torch.cat((z[..., 0], z[..., 1]), dim=-1)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind.startswith("rotary"):
        speed = [(axis, BASE ** (-j / pairs)) for axis, pairs in enumerate(_sections(case)) for j in range(pairs)]
        angle = torch.stack([s["positions"][:, axis].double() * f for axis, f in speed], dim=1)
        out = {name: _exact_turn(s[name].detach().double(), angle, case["interleaved"]) for name in ("q", "k")}
        if kind == "rotary_train":
            out.update({"g" + name: _exact_turn(s["grad_" + name].double(), -angle, case["interleaved"]) for name in ("q", "k")})
        return out
    group, scale, window = case["heads"] // case["key_heads"], case["dim"] ** -0.5, case["window"]
    if kind == "step":
        out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
        for b, n in enumerate(_lengths(case)):
            s["keys"][b, n], s["values"][b, n] = s["k"][b], s["v"][b]
            first = max(0, n - window) if window >= 0 else 0
            k, v = s["keys"][b, first:n + 1].double(), s["values"][b, first:n + 1].double()
            scores = torch.einsum("hgd,nhd->hgn", s["q"][b].double().view(case["key_heads"], group, -1), k) * scale
            out[b] = torch.einsum("hgn,nhd->hgd", torch.softmax(scores, dim=-1), v).reshape(case["heads"], -1)
        return {"out": out, "keys": s["keys"], "values": s["values"]}        # the caches hold copies: nothing is rounded
    train = kind == "attention_train"
    names = ("q", "k", "v", "grad") if train else ("q", "k", "v")
    t = {name: s[name].detach().double() for name in names}
    out = torch.zeros_like(t["q"])
    gq, gk, gv = torch.zeros_like(t["q"]), torch.zeros_like(t["k"]), torch.zeros_like(t["v"])
    ends = _ends(case)
    for begin, end in zip(ends, ends[1:]):
        for at in range(begin, end, 1024):
            to = min(end, at + 1024)
            low = begin if window < 0 else max(begin, at - window)
            high = to if case["causal"] else end if window < 0 else min(end, to + window)
            away = torch.arange(low, high, device=DEVICE)[None] - torch.arange(at, to, device=DEVICE)[:, None]
            hidden = torch.zeros_like(away, dtype=torch.bool)
            if case["causal"]:
                hidden |= away > 0
            if window >= 0:
                hidden |= (away > window) | (away < -window)
            for h in range(case["heads"]):
                q, k, v = t["q"][at:to, h], t["k"][low:high, h // group], t["v"][low:high, h // group]
                p = torch.softmax(torch.where(hidden, -math.inf, q @ k.t() * scale), dim=1)
                out[at:to, h] = p @ v
                if train:
                    g = t["grad"][at:to, h]
                    gp = g @ v.t()
                    gs = p * (gp - (p * gp).sum(dim=1, keepdim=True)) * scale
                    gq[at:to, h] = gs @ k
                    gk[low:high, h // group] += gs.t() @ q
                    gv[low:high, h // group] += p.t() @ g
    return {"out": out, "gq": gq, "gk": gk, "gv": gv} if train else out
