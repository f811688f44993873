"""The sequence operators (`htgs_b200.sequence`) as measurable cases: root-mean-square norm with the residual's addition, matrix
product in 8-bit floating point with a scale for each block of 128, and the gated linear recurrence.

Rows are Gaussians in the order of a space-filling curve (10^5 to 10^6 in a scene, one when a scene is extended token by token),
columns are the channels of a network that reads or refines them.
"""
import math

import torch

own = False

DEVICE = "cuda"
EPS = 1e-6
BLOCK = 128            # columns that share a scale
LARGEST = 448.0        # largest finite value of the 8-bit type (e4m3)
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _norm(kind, rows, width, type="bf16"):
    return {"kind": kind, "rows": rows, "width": width, "type": type}


def _product(kind, rows, width, out, type="bf16"):
    return {"kind": kind, "rows": rows, "width": width, "out": out, "type": type}


def _scan(kind, rows, width, type="bf16", sequences=1, reverse=False):
    return {"kind": kind, "rows": rows, "width": width, "type": type, "sequences": sequences, "reverse": reverse}


def listed():
    return [
        # One Gaussian is appended to a scene: the norm of one row, latency is all there is.
        dict(_norm("norm_8bit", 1, 1024), name="norm_token"),
        # Inference over a scene of 100 k Gaussians, the input of an 8-bit product.
        dict(_norm("norm_8bit", 100_000, 512), name="norm_scene"),
        # A training step's norm, forward and backward, wide rows in an odd number.
        dict(_norm("norm_train", 65_537, 1024), name="norm_train"),
        # The same in 32 bits over raw parameters and features joined to an odd width.
        dict(_norm("norm_train", 100_003, 333, "fp32"), name="norm_train_odd"),
        # One token through a projection: the weights are read once, latency counts.
        dict(_product("product", 1, 1024, 2048), name="product_token"),
        # A ragged handful of Gaussians, no size a multiple of the block.
        dict(_product("product", 4099, 1080, 1001, "fp16"), name="product_ragged"),
        # Projection of a whole scene at inference: value and gate side by side.
        dict(_product("product", 100_000, 1024, 2048), name="product_scene"),
        # A projection in a training step: the product and both of its gradients.
        dict(_product("product_train", 32_768, 512, 1024), name="product_train"),
        # One more token for each of 64 scenes kept open: the recurrence's step.
        dict(_scan("scan_step", 64, 1024, sequences=64), name="scan_step"),
        # Inference over one scene of a million Gaussians.
        dict(_scan("scan", 1_000_000, 128), name="scan_long"),
        # A training step's recurrence over a quarter of a million Gaussians, forward and backward.
        dict(_scan("scan_train", 262_144, 512), name="scan_train"),
        # Packed scenes of very different sizes, empty ones among them, read from the end, in 32 bits.
        dict(_scan("scan_train", 100_003, 97, "fp32", sequences=33, reverse=True), name="scan_packed"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm_8bit", "norm_train", "product", "product_train", "scan", "scan_train", "scan_step"])
    if kind.startswith("norm"):
        width, type = _log_uniform(rng, 33, 2048), rng.choice(list(TYPES))
        return _norm(kind, _log_uniform(rng, 1, min(200_000, 120_000_000 // BYTES[type] // width)), width, type)
    if kind.startswith("product"):
        width, out = _log_uniform(rng, 64, 2048), _log_uniform(rng, 64, 2048)
        most = (200_000_000_000 if kind == "product" else 17_000_000_000) // (width * out)
        return _product(kind, _log_uniform(rng, 1, max(1, min(100_000, most))), width, out, rng.choice(["bf16", "fp16"]))
    type = rng.choice(list(TYPES))
    width = _log_uniform(rng, 1, 1024)
    if kind == "scan_step":
        rows = _log_uniform(rng, 1, 4096)
        return _scan(kind, rows, width, type, sequences=rows)
    rows = _log_uniform(rng, 1, min(1_000_000, 260_000_000 // BYTES[type] // width))
    return _scan(kind, rows, width, type, sequences=rng.choice([1, 1, 2, 7, 64]), reverse=rng.choice([False, True]))


# ---- inputs -----------------------------------------------------------------------------------------------------------------


def _offsets(case, seed):
    """[sequences + 1] rows at which the packed sequences begin: random cuts, so lengths differ widely; the second cut falls on the
    first, so that one of three or more sequences is empty."""
    g = torch.Generator().manual_seed(seed)
    cuts = torch.sort((torch.rand(case["sequences"] - 1, generator=g, dtype=torch.float64) ** 2 * case["rows"]).long()).values
    if cuts.numel() > 1:
        cuts[1] = cuts[0]
    return torch.cat((torch.zeros(1, dtype=torch.long), cuts, torch.tensor([case["rows"]]))).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    type = TYPES[case["type"]]
    rows, width, kind = case["rows"], case["width"], case["kind"]

    def normal(*shape, scale=1.0, shift=0.0, as_type=type):
        return (torch.randn(shape, generator=g, device=DEVICE) * scale + shift).to(as_type)

    if kind.startswith("norm"):
        # a residual stream: some channels are far larger than the others, and rows of padding are zero
        spread = torch.exp(torch.randn(width, generator=g, device=DEVICE))
        s = {"case": case, "x": (normal(rows, width) * spread).to(type), "residual": (normal(rows, width) * spread * 0.3).to(type),
             "weight": normal(width, scale=0.1, shift=1.0)}
        if rows > 8:
            s["x"][5] = 0
            s["residual"][5] = 0
        if kind == "norm_train":
            s["grad_y"], s["grad_s"] = normal(rows, width), normal(rows, width)
            for name in ("x", "residual", "weight"):
                s[name].requires_grad_(True)
        return s
    if kind.startswith("product"):
        x = (normal(rows, width) * torch.exp(torch.randn(width, generator=g, device=DEVICE))).to(type)
        weight = normal(case["out"], width, scale=width ** -0.5)
        if kind == "product_train":
            return {"case": case, "x": x.requires_grad_(True), "weight": weight.requires_grad_(True), "grad_y": normal(rows, case["out"])}
        # the weights as a checkpoint holds them: 8-bit codes (rows begin on 16 bytes) and one exponent for each block of 128 x 128
        codes, exponents = _to_8bit(weight.float(), BLOCK)
        held = torch.zeros((case["out"], -(-width // 16) * 16), dtype=torch.float8_e4m3fn, device=DEVICE)[:, :width]
        held.copy_(codes.to(torch.float8_e4m3fn))
        scales = torch.zeros((exponents.shape[0], -(-exponents.shape[1] // 4) * 4), dtype=torch.uint8, device=DEVICE)[:, :exponents.shape[1]]
        scales.copy_((exponents + 127).to(torch.uint8))
        return {"case": case, "x": x, "codes": held, "scales": scales.view(torch.float8_e8m0fnu)}
    # values and gates of the recurrence lie side by side, as one projection writes them; a few gates are open or shut altogether
    both = torch.cat((normal(rows, width), normal(rows, width, scale=2.0, shift=2.0)), dim=1)
    both[:, width:][torch.rand((rows, width), generator=g, device=DEVICE) < 0.001] = 40.0
    both[:, width:][torch.rand((rows, width), generator=g, device=DEVICE) < 0.001] = -40.0
    s = {"case": case, "x": both[:, :width], "gate": both[:, width:], "initial": normal(case["sequences"], width, as_type=torch.float32)}
    if kind == "scan_step":
        return s
    s["offsets"] = _offsets(case, seed).to(DEVICE) if case["sequences"] > 1 else None
    if kind == "scan_train":
        s["grad_h"], s["grad_last"] = normal(rows, width), normal(case["sequences"], width, as_type=torch.float32)
        for name in ("x", "gate", "initial"):
            s[name] = s[name].detach().requires_grad_(True)
    return s


# ---- the framework's operators ------------------------------------------------------------------------------------------------


def _run_own(s):
    from htgs_b200 import sequence as seq
    case = s["case"]
    kind = case["kind"]
    if kind == "norm_8bit":
        q, stream = seq.add_rms_norm_fp8(s["x"], s["weight"], s["residual"], EPS)
        return {"y": q.dequantize(), "s": stream}
    if kind == "norm_train":
        y, stream = seq.add_rms_norm(s["x"], s["weight"], s["residual"], EPS)
        gx, gr, gw = torch.autograd.grad((y, stream), (s["x"], s["residual"], s["weight"]), (s["grad_y"], s["grad_s"]))
        return {"y": y, "s": stream, "gx": gx, "gr": gr, "gw": gw}
    if kind == "product":
        return seq.fp8_matmul(s["x"], seq.Fp8Matrix(s["codes"], s["scales"], rows_per_scale=BLOCK))
    if kind == "product_train":
        y = seq.fp8_linear(s["x"], s["weight"])
        gx, gw = torch.autograd.grad(y, (s["x"], s["weight"]), s["grad_y"])
        return {"y": y, "gx": gx, "gw": gw}
    if kind == "scan_step":
        state = s["initial"].clone()
        return {"h": seq.gated_scan_step(s["x"], s["gate"], state), "state": state}
    h, last = seq.gated_scan(s["x"], s["gate"], s["initial"], offsets=s["offsets"], reverse=case["reverse"])
    if kind == "scan":
        return {"h": h, "last": last}
    gx, gg, gi = torch.autograd.grad((h, last), (s["x"], s["gate"], s["initial"]), (s["grad_h"], s["grad_last"]))
    return {"h": h, "last": last, "gx": gx, "gg": gg, "gi": gi}


# ---- the plain forms ------------------------------------------------------------------------------------------------------------


def _to_8bit(v, rows_per_scale=1):
    """(values on the 8-bit grid, exponents): for each block of `rows_per_scale` x 128 the least exponent e with max |v| <= 448 * 2^e,
    and v * 2^-e rounded to e4m3."""
    rows, width = v.shape
    br, bc = -(-rows // rows_per_scale), -(-width // BLOCK)
    padded = torch.nn.functional.pad(v, (0, bc * BLOCK - width, 0, br * rows_per_scale - rows)).view(br, rows_per_scale, bc, BLOCK)
    mantissa, e = torch.frexp(padded.abs().amax(dim=(1, 3)))
    exponents = torch.where(mantissa > 0, e - 9 + (mantissa > LARGEST / 512).int(), 0)
    codes = torch.ldexp(padded, -exponents[:, None, :, None]).to(torch.float8_e4m3fn).float()
    return codes.view(br * rows_per_scale, bc * BLOCK)[:rows, :width], exponents


def _spread(exponents, rows_per_scale, rows, width):
    """2^exponent for each value of a [rows, width] matrix."""
    scales = torch.exp2(exponents.float())
    return scales.repeat_interleave(rows_per_scale, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :width]


def _through_8bit(v, rows_per_scale=1):
    codes, exponents = _to_8bit(v, rows_per_scale)
    return codes * _spread(exponents, rows_per_scale, *v.shape)


def _recur(a, b):
    """h_t = a_t h_{t-1} + b_t over the rows, by doubling: after each pass a row holds the composition of twice as many steps."""
    span = 1
    while span < b.shape[0]:
        b = torch.cat((b[:span], b[span:] + a[span:] * b[:-span]))
        a = torch.cat((a[:span], a[span:] * a[:-span]))
        span *= 2
    return b


def _run_plain(s):
    case = s["case"]
    kind, type = case["kind"], TYPES[case["type"]]
    if kind.startswith("norm"):
        w = s["weight"].float()
        u = s["x"].float() + s["residual"].float()
        rho = 1.0 / torch.sqrt((u * u).mean(dim=1, keepdim=True) + EPS)
        y = u * rho * w
        if kind == "norm_8bit":
            return {"y": _through_8bit(y).to(torch.bfloat16), "s": u.to(type)}
        z = s["grad_y"].float() * w
        unit = u * rho
        gu = (rho * (z - unit * (z * unit).mean(dim=1, keepdim=True)) + s["grad_s"].float()).to(type)
        return {"y": y.to(type), "s": u.to(type), "gx": gu, "gr": gu, "gw": (s["grad_y"].float() * unit).sum(dim=0).to(type)}
    if kind == "product":
        w = s["codes"].float() * _spread(s["scales"].view(torch.uint8).int() - 127, BLOCK, *s["codes"].shape)
        return (_through_8bit(s["x"].float()) @ w.t()).to(type)
    if kind == "product_train":
        x, w, gy = s["x"].float(), _through_8bit(s["weight"].float(), BLOCK), s["grad_y"].float()
        # each product's operands share a scale along 128 of the summed axis: rows of dy for dx, columns of dy and x for dW
        gw = _through_8bit(gy.t().contiguous()) @ _through_8bit(x.t().contiguous()).t()
        return {"y": (_through_8bit(x) @ w.t()).to(type), "gx": (_through_8bit(gy) @ w).to(type), "gw": gw.to(type)}
    x, gate, initial = s["x"].float(), s["gate"].float(), s["initial"]
    a, keep = 1.0 / (1.0 + torch.exp(-gate)), 1.0 / (1.0 + torch.exp(gate))   # keep = 1 - a
    if kind == "scan_step":
        h = a * initial + keep * x
        return {"h": h.to(type), "state": h}
    rows, flip = case["rows"], case["reverse"]
    ends = torch.tensor([0, rows], device=x.device) if s["offsets"] is None else s["offsets"].long()
    grad = kind == "scan_train"
    if grad:
        gh, glast = s["grad_h"].float(), s["grad_last"]
    if flip:   # the same recurrence over the rows, and over the sequences, from the end
        x, a, keep, initial, ends = x.flip(0), a.flip(0), keep.flip(0), initial.flip(0), rows - ends.flip(0)
        if grad:
            gh, glast = gh.flip(0), glast.flip(0)
    some = ends[1:] > ends[:-1]                                   # sequences that are not empty
    first, final = ends[:-1].clamp(max=rows - 1), (ends[1:] - 1).clamp(min=0)
    begins = torch.zeros(rows, 1, device=x.device).index_add_(0, first, some.float()[:, None]) > 0
    start = torch.zeros_like(x).index_add_(0, first, initial * some[:, None])       # initial state, at each sequence's first row
    h = _recur(a * ~begins, keep * x + a * start)
    last = torch.where(some[:, None], h[final], initial)
    out = {"h": h, "last": last}
    if grad:
        before = torch.where(begins, start, torch.cat((initial[:1], h[:-1])))
        given = gh.index_add(0, final, glast * some[:, None])
        later = torch.cat((a[1:] * ~begins[1:], torch.zeros_like(a[:1])))
        d = _recur(later.flip(0), given.flip(0)).flip(0)
        out.update(gx=keep * d, gg=d * (before - x) * a * keep, gi=torch.where(some[:, None], (a * d)[first], glast))
    if flip:
        out = {name: v.flip(0) for name, v in out.items()}
    return {name: v if name in ("last", "gi") else v.to(type) for name, v in out.items()}


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _run_plain(state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------------


def work(case):
    kind, rows, width, b = case["kind"], case["rows"], case["width"], BYTES[case["type"]]
    n = rows * width
    if kind == "norm_8bit":       # reads x, residual, weight; writes s and the 8-bit values as 16-bit numbers
        return {"bytes": n * (3 * b + 2) + width * b, "flops": 8 * n}
    if kind == "norm_train":      # reads x, residual, weight, dy, ds; writes y, s, the gradient of x and residual, and of the weight
        return {"bytes": n * 7 * b + 2 * width * b, "flops": 18 * n}
    if kind == "product":         # reads x, the codes and the exponents; writes y
        out = case["out"]
        return {"bytes": (n + rows * out) * b + width * out + -(-width // BLOCK) * -(-out // BLOCK), "flops": 2 * n * out}
    if kind == "product_train":   # reads x, the weight and dy; writes y and both gradients
        out = case["out"]
        return {"bytes": (2 * n + 2 * rows * out + 2 * width * out) * b, "flops": 6 * n * out}
    states = case["sequences"] * width * 4
    if kind == "scan_train":      # reads x, gate, dh and the states; writes h, dx, dgate and the states
        return {"bytes": n * 6 * b + 4 * states, "flops": 22 * n}
    return {"bytes": n * 3 * b + 2 * states, "flops": 7 * n}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------------


def _grid_8bit(v):
    """Nearest value with 4 significant bits and a least step of 2^-9, ties to even."""
    step = torch.exp2((torch.frexp(v)[1].double() - 1).clamp(min=-6) - 3)
    return torch.round(v / step) * step


def _exact_8bit(v, block_rows, block_cols=BLOCK):
    out = v.clone()
    for i in range(0, v.shape[1], block_cols):
        part = v[:, i:i + block_cols]
        top = part.abs().amax(dim=1)
        if block_rows > 1:
            top = torch.nn.functional.pad(top, (0, -len(top) % block_rows)).view(-1, block_rows).amax(dim=1).repeat_interleave(block_rows)[:len(top)]
        scale = torch.where(top > 0, torch.exp2(torch.ceil(torch.log2(top.clamp(min=1e-300) / LARGEST))), 1.0)[:, None]
        out[:, i:i + block_cols] = _grid_8bit(part / scale) * scale
    return out


def _exact_recurrence(c, b):
    """h_t = c_t h_{t-1} + b_t, step by step: all pieces of about sqrt(rows) steps side by side, then from piece to piece."""
    rows = b.shape[0]
    steps = max(1, math.isqrt(rows))
    pieces = -(-rows // steps)
    pad = pieces * steps - rows
    c = torch.nn.functional.pad(c, (0, 0, 0, pad)).view(pieces, steps, -1)
    b = torch.nn.functional.pad(b, (0, 0, 0, pad)).view(pieces, steps, -1)
    h, through = b.clone(), c.clone()
    for t in range(1, steps):
        h[:, t] += c[:, t] * h[:, t - 1]
        through[:, t] *= through[:, t - 1]
    for p in range(1, pieces):
        h[p] += through[p] * h[p - 1, -1]
    return h.view(pieces * steps, -1)[:rows]


def exact(case, seed):
    s = prepare(case, seed)
    v = {name: t.detach().double() for name, t in s.items() if isinstance(t, torch.Tensor) and name not in ("codes", "scales", "offsets")}
    kind = case["kind"]
    if kind.startswith("norm"):
        u = v["x"] + v["residual"]
        rho = torch.rsqrt(u.square().mean(dim=1) + EPS)[:, None]
        y = u * rho * v["weight"]
        if kind == "norm_8bit":
            return {"y": _exact_8bit(y, 1), "s": u}
        z = v["weight"] * v["grad_y"]
        gu = rho * z - u * rho ** 3 * (z * u).mean(dim=1, keepdim=True) + v["grad_s"]
        return {"y": y, "s": u, "gx": gu, "gr": gu, "gw": torch.einsum("mk,mk->k", v["grad_y"], u * rho)}
    if kind == "product":
        w = s["codes"].to(torch.float64)
        e = s["scales"].view(torch.uint8).double() - 127
        for i in range(e.shape[0]):
            for j in range(e.shape[1]):
                w[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] *= 2.0 ** e[i, j]
        return torch.einsum("mk,nk->mn", _exact_8bit(v["x"], 1), w)
    if kind == "product_train":
        x, w, gy = v["x"], _exact_8bit(v["weight"], BLOCK), v["grad_y"]
        return {"y": torch.einsum("mk,nk->mn", _exact_8bit(x, 1), w), "gx": torch.einsum("mn,nk->mk", _exact_8bit(gy, 1), w),
                "gw": torch.einsum("nm,km->nk", _exact_8bit(gy.t().contiguous(), 1), _exact_8bit(x.t().contiguous(), 1))}
    a = torch.sigmoid(v["gate"])
    keep = torch.sigmoid(-v["gate"])
    if kind == "scan_step":
        h = a * v["initial"] + keep * v["x"]
        return {"h": h, "state": h}
    ends = [0, case["rows"]] if s["offsets"] is None else s["offsets"].tolist()
    c, b = a.clone(), keep * v["x"]
    step = -1 if case["reverse"] else 1
    spans = [(q, lo, hi - 1) if step > 0 else (q, hi - 1, lo) for q, (lo, hi) in enumerate(zip(ends, ends[1:])) if hi > lo]   # (sequence, first row, last row)
    for q, begin, _ in spans:
        b[begin] += a[begin] * v["initial"][q]
        c[begin] = 0
    h = _exact_recurrence(c, b) if step > 0 else _exact_recurrence(c.flip(0), b.flip(0)).flip(0)
    last = v["initial"].clone()
    for q, _, end in spans:
        last[q] = h[end]
    if kind == "scan":
        return {"h": h, "last": last}
    before = torch.roll(h, step, 0)
    d, gi = v["grad_h"].clone(), v["grad_last"].clone()
    later = torch.roll(a, -step, 0)
    for q, begin, end in spans:
        before[begin] = v["initial"][q]
        d[end] += v["grad_last"][q]
        later[end] = 0
    d = _exact_recurrence(later.flip(0), d.flip(0)).flip(0) if step > 0 else _exact_recurrence(later, d)
    for q, begin, _ in spans:
        gi[q] = a[begin] * d[begin]
    return {"h": h, "last": last, "gx": keep * d, "gg": d * (before - v["x"]) * a * keep, "gi": gi}
