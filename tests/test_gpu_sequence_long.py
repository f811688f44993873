"""GPU: the recurrence over long sequences against its 64-bit form - chunks of 16, 32 and 64 rows, and a walk over them in clusters of blocks, in
runs of several chunks, and in runs longer than the registers hold.  (test_gpu_sequence.py has the short sequences, and the tolerances' derivation.)"""
import math

import numpy as np
import pytest

import sequence_reference as ref
from test_gpu_sequence import F, TINY, U, binding, draw, f64, near  # noqa: F401

pytestmark = pytest.mark.gpu


def linear(c, b):
    """h_t = c_t h_{t-1} + b_t from h_{-1} = 0, in 64 bits: pieces of about sqrt(rows) steps side by side, then from piece to piece."""
    rows, width = b.shape
    steps = max(1, math.isqrt(rows))
    pieces = -(-rows // steps)
    h, through = (np.concatenate((v, np.zeros((pieces * steps - rows, width)))).reshape(pieces, steps, width) for v in (b, c))
    for t in range(1, steps):
        h[:, t] += through[:, t] * h[:, t - 1]
        through[:, t] *= through[:, t - 1]
    for p in range(1, pieces):
        h[p] += through[p] * h[p - 1, -1]
    return h.reshape(pieces * steps, width)[:rows]


def long_scan(x, g, initial, offsets, gh, gl, reverse, kind):
    """[(value, bound)] of h, last and the three gradients: scan_bounds and backward_bounds of test_gpu_sequence.py, whose sums along a sequence are linear recurrences too."""
    rows, offsets = x.shape[0], np.asarray(offsets)
    if reverse:
        x, g, gh, initial, gl, offsets = x[::-1], g[::-1], gh[::-1], initial[::-1], gl[::-1], rows - offsets[::-1]
    a, rest = ref.gates(g)
    step = 2 * (8 + 1.2 * np.abs(g)) * 2 * F
    some = offsets[1:] > offsets[:-1]
    begin, end = offsets[:-1][some], offsets[1:][some] - 1
    c = a.copy()
    c[begin] = 0

    def forward(b, first):
        b = b.copy()
        b[begin] += a[begin] * first[some]
        return linear(c, b)
    h = forward(rest * x, initial)
    size = forward(rest * np.abs(x), np.abs(initial))
    off = linear(c, step * size)
    last, last_off = initial.copy(), np.zeros_like(initial)
    last[some], last_off[some] = h[end], off[end]
    before = np.concatenate((h[:1], h[:-1]))
    before_off = np.concatenate((off[:1], off[:-1])) + F * np.abs(before) + TINY["fp32"]
    before[begin], before_off[begin] = initial[some], 0.0

    later = np.concatenate((a[1:], a[:1]))                  # gate and step of the row behind, none at a sequence's end
    later_step = np.concatenate((step[1:], step[:1]))
    later[end] = later_step[end] = 0

    def backward(b):
        return linear(later[::-1], b[::-1])[::-1]
    d, d_size = gh.copy(), np.abs(gh)
    d[end] += gl[some]
    d_size[end] += np.abs(gl[some])
    d, d_size = backward(d), backward(d_size)
    behind = np.concatenate((d_size[1:], d_size[:1]))
    d_off = backward(F * d_size + later_step * later * behind)
    gx_off = rest * (d_off + step * d_size)
    ar = a * rest
    gg = d * (before - x) * ar
    gg_off = ar * (np.abs(before) + np.abs(x)) * (d_off + 2 * step * d_size) + ar * before_off * d_size
    gi, gi_off = gl.copy(), np.zeros_like(gl)
    gi[some], gi_off[some] = (a * d)[begin], (a * (d_off + step * d_size))[begin]
    out = [(v, o + u * np.abs(v) + t) for v, o, u, t in ((h, off, U[kind], TINY[kind]), (last, last_off, 2 * F, TINY["fp32"]), (rest * d, gx_off, U[kind], TINY[kind]),
                                                         (gg, gg_off, U[kind], TINY[kind]), (gi, gi_off, F, TINY["fp32"]))]
    return [(v[::-1], o[::-1]) for v, o in out] if reverse else out


def shape_of_walk(rows, width):
    """(rows of a chunk, chunks, blocks of a cluster, chunks of a run) by the launcher's rules, so that a change of them cannot drop a form unseen."""
    tiles, chunk = -(-width // 64), 64
    while rows > 64 and chunk > 16 and -(-rows // chunk) * tiles < 148 * 32:
        chunk //= 2
    chunks, parts = -(-rows // chunk), 1
    while parts < 8 and chunks > 1024 * parts:
        parts *= 2
    return chunk, chunks, parts, -(-chunks // (128 * parts))


def cuts(rows, chunk, seed):
    """Sequences of very different lengths, cut at borders of chunks and runs and beside them, empty ones and single rows among them."""
    rng = np.random.default_rng(seed)
    inside = [chunk, chunk, 7 * chunk, 7 * chunk + 1, 35 * chunk, rows // 2 // chunk * chunk, rows // 2 // chunk * chunk + 1, rows - 1] + list(rng.integers(1, rows, 5))
    return [0, 0] + sorted(int(c) for c in inside) + [rows, rows]


@pytest.mark.parametrize("kind,rows,width,walk", [
    ("bf16", 20_000, 64, (16, 1250, 2, 5)), ("fp32", 50_001, 1, (16, 3126, 4, 7)), ("fp16", 150_001, 3, (16, 9376, 8, 10)), ("bf16", 200_000, 64, (32, 6250, 8, 7)),
    ("bf16", 101_063, 130, (64, 1580, 2, 7)), ("fp32", 1_100_001, 2, (64, 17188, 8, 17)), ("bf16", 2_200_003, 2, (64, 34376, 8, 34))])
@pytest.mark.parametrize("packed,reverse", [(False, False), (True, False), (True, True)])
def test_scan_of_long_sequences(kind, rows, width, walk, packed, reverse):
    import torch
    from htgs_b200 import sequence as seq
    assert shape_of_walk(rows, width) == walk
    offsets = cuts(rows, walk[0], rows) if packed else [0, rows]
    n = len(offsets) - 1
    both = draw((rows, 2 * width), rows + width, kind)
    x, g = both[:, :width], both[:, width:]
    g.mul_(2).add_(4)                                     # long memories: a state goes on through many chunks
    initial, gh, gl = draw((n, width), 5), draw((rows, width), 6, kind), draw((n, width), 7)
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda") if packed else None
    leaves = [t.detach().requires_grad_(True) for t in (x, g, initial)]
    h, last = seq.gated_scan(*leaves, off, reverse)
    got = (h, last, *torch.autograd.grad((h, last), leaves, (gh, gl)))
    want = long_scan(f64(x), f64(g), f64(initial), offsets, f64(gh), f64(gl), reverse, kind)
    for value, (exact, bound), name in zip(got, want, ("h", "last", "grad_x", "grad_gate", "grad_initial")):
        near(value, exact, bound, name)
    with torch.no_grad():
        again = seq.gated_scan(x, g, initial, off, reverse)
    assert torch.equal(again[0], h) and torch.equal(again[1], last)


@pytest.mark.parametrize("reverse", [False, True])
def test_long_scan_keeps_nan_to_its_sequence(reverse):
    """A NaN in one sequence reaches every row behind it there, through chunks, runs and blocks of the walk, and no other sequence."""
    import torch
    from htgs_b200 import sequence as seq
    rows = 1_100_000
    offsets = [0, 64 * 17 * 128, 64 * 17 * 128, 400_003, 1_000_000, rows]
    x, g = draw((rows, 2), 1), draw((rows, 2), 2, "fp32", 1.0, 4.0)
    at = 500_000
    x[at, 0] = float("nan")
    leaves = [t.requires_grad_(True) for t in (x, g)]
    h, last = seq.gated_scan(*leaves, None, torch.tensor(offsets, dtype=torch.int32, device="cuda"), reverse)
    want = torch.zeros(rows, 2, dtype=torch.bool, device="cuda")
    want[400_003:at + 1 if reverse else 1_000_000, 0] = True
    if not reverse:
        want[400_003:at, 0] = False
    assert torch.equal(torch.isnan(h), want)
    assert torch.equal(torch.isnan(last), torch.tensor([[s == 3, False] for s in range(5)], device="cuda"))
    gh = torch.zeros_like(h)
    gh[at, 1] = float("nan")                              # backward it reaches what lies in front
    gx, gg = torch.autograd.grad(h, leaves, gh)
    want = torch.zeros(rows, 2, dtype=torch.bool, device="cuda")
    want[at:1_000_000, 1] = True
    if not reverse:
        want[:, 1] = False
        want[400_003:at + 1, 1] = True
    assert torch.equal(torch.isnan(gx)[:, 1], want[:, 1]) and torch.equal(torch.isnan(gg)[:, 1], want[:, 1])
