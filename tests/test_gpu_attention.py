"""GPU: rotary positions, attention over packed sequences and its step over a cache, against their 64-bit forms (attention_reference.py, which derives the tolerances)."""
import math

import pytest
import torch

import attention_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, params=["pybind", "ctypes"])
def binding(request, monkeypatch):
    """Every test runs over the compiled extension module and over ctypes."""
    from htgs_b200 import _native
    if request.param == "ctypes":
        monkeypatch.setattr(_native, "_pybind_modules", False)
    elif not _native.pybind_modules():
        pytest.skip("htgs_b200/pybind modules not built (python -m htgs_b200.build)")


DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def draw(shape, seed, kind, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(DTYPES[kind]).cuda()


def f64(t):
    return t.detach().double().cpu()


def near(got, want, bound, what=""):
    got = f64(got)
    assert got.shape == want.shape, what
    assert torch.equal(got.isnan(), want.isnan()), what
    off = (got.nan_to_num() - want.nan_to_num()).abs()
    bad = off > bound.nan_to_num()
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values, worst {float((off / bound)[bad].max())} of the bound, first at {bad.nonzero()[0].tolist()}"


def both_ways(q, k, v, grad, kind, ends=None, causal=False, window=None, scale=None, batch=None):
    """Forward and backward against the reference; q, k, v [rows, heads, width] (or with `batch` in front)."""
    from htgs_b200 import sequence as seq
    offsets = None if ends is None else torch.tensor(ends, dtype=torch.int32, device="cuda")
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = seq.attention(*leaves, offsets=offsets, causal=causal, window=window, scale=scale)
    with torch.no_grad():
        inference = seq.attention(q, k, v, offsets=offsets, causal=causal, window=window, scale=scale)
    if q.shape[-1] <= 64 or kind == "fp32":
        assert torch.equal(out, inference)
    grads = torch.autograd.grad(out, leaves, grad)
    flat = [f64(t).flatten(0, -3) for t in (q, k, v, grad)]
    rows = flat[0].shape[0]
    if q.dim() == 4:
        ends = list(range(0, rows + 1, q.shape[1]))
    want, bound = ref.attend(*flat[:3], ends or [0, rows], causal, window, q.shape[-1] ** -0.5 if scale is None else scale, kind, flat[3])
    # wider heads take a row's largest weight as 1 in training and as up to 2^8 else: other roundings of the weights, each at most u of them, which the bound has
    for name, t in zip(("out", "out", "gq", "gk", "gv"), (out, inference, *grads)):
        near(t.flatten(0, -3), want[name], bound[name], name)
    again = torch.autograd.grad(seq.attention(*leaves, offsets=offsets, causal=causal, window=window, scale=scale), leaves, grad)
    assert all(torch.equal(a, b) for a, b in zip(grads, again)), "the same inputs give the same bits"


def tensors(rows, heads, key_heads, width, kind, seed=1):
    return (draw((rows, heads, width), seed, kind, 1.5), draw((rows, key_heads, width), seed + 1, kind, 1.5), draw((rows, key_heads, width), seed + 2, kind),
            draw((rows, heads, width), seed + 3, kind))


# ---- rotary ----------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("rows,heads,key_heads,width,axes", [(1, 1, 1, 2, 1), (3, 2, 1, 6, 3), (9, 3, 0, 10, 4), (17, 4, 2, 16, 2), (33, 8, 2, 64, 3), (40, 3, 3, 40, 3), (5, 1, 1, 256, 1), (70, 5, 1, 36, 2)])
def test_rotary_forward_and_backward(rows, heads, key_heads, width, axes, kind, interleaved):
    from htgs_b200 import sequence as seq
    q, k = draw((rows, heads, width), 1, kind), draw((rows, key_heads, width), 2, kind) if key_heads else None
    g = torch.Generator().manual_seed(3)
    positions = torch.randint(-1_000_000, 1_000_000, (rows, 1), generator=g, dtype=torch.int32) if axes == 1 else torch.randn((rows, axes), generator=g) * 300
    pairs = width // 2
    sections = [pairs // axes + (a < pairs % axes) for a in range(axes)]
    angle = ref.angles(positions, sections, 10000.0)
    leaves = [t.requires_grad_(True) for t in (q, k) if t is not None]
    out = seq.rotary(q, k, positions.cuda(), interleaved=interleaved)
    assert (out[1] is None) == (k is None)
    grads = [draw(t.shape, 7 + i, kind) for i, t in enumerate(leaves)]
    back = torch.autograd.grad([t for t in out if t is not None], leaves, grads)
    for x, y, gy, gx in zip(leaves, out, grads, back):
        near(y, ref.turn(f64(x), angle, interleaved), ref.turn_bound(f64(x), kind, interleaved), "out")
        near(gx, ref.turn(f64(gy), -angle, interleaved), ref.turn_bound(f64(gy), kind, interleaved), "grad")


def test_rotary_views_sections_and_parts_of_the_gradient():
    from htgs_b200 import sequence as seq
    both = draw((2, 11, 7 * 24), 1, "bf16")
    q, k = both[..., :96].unflatten(-1, (4, 24)), both[..., 96:144].unflatten(-1, (2, 24))
    positions = (torch.randn((2, 11, 3), generator=torch.Generator().manual_seed(2)) * 50).cuda()
    a, b = seq.rotary(q, k, positions, sections=[5, 0, 7], base=100.0)
    angle = ref.angles(positions.cpu().flatten(0, 1), [5, 0, 7], 100.0)
    for x, y in ((q, a), (k, b)):
        assert y.shape == x.shape
        near(y.flatten(0, 1), ref.turn(f64(x).flatten(0, 1), angle, False), ref.turn_bound(f64(x).flatten(0, 1), "bf16", False))
    odd = draw((5, 3, 17), 3, "fp16")[..., 1:]                            # heads that begin on 2 bytes
    p = torch.arange(5, dtype=torch.int32, device="cuda")[:, None]
    for interleaved in (False, True):
        assert torch.equal(seq.rotary(odd, None, p, interleaved=interleaved)[0], seq.rotary(odd.contiguous(), None, p, interleaved=interleaved)[0])
    heads_first = draw((3, 5, 16), 4, "fp32").transpose(0, 1)
    assert torch.equal(seq.rotary(heads_first, None, p)[0], seq.rotary(heads_first.contiguous(), None, p)[0])
    ql, kl = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
    a, b = seq.rotary(ql, kl, positions)
    (gk,) = torch.autograd.grad(b, kl, torch.ones_like(b))                # nothing reaches q
    assert torch.equal(gk, torch.autograd.grad(seq.rotary(kl, None, positions)[0], kl, torch.ones_like(b))[0])
    empty = torch.empty((0, 2, 8), device="cuda")
    assert seq.rotary(empty, None, torch.empty((0, 2), device="cuda"))[0].shape == (0, 2, 8)
    with pytest.raises(RuntimeError, match="positions"):
        seq.rotary(q, k, positions.clone().requires_grad_(True))


# ---- attention --------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("causal,window", [(False, None), (True, None), (False, 0), (False, 50), (True, 130), (True, 1 << 40)])
@pytest.mark.parametrize("rows,heads,key_heads,width", [(1, 1, 1, 8), (7, 2, 1, 24), (130, 3, 3, 64), (300, 4, 2, 128), (521, 2, 1, 72)])
def test_attention_forward_and_backward(rows, heads, key_heads, width, causal, window, kind):
    both_ways(*tensors(rows, heads, key_heads, width, kind), kind, causal=causal, window=window)


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("width", [1, 5, 33, 100, 127])
def test_attention_of_odd_widths(kind, width):
    both_ways(*tensors(70, 4, 2, width, kind), kind, causal=True)


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("causal,window", [(False, None), (True, None), (False, 20), (True, 200)])
def test_packed_sequences(kind, causal, window):
    both_ways(*tensors(700, 4, 2, 32, kind), kind, ends=[0, 0, 1, 1, 3, 130, 258, 259, 515, 515, 700, 700], causal=causal, window=window)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_batches_scales_and_many_heads(kind):
    q, k, v, grad = (t.view(3, 45, *t.shape[1:]) for t in tensors(135, 8, 1, 16, kind))
    both_ways(q, k, v, grad, kind, causal=True, scale=0.7)
    both_ways(*tensors(40, 17, 17, 8, kind), kind)


def test_more_sequences_than_a_warp_searches_at_once():
    ends = [min(3 * i + i % 2, 3000) for i in range(1100)]
    ends[-1] = 3000
    both_ways(*tensors(3000, 1, 1, 16, "bf16"), "bf16", ends=sorted(ends))


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
def test_rows_of_no_sequence_get_zeros_and_leave_no_trace(kind):
    from htgs_b200 import sequence as seq
    q, k, v, grad = tensors(400, 2, 2, 64, kind)
    for t in (q, k, v, grad):
        t[:37] = float("nan")
        t[300:] = float("inf")
    offsets = torch.tensor([37, 100, 300], dtype=torch.int32, device="cuda")
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = seq.attention(*leaves, offsets=offsets, causal=True)
    grads = torch.autograd.grad(out, leaves, grad)
    # Beside values that are not finite a tile is summed up in another order than without them, each sum within the bound: n terms off by 2 F of their magnitudes, then one rounding.
    inner = [f64(t)[37:300] for t in (*leaves, grad)]
    want, bound = ref.attend(*inner[:3], [0, 63, 263], True, None, 0.125, kind, inner[3])
    for name, t in zip(("out", "gq", "gk", "gv"), (out, *grads)):
        near(t[37:300], want[name], bound[name], name)
        assert not t[:37].any() and not t[300:].any()


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_what_a_row_does_not_see_does_not_reach_it(kind, bad):
    """Rows 200 on of the values, keys and queries are not finite: rows before them, causal, and rows of the other sequences come out as if they were."""
    from htgs_b200 import sequence as seq
    rows, ends = 500, [0, 60, 390, 500]
    q, k, v, grad = tensors(rows, 2, 1, 64, kind)
    offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")

    def run(*given):
        leaves = [t.detach().clone().requires_grad_(True) for t in given[:3]]
        out = seq.attention(*leaves, offsets=offsets, causal=True, window=300)
        return (out, *torch.autograd.grad(out, leaves, given[3]))

    spoilt = [t.clone() for t in (q, k, v, grad)]
    for t in spoilt:
        t[200:390, :, 3] = bad
    dirty = run(*spoilt)
    want, bound = ref.attend(f64(q), f64(k), f64(v), ends, True, 300, 0.125, kind, f64(grad))          # as above: within the bound, not bit for bit
    other = torch.cat((torch.arange(60), torch.arange(390, rows)))
    for name, t in zip(("out", "gq", "gk", "gv"), dirty):
        near(t[other.cuda()], want[name][other], bound[name][other], name)
    for name, t in zip(("out", "gq"), dirty):           # keys before them are seen by queries behind: only these
        near(t[60:200], want[name][60:200], bound[name][60:200], name)
    assert dirty[0][200:390].isnan().any()


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_scores_that_are_not_finite_reach_the_rows_that_see_them(kind, bad):
    """One key's score is not finite, whichever column of a tile it is: NaN for NaN and plus infinity in every row that sees it, a weight of zero for minus infinity."""
    from htgs_b200 import sequence as seq
    rows = 390
    q, k, v, grad = tensors(rows, 1, 1, 16, kind)
    q[..., 0] = 1.0
    for j in (0, 1, 6, 7, 13, 40, 77, 127, 128, 200, 201, 259, 388):
        spoilt = k.clone()
        spoilt[j, 0, 0] = bad
        out = f64(seq.attention(q, spoilt, v, causal=True))
        want, bound = ref.attend(f64(q), f64(k), f64(v), [0, rows], True, None, 0.25, kind)
        near(out[:j], want["out"][:j], bound["out"][:j], f"{j}: rows before it")
        if bad != float("-inf"):
            assert out[j:].isnan().all(), j
        elif j:
            assert out[j:].isfinite().all(), j
            S = 0.25 * (f64(q)[j:, 0] @ f64(spoilt)[:, 0].t())
            P = torch.softmax(S.masked_fill(torch.arange(rows)[None] > torch.arange(j, rows)[:, None], -math.inf), dim=1)
            near(out[j:, 0], P @ f64(v)[:, 0], 2 * bound["out"][j:, 0] + 4 * ref.U[kind] * (P @ f64(v)[:, 0].abs()), f"{j}: rows behind it")        # fewer terms than the bound's, with weights up to twice and more


def test_scores_far_apart_and_large():
    """Scores from -2000 to 2000: no overflow, and one row's largest does not take another's."""
    kind = "bf16"
    q, k, v, grad = tensors(300, 1, 1, 64, kind)
    q[::7] *= 100
    k[::5] *= 4
    from htgs_b200 import sequence as seq
    out = seq.attention(q, k, v, causal=True)
    want, bound = ref.attend(f64(q), f64(k), f64(v), [0, 300], True, None, 0.125, kind)
    near(out, want["out"], bound["out"])


def test_a_long_row_of_small_weights():
    """One key holds half of the weight and 60000 others the rest, each too small for the smallest normal number of 16 bits."""
    from htgs_b200 import sequence as seq
    rows, width = 60001, 64
    for kind in ("fp16", "bf16"):
        q, k = torch.zeros((rows, 1, width), dtype=DTYPES[kind], device="cuda"), torch.zeros((rows, 1, width), dtype=DTYPES[kind], device="cuda")
        q[0, 0, 0], k[0, 0, 0] = 8.0, 11.0                           # score 11 = log(60000)
        v = draw((rows, 1, width), 1, kind, 0.1) + 1.0
        v[0] = 0.0
        out = seq.attention(q, k, v)[0, 0]
        p = math.exp(11.0) / (math.exp(11.0) + rows - 1)
        want = (1 - p) * f64(v)[1:, 0].mean(dim=0)
        assert ((f64(out) - want).abs() <= want.abs() * (2 * ref.U[kind] + 2 * rows * ref.SUM)).all(), kind       # weights and output rounded; two sums of as many terms as rows


def test_attention_without_rows_and_gradients_of_some_inputs():
    from htgs_b200 import sequence as seq
    e, f, g = (torch.empty((0, 2, 16), device="cuda", dtype=torch.bfloat16, requires_grad=True) for _ in range(3))
    out = seq.attention(e, f, g, window=1 << 80)
    assert out.shape == (0, 2, 16)
    out.sum().backward()
    assert all(t.grad.shape == t.shape for t in (e, f, g))
    q, k, v, grad = tensors(50, 2, 2, 16, "bf16")
    ql = q.clone().requires_grad_(True)
    (gq,) = torch.autograd.grad(seq.attention(ql, k, v), ql, grad)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    assert torch.equal(gq, torch.autograd.grad(seq.attention(*leaves), leaves, grad)[0])
    one = torch.ones((), device="cuda", dtype=torch.bfloat16).expand(50, 2, 16)           # a broadcast gradient
    a = torch.autograd.grad(seq.attention(*leaves), leaves, one)
    assert all(torch.equal(x, y) for x, y in zip(a, torch.autograd.grad(seq.attention(*leaves), leaves, one.contiguous())))
    shared = k[:, :1].expand(50, 2, 16).detach()                                              # heads that are one in memory
    assert torch.equal(seq.attention(q, shared, shared), seq.attention(q, shared.contiguous(), shared.contiguous()))
    out = seq.attention(*leaves)
    (g,) = torch.autograd.grad(out, leaves[0], grad, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.sum().backward()


def test_views_of_one_projection_and_heads_first():
    from htgs_b200 import sequence as seq
    both = draw((300, 6 * 40), 1, "bf16")
    q, k, v = (t.unflatten(1, (-1, 40)) for t in both.split([160, 40, 40], dim=1))
    out = seq.attention(q, k, v, causal=True)
    assert torch.equal(out, seq.attention(q.contiguous(), k.contiguous(), v.contiguous(), causal=True))
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert torch.equal(out, seq.attention(*turned, causal=True))
    odd = draw((300, 241), 1, "bf16")[:, 1:]
    odd.copy_(both)
    assert torch.equal(out, seq.attention(*(t.unflatten(1, (-1, 40)) for t in odd.split([160, 40, 40], dim=1)), causal=True))


def test_gradients_against_differences():
    """In 32 bits: (L(x + h e) - L(x - h e)) / 2 h along random directions."""
    from htgs_b200 import sequence as seq
    q, k, v, grad = tensors(40, 2, 1, 12, "fp32")
    positions = (torch.rand((40, 3), generator=torch.Generator().manual_seed(5)) * 20).cuda()
    ends = torch.tensor([0, 15, 40], dtype=torch.int32, device="cuda")

    def loss(q, k, v):
        q, k = seq.rotary(q, k, positions)
        return (seq.attention(q, k, v, offsets=ends, window=9).double() * grad.double()).sum()

    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    with torch.no_grad():
        for which in range(3):
            e = draw(leaves[which].shape, 20 + which, "fp32")
            h = 2.0 ** -7
            plus, minus = ([t + s * h * e if i == which else t for i, t in enumerate(leaves)] for s in (1, -1))
            # central differences: h^2 / 6 of the third derivative (a few tens here), and 32-bit noise of about 1e-5 over h
            slope, want = float(loss(*plus) - loss(*minus)) / (2 * h), float((grads[which].double() * e.double()).sum())
            assert abs(slope - want) <= 0.02 * max(1.0, abs(want)), which


# ---- one more row ------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("window", [None, 0, 40])
@pytest.mark.parametrize("capacity,heads,key_heads,width", [(1, 1, 1, 8), (40, 4, 2, 24), (300, 8, 1, 64), (700, 3, 3, 128), (2500, 20, 1, 40), (90, 2, 2, 13)])
def test_step(capacity, heads, key_heads, width, window, kind):
    from htgs_b200 import sequence as seq
    lengths = [0, capacity - 1, capacity // 2, -1, capacity, min(17, capacity - 1), capacity + 5, -7]
    batch = len(lengths)
    q, k, v = draw((batch, heads, width), 1, kind, 1.5), draw((batch, key_heads, width), 2, kind, 1.5), draw((batch, key_heads, width), 3, kind)
    keys, values = draw((batch, capacity, key_heads, width), 4, kind, 1.5), draw((batch, capacity, key_heads, width), 5, kind)
    for b, n in enumerate(lengths):            # what lies behind a sequence's rows never counts
        keys[b, max(n, 0):] = float("nan")
        values[b, max(n, 0):] = float("nan")
    before = keys.clone(), values.clone()
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = seq.attention_step(q, k, v, keys, values, n, window=window)
    assert torch.equal(n.cpu(), torch.tensor(lengths, dtype=torch.int32))
    for b, length in enumerate(lengths):
        if 0 <= length < capacity:
            before[0][b, length], before[1][b, length] = k[b], v[b]
            low = 0 if window is None else max(0, length - window)
            want, bound = ref.attend(f64(q[b])[None].expand(length + 1 - low, -1, -1), f64(keys[b, low:length + 1]), f64(values[b, low:length + 1]), [0, length + 1 - low], True, None,
                                     width ** -0.5, kind)
            near(out[b], want["out"][-1], bound["out"][-1], f"sequence {b}")
        else:
            assert out[b].isnan().all() if length >= capacity else not out[b].any()
    assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip((keys, values), before))


def test_steps_make_a_sequence():
    """Rotary and attention over whole sequences, and the same row by row over caches that lie heads first."""
    from htgs_b200 import sequence as seq
    batch, rows, heads, key_heads, width = 3, 50, 4, 2, 32
    q, k, v, _ = (t.view(batch, rows, *t.shape[1:]) for t in tensors(batch * rows, heads, key_heads, width, "fp32"))
    positions = torch.arange(rows, dtype=torch.int32, device="cuda")[None, :, None].expand(batch, rows, 1)
    whole = seq.attention(*seq.rotary(q, k, positions), v, causal=True, window=20)
    keys, values = (torch.full((batch, key_heads, rows, width), float("nan"), device="cuda").transpose(1, 2) for _ in range(2))
    lengths = torch.zeros(batch, dtype=torch.int32, device="cuda")
    for t in range(rows):
        qt, kt = seq.rotary(q[:, t], k[:, t], lengths[:, None])
        out = seq.attention_step(qt, kt, v[:, t], keys, values, lengths, window=20)
        assert torch.allclose(out, whole[:, t], rtol=1e-5, atol=1e-5)
        lengths += 1


def test_step_in_a_graph_and_on_another_stream():
    from htgs_b200 import sequence as seq
    batch, capacity, heads, width = 2, 3000, 2, 64
    q, k, v = (draw((batch, heads, width), i, "bf16") for i in range(3))
    keys, values = (draw((batch, capacity, heads, width), 4 + i, "bf16") for i in range(2))
    lengths = torch.tensor([0, 2500], dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        seq.attention_step(q, k, v, keys.clone(), values.clone(), lengths)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = seq.attention_step(q, k, v, keys, values, lengths)
            lengths += 1
    torch.cuda.current_stream().wait_stream(stream)
    lengths.copy_(torch.tensor([0, 2500]))
    plain = keys.clone(), values.clone(), lengths.clone()
    for _ in range(4):
        graph.replay()
        want = seq.attention_step(q, k, v, *plain)
        plain[2].add_(1)
        assert torch.equal(out, want)
    assert torch.equal(keys, plain[0]) and torch.equal(values, plain[1]) and lengths.tolist() == [4, 2504]


def test_a_captured_forward_and_backward():
    from htgs_b200 import sequence as seq
    q, k, v, grad = tensors(300, 4, 2, 64, "bf16")
    ends = torch.tensor([0, 100, 300], dtype=torch.int32, device="cuda")
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    run = lambda: (lambda out: (out, *torch.autograd.grad(out, leaves, grad)))(seq.attention(*leaves, offsets=ends, causal=True))  # noqa: E731
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            captured = run()
    torch.cuda.current_stream().wait_stream(stream)
    with torch.no_grad():
        for t in leaves:
            t.mul_(0.5)
        ends.copy_(torch.tensor([0, 250, 300]))
    graph.replay()
    for a, b in zip(captured, run()):
        assert torch.equal(a, b)


# ---- many pieces, several calls at once, large places, states of failure ---------------------------------------------------------------


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("heads,key_heads,width,causal,window", [(8, 8, 32, False, 100), (4, 2, 64, True, None), (6, 1, 48, False, None), (4, 2, 128, True, None), (2, 2, 96, False, 150)])
def test_copies_of_a_scene_get_the_same_bits(heads, key_heads, width, causal, window, kind):
    """So many pieces that every block goes through several: each copy of three sequences, one of them empty, comes out as the first, and the first as alone."""
    from htgs_b200 import sequence as seq
    lengths, copies = (431, 0, 130), 60
    one = [t.cpu() for t in tensors(sum(lengths), heads, key_heads, width, kind)]
    ends = [0]
    for _ in range(copies):
        for n in lengths:
            ends.append(ends[-1] + n)

    def run(parts, ends):
        leaves = [t.cuda().requires_grad_(True) for t in parts[:3]]
        out = seq.attention(*leaves, offsets=torch.tensor(ends, dtype=torch.int32, device="cuda"), causal=causal, window=window)
        return (out, *torch.autograd.grad(out, leaves, parts[3].cuda()))

    alone = run(one, ends[:4])
    for _ in range(3):
        for a, b in zip(alone, run([t.repeat(copies, 1, 1) for t in one], ends)):
            assert torch.equal(b.view(copies, *a.shape), a.expand(copies, *a.shape))
    want, bound = ref.attend(*(f64(t) for t in one[:3]), ends[:4], causal, window, width ** -0.5, kind, f64(one[3]))
    for name, t in zip(("out", "gq", "gk", "gv"), alone):
        near(t, want[name], bound[name], name)


def test_calls_of_several_threads_and_streams_at_once():
    import threading
    from htgs_b200 import sequence as seq
    cases = [(tensors(900, 4, 2, 64, "bf16", seed=1), {"causal": True}), (tensors(700, 2, 2, 128, "fp16", seed=9), {"window": 77})]

    def run(parts, how):
        leaves = [t.detach().requires_grad_(True) for t in parts[:3]]
        out = seq.attention(*leaves, **how)
        return (out, *torch.autograd.grad(out, leaves, parts[3]))

    serial = [run(*c) for c in cases]
    torch.cuda.synchronize()
    failures = []

    def work(which):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = run(*cases[which])
                torch.cuda.current_stream().synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, serial[which])):
                failures.append(which)
        except Exception as e:  # noqa: BLE001
            failures.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures


@pytest.mark.parametrize("factor", [2.0 ** -14, 1.0, 2.0 ** 13])
def test_half_precision_gradients_of_any_size(factor):
    """Gradients of scores are 10^-3 of the output's gradient and less; those of small output gradients would be below the smallest number of fp16, those of large ones pass its largest in a sum."""
    from htgs_b200 import sequence as seq
    for width in (64, 128):
        q, k, v, grad = tensors(700, 2, 1, width, "fp16")
        grad = (grad.float() * factor * 0.25).half()
        leaves = [t.requires_grad_(True) for t in (q, k, v)]
        got = torch.autograd.grad(seq.attention(*leaves), leaves, grad)
        want, bound = ref.attend(f64(q), f64(k), f64(v), [0, 700], False, None, width ** -0.5, "fp16", f64(grad))
        for name, t in zip(("gq", "gk", "gv"), got):
            near(t, want[name], bound[name], name)


def test_places_behind_two_to_the_31():
    """The last rows of a cache of 2.2e9 values, and rows of a projection 2^16 values apart."""
    from htgs_b200 import sequence as seq
    capacity, heads, width = 2_200_000, 8, 128
    keys, values = (torch.empty((1, capacity, heads, width), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q, k, v = (draw((1, heads, width), i, "bf16") for i in range(3))
    keys[:, -60:], values[:, -60:] = draw((1, 60, heads, width), 4, "bf16"), draw((1, 60, heads, width), 5, "bf16")
    out = seq.attention_step(q, k, v, keys, values, torch.tensor([capacity - 1], dtype=torch.int32, device="cuda"), window=50)
    assert torch.equal(keys[0, -1], k[0]) and torch.equal(values[0, -1], v[0])
    small = keys[:, -51:].clone(), values[:, -51:].clone()
    assert torch.equal(out, seq.attention_step(q, k, v, *small, torch.tensor([50], dtype=torch.int32, device="cuda")))
    del keys, values
    far = torch.empty((40_000, 1 << 16), dtype=torch.bfloat16, device="cuda")[:, :3 * 64]
    far.copy_(draw((40_000, 192), 6, "bf16"))
    parts = [t.unflatten(1, (1, 64)) for t in far.split(64, dim=1)]
    near_by = [t.contiguous() for t in parts]
    assert torch.equal(seq.attention(*parts, window=30), seq.attention(*near_by, window=30))
    p = torch.arange(40_000, dtype=torch.int32, device="cuda")[:, None]
    assert torch.equal(seq.rotary(parts[0], None, p)[0], seq.rotary(near_by[0], None, p)[0])


def test_a_wait_that_ran_out_is_reported_once():
    """The word that a kernel would set is set by hand."""
    from htgs_b200 import _native, sequence as seq
    q, k, v, _ = tensors(20, 1, 1, 16, "bf16")
    device = torch.cuda.current_device()
    seq.attention(q, k, v)
    word = _native.lib().htgs_attention_error_word(device)
    word[0] = 1
    with pytest.raises(RuntimeError, match="ran out"):
        seq.attention(q, k, v)
    seq.check_attention()
    word[0] = 1
    with pytest.raises(RuntimeError, match="ran out"):
        seq.check_attention(q.device)
    assert seq.attention(q, k, v).isfinite().all()


def test_refusals():
    from htgs_b200 import sequence as seq
    q, k, v, _ = tensors(20, 4, 2, 16, "bf16")
    n = torch.zeros(20, dtype=torch.int32, device="cuda")
    p = torch.zeros((20, 2), device="cuda")
    cache = torch.zeros((20, 5, 2, 16), dtype=torch.bfloat16, device="cuda")
    other = torch.zeros_like(cache)
    bad_values = [lambda: seq.attention(q, k[:10], v[:10]), lambda: seq.attention(q, k[:, :1].expand(20, 3, 16), v[:, :1].expand(20, 3, 16)), lambda: seq.attention(q, k, v[..., :8]),
                  lambda: seq.attention(q, k, v, window=-1), lambda: seq.attention(q, k, v, scale=0.0), lambda: seq.attention(q, k, v, scale=float("nan")),
                  lambda: seq.attention(q, k, v, offsets=n[:1]), lambda: seq.attention(q[None], k[None], v[None], offsets=n[:2]), lambda: seq.attention(q[:, 0], k[:, 0], v[:, 0]),
                  lambda: seq.attention(*(torch.zeros((4, 1, 129), device="cuda") for _ in range(3))),
                  lambda: seq.rotary(q[..., :15], None, p), lambda: seq.rotary(q, k[:10], p), lambda: seq.rotary(q, k, p[:10]), lambda: seq.rotary(q, k, p[:, :0]),
                  lambda: seq.rotary(q, k, p, sections=[8]), lambda: seq.rotary(q, k, p, sections=[9, -1]), lambda: seq.rotary(q, k, p, sections=[4, 3]), lambda: seq.rotary(q, k, p, base=0.0),
                  lambda: seq.rotary(q, k, p, base=float("inf")), lambda: seq.attention_step(q, k, v, cache, cache, n), lambda: seq.attention_step(q, k, v, cache[:, :, :1], other[:, :, :1], n),
                  lambda: seq.attention_step(q, k, v, cache, other, n[:3]), lambda: seq.attention_step(q, k, v, cache, other, n, window=-2),
                  lambda: seq.attention_step(q, k, v, cache[:, :1].expand(20, 5, 2, 16), other, n), lambda: seq.attention_step(q, k, v, cache.transpose(2, 3).contiguous().transpose(2, 3), other, n)]
    for i, call in enumerate(bad_values):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    bad_types = [lambda: seq.attention(q, k.half(), v), lambda: seq.attention(q.double(), k.double(), v.double()), lambda: seq.attention(q, k, v, offsets=n.long()), lambda: seq.attention(q, k, v, window=1.5),
                 lambda: seq.rotary(q, k, p.double()), lambda: seq.rotary(q, k, n.long()[:, None]), lambda: seq.attention_step(q, k, v, cache, other, n.long()), lambda: seq.attention(q, k, None)]
    for i, call in enumerate(bad_types):
        with pytest.raises(TypeError):
            call()
            pytest.fail(f"call {i} was not refused")
    wants = q.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="no gradient"):
        seq.attention_step(wants, k, v, cache, other, n)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q, torch.ones_like(q))
        for call in (lambda: seq.attention(dual, k, v), lambda: seq.rotary(dual, k, p), lambda: seq.attention_step(dual, k, v, cache, other, n)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_the_step_advances_the_caches_versions():
    from htgs_b200 import sequence as seq
    q, k, v, _ = tensors(3, 2, 2, 16, "bf16")
    keys, values = (torch.zeros((3, 5, 2, 16), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    before = keys._version, values._version
    seq.attention_step(q, k, v, keys, values, torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert keys._version > before[0] and values._version > before[1]
    with torch.inference_mode():
        inside = torch.zeros_like(keys), torch.zeros_like(values)
        seq.attention_step(q, k, v, *inside, torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert torch.equal(inside[0], keys)
