"""GPU: the paths through the attention kernels that ordinary inputs of ordinary sizes do not take."""
import math

import pytest
import torch

import attention_reference as ref
from test_gpu_attention import binding, draw, f64, near, tensors  # noqa: F401  (the fixture: every test runs over both bindings)
from test_gpu_attention_range import step_reference

pytestmark = pytest.mark.gpu

# ---- heads of more than 64: two tiles of queries to a block, and a backward pass of their own -----------------------------------------------


@pytest.mark.parametrize("width,heads,key_heads", [(72, 2, 1), (96, 3, 3), (128, 4, 2)])
@pytest.mark.parametrize("kind", ["fp16", "bf16"])
def test_rows_of_no_sequence_beside_wide_heads(kind, width, heads, key_heads):
    from htgs_b200 import sequence as seq
    q, k, v, grad = tensors(700, heads, key_heads, width, kind)
    for t in (q, k, v, grad):
        t[:37] = float("nan")
        t[600:] = float("inf")
    ends = [37, 100, 100, 420, 600]
    offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
    for causal, window in ((True, None), (False, 90), (False, None)):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = seq.attention(*leaves, offsets=offsets, causal=causal, window=window)
        grads = torch.autograd.grad(out, leaves, grad)
        inner = [f64(t)[37:600] for t in (q, k, v, grad)]
        want, bound = ref.attend(*inner[:3], [e - 37 for e in ends], causal, window, width ** -0.5, kind, inner[3])
        for name, t in zip(("out", "gq", "gk", "gv"), (out, *grads)):
            near(t[37:600], want[name], bound[name], name)
            assert not t[:37].any() and not t[600:].any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("which", ["all", "q", "k", "v", "grad"])
@pytest.mark.parametrize("width,heads,key_heads,window", [(72, 2, 1, 300), (128, 2, 2, 150)])
@pytest.mark.parametrize("kind", ["fp16", "bf16"])
def test_what_a_row_of_wide_heads_does_not_see_does_not_reach_it(kind, width, heads, key_heads, window, which, bad):
    """Some rows of one of the inputs, or of all, are not finite: the rows that do not see them, and the keys that no such row sees, come out as if they were."""
    from htgs_b200 import sequence as seq
    rows, ends, low, high = 900, [0, 60, 790, 900], 400, 440
    parts = dict(zip(("q", "k", "v", "grad"), tensors(rows, heads, key_heads, width, kind)))
    offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
    spoilt = {name: t.clone() for name, t in parts.items()}
    for name, t in spoilt.items():
        if which in ("all", name):
            t[low:high, :, 3] = bad
            t[low + 7, :, width - 1] = bad
    for causal in (True, False):
        want, bound = ref.attend(*(f64(parts[n]) for n in "qkv"), ends, causal, window, width ** -0.5, kind, f64(parts["grad"]))
        leaves = [spoilt[n].clone().requires_grad_(True) for n in "qkv"]
        out = seq.attention(*leaves, offsets=offsets, causal=causal, window=window)
        grads = torch.autograd.grad(out, leaves, spoilt["grad"])
        i = torch.arange(rows)
        sees = (i >= low - (0 if causal else window)) & (i < high + window) & (i >= 60) & (i < 790)          # rows that see a spoilt one, or are one
        seen = (i >= low - window) & (i < high + (0 if causal else window)) & (i >= 60) & (i < 790)          # keys that a spoilt row sees
        # a key's gradient is also of the rows that see it, which a spoilt key may have reached through their sums
        reached = torch.zeros(rows, dtype=torch.bool)
        for j in range(60, 790):
            first, last = max(60, j if causal else j - window), min(789, j + window)
            reached[j] = sees[first:last + 1].any()
        for name, t, touched in (("out", out, sees), ("gq", grads[0], sees), ("gk", grads[1], reached | seen), ("gv", grads[2], reached | seen)):
            clean = ~touched
            assert clean.sum() > 100
            near(t[clean.cuda()], want[name][clean], bound[name][clean], f"{name}, causal {causal}")
        if which in ("all", "q", "k") and not math.isinf(bad):
            assert out[low:high].isnan().any()


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_scores_of_wide_heads_that_are_not_finite(kind, bad):
    """One key's score is not finite, in either tile of queries and whichever column of a tile of keys."""
    from htgs_b200 import sequence as seq
    rows, width = 700, 128
    q, k, v, _ = tensors(rows, 1, 1, width, kind)
    q[..., 0] = 1.0
    want, bound = ref.attend(f64(q), f64(k), f64(v), [0, rows], True, None, width ** -0.5, kind)
    for j in (0, 1, 77, 127, 128, 255, 256, 300, 511, 698):
        spoilt = k.clone()
        spoilt[j, 0, 0] = bad
        out = seq.attention(q, spoilt, v, causal=True)
        near(out[:j], want["out"][:j], bound["out"][:j], f"{j}: rows before it")
        assert out[j:].isnan().all(), j


# ---- a step whose splits a second kernel joins ------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("batch,capacity,heads,key_heads,width,window", [(1, 40000, 8, 2, 64, None), (3, 33000, 4, 4, 128, None), (2, 50001, 5, 5, 32, 20000), (40, 3000, 8, 2, 40, None), (2, 30000, 40, 2, 72, None)])
def test_a_step_of_many_splits(batch, capacity, heads, key_heads, width, window, kind):
    """Long caches, filled from not at all to the last row; what lies behind a sequence's rows is not finite."""
    import ctypes
    from htgs_b200 import _native, sequence as seq
    g = torch.Generator(device="cuda").manual_seed(1)
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda").to({"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}[kind])  # noqa: E731
    q, k, v = normal(batch, heads, width), normal(batch, key_heads, width), normal(batch, key_heads, width)
    keys, values = normal(batch, capacity, key_heads, width), normal(batch, capacity, key_heads, width)
    fills = [capacity - 1, capacity // 3, 0, 129, -1, capacity, capacity // 2 + 1, 127, 4097 % capacity]
    lengths = [fills[b % len(fills)] for b in range(batch)]
    for b, n in enumerate(lengths):
        keys[b, max(n, 0):], values[b, max(n, 0):] = float("nan"), float("inf")
    step = _native.HtgsAttentionStep(*(t.data_ptr() for t in (q, k, v, keys, values, q)), q.stride(0), k.stride(0), v.stride(0), q.stride(1), k.stride(1), v.stride(1), keys.stride(0), values.stride(0),
                                     keys.stride(1), values.stride(1), keys.stride(2), values.stride(2), capacity, batch, heads, key_heads, width, {"fp32": 0, "fp16": 1, "bf16": 2}[kind],
                                     -1 if window is None else window, 0.1)
    assert _native.lib().htgs_attention_step_workspace_bytes(ctypes.byref(step)) > 0          # the second kernel has something to join
    before = keys.clone(), values.clone()
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = seq.attention_step(q, k, v, keys, values, n, window=window)
    for b, length in enumerate(lengths):
        if 0 <= length < capacity:
            before[0][b, length], before[1][b, length] = k[b], v[b]
            low = 0 if window is None else max(0, length - window)
            near(out[b], *step_reference(f64(q[b]), f64(keys[b, low:length + 1]), f64(values[b, low:length + 1]), kind), f"sequence {b}")
        else:
            assert out[b].isnan().all() if length >= capacity else not out[b].any()
    assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip((keys, values), before))
    again = seq.attention_step(q, k, v, keys, values, n, window=window)
    assert torch.equal(out.nan_to_num(7.0), again.nan_to_num(7.0))


# ---- heads and caches that begin anywhere ---------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("width", [1, 3, 8, 12, 24, 64])
def test_heads_and_caches_that_begin_on_any_value(width, kind):
    """Queries, keys, values, output gradients and both caches 0 to 5 values behind a multiple of 16 bytes, rows and heads an odd or even number of values apart: within the bounds, as their copies."""
    from htgs_b200 import sequence as seq

    def placed(shape, seed, begin, between):
        pitch = width + between
        row = shape[-2] * pitch + between
        wide = draw((shape[:-2].numel() * row + begin,), seed, kind)
        strides = [row]
        for n in reversed(shape[1:-2]):
            strides.insert(0, strides[0] * n)
        return wide.as_strided(shape, (*strides, pitch, 1), begin)

    rows, heads, key_heads, batch, capacity = 70, 4, 2, 3, 40
    for begin in range(6):
        for between in (0, 1, 2):
            q, k, v, grad = (placed(torch.Size((rows, n, width)), i, begin, between) for i, n in enumerate((heads, key_heads, key_heads, heads)))
            leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
            out = seq.attention(*leaves, causal=True)
            grads = torch.autograd.grad(out, leaves, grad)
            want, bound = ref.attend(f64(q), f64(k), f64(v), [0, rows], True, None, width ** -0.5, kind, f64(grad))
            for name, t in zip(("out", "gq", "gk", "gv"), (out, *grads)):
                near(t, want[name], bound[name], f"{name}, {begin} and {between}")
            keys, values = (placed(torch.Size((batch, capacity, key_heads, width)), 5 + i, begin, between) for i in range(2))
            lengths = torch.tensor([0, 17, capacity - 1], dtype=torch.int32, device="cuda")
            out = seq.attention_step(q[:batch], k[:batch], v[:batch], keys, values, lengths)
            for b, n in enumerate(lengths.tolist()):
                assert torch.equal(keys[b, n], k[b]) and torch.equal(values[b, n], v[b])
                near(out[b], *step_reference(f64(q[b]), f64(keys[b, :n + 1]), f64(values[b, :n + 1]), kind), f"sequence {b}, {begin} and {between}")
