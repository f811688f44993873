"""GPU: attention over values near the largest of their type, whose sums before they are divided by the weights' sum must not become infinite."""
import pytest
import torch

import attention_reference as ref
from test_gpu_attention import binding, draw, f64, near  # noqa: F401  (the fixture: every test runs over both bindings)

pytestmark = pytest.mark.gpu

# seven eighths of 2^126 (7.4e37): twice that is a 32-bit number, eight times is not
LARGE = 0.875 * 2.0 ** 126


def step_reference(q, k, v, kind):
    """The attention of one row of queries [heads, width] over all rows of k and v, and the bound of attention_reference.attend for it."""
    u, n, width, group = ref.U[kind], k.shape[0], q.shape[1], q.shape[0] // k.shape[1]
    k, v = k.repeat_interleave(group, dim=1), v.repeat_interleave(group, dim=1)
    S, largest = (torch.einsum("hd,nhd->hn", a, b) * width ** -0.5 for a, b in ((q, k), (q.abs(), k.abs())))
    P = torch.softmax(S, dim=1)
    off = largest.amax(dim=1, keepdim=True) * (width * ref.SUM + 8 * ref.F) * 2 + 2.0 ** -20 + n * ref.SUM
    want, spread = torch.einsum("hn,nhd->hd", P, v), torch.einsum("hn,nhd->hd", P, v.abs())
    return want, u * want.abs() + (u + off + n * ref.SUM) * spread + ref.TINY[kind]


def values(rows, heads, width, kind, seed):
    """Of one sign in each column, and a factor of two apart."""
    g = torch.Generator().manual_seed(seed)
    v = (1 + torch.rand((rows, heads, width), generator=g)) * (LARGE / 2) * torch.where(torch.arange(width) % 2 == 0, 1.0, -1.0)
    return v.to({"fp32": torch.float32, "bf16": torch.bfloat16}[kind]).cuda()


def rising(rows, heads, key_heads, width, kind):
    """Queries and keys whose scores rise along the rows by about 8 in all, so that weights go on past an early maximum."""
    q, k = draw((rows, heads, width), 1, kind, 0.1), draw((rows, key_heads, width), 2, kind, 0.1)
    q[..., 0] = 1.0
    k[..., 0] = torch.linspace(-3.0, 2.5, rows).to(k.dtype).cuda()[:, None] * width ** 0.5
    return q, k


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("flat", [True, False])
@pytest.mark.parametrize("rows,heads,key_heads,width,causal,window,ends", [(1500, 2, 1, 64, True, None, None), (900, 1, 1, 128, False, 300, None), (1100, 2, 2, 24, False, None, [0, 5, 5, 700, 1100]),
                                                                          (400, 1, 1, 13, True, 100, None)])
def test_sums_of_large_values_stay_finite(rows, heads, key_heads, width, causal, window, ends, flat, kind):
    """Every result is at most the largest value, and finite; the gradients, with an output gradient that keeps them in range, are right too."""
    from htgs_b200 import sequence as seq
    q, k = rising(rows, heads, key_heads, width, kind)
    if flat:
        q, k = torch.zeros_like(q), torch.zeros_like(k)
    v, grad = values(rows, key_heads, width, kind, 3), draw((rows, heads, width), 4, kind, 2.0 ** -20)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    offsets = None if ends is None else torch.tensor(ends, dtype=torch.int32, device="cuda")
    out = seq.attention(*leaves, offsets=offsets, causal=causal, window=window)
    with torch.no_grad():
        inference = seq.attention(*leaves, offsets=offsets, causal=causal, window=window)
    grads = torch.autograd.grad(out, leaves, grad)
    want, bound = ref.attend(*(f64(t) for t in leaves), ends or [0, rows], causal, window, width ** -0.5, kind, f64(grad))
    for name, t in zip(("out", "out", "gq", "gk", "gv"), (out, inference, *grads)):
        assert want[name].abs().max() < 2.0 ** 127
        near(t, want[name], bound[name], name)


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_small_values_keep_their_bits(kind):
    """The other end: values of 2^-90, 2000 of them to a row, as far above the smallest normal number as the weights go below 1."""
    from htgs_b200 import sequence as seq
    rows, width = 2000, 64
    q, k = rising(rows, 1, 1, width, kind)
    v = draw((rows, 1, width), 3, kind) * 2.0 ** -90
    out = seq.attention(q, k, v)
    want, bound = ref.attend(f64(q), f64(k), f64(v), [0, rows], False, None, 0.125, kind)
    near(out, want["out"], bound["out"])


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("flat", [True, False])
@pytest.mark.parametrize("batch,capacity,heads,key_heads,width,window", [(1, 70, 2, 1, 64, None), (2, 1500, 4, 2, 128, None), (1, 40000, 4, 1, 64, None), (3, 900, 1, 1, 13, None), (2, 60000, 2, 2, 32, 5000),
                                                                        (9, 6000, 16, 8, 128, None)])
def test_a_step_over_large_values_stays_finite(batch, capacity, heads, key_heads, width, window, flat, kind):
    """Alone, in a cluster of splits and in splits that a second kernel joins."""
    from htgs_b200 import sequence as seq
    q, k, v = draw((batch, heads, width), 1, kind), draw((batch, key_heads, width), 2, kind), values(batch, key_heads, width, kind, 3)
    if flat:
        q.zero_()
    keys = draw((batch, capacity, key_heads, width), 4, kind)
    vals = values(batch * capacity, key_heads, width, kind, 5).view(batch, capacity, key_heads, width)
    lengths = torch.tensor([capacity - 1 - 3 * b for b in range(batch)], dtype=torch.int32, device="cuda")
    out = seq.attention_step(q, k, v, keys, vals, lengths, window=window)
    for b, n in enumerate(lengths.tolist()):
        low = 0 if window is None else max(0, n - window)
        want, bound = step_reference(f64(q[b]), f64(keys[b, low:n + 1]), f64(vals[b, low:n + 1]), kind)
        near(out[b], want, bound)
