"""GPU: the gradients of attention are as exact as the kernels' roundings allow, where one rounding more would show.

D of a row is the product of its output's gradient with its output; it goes into the gradient of each of the row's scores, whose sum over the row is zero.  So where keys have a common part, an error of D
or of the score gradients meets that part, and what it ought to be does not.  The forward pass therefore keeps what the output's rounding took away (all 16-bit heads), and score gradients go into their sums
in two parts (heads of up to 64).  attention_reference.attend bounds each rounding by its largest and cannot tell whether one is there; here the kernels are compared with emulations of
themselves in 64 bits, with the same roundings and with one more."""
import math

import pytest
import torch

import attention_reference as ref
from test_gpu_attention import DTYPES, binding, draw, f64  # noqa: F401  (the fixture: every test runs over both bindings)


def emulate(q, k, v, grad, kind, kept_rest, two_parts):
    """(gq, gk) of one sequence and head in 64 bits but for these roundings: weights, the output's rounding (in D, unless what it takes away is kept: then of that), score gradients (in one part or
    two) and the results."""
    rounded = lambda t: t.to(DTYPES[kind]).double()  # noqa: E731
    scale = q.shape[1] ** -0.5
    # weights carry powers of two in the kernels: in fp16 no small ones are lost, so they are lifted here too
    P = torch.softmax(scale * q @ k.t(), dim=1)
    lift = 2.0 ** 14 if kind == "fp16" else 1.0
    O = rounded(P * lift) / lift @ v
    D = rounded(O) + (rounded(O - rounded(O)) if kept_rest else 0.0)
    dS = P * (grad @ v.t() - (grad * D).sum(dim=1, keepdim=True))
    lift = 2.0 ** (13 - math.floor(math.log2(dS.abs().max()))) if kind == "fp16" else 1.0
    parts = rounded(dS * lift)
    if two_parts:
        parts = parts + rounded(dS * lift - parts)
    parts = parts / lift
    return rounded(scale * parts @ k), rounded(scale * parts.t() @ q)


def inputs(width, kind, common, rows=400):
    """One head; with `common`, keys and values have a common part."""
    q, k, v, grad = (draw((rows, 1, width), seed, kind) for seed in (1, 2, 3, 4))
    return (q, k + 8, v + 4, grad) if common else (q, k, v, grad)


def errors(parts, kind, got=None, **how):
    q, k, v, grad = (f64(t)[:, 0] for t in parts)
    want, _ = ref.attend(*(t[:, None] for t in (q, k, v)), [0, q.shape[0]], False, None, q.shape[1] ** -0.5, kind, grad[:, None])
    got = emulate(q, k, v, grad, kind, **how) if got is None else got
    return [float((g - want[name].squeeze(1)).norm() / want[name].norm()) for g, name in zip(got, ("gq", "gk"))]


@pytest.mark.gpu
@pytest.mark.parametrize("common", [True, False])
@pytest.mark.parametrize("width,kind", [(32, "bf16"), (64, "bf16"), (64, "fp16"), (128, "bf16"), (96, "fp16")])
def test_gradients_without_the_roundings_that_are_kept_out(width, kind, common):
    """The kernels' error is nearer, by its logarithm, to that of their own roundings than to that with one more: with common parts the output's in D, without them the score gradients'."""
    from htgs_b200 import sequence as seq
    narrow = width <= 64
    if not (common or narrow):
        pytest.skip("score gradients of wider heads are in one part")
    parts = inputs(width, kind, common)
    leaves = [t.requires_grad_(True) for t in parts[:3]]
    got = torch.autograd.grad(seq.attention(*leaves), leaves[:2], parts[3])
    off = errors(parts, kind, [f64(g)[:, 0] for g in got])
    own = errors(parts, kind, kept_rest=True, two_parts=narrow)
    more = errors(parts, kind, kept_rest=not common, two_parts=narrow and common)
    for i, name in enumerate(("gq", "gk")):
        assert off[i] <= math.sqrt(own[i] * more[i]), f"{name}: off by {off[i]:.2e} of its size, {own[i]:.2e} by its own roundings and {more[i]:.2e} with one more"
