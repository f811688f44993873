"""Rotary positions and attention in 64 bits, from their definitions, with bounds on what rounding may do, for the tests (torch on the CPU, small sizes)."""
import math

import torch

F = 2.0 ** -24
U = {"fp32": 2.0 ** -24, "fp16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"fp32": 2.0 ** -149, "fp16": 2.0 ** -24, "bf16": 2.0 ** -133}      # spacing of the smallest numbers
# A sum on the tensor cores may drop what lies below its largest term's last place instead of rounding: two F for each of its terms.
SUM = 2 * F


def angles(positions, sections, base):
    """[rows, pairs] angles."""
    speeds = [(axis, base ** (-i / n)) for axis, n in enumerate(sections) for i in range(n)]
    return torch.stack([positions[:, axis].double() * speed for axis, speed in speeds], dim=1)


def turn(x, angle, interleaved):
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else x.chunk(2, dim=-1)
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    parts = (a * c - b * s, a * s + b * c)
    return torch.stack(parts, dim=-1).flatten(-2) if interleaved else torch.cat(parts, dim=-1)


def turn_bound(x, kind, interleaved):
    """An angle is off by 2^-25 (it is rounded to 32 bits where it is at most an eighth of a turn, 0.79) and cosine and sine by two units in the last place: 2^-22 together, of both values of
    the pair; the two products and their sum by 3 F of them."""
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else x.chunk(2, dim=-1)
    both = (a.abs() + b.abs()) * (4 * F + 3 * F + U[kind]) + TINY[kind]
    return torch.stack((both, both), dim=-1).flatten(-2) if interleaved else torch.cat((both, both), dim=-1)


def visible(n, causal, window):
    away = torch.arange(n)[None] - torch.arange(n)[:, None]          # of column from row
    seen = torch.ones((n, n), dtype=torch.bool)
    if causal:
        seen &= away <= 0
    if window is not None:
        seen &= away.abs() <= window
    return seen


def attend(q, k, v, ends, causal, window, scale, kind, grad=None):
    """out (and, with `grad`, the gradients gq, gk, gv) in 64 bits and a bound for each, from 64-bit tensors [rows, heads, width].

    Where roundings happen: scores are sums of `width` products; an exponential is off by 2^-21 and what its argument is off by; weights and score gradients are rounded to the type (u);
    sums over n rows; the output is rounded to the type (u); the row's D is a product with that output."""
    u, rows, heads, width = U[kind], q.shape[0], q.shape[1], q.shape[2]
    group = heads // k.shape[1]
    out = {name: torch.zeros_like(t) for name, t in (("out", q), ("gq", q), ("gk", k), ("gv", v))}
    bound = {name: torch.zeros_like(t) for name, t in out.items()}
    for lo, hi in zip(ends[:-1], ends[1:]):
        n = hi - lo
        if n <= 0:
            continue
        seen = visible(n, causal, window)
        for h in range(heads):
            at = (slice(lo, hi), h)
            kat = (slice(lo, hi), h // group)
            Q, K, V = q[at], k[kat], v[kat]
            S = scale * (Q @ K.t())
            P = torch.softmax(torch.where(seen, S, -math.inf), dim=1)
            off = torch.where(seen, scale * (Q.abs() @ K.abs().t()) * (width * SUM + 8 * F), 0.0).amax(dim=1, keepdim=True) * 2 + 2.0 ** -20 + n * SUM       # of a weight, relative
            O = P @ V
            spread = P @ V.abs()
            O_bound = u * O.abs() + (u + off + n * SUM) * spread + TINY[kind]
            out["out"][at], bound["out"][at] = O, O_bound
            if grad is None:
                continue
            G = grad[at]
            D = (G * O).sum(dim=1, keepdim=True)
            dP = G @ V.t()
            dS = P * (dP - D)
            lse = torch.logsumexp(torch.where(seen, S, -math.inf), dim=1, keepdim=True)
            off = off + 4 * F * lse.abs()
            D_off = (G.abs() * (O_bound + width * SUM * O.abs())).sum(dim=1, keepdim=True)
            dS_off = P * ((off + u) * (dP - D).abs() + (G.abs() @ V.abs().t()) * width * SUM + D_off)
            few = n * SUM
            out["gq"][at] = scale * (dS @ K)
            bound["gq"][at] = scale * ((dS_off + few * dS.abs()) @ K.abs())
            out["gk"][kat] += scale * (dS.t() @ Q)
            bound["gk"][kat] += scale * ((dS_off + group * few * dS.abs()).t() @ Q.abs())
            out["gv"][kat] += P.t() @ G
            bound["gv"][kat] += ((off + u + group * few) * P).t() @ G.abs()
    for name in ("gq", "gk", "gv"):
        bound[name] += u * out[name].abs() + TINY[kind]
    return out, bound
