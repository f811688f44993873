"""The sequence operators in 64 bits, from their definitions, for the tests (numpy, small sizes)."""
import numpy as np

BLOCK = 128


def norm(x, weight, residual, eps):
    u = x + (0.0 if residual is None else residual)
    rho = 1.0 / np.sqrt(np.mean(u * u, axis=1, keepdims=True) + eps)
    return u * rho * weight, u, rho


def norm_backward(grad_y, grad_sum, u, rho, weight):
    unit, z = u * rho, grad_y * weight
    return rho * (z - unit * np.mean(z * unit, axis=1, keepdims=True)) + grad_sum, np.sum(grad_y * unit, axis=0)


def e4m3(v):
    """Nearest E4M3 value, ties to even; what is not finite becomes NaN."""
    finite = np.isfinite(v)
    w = np.where(finite, v, 0.0)
    exponent = np.maximum(np.frexp(w)[1] - 1, -6)
    step = np.exp2(exponent - 3.0)
    return np.where(finite, np.round(w / step) * step, np.nan)


def quantize(v, rows_per_scale=1):
    """(codes as values, exponents): the least e >= -127 with max |finite v| <= 448 * 2^e per block; 0 for zeros."""
    rows, width = v.shape
    shape = (-(-rows // rows_per_scale), -(-width // BLOCK))
    codes, exponents = np.zeros_like(v), np.zeros(shape, dtype=np.int64)
    for i in range(shape[0]):
        for j in range(shape[1]):
            at = (slice(i * rows_per_scale, (i + 1) * rows_per_scale), slice(j * BLOCK, (j + 1) * BLOCK))
            block = v[at]
            most = np.max(np.abs(block[np.isfinite(block)]), initial=0.0)
            e = 0
            if most > 0:
                e = int(np.floor(np.log2(most))) - 10
                while most > 448.0 * 2.0 ** e:
                    e += 1
                e = max(e, -127)
            exponents[i, j] = e
            codes[at] = e4m3(block * 2.0 ** -e)
    return codes, exponents


def dequantize(codes, exponents, rows_per_scale=1):
    scale = np.exp2(exponents.astype(np.float64)).repeat(rows_per_scale, 0).repeat(BLOCK, 1)
    return codes * scale[:codes.shape[0], :codes.shape[1]]


def gates(gate):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-gate)), 1.0 / (1.0 + np.exp(gate))


def spans(offsets, reverse):
    """(sequence, its rows in the order in which they are gone through)."""
    for s, (lo, hi) in enumerate(zip(offsets[:-1], offsets[1:])):
        yield s, (range(hi - 1, lo - 1, -1) if reverse else range(lo, hi))


def scan(x, gate, initial, offsets, reverse=False):
    a, rest = gates(gate)
    h, last = np.zeros_like(x), initial.copy()
    for s, rows in spans(offsets, reverse):
        for t in rows:
            last[s] = a[t] * last[s] + rest[t] * x[t]
            h[t] = last[s]
    return h, last


def scan_backward(x, gate, initial, offsets, grad_h, grad_last, reverse=False):
    a, rest = gates(gate)
    h, _ = scan(x, gate, initial, offsets, reverse)
    grad_x, grad_gate, grad_initial = np.zeros_like(x), np.zeros_like(x), grad_last.copy()
    for s, rows in spans(offsets, reverse):
        rows = list(rows)
        for i in range(len(rows) - 1, -1, -1):
            t = rows[i]
            before = h[rows[i - 1]] if i else initial[s]
            d = grad_h[t] + grad_initial[s]
            grad_x[t] = rest[t] * d
            grad_gate[t] = d * (before - x[t]) * a[t] * rest[t]
            grad_initial[s] = a[t] * d
    return grad_x, grad_gate, grad_initial
