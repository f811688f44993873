"""GPU: the sequence operators (htgs_b200.sequence) against their 64-bit forms (sequence_reference.py).

Tolerances.  U[type] is the largest relative error of a rounding to the type (2^-9, 2^-12, 2^-25 would be half of a unit; the full 2^-8, 2^-11, 2^-24 is
used), and F = 2^-24 that of one 32-bit operation.  A 32-bit sum of n products is off by at most n * F times the sum of their magnitudes, whatever its order."""
import numpy as np
import pytest

import sequence_reference as ref

pytestmark = pytest.mark.gpu

F = 2.0 ** -24
U = {"fp32": 2.0 ** -24, "fp16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"fp32": 2.0 ** -149, "fp16": 2.0 ** -24, "bf16": 2.0 ** -133}      # spacing of the smallest numbers


@pytest.fixture(autouse=True, params=["pybind", "ctypes"])
def binding(request, monkeypatch):
    """Every test runs over the compiled extension module and over ctypes."""
    from htgs_b200 import _native
    if request.param == "ctypes":
        monkeypatch.setattr(_native, "_pybind_modules", False)
    elif not _native.pybind_modules():
        pytest.skip("htgs_b200/pybind modules not built (python -m htgs_b200.build)")


def dtype(name):
    import torch
    return {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}[name]


def draw(shape, seed, kind="fp32", scale=1.0, shift=0.0):
    import torch
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale + shift).to(dtype(kind)).cuda()


def f64(t):
    return t.detach().double().cpu().numpy()


def near(got, want, bound, what=""):
    got = f64(got)
    assert got.shape == want.shape, what
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    off = np.abs(np.nan_to_num(got) - np.nan_to_num(want))
    bad = off > np.nan_to_num(bound)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} values, worst {np.max(off[bad] / np.broadcast_to(bound, off.shape)[bad])} of the bound"


# ---- norm ------------------------------------------------------------------------------------------------------------------------


def norm_bounds(y, u, kind, width):
    # mean: (width + 2) F at most, of which rho gets half; rsqrt 2 F; two products 2 F
    return (U[kind] + (width / 2 + 8) * F) * np.abs(y) + TINY[kind], (U[kind] + F) * np.abs(u) + TINY[kind]


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 7), (9, 128), (5, 130), (17, 256), (8, 333), (33, 512), (6, 1000), (7, 1024), (4, 1032), (3, 2049), (2, 4104), (5, 8192)])
def test_norm_forward_and_backward(kind, rows, width):
    import torch
    from htgs_b200 import sequence as seq
    eps = 1e-5
    x, r, w = (draw(s, 10 + i, kind, sc, sh).requires_grad_(True) for i, (s, sc, sh) in enumerate((((rows, width), 1, 0), ((rows, width), 0.5, 0), ((width,), 0.2, 1))))
    gy, gs = draw((rows, width), 20, kind), draw((rows, width), 21, kind)
    y64, u64, rho = ref.norm(f64(x), f64(w), f64(r), eps)
    y_bound, s_bound = norm_bounds(y64, u64, kind, width)
    with torch.no_grad():
        y, s = seq.add_rms_norm(x, w, r, eps)
        near(y, y64, y_bound, "y")
        near(s, u64, s_bound, "stream")
    y2, s2 = seq.add_rms_norm(x, w, r, eps)
    assert torch.equal(y, y2) and torch.equal(s, s2)
    gx, gr, gw = torch.autograd.grad((y2, s2), (x, r, w), (gy, gs))
    gx64, gw64 = ref.norm_backward(f64(gy), f64(gs), u64, rho, f64(w))
    unit, z = np.abs(u64 * rho), np.abs(f64(gy) * f64(w))
    rough = U[kind] + (2 * width + 16) * F          # the stream is read back rounded; sums over the row
    bound = U[kind] * np.abs(gx64) + rough * (rho * (z + 2 * unit * np.mean(z * unit, axis=1, keepdims=True)) + np.abs(f64(gs))) + TINY[kind]
    near(gx, gx64, bound, "grad_x")
    assert torch.equal(gx, gr)
    near(gw, gw64, U[kind] * np.abs(gw64) + (U[kind] + (rows + width + 8) * F) * np.sum(np.abs(f64(gy)) * unit, axis=0) + TINY[kind], "grad_weight")


def test_norm_without_residual_views_and_parts_of_the_gradient():
    import torch
    from htgs_b200 import sequence as seq
    both = draw((6, 2, 96), 1, "bf16")
    x = both[:, 1]                                    # rows 192 apart
    w = draw((96,), 2, "bf16", 0.1, 1.0)
    y, s = seq.add_rms_norm(x, w)
    assert s is x
    y64, u64, rho = ref.norm(f64(x), f64(w), None, 1e-6)
    near(y, y64, norm_bounds(y64, u64, "bf16", 96)[0])
    flat, _ = seq.add_rms_norm(both, w)
    assert flat.shape == both.shape and torch.equal(flat[:, 1], y)
    odd = draw((5, 97), 3, "fp16")[:, 1:]             # rows that begin on 2 bytes only
    yo, _ = seq.add_rms_norm(odd, w.half())
    assert torch.equal(yo, seq.add_rms_norm(odd.contiguous(), w.half())[0])
    xg = draw((4, 40), 4).requires_grad_(True)
    wg = draw((40,), 5).requires_grad_(True)
    y, s = seq.add_rms_norm(xg, wg, xg.detach())
    s.sum().backward()                                # nothing reaches y
    assert torch.equal(xg.grad, torch.ones_like(xg)) and torch.equal(wg.grad, torch.zeros_like(wg))
    y, _ = seq.add_rms_norm(xg, wg)
    (gx,) = torch.autograd.grad(y, xg, torch.ones_like(y).t().contiguous().t())
    gx64, _ = ref.norm_backward(np.ones((4, 40)), 0.0, f64(xg), ref.norm(f64(xg), f64(wg), None, 1e-6)[2], f64(wg))
    near(gx, gx64, 1e-5 * np.ones((4, 40)))


def test_norm_of_zeros_large_values_and_nan():
    import torch
    from htgs_b200 import sequence as seq
    x = draw((4, 200), 6)
    x[0] = 0
    x[1] *= 1e15
    x[2, 3] = float("nan")
    x[3, 7] = float("inf")
    w = torch.ones(200, device="cuda")
    y, _ = seq.add_rms_norm(x, w, eps=1e-6)
    assert torch.equal(y[0], torch.zeros_like(y[0])) and abs(y[1].square().mean().item() - 1) < 1e-4
    assert torch.isnan(y[2]).all() and torch.isnan(y[3, 7]) and (y[3, :7] == 0).all()
    q, _ = seq.add_rms_norm_fp8(x, w)
    d = q.dequantize()
    assert (d[0] == 0).all() and torch.isnan(d[2]).all() and torch.isnan(d[3, 7]) and (d[3, :7] == 0).all()
    empty, _ = seq.add_rms_norm(torch.empty(0, 200, device="cuda"), w)
    assert empty.shape == (0, 200)
    none = torch.empty(0, 200, device="cuda", requires_grad=True)
    weight = w.clone().requires_grad_(True)
    y, _ = seq.add_rms_norm(none, weight)
    assert torch.equal(torch.autograd.grad(y.sum(), weight)[0], torch.zeros_like(w))


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 100), (5, 128), (9, 129), (4, 333), (2, 1024), (3, 1160), (2, 4100)])
def test_norm_into_8_bits(kind, rows, width):
    import torch
    from htgs_b200 import sequence as seq
    x, r, w = draw((rows, width), 30, kind), draw((rows, width), 31, kind), draw((width,), 32, kind, 0.2, 1.0)
    q, s = seq.add_rms_norm_fp8(x, w, r)
    y64, u64, _ = ref.norm(f64(x), f64(w), f64(r), 1e-6)
    got = f64(q.dequantize(torch.float32))
    scale = np.exp2(q.scales.view(torch.uint8).cpu().numpy().astype(np.float64) - 127).repeat(128, 1)[:, :width]
    # half a step: 2^-4 of the value, 2^-10 of the scale among the subnormals; and y's own error moves it by no more than itself
    near(q.dequantize(torch.float32), y64, np.maximum(np.abs(y64) * 2.0 ** -4, scale * 2.0 ** -10) + (width + 16) * F * np.abs(y64), "values")
    again, exponents = ref.quantize(got)
    assert np.array_equal(ref.dequantize(again, exponents), got)                # on the grid
    top = np.abs(y64).reshape(rows, width)
    for j in range(-(-width // 128)):
        most = top[:, j * 128:(j + 1) * 128].max(axis=1)
        assert (most <= 448 * scale[:, j * 128] * (1 + 1e-4)).all() and (most > 224 * scale[:, j * 128] * (1 - 1e-4)).all()
    assert torch.equal(s, seq.add_rms_norm(x, w, r)[1])


# ---- 8-bit matrices ------------------------------------------------------------------------------------------------------------------


def codes_of(q):
    """(codes as values, exponents) of an Fp8Matrix."""
    import torch
    return q.codes.contiguous().cpu().float().double().numpy(), q.scales.contiguous().view(torch.uint8).cpu().numpy().astype(np.int64) - 127


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("rows_per_scale", [1, 128])
@pytest.mark.parametrize("rows,width", [(1, 1), (2, 128), (130, 8), (127, 257), (129, 300), (5, 1024), (256, 384)])
def test_quantize_is_exact(kind, rows_per_scale, rows, width):
    import torch
    from htgs_b200 import sequence as seq
    x = draw((rows, width), rows + width, kind) * torch.exp(3 * torch.randn(width, device="cuda", generator=torch.Generator("cuda").manual_seed(1))).to(dtype(kind))
    x[0] = 0
    if rows > 3:
        x[2, 0], x[3, 0] = float("nan"), float("-inf")
        x[1, width // 2] = 1.75 * 2.0 ** 10            # the largest code of its block, or close to it
    for transpose in (False, True):
        q = seq.quantize_fp8(x, rows_per_scale, transpose)
        codes, exponents = codes_of(q)
        want = f64(x).T.copy() if transpose else f64(x)
        want_codes, want_exponents = ref.quantize(want, rows_per_scale)
        assert np.array_equal(exponents, want_exponents)
        assert np.array_equal(codes, want_codes, equal_nan=True)
        values = ref.dequantize(want_codes, want_exponents, rows_per_scale)
        assert np.array_equal(f64(q.dequantize(torch.float32)), values, equal_nan=True)
        assert np.array_equal(f64(q.dequantize()), values, equal_nan=True)


ANYWHERE = [("fp32", 20000, 45), ("bf16", 20000, 131), ("fp16", 6001, 250), ("fp32", 9001, 257), ("bf16", 6001, 383), ("fp16", 5001, 511), ("bf16", 4001, 514), ("fp32", 3001, 777),
            ("bf16", 3001, 1023), ("fp16", 1501, 1111), ("fp32", 1501, 1111), ("bf16", 1201, 1999), ("fp32", 701, 2051), ("bf16", 701, 5003), ("fp16", 301, 8191)]


@pytest.mark.parametrize("kind,rows,width", ANYWHERE)
def test_norm_of_many_rows_that_begin_anywhere(kind, rows, width):
    """Rows inside a matrix whose other columns are NaN, on addresses of every kind, and enough of them that a warp deals with several."""
    import torch
    from htgs_b200 import sequence as seq
    def inside(seed, scale):
        whole = torch.full((rows, width + 3), float("nan"), dtype=dtype(kind), device="cuda")
        whole[:, 1:-2] = draw((rows, width), seed, kind, scale)
        return whole[:, 1:-2]
    x, r, gy, gs = inside(70, 1.0), inside(71, 0.5), inside(72, 1.0), inside(73, 1.0)
    w = draw((width + 1,), 74, kind, 0.2, 1.0)[1:]
    y64, u64, rho = ref.norm(f64(x), f64(w), f64(r), 1e-6)
    y_bound, s_bound = norm_bounds(y64, u64, kind, width)
    x, r, w = (t.detach().requires_grad_(True) for t in (x, r, w))
    y, s = seq.add_rms_norm(x, w, r)
    near(y, y64, y_bound, "y")
    near(s, u64, s_bound, "stream")
    gx, gr, gw = torch.autograd.grad((y, s), (x, r, w), (gy, gs))
    gx64, gw64 = ref.norm_backward(f64(gy), f64(gs), u64, rho, f64(w))
    unit, z = np.abs(u64 * rho), np.abs(f64(gy) * f64(w))
    bound = U[kind] * np.abs(gx64) + (U[kind] + (2 * width + 16) * F) * (rho * (z + 2 * unit * np.mean(z * unit, axis=1, keepdims=True)) + np.abs(f64(gs))) + TINY[kind]
    near(gx, gx64, bound, "grad_x")
    near(gw, gw64, U[kind] * np.abs(gw64) + (U[kind] + (rows + width + 8) * F) * np.sum(np.abs(f64(gy)) * unit, axis=0) + TINY[kind], "grad_weight")
    with torch.no_grad():
        q, s8 = seq.add_rms_norm_fp8(x, w, r)
        scale = np.exp2(q.scales.view(torch.uint8).cpu().numpy().astype(np.float64) - 127).repeat(128, 1)[:, :width]
        near(q.dequantize(torch.float32), y64, np.maximum(np.abs(y64) * 2.0 ** -4, scale * 2.0 ** -10) + (width + 16) * F * np.abs(y64), "values")
        assert torch.equal(s8, s)


@pytest.mark.parametrize("kind,rows,width", ANYWHERE)
def test_quantize_many_rows_that_begin_anywhere(kind, rows, width):
    import torch
    from htgs_b200 import sequence as seq
    whole = torch.full((rows, width + 3), float("inf"), dtype=dtype(kind), device="cuda")
    whole[:, 1:-2] = draw((rows, width), 75, kind)
    x = whole[:, 1:-2]
    x[:, :5] *= 64
    x[rows // 2, width // 2], x[rows // 3, width - 1] = float("nan"), float("inf")
    for transpose in (False, True):
        q = seq.quantize_fp8(x, 1, transpose)
        codes, exponents = codes_of(q)
        want = ref.quantize(f64(x).T.copy() if transpose else f64(x))
        assert np.array_equal(exponents, want[1]) and np.array_equal(codes, want[0], equal_nan=True)
    q = seq.quantize_fp8(x)
    values = ref.dequantize(*ref.quantize(f64(x)))
    assert np.array_equal(f64(q.dequantize()), values, equal_nan=True)
    assert np.array_equal(f64(q.dequantize(torch.float32)), values, equal_nan=True)


def test_quantize_at_the_ends_of_the_range():
    import torch
    from htgs_b200 import sequence as seq
    x = torch.tensor([[3.4028234663852886e38, 1.0, 0, -1e38], [2.0 ** -149, 2.0 ** -140, 0, 0], [2.0 ** -126, -2.0 ** -127, 0, 0], [448.0, 449.0, -0.0, 1e-3],
                      [float("inf"), float("nan"), float("-inf"), 2.0]], device="cuda")
    q = seq.quantize_fp8(x)
    want = ref.quantize(f64(x))
    codes, exponents = codes_of(q)
    assert np.array_equal(exponents, want[1]) and np.array_equal(codes, want[0], equal_nan=True)
    with np.errstate(over="ignore"):                   # the largest float rounds up to 2^128, which 32 bits do not hold
        values = ref.dequantize(*want).astype(np.float32).astype(np.float64)
    assert np.array_equal(f64(q.dequantize(torch.float32)), values, equal_nan=True)


def product_bound(a, b, kind):
    exact = a @ b.T
    return exact, U[kind] * np.abs(exact) + (a.shape[1] + 2) * 2 * F * (np.abs(a) @ np.abs(b).T) + TINY[kind]     # 2 F: an addition that cuts off


SIZES = [(1, 1, 1), (1, 8, 16), (1, 1000, 1024), (3, 129, 127), (8, 256, 512), (9, 64, 130), (31, 72, 1100), (64, 136, 384), (100, 300, 640), (128, 128, 128), (129, 257, 129),
         (200, 520, 2056), (300, 1001, 392), (513, 96, 1536),
         (2, 130, 8200), (5, 33, 16500), (40, 300, 8200), (130, 140, 4100), (64, 64, 33000)]


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("rows,out,width", SIZES)
def test_product(kind, rows, out, width):
    import torch
    from htgs_b200 import sequence as seq
    x = draw((rows, width), 3, kind) * torch.exp(torch.randn(width, device="cuda", generator=torch.Generator("cuda").manual_seed(5))).to(dtype(kind))
    w = draw((out, width), 4, kind, width ** -0.5)
    wq = seq.quantize_fp8(w, 128)
    y = seq.fp8_matmul(x, wq)
    assert y.dtype == x.dtype
    a, b = ref.dequantize(*ref.quantize(f64(x))), ref.dequantize(*ref.quantize(f64(w), 128), 128)
    exact, bound = product_bound(a, b, kind)
    near(y, exact, bound, "x W^T")
    rows_scaled = seq.quantize_fp8(w, 1)              # a scale for each row of both
    near(seq.fp8_matmul(seq.quantize_fp8(x), rows_scaled, torch.float32), *product_bound(a, ref.dequantize(*ref.quantize(f64(w))), "fp32"), "row scales")
    near(seq.fp8_matmul(seq.quantize_fp8(x, 128), wq, torch.float32), *product_bound(ref.dequantize(*ref.quantize(f64(x), 128), 128), b, "fp32"), "block scales")


@pytest.mark.parametrize("rows,out,width", [(2500, 2301, 640), (40_001, 200, 129), (385, 4100, 1030)])
def test_product_of_many_tiles(rows, out, width):
    """More tiles than SMs, so that each block computes several; sizes that leave the last tiles ragged."""
    import torch
    from htgs_b200 import sequence as seq
    x, w = draw((rows, width), 3, "bf16"), draw((out, width), 4, "bf16", width ** -0.5)
    y = seq.fp8_matmul(x, seq.quantize_fp8(w, 128))
    a, b = ref.dequantize(*ref.quantize(f64(x))), ref.dequantize(*ref.quantize(f64(w), 128), 128)
    near(y, *product_bound(a, b, "bf16"))
    assert torch.equal(y, seq.fp8_matmul(x, seq.quantize_fp8(w, 128)))


def test_product_of_views_strides_and_empty_matrices():
    import torch
    from htgs_b200 import sequence as seq
    w = draw((40, 200), 1, "bf16", 0.1)
    wq = seq.quantize_fp8(w, 128)
    x = draw((6, 3, 200), 2, "bf16")
    y = seq.fp8_matmul(x, wq)
    assert y.shape == (6, 3, 40)
    assert torch.equal(seq.fp8_matmul(x[:, 1], wq), y[:, 1]) and torch.equal(seq.fp8_matmul(x.transpose(0, 1), wq), y.transpose(0, 1))
    odd = draw((7, 201), 3, "bf16")[:, 1:]
    assert torch.equal(seq.fp8_matmul(odd, wq), seq.fp8_matmul(odd.contiguous(), wq))
    assert seq.fp8_matmul(x[:0], wq).shape == (0, 3, 40)
    # codes and scales inside larger tensors, with other bytes (NaN codes) around them
    held = torch.full((40, 256), 0x7f, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    held[:, 16:216].copy_(wq.codes)
    scales = torch.full((1, 12), 0xff, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    scales[:, 4:6].copy_(wq.scales)
    again = seq.Fp8Matrix(held[:, 16:216], scales[:, 4:6], 128)
    assert torch.equal(seq.fp8_matmul(x, again), y)
    big = torch.cat([x.reshape(18, 200)] * 20)
    assert torch.equal(seq.fp8_matmul(big, again), seq.fp8_matmul(big, wq))
    zero = seq.quantize_fp8(torch.empty(5, 0, device="cuda"))
    assert torch.equal(seq.fp8_matmul(zero, seq.quantize_fp8(torch.empty(3, 0, device="cuda"), 128)), torch.zeros(5, 3, dtype=torch.bfloat16, device="cuda"))


def test_product_keeps_nan_to_its_row_and_column():
    import torch
    from htgs_b200 import sequence as seq
    for rows in (4, 300):
        x, w = draw((rows, 256), 1), draw((150, 256), 2)
        x[1, 5], w[7, 200], x[3, 9] = float("nan"), float("inf"), float("inf")
        y = seq.fp8_matmul(seq.quantize_fp8(x), seq.quantize_fp8(w, 1))
        want = torch.zeros(rows, 150, dtype=torch.bool, device="cuda")
        want[1] = want[3] = True
        want[:, 7] = True
        assert torch.equal(torch.isnan(y), want)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,out,width", [(1, 1, 1), (5, 130, 72), (200, 96, 130), (1000, 136, 256), (4097, 128, 64)])
def test_linear_gradients(kind, rows, out, width):
    import torch
    from htgs_b200 import sequence as seq
    x, w, gy = draw((rows, width), 1, kind).requires_grad_(True), draw((out, width), 2, kind, 0.1).requires_grad_(True), draw((rows, out), 3, kind)
    y = seq.fp8_linear(x, w)
    gx, gw = torch.autograd.grad(y, (x, w), gy)
    rowwise, tilewise = lambda v: ref.dequantize(*ref.quantize(v)), lambda v: ref.dequantize(*ref.quantize(v, 128), 128)  # noqa: E731
    near(y, *product_bound(rowwise(f64(x)), tilewise(f64(w)), kind), "y")
    near(gx, *product_bound(rowwise(f64(gy)), tilewise(f64(w)).T, kind), "grad_x")
    near(gw, *product_bound(rowwise(f64(gy).T.copy()), rowwise(f64(x).T.copy()), kind), "grad_weight")
    with torch.no_grad():
        assert torch.equal(seq.fp8_linear(x, w), y)
    only_w, = torch.autograd.grad(seq.fp8_linear(x.detach(), w), w, gy)
    only_x, = torch.autograd.grad(seq.fp8_linear(x, w.detach()), x, gy)
    assert torch.equal(only_w, gw) and torch.equal(only_x, gx)


# ---- recurrence --------------------------------------------------------------------------------------------------------------------------


def scan_bounds(x, g, initial, offsets, reverse, kind):
    """(h, last) and their bounds.  exp(-g) is off by (2 + 1.2 |g|) units of 2^-23 at most (the bound that CUDA gives for its fast exponential), a and 1 - a by
    that and 4 more; each step adds its own error to a times the last one's.  Twice that, for steps that are composed before they meet the state."""
    a, rest = ref.gates(g)
    step = 2 * (8 + 1.2 * np.abs(g)) * 2 * F
    h, last = ref.scan(x, g, initial, offsets, reverse)
    bound, bound_last = np.zeros_like(x), np.zeros_like(initial)
    for s, rows in ref.spans(offsets, reverse):
        size, off = np.abs(initial[s]), np.zeros(x.shape[1])
        for t in rows:
            off = a[t] * off + step[t] * (a[t] * size + rest[t] * np.abs(x[t]))
            size = a[t] * size + rest[t] * np.abs(x[t])
            bound[t] = off
        bound_last[s] = off
    return h, last, bound + U[kind] * np.abs(h) + TINY[kind], bound_last + 2 * F * np.abs(last)


def backward_bounds(x, g, initial, offsets, gh, gl, reverse, kind):
    """Bounds of the gradients by the same rule, along the recurrence of E and through h."""
    a, rest = ref.gates(g)
    step = 2 * (8 + 1.2 * np.abs(g)) * 2 * F
    h, _, h_bound, _ = scan_bounds(x, g, initial, offsets, reverse, "fp32")
    grads = ref.scan_backward(x, g, initial, offsets, gh, gl, reverse)
    bx, bg, bi = np.zeros_like(x), np.zeros_like(x), np.zeros_like(initial)
    for s, rows in ref.spans(offsets, reverse):
        rows = list(rows)
        size, off = np.abs(gl[s]), np.zeros(x.shape[1])
        for i in range(len(rows) - 1, -1, -1):
            t = rows[i]
            before, before_off = (h[rows[i - 1]], h_bound[rows[i - 1]]) if i else (initial[s], 0.0)
            size, off = size + np.abs(gh[t]), off + F * (size + np.abs(gh[t]))
            bx[t] = rest[t] * (off + step[t] * size)
            ar = a[t] * rest[t]
            bg[t] = ar * (np.abs(before) + np.abs(x[t])) * (off + 2 * step[t] * size) + ar * before_off * size
            size, off = a[t] * size, a[t] * off + step[t] * a[t] * size
        bi[s] = off
    return [(v, b + U[k] * np.abs(v) + TINY[k]) for v, b, k in zip(grads, (bx, bg, bi), (kind, kind, "fp32"))]


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("rows,width,offsets", [
    (1, 1, None), (1, 64, None), (2, 5, None), (15, 33, None), (16, 64, None), (127, 3, None), (128, 2, None), (129, 66, None), (300, 130, None), (1000, 7, None),
    (300, 8, [0, 0, 1, 1, 130, 128 + 128, 300, 300]), (257, 6, [0, 128, 256, 257]), (40, 34, [0, 40, 40]), (5, 4, [0, 1, 2, 3, 4, 5]), (500, 2, [0] * 40 + [499, 500])])
@pytest.mark.parametrize("reverse", [False, True])
def test_scan_forward_and_backward(kind, rows, width, offsets, reverse):
    import torch
    from htgs_b200 import sequence as seq
    ends = [0, rows] if offsets is None else offsets
    n = len(ends) - 1
    both = draw((rows, 2 * width), rows + width, kind)
    x, g = both[:, :width], both[:, width:]
    with torch.no_grad():
        g.mul_(3).add_(2)
        g[torch.rand(g.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(3)) < 0.02] = 40.0
        g[torch.rand(g.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(4)) < 0.02] = -60.0
    initial, gh, gl = draw((n, width), 5), draw((rows, width), 6, kind), draw((n, width), 7)
    off = None if offsets is None else torch.tensor(offsets, dtype=torch.int32, device="cuda")
    h64, last64, h_bound, last_bound = scan_bounds(f64(x), f64(g), f64(initial), ends, reverse, kind)
    h, last = seq.gated_scan(x, g, initial, off, reverse)
    near(h, h64, h_bound, "h")
    near(last, last64, last_bound, "last")
    leaves = [t.detach().requires_grad_(True) for t in (x, g, initial)]
    h2, last2 = seq.gated_scan(*leaves, off, reverse)
    assert torch.equal(h, h2) and torch.equal(last, last2)
    grads = torch.autograd.grad((h2, last2), leaves, (gh, gl))
    for got, (want, bound), name in zip(grads, backward_bounds(f64(x), f64(g), f64(initial), ends, f64(gh), f64(gl), reverse, kind), ("grad_x", "grad_gate", "grad_initial")):
        near(got, want, bound, name)
    again = torch.autograd.grad(seq.gated_scan(*leaves, off, reverse), leaves, (gh, gl))
    assert all(torch.equal(p, q) for p, q in zip(grads, again))


def test_scan_of_batches_defaults_and_parts_of_the_gradient():
    import torch
    from htgs_b200 import sequence as seq
    x, g = draw((3, 50, 20), 1), draw((3, 50, 20), 2, "fp32", 2.0, 1.0)
    h, last = seq.gated_scan(x, g)
    assert h.shape == x.shape and last.shape == (3, 20)
    for b in range(3):
        h64, last64, h_bound, last_bound = scan_bounds(f64(x[b]), f64(g[b]), np.zeros((1, 20)), [0, 50], False, "fp32")
        near(h[b], h64, h_bound, "h")
        near(last[b:b + 1], last64, last_bound, "last")
    packed, _ = seq.gated_scan(x.reshape(150, 20), g.reshape(150, 20), offsets=torch.tensor([0, 50, 100, 150], dtype=torch.int32, device="cuda"))
    assert torch.equal(packed, h.reshape(150, 20))
    strided, _ = seq.gated_scan(x.transpose(1, 2).contiguous().transpose(1, 2), g)
    assert torch.equal(strided, h)
    xg = x.clone().requires_grad_(True)
    h, last = seq.gated_scan(xg, g)
    from_last, = torch.autograd.grad(last.sum(), xg)
    h, last = seq.gated_scan(xg, g)
    from_h, = torch.autograd.grad(h[:, -1].sum(), xg)
    assert torch.allclose(from_last, from_h, rtol=1e-5, atol=1e-7)
    none, last = seq.gated_scan(torch.empty(0, 4, device="cuda"), torch.empty(0, 4, device="cuda"), torch.ones(2, 4, device="cuda"),
                                torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert none.shape == (0, 4) and torch.equal(last, torch.ones(2, 4, device="cuda"))


def test_scan_of_far_rows():
    """Rows further apart than the kernels reach are copied first; a single row's stride says nothing."""
    import torch
    from htgs_b200 import sequence as seq
    far = torch.empty(3, (1 << 22) + 8, device="cuda")
    far[:, :4] = draw((3, 4), 1)
    x, g = far[:, :4], draw((3, 4), 2)
    for n in (3, 1):
        h, last = seq.gated_scan(x[:n], g[:n])
        want, want_last = seq.gated_scan(x[:n].contiguous() + 0, g[:n] + 0)
        assert torch.equal(h, want) and torch.equal(last, want_last)


@pytest.mark.parametrize("reverse", [False, True])
def test_scan_keeps_nan_to_its_sequence_and_channel(reverse):
    import torch
    from htgs_b200 import sequence as seq
    offsets = [0, 100, 150, 400, 600]
    x, g = draw((600, 40), 1), draw((600, 40), 2, "fp32", 1.0, 1.0)
    initial = draw((4, 40), 3)
    x[120, 3], g[300, 5], initial[3, 7], x[50, 9] = float("nan"), float("nan"), float("inf"), float("inf")
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    leaves = [t.requires_grad_(True) for t in (x, g, initial)]
    h, last = seq.gated_scan(*leaves, off, reverse)
    gh = draw((600, 40), 4)
    gh[420, 11] = float("nan")
    grads = torch.autograd.grad((h, last), leaves, (gh, torch.ones_like(last)))
    with np.errstate(invalid="ignore"):
        h64, last64 = ref.scan(f64(x), f64(g), f64(initial), offsets, reverse)
        want = ref.scan_backward(f64(x), f64(g), f64(initial), offsets, f64(gh), np.ones((4, 40)), reverse)
    for got, w in zip((h, last, *grads), (h64, last64, *want)):
        got = f64(got)
        assert np.array_equal(np.isfinite(got), np.isfinite(w))


def test_scan_gradient_against_differences():
    """Directional derivatives of sum(weights * outputs), by differences of the GPU's own outputs: step 2^-6; the third derivative and 32-bit outputs
    leave about 1e-4 of the sum of magnitudes."""
    import torch
    from htgs_b200 import sequence as seq
    off = torch.tensor([0, 70, 70, 300], dtype=torch.int32, device="cuda")
    leaves = [draw((300, 6), 1).requires_grad_(True), draw((300, 6), 2, "fp32", 1.0, 1.0).requires_grad_(True), draw((3, 6), 3).requires_grad_(True)]
    wh, wl = draw((300, 6), 4), draw((3, 6), 5)
    value = lambda *v: sum((o.double() * w.double()).sum().item() for o, w in zip(seq.gated_scan(*v, off, True), (wh, wl)))  # noqa: E731
    grads = torch.autograd.grad(seq.gated_scan(*leaves, off, True), leaves, (wh, wl))
    for i, g in enumerate(grads):
        direction = draw(g.shape, 50 + i)
        eps = 2.0 ** -6
        moved = [[t.detach() + (eps * sign * direction if j == i else 0) for j, t in enumerate(leaves)] for sign in (1, -1)]
        numeric = (value(*moved[0]) - value(*moved[1])) / (2 * eps)
        assert abs(numeric - (g.double() * direction.double()).sum().item()) <= 1e-4 * (g.double() * direction.double()).abs().sum().item()


def test_norm_gradient_against_differences():
    import torch
    from htgs_b200 import sequence as seq
    leaves = [draw((20, 70), 1).requires_grad_(True), draw((70,), 2, "fp32", 0.2, 1.0).requires_grad_(True), draw((20, 70), 3).requires_grad_(True)]
    wy, ws = draw((20, 70), 4), draw((20, 70), 5)
    value = lambda *v: sum((o.double() * w.double()).sum().item() for o, w in zip(seq.add_rms_norm(*v), (wy, ws)))  # noqa: E731
    grads = torch.autograd.grad(seq.add_rms_norm(*leaves), leaves, (wy, ws))
    for i, g in enumerate(grads):
        direction = draw(g.shape, 50 + i)
        eps = 2.0 ** -7
        moved = [[t.detach() + (eps * sign * direction if j == i else 0) for j, t in enumerate(leaves)] for sign in (1, -1)]
        numeric = (value(*moved[0]) - value(*moved[1])) / (2 * eps)
        assert abs(numeric - (g.double() * direction.double()).sum().item()) <= 1e-4 * (g.double() * direction.double()).abs().sum().item()


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 65), (64, 1024), (1000, 33)])
def test_step(kind, rows, width):
    import torch
    from htgs_b200 import sequence as seq
    both = draw((rows, 2 * width), 1, kind, 2.0)
    held = draw((rows, width + 3), 2)
    state = held[:, :width]
    before = f64(held)
    h64, last64, h_bound, last_bound = scan_bounds(f64(both[:, :width]), f64(both[:, width:]), before[:, :width], list(range(rows + 1)), False, kind)
    h = seq.gated_scan_step(both[:, :width], both[:, width:], state)
    near(h, h64, h_bound, "h")
    near(state, last64, last_bound, "state")
    assert np.array_equal(f64(held[:, width:]), before[:, width:])
    assert seq.gated_scan_step(both[:0, :width], both[:0, width:], state[:0]).shape == (0, width)


def test_steps_follow_a_sequence():
    """A sequence's steps one by one are the sequence."""
    import torch
    from htgs_b200 import sequence as seq
    x, g = draw((30, 2, 16), 1), draw((30, 2, 16), 2)
    state = torch.zeros(2, 16, device="cuda")
    steps = torch.stack([seq.gated_scan_step(x[t], g[t], state) for t in range(30)])
    h, last = seq.gated_scan(x.transpose(0, 1), g.transpose(0, 1))
    assert torch.allclose(steps.transpose(0, 1), h, rtol=1e-5, atol=1e-6) and torch.allclose(state, last, rtol=1e-5, atol=1e-6)


# ---- all of them -----------------------------------------------------------------------------------------------------------------------------


def test_refusals():
    import torch
    from htgs_b200 import sequence as seq
    x, w = draw((4, 64), 1), draw((64,), 2)
    q = seq.quantize_fp8(x)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    for error, call in [
        (ValueError, lambda: seq.add_rms_norm(x, w[:63])), (TypeError, lambda: seq.add_rms_norm(x, w.half())), (TypeError, lambda: seq.add_rms_norm(x.double(), w.double())),
        (ValueError, lambda: seq.add_rms_norm(x, w, x[:3])), (ValueError, lambda: seq.add_rms_norm(x, w.cpu())), (TypeError, lambda: seq.add_rms_norm(x, w, x.bfloat16())),
        (ValueError, lambda: seq.add_rms_norm(draw((1, 8193), 1), draw((8193,), 1))), (ValueError, lambda: seq.add_rms_norm(x[:, :0], w[:0])),
        (RuntimeError, lambda: seq.add_rms_norm(x, w, eps=-1.0)), (RuntimeError, lambda: seq.add_rms_norm_fp8(x.clone().requires_grad_(True), w)),
        (ValueError, lambda: seq.quantize_fp8(x, 2)), (ValueError, lambda: seq.quantize_fp8(x[None], 1, True)), (TypeError, lambda: seq.quantize_fp8(x.int())),
        (TypeError, lambda: seq.Fp8Matrix(x, q.scales)), (TypeError, lambda: seq.Fp8Matrix(q.codes, x)), (ValueError, lambda: seq.Fp8Matrix(q.codes, q.scales, 64)),
        (ValueError, lambda: seq.Fp8Matrix(q.codes, q.scales[:3])), (ValueError, lambda: seq.Fp8Matrix(q.codes.t(), q.scales)),
        (ValueError, lambda: seq.Fp8Matrix(torch.zeros(4, 65, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, 1:], q.scales)),
        (ValueError, lambda: seq.Fp8Matrix(torch.zeros(4, 65, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, :64], q.scales)),
        (ValueError, lambda: seq.Fp8Matrix(q.codes[0], q.scales)),
        (ValueError, lambda: seq.fp8_matmul(x[:, :32], q)), (TypeError, lambda: seq.fp8_matmul(x, x)), (TypeError, lambda: seq.fp8_matmul(x, q, torch.float64)),
        (ValueError, lambda: seq.fp8_matmul(seq.quantize_fp8(x[:, :32]), q)), (RuntimeError, lambda: seq.fp8_matmul(x.clone().requires_grad_(True), q)),
        (ValueError, lambda: seq.fp8_linear(x, w)), (ValueError, lambda: seq.fp8_linear(x, draw((8, 32), 1))), (TypeError, lambda: seq.fp8_linear(x, draw((8, 64), 1, "bf16"))),
        (TypeError, lambda: q.dequantize(torch.float64)),
        (ValueError, lambda: seq.gated_scan(x, x[:3])), (TypeError, lambda: seq.gated_scan(x, x.half())), (ValueError, lambda: seq.gated_scan(x[0], x[0])),
        (ValueError, lambda: seq.gated_scan(x, x, torch.zeros(2, 64, device="cuda"))), (TypeError, lambda: seq.gated_scan(x, x, torch.zeros(1, 64, device="cuda").half())),
        (TypeError, lambda: seq.gated_scan(x, x, None, i32(0, 4).long())), (ValueError, lambda: seq.gated_scan(x, x, None, i32(0))),
        (ValueError, lambda: seq.gated_scan(x[None], x[None], None, i32(0, 4))), (ValueError, lambda: seq.gated_scan(x[:, :0], x[:, :0])),
        (ValueError, lambda: seq.gated_scan_step(x, x, torch.zeros(4, 63, device="cuda"))), (TypeError, lambda: seq.gated_scan_step(x, x, x.half())),
        (ValueError, lambda: seq.gated_scan_step(x, x, torch.zeros(64, 4, device="cuda").t())),
        (RuntimeError, lambda: seq.gated_scan_step(x, x.clone().requires_grad_(True), torch.zeros(4, 64, device="cuda")))]:
        with pytest.raises(error):
            call()


def test_other_streams_and_graphs():
    """Every operator runs on the current stream, and a captured graph of all of them gives the same bits on new inputs."""
    import torch
    from htgs_b200 import sequence as seq
    x, r, w = draw((700, 256), 1, "bf16"), draw((700, 256), 2, "bf16"), draw((256,), 3, "bf16")
    weight = seq.quantize_fp8(draw((512, 256), 4, "bf16", 0.06), 128)
    back = seq.quantize_fp8(draw((256, 256), 5, "bf16", 0.06), 128)

    def block():
        q, stream = seq.add_rms_norm_fp8(x, w, r)
        both = seq.fp8_matmul(q, weight)
        h, last = seq.gated_scan(both[:, :256], both[:, 256:])
        return stream, seq.fp8_matmul(h, back), last

    want = block()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = block()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = block()
    for seed in (8, 9):
        x.copy_(draw((700, 256), seed, "bf16"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(kept, block()))
