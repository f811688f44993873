"""GPU: the forms of the sequence operators that large sizes take, chosen from the launchers' rules - pairs of SMs, column tiles of 224 and sums split in two in the
8-bit product, persistent kernels that go round more than once on aligned rows - against 64-bit forms (elementary torch operations in double on the GPU).

Tolerances: as in test_gpu_sequence.py, with the sums' real depths.  A row's statistic is a sum of at most 64 terms in a lane (32 columns of a warp), five steps between
lanes and eight warps: 77 F, of which rho gets half, besides the mean's and the root's own 4 F.  A column of grad_weight is summed over the rows of a block, then over
blocks by 32 slices of up to 38 in four parts and five steps: with up to 40 rows of a block 80 F and rho's.  Outputs are rounded once."""
import numpy as np
import pytest

import sequence_reference as ref
from test_gpu_sequence import ANYWHERE, F, TINY, U, binding, codes_of, draw, dtype, f64, near, product_bound  # noqa: F401

pytestmark = pytest.mark.gpu

RHO = (77 / 2 + 4) * F


def close(got, want, bound, what=""):
    import torch
    assert got.shape == want.shape, what
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    over = ((got.double() - want).abs() / bound).nan_to_num()
    assert over.max().item() <= 1, f"{what}: worst {over.max().item()} of the bound"


# ---- product -----------------------------------------------------------------------------------------------------------------------


def form_of_product(rows, out, width):
    """The launcher's rule (matmul_typed), so that a change of it cannot drop a form from these tests unseen."""
    if rows <= 8:
        return "rows"
    up = lambda n, d: -(-n // d)  # noqa: E731
    tiles = lambda r, c: up(rows, r) * up(out, c)  # noqa: E731
    blocks, parts = up(width, 128), 1
    while parts < 8 and blocks >= 32 and blocks >= 16 * parts and tiles(128, 128) * parts * 2 <= (148 if parts < 4 else 64):
        parts *= 2
    if parts > 1:
        return f"split {parts}"
    if tiles(256, 224) >= 16 * 74:
        return "pair"
    return "single 128" if up(tiles(128, 128), 148) * 128 <= up(tiles(128, 224), 148) * 224 else "single 224"


def decoded(q):
    """An Fp8Matrix in 64 bits, by torch."""
    import torch
    scales = torch.exp2(q.scales.contiguous().view(torch.uint8).double() - 127).repeat_interleave(q.rows_per_scale, 0).repeat_interleave(128, 1)
    return q.codes.float().double() * scales[:q.codes.shape[0], :q.codes.shape[1]]


@pytest.mark.parametrize("form,rows,out,width", [
    ("pair", 75_900, 1001, 136),          # the last pair's second block has no rows; rows of the output begin anywhere
    ("pair", 76_031, 1008, 300),          # it lacks one; 1008 = 4 * 224 + 112
    ("pair", 30_209, 2240, 1030),         # one row in the last pair; whole column tiles
    ("pair", 303_000, 130, 64),           # the second half of the rows of b is nearly empty
    ("single 224", 12_795, 210, 300), ("single 224", 12_800, 224, 128), ("single 224", 6_300, 447, 1000),
    ("split 2", 7_677, 100, 4091), ("split 2", 2_500, 384, 4096), ("split 4", 1_000, 250, 6000), ("split 8", 250, 300, 16_500),
    ("single 128", 300, 520, 2056), ("single 128", 40_001, 200, 129)])
@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("rows_per_scale", [1, 128])
def test_product_in_each_form(form, rows, out, width, kind, rows_per_scale):
    import torch
    from htgs_b200 import sequence as seq
    assert form_of_product(rows, out, width) == form
    g = torch.Generator("cuda").manual_seed(rows + out)
    x = torch.randn((rows, width), device="cuda", generator=g) * torch.exp(torch.randn(width, device="cuda", generator=g)) * torch.exp(torch.randn((rows, 1), device="cuda", generator=g))
    w = torch.randn((out, width), device="cuda", generator=g) * width ** -0.5 * torch.exp(torch.randn((out, 1), device="cuda", generator=g))
    a, b = seq.quantize_fp8(x), seq.quantize_fp8(w, rows_per_scale)
    a64, b64 = decoded(a), decoded(b)
    y = seq.fp8_matmul(a, b, dtype(kind))
    exact, sizes = a64 @ b64.t(), a64.abs() @ b64.abs().t()
    close(y, exact, U[kind] * exact.abs() + (width + 2) * 2 * F * sizes + TINY[kind])      # product_bound
    assert torch.equal(y, seq.fp8_matmul(a, b, dtype(kind)))


def test_forms_of_the_product():
    """What a whole scene's projection and a training step's take."""
    assert form_of_product(100_000, 2048, 1024) == "pair"
    assert form_of_product(512, 1024, 32_768) == "split 4" and form_of_product(32_768, 1024, 512) == "single 128"


@pytest.mark.parametrize("rows,out,width", [(5, 130, 72), (200, 96, 130), (1000, 136, 256), (4097, 128, 64)])
def test_linear_gradients_in_fp16(rows, out, width):
    import torch
    from htgs_b200 import sequence as seq
    x, w, gy = draw((rows, width), 1, "fp16").requires_grad_(True), draw((out, width), 2, "fp16", 0.1).requires_grad_(True), draw((rows, out), 3, "fp16")
    y = seq.fp8_linear(x, w)
    gx, gw = torch.autograd.grad(y, (x, w), gy)
    rowwise, tilewise = lambda v: ref.dequantize(*ref.quantize(v)), lambda v: ref.dequantize(*ref.quantize(v, 128), 128)  # noqa: E731
    near(y, *product_bound(rowwise(f64(x)), tilewise(f64(w)), "fp16"), "y")
    near(gx, *product_bound(rowwise(f64(gy)), tilewise(f64(w)).T, "fp16"), "grad_x")
    near(gw, *product_bound(rowwise(f64(gy).T.copy()), rowwise(f64(x).T.copy()), "fp16"), "grad_weight")


# ---- norm --------------------------------------------------------------------------------------------------------------------------


# 16-byte groups in narrow and wide blocks, 4-byte pairs, single values of narrow rows; enough rows that a block goes round several times, and a remainder
ALIGNED = [("bf16", 5003, 1024), ("fp16", 9001, 512), ("fp32", 5003, 512), ("fp32", 20_001, 100), ("bf16", 3001, 2048), ("fp32", 1201, 4096), ("fp16", 601, 8192), ("fp16", 25_001, 250),
           ("bf16", 7001, 1002), ("fp32", 20_001, 101), ("bf16", 30_001, 33)]


@pytest.mark.parametrize("kind,rows,width", ALIGNED + ANYWHERE)
def test_norm_gradients_lose_no_row(kind, rows, width):
    """grad_x of every row, and grad_weight from some rows at a time: the gradients of the others are zero, so that one that were lost or counted twice would show, in
    16-bit outputs too."""
    import torch
    from htgs_b200 import sequence as seq
    eps = 1e-6
    x, r, gs = draw((rows, width), 1, kind), draw((rows, width), 2, kind, 0.5), draw((rows, width), 4, kind)
    w, gy = draw((width,), 5, kind, 0.2, 1.0), draw((rows, width), 3, kind)
    if (kind, rows, width) in ANYWHERE:                    # rows on addresses of every kind
        x, r, gs, gy = (torch.nn.functional.pad(t, (1, 2), value=float("nan"))[:, 1:-2] for t in (x, r, gs, gy))
    leaves = [t.detach().requires_grad_(True) for t in (x, w, r)]
    y, s = seq.add_rms_norm(*leaves, eps)
    u = x.double() + r.double()
    rho = (u.square().mean(dim=1, keepdim=True) + eps).rsqrt()
    unit, wd = u * rho, w.double()
    close(y, unit * wd, (U[kind] + RHO + 4 * F) * (unit * wd).abs() + TINY[kind], "y")

    def gradients(gy, gs):
        gx, gw, gr = torch.autograd.grad((y, s), leaves, (gy, gs), retain_graph=True)
        assert torch.equal(gx, gr)
        z, terms = gy.double() * wd, gy.double() * unit
        slope = (z * unit).mean(dim=1, keepdim=True)
        want = rho * (z - unit * slope) + gs.double()
        rough = rho * (z.abs() + 2 * unit.abs() * (z * unit).abs().mean(dim=1, keepdim=True)) + gs.double().abs()
        close(gx, want, U[kind] * want.abs() + (77 * F + 3 * RHO + 8 * F) * rough + TINY[kind], "grad_x")
        total = terms.sum(dim=0)
        close(gw, total, U[kind] * total.abs() + (80 * F + RHO + 4 * F) * terms.abs().sum(dim=0) + TINY[kind], "grad_weight")
    gradients(gy, gs)
    group = torch.arange(rows, device="cuda") // 16
    g = torch.Generator().manual_seed(rows)
    last = int(group[-1].item())
    for k in sorted({0, 1, last - 1, last, *(int(v) for v in torch.randint(0, last, (12,), generator=g))}):
        gradients(torch.where((group == k)[:, None], gy, torch.zeros_like(gy)), gs)
    stripes = torch.arange(rows, device="cuda") % 97
    for k in (0, 41):
        gradients(torch.where((stripes == k)[:, None], gy, torch.zeros_like(gy)), gs)


# ---- coding ------------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("kind,rows,width", [("bf16", 60_003, 256), ("fp16", 30_001, 384), ("fp32", 60_003, 128), ("bf16", 9_001, 1024), ("fp32", 90_001, 8)])
def test_coding_of_many_aligned_rows(kind, rows, width):
    """Enough that a warp deals with several groups of rows; what is special lies in the last ones too.  Coded and decoded exactly."""
    import torch
    from htgs_b200 import sequence as seq
    x = draw((rows, width), rows, kind)
    x[:, :3] *= 64
    x[rows - 1] = 0
    x[rows - 2, width // 2], x[rows - 3, width - 1], x[rows // 2, 0] = float("nan"), float("-inf"), float("inf")
    q = seq.quantize_fp8(x)
    codes, exponents = codes_of(q)
    want = ref.quantize(f64(x))
    assert np.array_equal(exponents, want[1]) and np.array_equal(codes, want[0], equal_nan=True)
    values = ref.dequantize(*want)
    for to in (torch.bfloat16, torch.float32):
        assert np.array_equal(f64(q.dequantize(to)), values, equal_nan=True)
    half = torch.tensor(values, device="cuda").to(torch.float16)
    assert torch.equal(q.dequantize(torch.float16).nan_to_num(7.0), half.nan_to_num(7.0))
