"""GPU: the sequence operators at the ends of their range, and what autograd knows of them.  (Tolerances as in test_gpu_sequence.py.)"""
import numpy as np
import pytest

import sequence_reference as ref
from test_gpu_sequence import binding, draw, f64, near, product_bound  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,out,width", [(1, 40, 128), (3, 33, 300), (8, 65, 1000), (300, 136, 260)])
@pytest.mark.parametrize("size_x,size_w", [(1e36, 1e-2), (1e30, 1e-30), (3e37, 1e-25), (1e-37, 1e30), (1e-30, 1e36), (1e-10, 1e-25)])
def test_product_of_large_and_small_values(kind, rows, out, width, size_x, size_w):
    """Scales whose product is in range although one of them, times a sum of codes, is not."""
    import torch
    from htgs_b200 import sequence as seq
    x, w = draw((rows, width), 3, kind, size_x / 8), draw((out, width), 4, kind, size_w)
    a, b = ref.dequantize(*ref.quantize(f64(x))), ref.dequantize(*ref.quantize(f64(w), 128), 128)
    assert np.isfinite(f64(x)).all() and np.abs(a @ b.T).max() < 1e38
    q = seq.quantize_fp8(w, 128)
    near(seq.fp8_matmul(x, q), *product_bound(a, b, kind), "values")
    near(seq.fp8_matmul(seq.quantize_fp8(x), q, torch.float32), *product_bound(a, b, "fp32"), "codes")


def test_product_with_scales_that_are_nan():
    import torch
    from htgs_b200 import sequence as seq
    x, w = draw((4, 300), 1), draw((9, 300), 2)
    q = seq.quantize_fp8(w, 1)
    q.scales.view(torch.uint8)[3, 1] = 255
    want = torch.zeros(4, 9, dtype=torch.bool, device="cuda")
    want[:, 3] = True
    for rows in (1, 4):
        assert torch.equal(torch.isnan(seq.fp8_matmul(x[:rows], q)), want[:rows])
        assert torch.equal(torch.isnan(seq.fp8_matmul(seq.quantize_fp8(x[:rows]), q)), want[:rows])


def test_forward_mode_derivatives_are_refused():
    """No operator has one, and none drops a tangent without a word."""
    import torch
    import torch.autograd.forward_ad as fw
    from htgs_b200 import sequence as seq
    x, w, r, square = draw((4, 64), 1), draw((64,), 2), draw((4, 64), 3), draw((64, 64), 4)
    initial, q = draw((1, 64), 5), seq.quantize_fp8(draw((64, 64), 4), 128)
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: seq.add_rms_norm(dual(x), w, r), lambda: seq.add_rms_norm(x, dual(w)), lambda: seq.add_rms_norm(x, w, dual(r)),
                     lambda: seq.add_rms_norm_fp8(dual(x), w), lambda: seq.fp8_matmul(dual(x), q), lambda: seq.fp8_linear(dual(x), square), lambda: seq.fp8_linear(x, dual(square)),
                     lambda: seq.gated_scan(dual(x), r), lambda: seq.gated_scan(x, dual(r)), lambda: seq.gated_scan(x, r, dual(initial)),
                     lambda: seq.gated_scan_step(dual(x), r, torch.zeros_like(x)), lambda: seq.gated_scan_step(x, r, dual(torch.zeros_like(x)))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()
        seq.add_rms_norm(x, w, r)
    seq.add_rms_norm(x, w, r)


def test_step_tells_autograd_of_its_state():
    """A state that another operator keeps for its gradient: the step overwrites it, and that gradient is refused."""
    import torch
    from htgs_b200 import sequence as seq
    x, g, state = draw((3, 16), 1), draw((3, 16), 2), draw((3, 20), 3)[:, :16]
    factor = draw((3, 16), 4).requires_grad_(True)
    y = (factor * state).sum()
    before = state._version
    seq.gated_scan_step(x, g, state)
    assert state._version == before + 1
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()
    with torch.inference_mode():
        inner = torch.zeros(3, 16, device="cuda")
        seq.gated_scan_step(x, g, inner)
    seq.gated_scan_step(x, g, inner)                       # nothing can have kept it


def operators_with_gradients():
    from htgs_b200 import sequence as seq
    x, other, vector, square = draw((5, 32), 1), draw((5, 32), 2), draw((32,), 3), draw((32, 32), 4)
    return {"norm": (lambda v: seq.add_rms_norm(v, vector, other)[0], x), "norm's weight": (lambda v: seq.add_rms_norm(x, v)[0], vector),
            "linear": (lambda v: seq.fp8_linear(v, square), x), "linear's weight": (lambda v: seq.fp8_linear(x, v), square),
            "scan": (lambda v: seq.gated_scan(v, other)[0], x), "gate": (lambda v: seq.gated_scan(x, v)[0], other)}


def test_first_derivatives_with_a_graph_and_no_second_ones():
    """create_graph=True is no error by itself.  A second derivative is one, also where the first one's gradient wants none itself: it is not left out of a sum."""
    import torch
    for name, (f, leaf) in operators_with_gradients().items():
        v = leaf.clone().requires_grad_(True)
        want, = torch.autograd.grad(f(v).square().sum(), v)
        y = f(v)
        got, = torch.autograd.grad(y.square().sum(), v, create_graph=True)
        assert torch.equal(got, want), name
        with pytest.raises(RuntimeError, match="second derivative"):
            got.sum().backward()
        assert v.grad is None or torch.equal(v.grad, torch.zeros_like(v))
        y = f(v)
        got, = torch.autograd.grad(y.sum(), v, create_graph=True)
        with pytest.raises(RuntimeError, match="second derivative"):
            (y.square().sum() + got.square().sum()).backward()


def test_what_a_gradient_needs_is_kept_as_saved_tensors():
    """They are freed by the backward pass, which is refused the second time, and hooks on saved tensors see them."""
    import torch
    for name, (f, leaf) in operators_with_gradients().items():
        v = leaf.clone().requires_grad_(True)
        seen = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t.dtype) or t, lambda t: t):
            y = f(v)
        assert seen, name
        y.sum().backward()
        with pytest.raises(RuntimeError, match="second time"):
            y.sum().backward()
    assert torch.float8_e4m3fn not in seen                 # the recurrence keeps its inputs and states


def test_a_wait_that_ran_out_is_reported_once_and_for_its_device():
    """The word that a kernel sets is set here on the host."""
    import torch
    from htgs_b200 import _native, sequence as seq
    lib = _native.lib()
    x, w = draw((20, 128), 1), draw((16, 128), 2)
    q = seq.quantize_fp8(w, 128)
    want, few = seq.fp8_matmul(x, q), seq.fp8_matmul(x[:2], q)
    word, other = (lib.htgs_fp8_matmul_error_word(device) for device in (0, 1))
    for call in (lambda: seq.fp8_matmul(x, q), lambda: seq.fp8_matmul(x[:2], q), lambda: seq.fp8_matmul(seq.quantize_fp8(x[:2]), q), lambda: seq.fp8_linear(x, w),
                 lambda: seq.check_products(), lambda: seq.check_products(x.device)):
        word[0] = 1
        with pytest.raises(RuntimeError, match="wait in an earlier product"):
            call()
        assert word[0] == 0
        seq.check_products()
        assert torch.equal(seq.fp8_matmul(x, q), want)
    other[0] = 1                                           # another device's
    assert torch.equal(seq.fp8_matmul(x, q), want) and torch.equal(seq.fp8_matmul(x[:2], q), few)
    seq.check_products("cuda:0")
    assert lib.htgs_fp8_matmul_status(1) == _native.HTGS_ERR_DEVICE_FLAG and lib.htgs_fp8_matmul_status(1) == 0
    for device in (-1, 64):
        assert lib.htgs_fp8_matmul_status(device) == _native.HTGS_ERR_INVALID_ARGUMENT and not lib.htgs_fp8_matmul_error_word(device)


def test_more_rows_than_a_grid_has_in_one_direction():
    """65536 blocks of 128 rows and a few more: coded by blocks and transposed, and through the linear layer's gradients."""
    import torch
    from htgs_b200 import sequence as seq
    rows, begin = 65536 * 128 + 130, 65536 * 128 - 128           # what is not zero lies at the end
    x, gy, w = torch.zeros(rows, 16, dtype=torch.bfloat16, device="cuda"), torch.zeros(rows, 24, dtype=torch.bfloat16, device="cuda"), draw((24, 16), 3, "bf16")
    x[begin:], gy[begin:] = draw((rows - begin, 16), 1, "bf16"), draw((rows - begin, 24), 2, "bf16")
    blocks, turned = seq.quantize_fp8(x, 128), seq.quantize_fp8(x, 1, True)
    end = f64(x[begin:])
    for q, part, want, per in ((blocks, slice(begin, None), ref.quantize(end, 128), 128), (turned, slice(None), ref.quantize(end.T.copy()), 1)):
        codes = q.codes[part] if per == 128 else q.codes[:, begin:]
        scales = q.scales[begin // 128:] if per == 128 else q.scales[:, begin // 128:]
        assert np.array_equal(codes.float().double().cpu().numpy(), want[0])
        assert np.array_equal(scales.contiguous().view(torch.uint8).cpu().numpy().astype(np.int64) - 127, want[1])
    assert not blocks.codes[:begin].view(torch.uint8).any() and not turned.codes[:, :begin].view(torch.uint8).any()
    leaves = [t.requires_grad_(True) for t in (x, w)]
    gx, gw = torch.autograd.grad(seq.fp8_linear(*leaves), leaves, gy)
    rowwise, tilewise = lambda v: ref.dequantize(*ref.quantize(v)), lambda v: ref.dequantize(*ref.quantize(v, 128), 128)  # noqa: E731
    g = f64(gy[begin:])
    near(gw, *product_bound(rowwise(g.T.copy()), rowwise(end.T.copy()), "bf16"), "grad_weight")
    near(gx[begin:], *product_bound(rowwise(g), tilewise(f64(w)).T, "bf16"), "grad_x")
