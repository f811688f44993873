"""CPU: the 64-bit forms of the sequence operators that the GPU tests compare with - their gradients against central differences, their
8-bit rounding against torch's."""
import numpy as np
import pytest

import sequence_reference as ref


def differences(f, v, weights, eps=1e-6):
    """d sum(weights * f(v)) / dv by central differences; error about eps^2 + 2^-52 / eps = 2e-10 of the values' size."""
    grad = np.zeros_like(v)
    for i in np.ndindex(*v.shape):
        keep = v[i]
        v[i] = keep + eps
        hi = sum(np.sum(w * o) for w, o in zip(weights, f()))
        v[i] = keep - eps
        lo = sum(np.sum(w * o) for w, o in zip(weights, f()))
        v[i] = keep
        grad[i] = (hi - lo) / (2 * eps)
    return grad


def test_norm_gradient():
    rng = np.random.default_rng(1)
    x, r, w, gy, gs = rng.normal(size=(3, 7)), rng.normal(size=(3, 7)), rng.normal(size=7), rng.normal(size=(3, 7)), rng.normal(size=(3, 7))
    y, u, rho = ref.norm(x, w, r, 1e-3)
    gx, gw = ref.norm_backward(gy, gs, u, rho, w)
    both = lambda: ref.norm(x, w, r, 1e-3)[:2]  # noqa: E731
    assert np.allclose(gx, differences(both, x, (gy, gs)), atol=1e-8)
    assert np.allclose(gx, differences(both, r, (gy, gs)), atol=1e-8)
    assert np.allclose(gw, differences(both, w, (gy, gs)), atol=1e-8)


@pytest.mark.parametrize("reverse", [False, True])
def test_scan_gradient(reverse):
    rng = np.random.default_rng(2)
    offsets = [0, 4, 4, 5, 9]
    x, g, h0 = rng.normal(size=(9, 3)), rng.normal(size=(9, 3)) * 2, rng.normal(size=(4, 3))
    gh, gl = rng.normal(size=(9, 3)), rng.normal(size=(4, 3))
    grads = ref.scan_backward(x, g, h0, offsets, gh, gl, reverse)
    both = lambda: ref.scan(x, g, h0, offsets, reverse)  # noqa: E731
    for got, v in zip(grads, (x, g, h0)):
        assert np.allclose(got, differences(both, v, (gh, gl)), atol=1e-8)


def test_rounding_to_8_bits_is_torchs():
    import torch
    v = torch.cat((torch.linspace(-448, 448, 200_001, dtype=torch.float32), torch.logspace(-5, 2, 50_001)))
    assert np.array_equal(ref.e4m3(v.double().numpy()), v.to(torch.float8_e4m3fn).double().numpy())
    ties = torch.arange(-512, 513, dtype=torch.float32) / 1024          # ties among the subnormals and the smallest normals
    assert np.array_equal(ref.e4m3(ties.double().numpy()), ties.to(torch.float8_e4m3fn).double().numpy())
