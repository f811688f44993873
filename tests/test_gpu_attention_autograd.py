"""GPU: rotary positions and attention within autograd, as other operators of torch are: results changed in place, gradients of some inputs, overlapping inputs."""
import pytest
import torch

from test_gpu_attention import binding, draw, tensors  # noqa: F401  (the fixture: every test runs over both bindings)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch", [False, True])
def test_results_may_be_changed_in_place(batch):
    """A residual that is added, or a factor, and its gradient; what the backward pass needs may not change, and then it says so."""
    from htgs_b200 import sequence as seq
    q, k, v, grad = (t.view(2, 20, *t.shape[1:]) if batch else t for t in tensors(40, 4, 2, 16, "bf16"))
    positions = torch.rand((*q.shape[:-2], 3), generator=torch.Generator().manual_seed(1)).cuda()
    ql, kl, vl = (t.clone().requires_grad_(True) for t in (q, k, v))
    a, b = seq.rotary(ql, kl, positions)
    a.mul_(2.0)
    b.flatten(-2).mul_(0.5)
    got = torch.autograd.grad((a, b), (ql, kl), (grad, k))
    c, d = seq.rotary(ql, kl, positions)
    want = torch.autograd.grad((c * 2.0, d * 0.5), (ql, kl), (grad, k))
    assert all(torch.equal(x, y) for x, y in zip((a, b, *got), (c * 2.0, d * 0.5, *want)))
    out = seq.attention(ql, kl, vl)
    plain = out.detach().clone()
    out.add_(1.0)
    assert torch.equal(out, plain + 1.0)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(out, ql, grad)
