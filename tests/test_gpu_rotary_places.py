"""GPU: rotary positions of heads that begin anywhere, and of rows of more values than a block's threads load at once."""
import pytest
import torch

import attention_reference as ref
from test_gpu_attention import binding, draw, f64, near  # noqa: F401  (the fixture: every test runs over both bindings)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("width", [2, 4, 6, 12, 20, 36, 64])
def test_rotary_of_heads_that_begin_on_any_value(width, kind, interleaved):
    """A view that begins 0 to 5 values behind a multiple of 16 bytes, rows and heads an odd or even number of values apart: the same bits as of its copy."""
    from htgs_b200 import sequence as seq
    rows, heads = 7, 3
    positions = (torch.rand((rows, 1), generator=torch.Generator().manual_seed(3)) * 1000).cuda()
    for begin in range(6):
        for between in (0, 1, 2):                     # values between heads, and as many between rows
            pitch = width + between
            wide = draw((rows, heads * pitch + between + begin), begin, kind)
            x = wide.as_strided((rows, heads, width), (wide.stride(0), pitch, 1), begin)
            assert torch.equal(seq.rotary(x, None, positions, interleaved=interleaved)[0], seq.rotary(x.contiguous(), None, positions, interleaved=interleaved)[0])
            leaf = x.contiguous().requires_grad_(True)
            out = seq.rotary(leaf, None, positions, interleaved=interleaved)[0]
            assert torch.equal(*(torch.autograd.grad(out, leaf, g, retain_graph=True)[0] for g in (x, x.contiguous())))          # such a gradient
    near(out, ref.turn(f64(leaf), ref.angles(positions.cpu(), [width // 2], 10000.0), interleaved), ref.turn_bound(f64(leaf), kind, interleaved))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("kind,heads,key_heads,width,axes,spare", [("bf16", 64, 8, 128, 3, 0), ("fp16", 70, 1, 128, 1, 0), ("fp32", 40, 9, 128, 2, 0), ("bf16", 9, 2, 124, 3, 1), ("fp16", 33, 0, 34, 4, 1),
                                                                   ("fp32", 6, 5, 256, 2, 1)])
def test_rotary_of_rows_of_many_values(kind, heads, key_heads, width, axes, spare, interleaved):
    """More than 512 pieces to a row; with `spare`, heads that begin on no more than a value, so that a piece is a pair."""
    from htgs_b200 import sequence as seq
    rows = 5
    both = draw((rows, (heads + key_heads) * width + spare), 1, kind)[:, spare:]
    q, k = both[:, :heads * width].unflatten(1, (heads, width)), both[:, heads * width:].unflatten(1, (key_heads, width)) if key_heads else None
    positions = (torch.rand((rows, axes), generator=torch.Generator().manual_seed(3)) * 1000).cuda()
    sections = [width // 2 // axes + (a < width // 2 % axes) for a in range(axes)]
    angle = ref.angles(positions.cpu(), sections, 10000.0)
    leaves = [t.detach().requires_grad_(True) for t in (q, k) if t is not None]
    out = [t for t in seq.rotary(leaves[0], leaves[1] if key_heads else None, positions, interleaved=interleaved) if t is not None]
    grads = [draw((*t.shape[:2], width + spare), 7 + i, kind)[..., spare:] for i, t in enumerate(leaves)]
    back = torch.autograd.grad(out, leaves, grads)
    for x, y, gy, gx in zip(leaves, out, grads, back):
        near(y, ref.turn(f64(x), angle, interleaved), ref.turn_bound(f64(x), kind, interleaved), "out")
        near(gx, ref.turn(f64(gy), -angle, interleaved), ref.turn_bound(f64(gy), kind, interleaved), "grad")
