"""GPU: the refiner with attention in its layers - norm, 8-bit products, recurrence, rotary positions and attention together, in front of the rasterizer."""
import pytest

from test_gpu_refiner import raw_scene, render

pytestmark = pytest.mark.gpu


def test_training_through_the_rasterizer():
    """It runs, and finite gradients reach every weight."""
    import torch
    from htgs_b200.refiner import GaussianRefiner
    torch.manual_seed(0)
    scene, raw, sh_rest = raw_scene()
    with torch.no_grad():
        target = render(scene, raw, sh_rest)
    raw["sh_0"] = raw["sh_0"] + 0.4
    model = GaussianRefiner(64, 2, step=0.1, heads=4, key_heads=2, window=40).cuda()
    for _ in range(2):
        model.zero_grad()
        (render(scene, model(raw), sh_rest) - target).square().mean().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().max().item() > 0 for p in model.parameters())


def test_weights_without_attention_are_drawn_as_before():
    import torch
    from htgs_b200.refiner import GaussianRefiner
    torch.manual_seed(1)
    plain = GaussianRefiner(64, 2)
    torch.manual_seed(1)
    with_heads = GaussianRefiner(64, 2, heads=2)
    state = with_heads.state_dict()
    assert all(torch.equal(value, state[name]) for name, value in plain.state_dict().items())


def test_coded_weights_follow_the_training_forward():
    """As without attention: activations differ by the 16-bit rounding of the norm's output in front of its coding, the change that the network makes by half a step of a code at most."""
    import torch
    from htgs_b200.refiner import PARAMETERS, GaussianRefiner
    torch.manual_seed(1)
    _, raw, _ = raw_scene()
    model = GaussianRefiner(128, 2, step=1.0, heads=4, window=100).cuda()
    with torch.no_grad():
        a = model(raw)
    b = model.freeze().infer(raw)
    for name, _ in PARAMETERS:
        change, other = a[name] - raw[name], b[name] - raw[name]
        assert change.abs().max().item() > 0
        assert (change - other).norm().item() <= 2.0 ** -4 * change.norm().item(), name


def test_packed_scenes_are_refined_as_each_alone():
    import torch
    from htgs_b200.refiner import PARAMETERS, GaussianRefiner
    torch.manual_seed(3)
    (_, one, _), (_, two, _) = raw_scene(700, seed=3), raw_scene(901, seed=4)
    model = GaussianRefiner(64, 2, step=1.0, heads=2, window=64).cuda().freeze()
    offsets = torch.tensor([0, 700, 1601], dtype=torch.int32, device="cuda")
    results = []
    for factor in (1.0, 1000.0):
        both = {name: torch.cat([one[name], two[name] * (factor if name == "positions" else 1.0)]) for name, _ in PARAMETERS}
        results.append(model.infer(both, offsets))
    for name, _ in PARAMETERS:
        assert torch.equal(results[0][name][:700], results[1][name][:700]), name
    empty = {name: t[:0] for name, t in one.items()}
    assert all(model.infer(empty)[name].shape[0] == 0 for name, _ in PARAMETERS)


def test_heads_have_to_fit():
    from htgs_b200.refiner import GaussianRefiner
    for k in ({"heads": 3}, {"heads": 64}, {"heads": 4, "key_heads": 3}, {"heads": 4, "key_heads": 0}):
        with pytest.raises(ValueError):
            GaussianRefiner(64, 1, **k)
    with pytest.raises(ValueError):
        GaussianRefiner(512, 1, heads=2)
