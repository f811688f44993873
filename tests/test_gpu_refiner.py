"""GPU: the sequence operators used together - the refiner in front of the rasterizer, in training and with coded weights."""
import pytest

pytestmark = pytest.mark.gpu


def raw_scene(n=3000, size=96, seed=5):
    import torch
    import harness
    from htgs_b200 import scenes
    scene = scenes.tiny_scene(n=n, size=size, seed=seed, sh_degree=1)
    t = harness.scene_tensors(scene)
    raw = {"positions": t[0], "scales": t[1].log(), "rotations": t[2], "opacities": torch.special.logit(t[3].clamp(1e-4, 1 - 1e-4)), "sh_0": t[4]}
    return scene, raw, t[5]


def render(scene, raw, sh_rest):
    import torch
    import harness
    from htgs_b200 import glue
    ours = harness.ours()
    s, r, o = glue.activate(raw["scales"], raw["rotations"], raw["opacities"])
    st = harness.settings_for(ours, scene, scene.views[0], 0, 8)
    return ours.diff_rasterize(raw["positions"], s, r, o, raw["sh_0"], sh_rest, torch.empty(0, device="cuda"), st, False)


def test_training_through_the_rasterizer():
    """Gradients reach every weight, and a few steps bring a scene with disturbed colours nearer to its image."""
    import torch
    from htgs_b200.refiner import GaussianRefiner
    torch.manual_seed(0)
    scene, raw, sh_rest = raw_scene()
    with torch.no_grad():
        target = render(scene, raw, sh_rest)
    raw["sh_0"] = raw["sh_0"] + 0.4
    model = GaussianRefiner(64, 2, step=0.1).cuda()
    optimizer = torch.optim.Adam(model.parameters(), lr=5e-3)
    losses = []
    for _ in range(25):
        optimizer.zero_grad()
        loss = (render(scene, model(raw), sh_rest) - target).square().mean()
        loss.backward()
        losses.append(loss.item())
        assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())
        optimizer.step()
    assert all(p.grad.abs().max().item() > 0 for p in model.parameters())
    assert losses[-1] < 0.5 * losses[0]


def test_coded_weights_follow_the_training_forward():
    """Both code the same weights; activations differ by the 16-bit rounding of the norm's output in front of its coding, which moves codes by a step (2^-3 of a value at
    most) here and there: the change that the network makes agrees within half of that."""
    import torch
    from htgs_b200.refiner import PARAMETERS, GaussianRefiner
    torch.manual_seed(1)
    _, raw, _ = raw_scene()
    model = GaussianRefiner(128, 3, step=1.0).cuda()
    with torch.no_grad():
        a = model(raw)
    b = model.freeze().infer(raw)
    for name, _ in PARAMETERS:
        change, other = a[name] - raw[name], b[name] - raw[name]
        assert change.abs().max().item() > 0
        assert (change - other).norm().item() <= 2.0 ** -4 * change.norm().item(), name


def test_packed_scenes_do_not_see_one_another():
    import torch
    from htgs_b200.refiner import PARAMETERS, GaussianRefiner
    torch.manual_seed(2)
    (_, one, _), (_, two, _) = raw_scene(700, seed=3), raw_scene(901, seed=4)
    model = GaussianRefiner(64, 2, step=1.0).cuda().freeze()
    both = {name: torch.cat([one[name], two[name]]) for name, _ in PARAMETERS}
    offsets = torch.tensor([0, 700, 1601], dtype=torch.int32, device="cuda")
    first = model.infer(both, offsets)
    moved = {**both, "sh_0": torch.cat([one["sh_0"], two["sh_0"] * 3 + 1])}
    second = model.infer(moved, offsets)
    for name, _ in PARAMETERS:
        assert torch.equal(first[name][:700], second[name][:700]), name
    assert not torch.equal(first["positions"][700:], second["positions"][700:])


def test_packed_scenes_are_refined_as_each_alone_wherever_the_others_lie():
    import torch
    from htgs_b200.refiner import PARAMETERS, GaussianRefiner
    torch.manual_seed(3)
    (_, one, _), (_, two, _) = raw_scene(700, seed=3), raw_scene(901, seed=4)
    model = GaussianRefiner(64, 2, step=1.0).cuda().freeze()
    offsets = torch.tensor([0, 700, 1601], dtype=torch.int32, device="cuda")
    results = []
    for factor in (1.0, 1000.0):
        both = {name: torch.cat([one[name], two[name] * (factor if name == "positions" else 1.0)]) for name, _ in PARAMETERS}
        results.append(model.infer(both, offsets))
    for name, _ in PARAMETERS:
        assert torch.equal(results[0][name][:700], results[1][name][:700]), name


def test_near_positions_are_told_apart():
    """Gaussians a fortieth apart between 1 and 2, with nothing else to tell them by and no recurrence: 8-bit numbers there are an eighth apart, which would leave nine
    different changes; the coding of the norm's output may take a few of the 41 away."""
    import torch
    from htgs_b200.refiner import PARAMETERS, GaussianRefiner
    torch.manual_seed(4)
    model = GaussianRefiner(64, 0, step=1.0).cuda()
    raw = {name: torch.ones(41, *((width,) if name != "sh_0" else (1, 3)), device="cuda") for name, width in PARAMETERS}
    raw["positions"] = torch.cat((torch.linspace(1.0, 2.0, 41, device="cuda")[:, None], torch.ones(41, 2, device="cuda")), dim=1)
    with torch.no_grad():
        for result in (model(raw), model.freeze().infer(raw)):
            change = torch.cat([(result[name] - raw[name]).reshape(41, -1) for name, _ in PARAMETERS[1:]], dim=1)
            assert torch.unique(change, dim=0).shape[0] > 20


def test_infer_stays_with_the_weights_that_were_coded():
    import torch
    from htgs_b200.refiner import GaussianRefiner
    torch.manual_seed(5)
    _, raw, _ = raw_scene(300)
    model = GaussianRefiner(64, 2).cuda().freeze()
    before = model.infer(raw)
    with torch.no_grad():
        for p in (model.embed, model.head, *model.enter, *model.leave):
            p.mul_(2)
    assert all(torch.equal(before[name], value) for name, value in model.infer(raw).items())
    assert not torch.equal(before["positions"], model.freeze().infer(raw)["positions"])
