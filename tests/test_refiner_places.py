"""The refiner's attention takes Gaussians' places from positions of any type that the refiner without attention takes."""
import pytest
import torch

from htgs_b200.refiner import PARAMETERS, GaussianRefiner, curve_order


@pytest.mark.parametrize("offsets", [None, [0, 4, 10]])
@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.float16, torch.bfloat16])
def test_places_are_32_bit_numbers_within_the_box(dtype, offsets):
    model = GaussianRefiner(64, 1, heads=2)
    positions = torch.randn((10, 3), generator=torch.Generator().manual_seed(1)).to(dtype)
    offsets = None if offsets is None else torch.tensor(offsets, dtype=torch.int32)
    places = model._places(positions, offsets, curve_order(positions, offsets))
    assert places.dtype == torch.float32 and places.shape == (10, 3) and places.min() == 0 and 1023 < places.max() <= 1024


@pytest.mark.gpu
def test_a_scene_of_64_bit_positions_is_refined():
    torch.manual_seed(1)
    g = torch.Generator().manual_seed(2)
    raw = {name: torch.randn((300, width), generator=g).cuda() for name, width in PARAMETERS}
    model = GaussianRefiner(64, 2, step=1.0, heads=2, window=20).cuda().freeze()
    wide = {**raw, "positions": raw["positions"].double()}
    for refine in (model, model.infer):
        with torch.no_grad():
            a, b = refine(raw), refine(wide)
        for name, _ in PARAMETERS:
            # Places are off by 2^-13 at most where the box is computed in 64 bits (half a unit of 1024's last place and of each step before): the same network, whose 8-bit codes differ by a step here and there.
            change, other = a[name] - raw[name], (b[name] - raw[name]).to(a[name].dtype)
            assert change.abs().max().item() > 0
            assert (change - other).norm().item() <= 2.0 ** -4 * change.norm().item(), name
