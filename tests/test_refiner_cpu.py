"""CPU: the order of the Gaussians along the curve, and the refiner's refusals."""
import pytest
import torch

from htgs_b200 import refiner


def test_curve_order_is_a_permutation_that_keeps_neighbours_together():
    g = torch.Generator().manual_seed(1)
    grid = torch.stack(torch.meshgrid(*[torch.arange(8.0)] * 3, indexing="ij"), dim=-1).reshape(-1, 3)
    shuffled = grid[torch.randperm(512, generator=g)]
    order = refiner.curve_order(shuffled)
    assert torch.equal(torch.sort(order).values, torch.arange(512))
    path = shuffled[order]
    # the curve goes through each octant before the next: 8 runs of 64
    octant = (path >= 4).long() @ torch.tensor([1, 2, 4])
    assert torch.equal(octant, torch.arange(8).repeat_interleave(64))


def test_curve_order_of_packed_scenes_stays_in_each():
    g = torch.Generator().manual_seed(2)
    positions = torch.rand((100, 3), generator=g)
    offsets = torch.tensor([0, 30, 30, 100], dtype=torch.int32)
    order = refiner.curve_order(positions, offsets)
    assert torch.equal(torch.sort(order[:30]).values, torch.arange(30)) and torch.equal(torch.sort(order[30:]).values, torch.arange(30, 100))


def test_order_of_equal_and_of_no_positions():
    assert torch.equal(refiner.curve_order(torch.ones(5, 3)), torch.arange(5))
    assert refiner.curve_order(torch.empty(0, 3)).shape == (0,)


def test_infer_needs_coded_weights():
    with pytest.raises(RuntimeError):
        refiner.GaussianRefiner(32, 1).infer({})


def separate_orders(parts):
    """The orders that scenes get alone, one behind the other."""
    begin, orders = 0, []
    for p in parts:
        orders.append(refiner.curve_order(p) + begin)
        begin += p.shape[0]
    return torch.cat(orders)


def test_curve_order_of_packed_scenes_is_that_of_each_alone():
    g = torch.Generator().manual_seed(3)
    parts = [torch.rand((500, 3), generator=g), torch.rand((300, 3), generator=g) * 5000.0 - 1000.0, torch.empty(0, 3), torch.rand((1, 3), generator=g) * 1e-6,
             torch.rand((200, 3), generator=g) * torch.tensor([1e-3, 1.0, 1e4])]
    offsets = torch.tensor([0, 500, 800, 800, 801, 1001], dtype=torch.int32)
    assert torch.equal(refiner.curve_order(torch.cat(parts), offsets), separate_orders(parts))


def test_positions_that_are_not_finite_leave_the_others_in_order():
    g = torch.Generator().manual_seed(4)
    positions = torch.rand((400, 3), generator=g)
    alone = refiner.curve_order(positions)
    for value in (float("nan"), float("inf"), float("-inf")):
        for axis in range(3):
            odd = torch.cat((positions, torch.full((1, 3), 0.5)))
            odd[400, axis] = value
            order = refiner.curve_order(odd)
            assert torch.equal(order[order != 400], alone)
    nothing = torch.full((3, 3), float("nan"))
    assert torch.equal(refiner.curve_order(nothing), torch.arange(3))
    parts = [positions, odd]
    assert torch.equal(refiner.curve_order(torch.cat(parts), torch.tensor([0, 400, 801], dtype=torch.int32)), separate_orders(parts))


def test_a_few_far_positions_leave_the_others_near_one_another():
    """Steps along the curve through 10 000 points of a unit cube are about as long as its cells, without and with one point ten thousand times as far away (in a
    random order they would be 0.66 on average)."""
    g = torch.Generator().manual_seed(5)
    positions = torch.rand((10_000, 3), generator=g)
    for points in (positions, torch.cat((positions, torch.full((1, 3), 1e4))), torch.cat((torch.tensor([[-1e4, 0.5, 2.0]]), positions))):
        order = refiner.curve_order(points)
        path = points[order]
        path = path[(path.abs() <= 1).all(dim=1)]
        assert path.shape[0] == 10_000 and (path[1:] - path[:-1]).norm(dim=1).mean().item() < 0.15


def test_curve_order_is_that_of_the_interleaved_cells():
    g = torch.Generator().manual_seed(6)
    positions = torch.randint(0, 2 ** 20, (2000, 3), generator=g).float()
    positions[0], positions[1] = 0.0, 2.0 ** 20 - 1
    cells = [[int(c) for c in p] for p in positions]
    code = [sum((c >> bit & 1) << (3 * bit + axis) for bit in range(20) for axis, c in enumerate(cell)) for cell in cells]
    assert refiner.curve_order(positions).tolist() == sorted(range(2000), key=lambda i: code[i])
