"""CPU: the 64-bit form for long sequences, with its bounds, agrees with the one that goes row by row."""
import numpy as np
import pytest

import test_gpu_sequence as short
import test_gpu_sequence_long as long


@pytest.mark.parametrize("rows,offsets", [(1, [0, 1]), (2, [0, 0, 1, 2, 2]), (57, [0, 57]), (200, [0, 0, 16, 17, 17, 90, 200, 200])])
@pytest.mark.parametrize("reverse", [False, True])
def test_long_form_is_the_row_by_row_form(rows, offsets, reverse):
    rng = np.random.default_rng(rows)
    x, g, gh = rng.normal(size=(rows, 3)), rng.normal(size=(rows, 3)) * 2 + 2, rng.normal(size=(rows, 3))
    initial, gl = rng.normal(size=(len(offsets) - 1, 3)), rng.normal(size=(len(offsets) - 1, 3))
    h, last, h_bound, last_bound = short.scan_bounds(x, g, initial, offsets, reverse, "bf16")
    want = [(h, h_bound), (last, last_bound)] + short.backward_bounds(x, g, initial, offsets, gh, gl, reverse, "bf16")
    got = long.long_scan(x, g, initial, offsets, gh, gl, reverse, "bf16")
    for (v, b), (w, c) in zip(got, want):
        assert np.allclose(v, w, rtol=1e-12, atol=1e-12)
        assert np.allclose(b, c, rtol=1e-6, atol=1e-30)


def test_walks_of_the_long_sequences():
    for case in next(m for m in long.test_scan_of_long_sequences.pytestmark if m.args[0].startswith("kind")).args[1]:
        assert long.shape_of_walk(case[1], case[2]) == case[3]
