"""CPU: how attention_step splits a sequence's cache goes by the rows that the call may have to read, and by no other number of them."""
import ctypes

import pytest

from htgs_b200 import _native


def splits(**k):
    """The splits that the second kernel joins, by the workspace that holds their parts; 1 where there are none, or where a cluster joins them."""
    values = {"q": 64, "k": 64, "v": 64, "keys": 64, "values": 128, "lengths": 64, "strides": 4096, "capacity": 1, "batch": 1, "heads": 1, "key_heads": 1, "width": 64, "type": 2, "window": -1} | k
    v = values
    step = _native.HtgsAttentionStep(*(v[n] for n in ("q", "k", "v", "keys", "values", "lengths")), *(v["strides"],) * 12, *(v[n] for n in ("capacity", "batch", "heads", "key_heads", "width", "type", "window")), 0.5)
    size = _native.lib().htgs_attention_step_workspace_bytes(ctypes.byref(step))
    part = v["batch"] * v["heads"] * (4 + (v["width"] + 3) // 4 * 4) * 4
    assert size % part == 0
    return max(size // part, 1)


def plan(batch, blocks, rows, places, tiles):
    """The rule: rows of a full cache, or of the window; a block costs 128 rows more than its own, 256 while it takes from others; a cluster's join 128, a kernel's 512."""
    best = None
    for n in range(1, 257):
        if n > 1 and rows < n * 128:
            break
        cluster = tiles and 1 < n <= 8 and blocks * n <= places // 2
        time = (blocks * n + places - 1) // places * (rows // n + 128) if batch == 1 else blocks * (rows + 256 * n) // places + rows // n
        cost = time + (0 if n == 1 else 128 if cluster else 512)
        if best is None or cost < best[0]:
            best = cost, 1 if cluster else n
    return best[1]


@pytest.mark.parametrize("window", [-1, 5000])
@pytest.mark.parametrize("capacity", [1, 900, 4096, 33000, 60000, 200000, 1 << 20])
@pytest.mark.parametrize("heads,key_heads,width", [(8, 2, 64), (8, 8, 32), (40, 2, 128), (4, 1, 96)])
def test_splits_go_by_the_rows_that_may_be_read(heads, key_heads, width, capacity, window):
    chunks = (heads // key_heads + 15) // 16
    rows = (min(window + 1, capacity) if window >= 0 else capacity) + 1
    for batch in (1, 2, 3, 5, 8, 32):
        for kind in (0, 2):
            blocks = batch * (key_heads * chunks if kind else heads)
            want = plan(batch, blocks, rows, 148 * ((4 if width <= 32 else 2) if kind else 8), kind != 0)
            assert splits(batch=batch, heads=heads, key_heads=key_heads, width=width, capacity=capacity, window=window, type=kind) == want, (batch, kind)
