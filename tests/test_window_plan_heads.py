"""CPU tests of the plans of busy steps, whose row items take two or four kv heads: the same cover of every visible tile, the same
merges."""
import numpy as np
import pytest

from tests import test_window_plan as base
from tests.window_util import make_case

# Single sequences, shortest and longest context, window, sinks, kv heads of an item, and whether some tokens are split.
BUSY = [(300, 300, 310, 0, 0, 2, False), (180, 60, 900, 0, 0, 2, True), (256, 500, 520, 0, 0, 4, False), (130, 60, 2500, 0, 0, 4, True),
        (60, 3000, 5000, 1500, 70, 2, True), (256, 3000, 5000, 500, 4, 4, False)]


@pytest.mark.parametrize("shape", [(16, 8, 256), (8, 8, 128), (8, 4, 512), (64, 8, 128)])
@pytest.mark.parametrize("busy", BUSY)
def test_items_of_two_and_four_heads_cover_every_visible_tile_once(busy, shape, monkeypatch):
    runs, lo, hi, window, sinks, heads, split = busy
    lens = [(int(c), 3 if i % 31 == 7 and shape[0] <= 5 * shape[1] else 1) for i, c in enumerate(np.linspace(lo, hi, runs))]
    case = make_case(1, lens, window=window, sinks=sinks)
    st, _, info = base.plan(case, nq=shape[0], nkv=shape[1], d=shape[2])
    assert st == 0 and info[14] == 0 and info[25] == heads
    assert (info[1] > 0) == split
    monkeypatch.setattr(base, "STEPS", [(lens, window, sinks)])
    base.test_items_cover_every_visible_tile_once(shape, 0)
