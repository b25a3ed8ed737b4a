"""The launches of 4-bit products that the GPU tests run, held against the rules (host code; no GPU is touched)."""
import pytest

from tests.w4_plans import BATCH, FEW, PLANS, STREAM, TILE, plan


@pytest.mark.parametrize("shape", PLANS)
def test_the_plan_of_a_shape(shape):
    assert plan(*shape) == PLANS[shape]


def test_a_shape_that_is_refused_has_no_plan():
    assert [plan(*s) for s in ((0, 16, 128), (1, 0, 128), (1, 16, 100), (1 << 20, 16, 128))] == [None] * 4


def test_every_kernel_is_run():
    few, batch, long_batch, tile = set(), set(), set(), set()
    for (m, _, k), (kind, nt, waves, splits, span) in PLANS.items():
        if kind == FEW:
            few.add((nt, k > 4096, m <= 4))
        elif kind == BATCH:
            one = (1 if m <= 16 else 2 if m <= 32 else 4, nt, waves, splits > 1)
            batch.add(one)
            # A window of scales has 8, 16 or 32 steps (groups of 32, 64, 128): it is loaded again in a longer span.
            long_batch |= {one} if span > 32 else set()
        elif kind == TILE:
            tile.add((nt, splits > 1, span % 3))  # chunks of 64 k behind the last six: 0, 2 or 4
    assert few >= {(1, False, True), (1, False, False), (1, True, True), (2, False, True), (2, False, False), (4, False, False)}
    assert batch == long_batch == {(tm, nt, waves, split) for tm, nt, waves in ((1, 1, 4), (2, 1, 4), (4, 1, 4), (1, 1, 16), (2, 2, 16), (4, 1, 8))
                                   for split in (False, True)}
    assert {t[:2] for t in tile} == {(nt, split) for nt in (1, 2) for split in (False, True)}
    assert {(t[0], t[2]) for t in tile} == {(nt, rest) for nt in (1, 2) for rest in (0, 1, 2)}


def test_streams_with_x_in_one_and_in_several_chunks():
    """56 KiB hold 56 KiB / tokens / 256 steps, less a row's padding."""
    chunks = {k // 128 > (56 * 1024 // m - 16) // 512 * 2 for (m, _, k), p in PLANS.items() if p[0] == STREAM}
    assert chunks == {False, True}
