"""Rows of one large weight and a million small ones: what the integers of the third launch leave of the small ones.

A weight is held to half a unit of max(2^-51 of the largest, 2^-55 of the row's sum), so that a border between two tokens
lies within vocab times that, 2^-32 of the sum at 2^20 tokens; TOL allows for twice as much."""
import numpy as np
import pytest

from tests import step_util as S
from tests.gpu_util import announce
from tests.test_gpu_sample import _call

pytestmark = pytest.mark.gpu

TOL = 2.0 ** -31


def _tail(vocab, lowest, highest):
    """The largest logit last; the others from the lowest on, in order."""
    z = np.linspace(lowest, highest, vocab)
    z[-1] = 0.0
    return z.astype(np.float32)


def _draws(z, asked, us):
    got = _call(np.tile(z, len(us)), z.size, z.size, [asked] * len(us), us)
    t, k, p, floor = (float(np.float32(v)) for v in asked)
    w = S.sample_weights(z.astype(np.float64), t, int(k), p, floor)
    return got, w


@pytest.mark.parametrize("vocab", [1 << 18, 1 << 20])
@pytest.mark.parametrize("asked", ["top_k", "min_p", "top_k and top_p"])
@pytest.mark.parametrize("lowest,highest", [(-29.91, -29.91), (-31.0, -29.0), (-20.7, -20.7)])
def test_draws_among_the_small_ones(vocab, asked, lowest, highest):
    announce(f"sample units vocab={vocab} {asked} {lowest} {highest}")
    z = _tail(vocab, lowest, highest)
    asked = {"top_k": (1.0, vocab - 1, 1.0, 0.0), "min_p": (1.0, 0, 1.0, 1e-14), "top_k and top_p": (1.0, vocab - 1, 1 - 2.0 ** -24, 0.0)}[asked]
    tail = float(np.exp(z[:-1].astype(np.float64)).sum())
    us = [float(np.float32(tail * part)) for part in (0.02, 0.25, 0.5, 0.75, 0.98, 1.5)]
    got, w = _draws(z, asked, us)
    sums = np.cumsum(w)
    for g, u in zip(got, us):
        goal = u * sums[-1]
        assert w[g] > 0 and sums[g] - w[g] - TOL * sums[-1] <= goal <= sums[g] + TOL * sums[-1], (int(g), u)
    assert got[-1] == vocab - 1


@pytest.mark.parametrize("vocab", [1 << 18, 1 << 20])
@pytest.mark.parametrize("lowest,highest", [(-40.0, -22.0), (-30.0, -26.0), (-28.0, -27.9)])
@pytest.mark.parametrize("part", [0.5, 0.05])
def test_cuts_among_the_small_ones(vocab, lowest, highest, part):
    """u of 0 draws the lowest index that is kept: the last token of the prefix, as the small ones are in order."""
    announce(f"sample units cut vocab={vocab} {lowest} {highest} {part}")
    z = _tail(vocab, lowest, highest)
    w = np.exp(z.astype(np.float64))
    share = float(w[:-1].sum() / w.sum())
    top_p = float(np.float32(1 - part * share))
    top_p = min(top_p, 1 - 2.0 ** -24)  # the largest below 1 that f32 holds
    assert 1 - share < top_p
    got, kept = _draws(z, (1.0, 0, top_p, 0.0), [0.0])
    g, total = int(got[0]), w.sum()
    above = w[g + 1:].sum()  # all that come before it in order
    assert above - TOL * total <= top_p * total <= above + w[g] + TOL * total, (g, int(np.flatnonzero(kept)[0]))
