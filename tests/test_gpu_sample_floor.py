"""min_p of 1 and more keeps the largest logits alone, however near the others come: the weight of a logit that is smaller is
below 1, though it may round to 1 in 64 bits."""
import numpy as np
import pytest

from tests.gpu_util import announce
from tests.test_gpu_sample import _call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("asked", [(1.0, 0, 1.0, 1.0), (1.0, 50, 1.0, 1.0), (1.0, 0, 0.9, 1.5), (1e30, 0, 1.0, 1.0), (1e30, 1500, 0.99, 1.0),
                                   (float("inf"), 0, 1.0, 1.0), (float("inf"), 0, 0.7, float("inf")), (0.5, 0, 1.0, 2.0)])
@pytest.mark.parametrize("vocab", [2, 300, 5000, 70001])
def test_the_largest_alone(vocab, asked):
    announce(f"sample floor vocab={vocab} {asked}")
    rng = np.random.default_rng(vocab)
    z = (1e-30 * (1 + 1e-3 * rng.random((6, vocab)))).astype(np.float32)
    z[3] = rng.standard_normal(vocab)
    z[4:] += np.float32(1.0)  # one value: all are the largest
    u = rng.random(6).astype(np.float32)
    got = _call(z, vocab, vocab, [asked] * 6, u)
    for row in range(4):
        assert z[row, got[row]] == z[row].max(), row
    if asked[2] >= 1 and not asked[1]:
        assert [int(g) for g in got[4:]] == [int(float(v) * vocab) for v in u[4:]]
