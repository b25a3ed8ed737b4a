"""Vocabularies of up to 2,048 tokens, all of which are candidates: cuts and draws where the bins that a cut is looked for
in hold many of them (logits in a narrow range, equal ones, masks of the type's lowest value, low temperatures)."""
import numpy as np
import pytest

from tests import step_util as S
from tests.gpu_util import announce
from tests.test_gpu_sample import MIX, _check

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _the_largest_alone_from_a_floor_of_one(monkeypatch):
    """exp(-d) is below 1 for every d > 0, but 1 in 64 bits for those below 2^-53: a floor of 1 keeps the largest logits alone."""
    plain = S.sample_weights

    def weights(z, t, k, p, floor):
        w = plain(z, t, k, p, floor)
        return np.where(z == np.nanmax(z), w, 0.0) if floor >= 1 else w

    monkeypatch.setattr(S, "sample_weights", weights)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("vocab", [300, 1000, 1500, 2041, 2047, 2048, 2049])
def test_many_candidates_of_one_bin(vocab, f32):
    announce(f"sample small vocab={vocab} f32={f32}")
    rng = np.random.default_rng(vocab)
    low = -3.4028234663852886e38 if f32 else -3.3895313892515355e38
    z = rng.standard_normal((16, vocab))
    z[1] = 20 + 0.01 * z[1]                                      # within half an octave
    z[2] = np.where(rng.random(vocab) < 0.9, low, 20 + z[2])     # and far below
    z[3] = np.where(rng.random(vocab) < 0.5, low, 1.0)           # two values
    z[4] = 3.0                                                   # one
    z[5] = np.where(np.arange(vocab) == vocab // 2, 9.0, -2.0)   # one above equal ones
    z[6] = np.where(rng.random(vocab) < 0.7, -np.inf, z[6])
    z[7] = np.round(z[7])
    z[8] *= 1e-30
    z[9] = np.where(rng.random(vocab) < 0.3, np.nan, 100 * z[9])
    z[10, :5] = np.inf
    z[11] = np.linspace(-30, 30, vocab)
    z[12] = np.exp(3 * z[12])
    z[13] = -np.exp(3 * z[13])
    asked = MIX + [(1.0, vocab - 1, 0.6, 0.0), (0.01, 40, 1.0, 0.0), (0.01, vocab // 2, 0.5, 0.0), (50.0, vocab // 3, 0.9, 0.0), (1.0, 260, 1.0, 0.5)]
    for i in range(0, len(asked), 3):
        with np.errstate(over="ignore"):
            _check(z, [asked[(r + i) % len(asked)] for r in range(16)], rng.random(16), f32, pad=i % 5, offset=i % 3)
