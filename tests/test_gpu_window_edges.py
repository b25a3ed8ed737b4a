"""The window and 8-bit cache operators where their numbers are at an end: blocks that grow from a scale of 0."""
import numpy as np
import pytest

from tests.gpu_util import announce
from tests.test_gpu_kv8_write import Cache, make_plan, same_codes, tables, write
from tests.window_util import bf16, code_values, make_case, round_code, to_codes

pytestmark = pytest.mark.gpu

WRITE = (2, 1, 128, 8, 64)  # q and kv heads, head_dim, rotated pairs of dims 0-7 and 64-71


def steps_of(lens, shape, kv, cache, cos, sin, *steps):
    """Writes each (k, v) of `steps` as the tokens of `lens` in turn on the pages of one sequence."""
    whole = make_case(1, [(0, 64)])
    for (c, n), (k, v) in zip(lens, steps):
        case = make_case(1, [(c, n)])
        case.table.base_rows, case.pages, case.rows = list(whole.pages[0]), whole.pages, whole.rows
        q = np.ones((n, shape[0], shape[2]), dtype=np.float32)
        write(make_plan(case, shape, 32), cache, q, k, v, None, cos, sin, shape)
    return whole


@pytest.mark.parametrize("kv", ["e4m3", "int8"])
def test_a_block_that_grows_from_a_scale_of_zero(kv):
    """Rows of zeros, infinities and NaN, then a token with a scale: what was worth 0 stays worth 0, NaN stays NaN in e4m3."""
    announce(f"kv8 growth from zero {kv}")
    rng = np.random.default_rng(2)
    zero = np.zeros((2, 1, 128), dtype=np.float32)
    zero[0, 0, 20], zero[0, 0, 21], zero[1, 0, 22], zero[1, 0, 23] = np.inf, -np.inf, np.nan, np.inf
    token = bf16(rng.standard_normal((1, 1, 128)))
    cos, sin = tables(make_case(1, [(0, 64)]), 8)
    cache = Cache(4 * 64, 1, 128, kv, 32, 3)
    whole = steps_of([(32, 2), (34, 1)], WRITE, kv, cache, cos, sin, (zero, zero), (token, token))
    row = whole.row(0, np.arange(32, 35))
    for i in range(2):
        raw, scales = cache.got(i)
        assert scales[row[0] // 32, 0] > 0
        held = code_values(raw[row], kv)
        old = held[:2].copy()
        if kv == "e4m3":
            assert np.isnan(old[1, 22])
            old[1, 22] = 0.0
        assert (old == 0.0).all(), np.argwhere(old != 0.0).tolist()
        s = float(scales[row[0] // 32, 0])
        if i == 1:
            same_codes(raw[row[2]], to_codes(round_code(token[0, 0] / np.float64(s), kv), kv), kv, "token")
