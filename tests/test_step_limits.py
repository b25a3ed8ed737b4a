"""Sizes that the entry points behind the attention take, against what one launch takes (a grid has less than 2^32 threads);
every call here ends in an argument check."""
import pytest

from inferno_amd import _lib
from tests.test_step_refusals import EINVAL, sample


@pytest.mark.parametrize("kind,fits,past", [(1, 15 * 4096 - 7, 15 * 4096), (0, 15 * 8192 - 7, 15 * 8192)])
def test_sample_grid(kind, fits, past):
    """2^20 rows of 15 pieces of 16 KiB, and of 16: 2^24 workgroups of 256 threads.  (min_p in the place of the tokens ends the
    call that fits.)"""
    rows, far = 1 << 20, 1 << 50
    args = dict(rows=rows, kind=kind, uniform=2 * far, tokens=3 * far, min_p=3 * far, workspace=4 * far, workspace_bytes=1 << 48)
    assert sample(vocab=past, stride=past, **args) == EINVAL and "pieces" in _lib.last_error()
    assert sample(vocab=fits, stride=fits, **args) == EINVAL and "overlap" in _lib.last_error()
    assert sample(vocab=1 << 15, stride=1 << 15, **args) == EINVAL and "overlap" in _lib.last_error()  # the 2^35 of the header
    assert sample(vocab=1 << 20, stride=1 << 20, **{**args, "rows": 1 << 15}) == EINVAL and "overlap" in _lib.last_error()
