"""Norms around a block over more rows than one launch takes: its grid has less than 2^32 threads."""
import pytest

from inferno_amd import attention as A
from tests.gpu_util import announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,hidden,per_launch", [(1 << 24, 1032, 2 ** 24 - 1), ((1 << 22) + 2, 8200, 2 ** 22 - 1)])
def test_rows_past_one_launch(rows, hidden, per_launch):
    """In place (70 and 140 GB); the rows looked at lie around the launches' ends, the others hold anything.  Each is as in a
    call of its own few rows."""
    import torch

    announce(f"norm_residual rows={rows} hidden={hidden}")
    at = [0, 1, rows // 2, per_launch - 1, *range(per_launch, rows)]
    gen = torch.Generator(device="cuda").manual_seed(hidden)

    def normal(*size):
        return torch.randn(*size, generator=gen, device="cuda").to(torch.bfloat16)

    y, r, gate, post, pre = normal(len(at), hidden), normal(len(at), hidden), normal(hidden), normal(hidden), normal(hidden)
    keep = dict(hidden=hidden, eps=1e-6, post_weight=post, gate=gate, pre_weight=pre, residual_scale=0.75, block_scale=0.5)
    want_r, want_x = torch.empty_like(r), torch.empty_like(y)
    A.dispatch_norm_residual(y, r, want_r, want_x, seq_len=len(at), **keep)
    big_y, big_r = (torch.empty(rows, hidden, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    for i, row in enumerate(at):
        big_y[row], big_r[row] = y[i], r[i]
    A.dispatch_norm_residual(big_y, big_r, big_r, big_y, seq_len=rows, **keep)
    torch.cuda.synchronize()
    for i, row in enumerate(at):
        assert torch.equal(big_r[row], want_r[i]) and torch.equal(big_y[row], want_x[i]), row
    del big_y, big_r
    torch.cuda.empty_cache()
