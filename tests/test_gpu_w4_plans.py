"""Every launch of the 4-bit products (tests/w4_plans.py) in both formats and all groups against sums in 64 bits: wide heads,
rows of more steps than a window of scales has, spans whose last one is shorter, both tiles."""
import pytest

from inferno_amd import attention as A
from tests import step_util as S
from tests.gpu_util import announce
from tests.w4_plans import PLANS, plan

pytestmark = pytest.mark.gpu


def _weight(codes, scales, group, fmt):
    """Some rows of the weight in 64 bits, on the GPU."""
    import torch

    table = torch.tensor(S.VALUES[fmt], dtype=torch.float64, device="cuda")
    w = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device="cuda")
    w[:, 0::2], w[:, 1::2] = table[(codes & 15).long()], table[(codes >> 4).long()]
    return w.view(codes.shape[0], -1, group).mul_(scales.double()[..., None]).view(codes.shape[0], -1)


@pytest.mark.parametrize("fmt", ["int4", "e2m1"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("shape", PLANS, ids=str)
def test_against_64_bits(shape, group, fmt):
    """The bound is that of step_util.w4_bound."""
    import torch

    announce(f"w4 plan {shape} group={group} {fmt}")
    assert plan(*shape) == PLANS[shape]
    m, n, k = shape
    gen = torch.Generator(device="cuda").manual_seed(m + n + k + group)

    def normal(*size):
        return torch.randn(*size, generator=gen, device="cuda")

    x = (normal(m, k) * torch.exp(0.7 * normal(k))).to(torch.bfloat16)
    codes = torch.randint(0, 256, (n, k // 2), generator=gen, device="cuda", dtype=torch.uint8)
    scales = (0.01 * torch.exp(0.5 * normal(n, k // group))).to(torch.bfloat16)
    guard = 64
    out = torch.full((m * n + guard,), 7.0, device="cuda", dtype=torch.bfloat16)
    ws = A.w4_gemm_workspace(n, k, m)
    if ws is not None:
        ws.fill_(float("nan"))
    A.dispatch_w4_gemm_cols(x, codes, scales, out, rows=n, cols=k, seq_len=m, group=group, w_format=fmt, workspace=ws)
    assert bool((out[m * n:] == 7.0).all())
    got = out[:m * n].view(m, n)
    xf = x.double()
    steps = k + k // group + 2
    for n0 in range(0, n, max(1, (1 << 26) // k)):
        rows = slice(n0, n0 + max(1, (1 << 26) // k))
        w = _weight(codes[rows], scales[rows], group, fmt)
        exact = xf @ w.t().contiguous()
        bound = 2.0 ** -8 * exact.abs() + steps * 2.0 ** -23 * (xf.abs() @ w.abs().t().contiguous()) + 2.0 ** -133
        over = (got[:, rows].double() - exact).abs() - bound
        assert bool((over <= 0).all()), (n0, float(over.max()), int((over > 0).sum()))


def test_the_same_bits_every_time():
    """A launch of each kind with work of other kinds between: sums are taken in an order of their own, never in that of time."""
    import torch

    announce("w4 repeated")
    gen = torch.Generator(device="cuda").manual_seed(7)
    n, k = 2816, 4096
    codes = torch.randint(0, 256, (n, k // 2), generator=gen, device="cuda", dtype=torch.uint8)
    scales = (0.01 * torch.randn(n, k // 64, generator=gen, device="cuda")).to(torch.bfloat16)
    x = torch.randn(300, k, generator=gen, device="cuda").to(torch.bfloat16)
    seen = {}
    for i in range(8):
        for m in (1, 4, 16, 17, 61, 65, 300):
            out, ws = torch.empty(m, n, device="cuda", dtype=torch.bfloat16), A.w4_gemm_workspace(n, k, m)
            A.dispatch_w4_gemm_cols(x, codes, scales, out, rows=n, cols=k, seq_len=m, group=64, w_format="int4", workspace=ws)
            assert torch.equal(seen.setdefault(m, out), out), (i, m)
