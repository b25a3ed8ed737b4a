"""Products with 4-bit weights and group scales against the same sums in 64 bits."""
import numpy as np
import pytest

from inferno_amd import attention as A
from inferno_amd._lib import InfernoHipError
from tests import step_util as S
from tests.gpu_util import announce, empty_dev, from_dev, to_dev

pytestmark = pytest.mark.gpu


def _run(x, codes, scales, group, fmt, workspace=True):
    m, k = x.shape
    n = codes.shape[0]
    guard = 64
    out = to_dev(np.full(m * n + guard, 0x4242, np.uint16))
    ws = A.w4_gemm_workspace(n, k, m) if workspace else None
    if ws is not None:
        ws.fill_(float("nan"))
    A.dispatch_w4_gemm_cols(to_dev(x), to_dev(codes), to_dev(scales), out, rows=n, cols=k, seq_len=m,
                            group=group, w_format=fmt, workspace=ws)
    got = from_dev(out, np.uint16)
    assert np.all(got[m * n:] == 0x4242)
    return got[:m * n].reshape(m, n)


def _check(x, codes, scales, group, fmt):
    got = S.f64(_run(x, codes, scales, group, fmt))
    xf, w = S.f64(x), S.w4_weight(codes, scales, group, fmt)
    exact = xf @ w.T
    bad = np.abs(got - exact) - S.w4_bound(xf, w, exact, group)
    assert np.all(bad <= 0), (float(bad.max()), np.argwhere(bad > 0)[:5])


SHAPES = [(1, 1, 128), (1, 16, 128), (1, 2816, 4096), (2, 17, 256), (3, 65, 384), (4, 48, 1024),
          (5, 33, 2816), (7, 300, 640), (8, 31, 8192), (15, 100, 1152), (16, 2816, 8192),
          (17, 50, 512), (31, 257, 2816), (32, 80, 4096), (33, 511, 1280), (48, 64, 128),
          (61, 2816, 4096), (64, 1000, 256), (65, 130, 2816), (100, 257, 512), (127, 96, 384),
          (128, 128, 128), (129, 129, 1024), (200, 2816, 640), (255, 63, 2816), (300, 400, 4096),
          (513, 2816, 512), (1000, 1111, 896), (2050, 300, 256),
          # Many columns: streams of weights, one to 64 tokens, odd steps and x in more than one chunk.
          (1, 32768, 256), (4, 33001, 384), (3, 40000, 128), (2, 32769, 16512), (5, 32800, 384), (16, 33333, 640), (17, 32768, 256),
          (32, 32999, 896), (33, 32770, 512), (64, 40001, 384)]


@pytest.mark.parametrize("fmt", ["int4", "e2m1"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_against_64_bits(m, n, k, group, fmt):
    announce(f"w4 m={m} n={n} k={k} group={group} {fmt}")
    _check(*S.random_w4(np.random.default_rng(m * 31 + n + k + group), m, n, k, group), group, fmt)


@pytest.mark.parametrize("fmt", ["int4", "e2m1"])
@pytest.mark.parametrize("m", [1, 16, 40, 64, 150, 700])
def test_integer_sums_are_exact(m, fmt):
    """Small whole numbers under scales of powers of two: every sum is exact, so the output is its one
    rounding; all sixteen codes at every place of a word."""
    announce(f"w4 exact m={m} {fmt}")
    rng = np.random.default_rng(m)
    n, k, group = 272, 1024, 64
    x = rng.integers(-4, 5, (m, k)).astype(np.float32)
    codes = rng.integers(0, 256, (n, k // 2), dtype=np.uint8)
    scales = S.f32_to_bf16(2.0 ** rng.integers(-2, 3, (n, k // group)))
    got = _run(S.f32_to_bf16(x), codes, scales, group, fmt)
    exact = x.astype(np.float64) @ S.w4_weight(codes, scales, group, fmt).T
    assert np.array_equal(got, S.f32_to_bf16(exact.astype(np.float32)))


@pytest.mark.parametrize("fmt", ["int4", "e2m1"])
@pytest.mark.parametrize("m,n,k,group", [(1, 64, 256, 32), (20, 64, 256, 64), (200, 64, 256, 128), (300, 130, 512, 32)])
def test_each_column_and_group_by_itself(m, n, k, group, fmt):
    """x of one 1 a token and codes and scales that differ at every place: an output is one weight."""
    announce(f"w4 single columns m={m} {fmt} group={group}")
    rng = np.random.default_rng(m + group)
    cols = rng.permutation(np.tile(np.arange(k), -(-m // k))[:m]) if m > 1 else np.array([k - 1])
    x = np.zeros((m, k), np.float32)
    x[np.arange(m), cols] = 1
    codes = rng.integers(0, 256, (n, k // 2), dtype=np.uint8)
    scales = S.f32_to_bf16(rng.standard_normal((n, k // group)))
    got = _run(S.f32_to_bf16(x), codes, scales, group, fmt)
    want = S.w4_weight(codes, scales, group, fmt)[:, cols].T  # a code times a scale: exact in f32
    assert np.array_equal(S.f64(got), S.f64(S.f32_to_bf16(want.astype(np.float32))))


@pytest.mark.parametrize("m", [1, 16, 33, 64, 130])
def test_infinities_and_nan_stay_in_their_token_and_row(m):
    announce(f"w4 special values m={m}")
    rng = np.random.default_rng(m)
    n, k, group = 80, 512, 64
    x, codes, scales = S.random_w4(rng, m, n, k, group)
    clean = _run(x, codes, scales, group, "int4")
    x2, s2 = x.copy(), scales.copy()
    row = m // 2
    x2[row, 77] = 0x7F80   # +inf: inf * code is +-inf, or NaN where the code is 0
    s2[5, 3] = 0x7FC0      # a NaN scale
    got = _run(x2, codes, s2, group, "int4")
    keep = np.ones((m, n), bool)
    keep[row], keep[:, 5] = False, False
    assert np.array_equal(got[keep], clean[keep])
    assert np.all(np.isnan(S.f64(got[:, 5])))
    c = S.INT4[(codes[:, 77 // 2] >> 4) & 15] * S.f64(scales[:, 1])
    want = np.where(c == 0, np.nan, np.where(c > 0, np.inf, -np.inf))
    seen = np.delete(np.arange(n), 5)
    assert np.array_equal(S.f64(got[row])[seen], want[seen], equal_nan=True)


@pytest.mark.parametrize("m", [1, 64, 200])
def test_scales_of_any_size(m):
    """Zero, negative, the smallest and large scales; codes of only the largest value."""
    announce(f"w4 scales m={m}")
    rng = np.random.default_rng(m + 5)
    n, k, group = 96, 256, 32
    x, codes, _ = S.random_w4(rng, m, n, k, group)
    pick = np.array([0.0, -0.0, 1e-30, -1e-30, 3e30, -2e30, 1.0, -1.0, 2.0 ** -126, 2.0 ** -133])
    scales = S.f32_to_bf16(pick[rng.integers(0, 4, (n, k // group))])
    big = S.f32_to_bf16(pick[rng.integers(4, 8, (n, k // group))])
    for s in (scales, big):
        _check(x, codes, s, group, "int4")
        _check(x, codes, s, group, "e2m1")
    _check(x, np.full_like(codes, 0x88), big, group, "int4")
    _check(x, np.full_like(codes, 0xF7), big, group, "e2m1")


def test_no_tokens():
    out = to_dev(np.full(64, 0x4242, np.uint16))
    A.dispatch_w4_gemm_cols(out, empty_dev(64 * 64, np.uint8), empty_dev(64, np.uint16), out, rows=64, cols=128, seq_len=0,
                            group=128, w_format="int4")
    assert np.all(from_dev(out, np.uint16) == 0x4242)


@pytest.mark.parametrize("m,n,k", [(1, 2816, 4096), (16, 2816, 8192), (64, 1000, 2816), (300, 2816, 2816)])
def test_captured_and_on_another_stream(m, n, k):
    """Replays with other inputs in the same buffers and eager work of the same kind in between."""
    import torch

    announce(f"w4 graph m={m}")
    rng = np.random.default_rng(k)
    group, fmt = 64, "e2m1"
    x, codes, scales = S.random_w4(rng, m, n, k, group)
    xs = [x] + [np.roll(x, i + 1, axis=1) for i in range(3)]
    want = [_run(v, codes, scales, group, fmt) for v in xs]
    dx, dc, ds = to_dev(x), to_dev(codes), to_dev(scales)
    out, ws = empty_dev(m * n, np.uint16), A.w4_gemm_workspace(n, k, m)

    def call():
        A.dispatch_w4_gemm_cols(dx, dc, ds, out, rows=n, cols=k, seq_len=m, group=group, w_format=fmt, workspace=ws)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
    stream.synchronize()
    assert np.array_equal(from_dev(out, np.uint16).reshape(m, n), want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in (1, 2, 3, 0):
        dx.copy_(to_dev(xs[i]))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(from_dev(out, np.uint16).reshape(m, n), want[i]), i
        assert np.array_equal(_run(xs[0], codes, scales, group, fmt), want[0])
    del graph


def test_refusals():
    x, codes, scales, out = (empty_dev(n, t) for n, t in ((4 * 256, np.uint16), (64 * 128, np.uint8), (64 * 8, np.uint16), (4 * 64, np.uint16)))

    def call(**kw):
        args = dict(rows=64, cols=256, seq_len=4, group=32, w_format="int4")
        t = dict(x=x, codes=codes, scales=scales, output=out)
        t.update({k: kw.pop(k) for k in list(kw) if k in t})
        A.dispatch_w4_gemm_cols(t["x"], t["codes"], t["scales"], t["output"], **{**args, **kw})

    call()
    for bad in (dict(group=48), dict(w_format="int8"), dict(rows=65), dict(seq_len=5), dict(x=x.cpu()), dict(scales=codes),
                dict(codes=codes.view(64, 128)[:, ::2]), dict(x=x.float()), dict(output=out.half())):
        with pytest.raises(ValueError):
            call(**bad)
    for bad in (dict(cols=192), dict(rows=0), dict(cols=0), dict(x=x[1:], seq_len=3), dict(seq_len=-1)):
        with pytest.raises(InfernoHipError):
            call(**bad)


@pytest.mark.parametrize("m,k", [(61, 4096), (300, 4096), (16, 8192)])
def test_calls_at_once_and_graphs_that_share_a_workspace(m, k):
    """Two streams with a workspace each; then two graphs over one workspace, replayed in turn."""
    import torch

    announce(f"w4 at once m={m} k={k}")
    n, group, fmt = 2816, 64, "int4"
    cases = [S.random_w4(np.random.default_rng(s), m, n, k, group) for s in (1, 2)]
    want = [_run(*c, group, fmt) for c in cases]
    dev = [[to_dev(t) for t in c] for c in cases]
    outs = [empty_dev(m * n, np.uint16) for _ in cases]
    spaces = [A.w4_gemm_workspace(n, k, m) for _ in cases]
    assert spaces[0] is not None
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()

    def call(i, ws):
        A.dispatch_w4_gemm_cols(*dev[i], outs[i], rows=n, cols=k, seq_len=m, group=group, w_format=fmt, workspace=ws)

    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                call(i, spaces[i])
    torch.cuda.synchronize()
    for i in range(2):
        assert np.array_equal(from_dev(outs[i], np.uint16).reshape(m, n), want[i])
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(i, spaces[0])
        graphs.append(g)
    for i in (0, 1, 1, 0, 1):
        outs[i].zero_()
        graphs[i].replay()
        torch.cuda.synchronize()
        assert np.array_equal(from_dev(outs[i], np.uint16).reshape(m, n), want[i])
    del graphs


@pytest.mark.parametrize("m,n,k", [(8, 300, 8320), (16, 65, 16384), (5, 2816, 12288), (64, 48, 32768), (2, 20000, 512), (16, 20000, 256),
                                   (3, 6000, 8192), (90, 16, 65536), (130, 2816, 8192), (1, 3, 131072)])
def test_long_rows_and_other_plans(m, n, k):
    """Past the sizes of the other tests: spans of long rows, the columns between the kernels' ranges."""
    announce(f"w4 long m={m} n={n} k={k}")
    for group, fmt in ((32, "int4"), (128, "e2m1")):
        _check(*S.random_w4(np.random.default_rng(m + n + k), m, n, k, group), group, fmt)


def test_a_workspace_that_is_too_small():
    x, codes, scales, out = (empty_dev(n, t) for n, t in ((64 * 4096, np.uint16), (2816 * 2048, np.uint8), (2816 * 128, np.uint16), (64 * 2816, np.uint16)))
    ws = A.w4_gemm_workspace(2816, 4096, 64)
    args = dict(rows=2816, cols=4096, seq_len=64, group=32, w_format="int4")
    A.dispatch_w4_gemm_cols(x, codes, scales, out, workspace=ws, **args)
    for bad in (None, ws[:-1], ws[1:]):
        with pytest.raises(InfernoHipError):
            A.dispatch_w4_gemm_cols(x, codes, scales, out, workspace=bad, **args)
