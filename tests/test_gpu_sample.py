"""Sampling with temperature, top-k, top-p and min-p: the token of every row is the one of the
definition in 64 bits.  Numbers u and top_p are taken away from borders between two tokens (1e-9 of
the whole), so that the token does not hang on the rounding of the reference's sums."""
import numpy as np
import pytest

from inferno_amd import attention as A
from inferno_amd._lib import InfernoHipError
from tests import step_util as S
from tests.gpu_util import announce, empty_dev, from_dev, to_dev

pytestmark = pytest.mark.gpu

CLEAR = 1e-9
OFF = (1.0, 0, 1.0, 0.0)


def _clear_top_p(z, t, k, p):
    """A top_p near p whose cut lies clear of the sums of the ordered weights."""
    if not p < 1 or not t > 0:
        return p
    w = np.sort(S.sample_weights(z, t, k, 1.0, 0.0))[::-1]
    if w[0] == 0:
        return p
    sums = np.cumsum(w) / w.sum()
    for _ in range(100):
        p = float(np.float32(p))
        if np.min(np.abs(sums - p)) > CLEAR:
            return p
        p = p * (1 - 1e-5)
    raise AssertionError("no clear top_p")


def _prepare(z, asked, u):
    """(asked with clear cuts, clear u, tokens) for rows z (64 bits)."""
    out, us, want = [], [], []
    for row, (t, k, p, floor), v in zip(z, asked, u):
        t, floor = float(np.float32(t)), float(np.float32(floor))
        p = _clear_top_p(row, t, k, p)
        w = S.sample_weights(row, t, k, p, floor)
        for _ in range(1000):
            v = float(np.float32(v))
            token, gap = S.sample_token(w, v)
            if gap > CLEAR or not 0 < v < 1:
                break
            v = (v * 0.731 + 0.1237) % 1.0
        else:
            raise AssertionError("no clear u")
        out.append((t, k, p, floor))
        us.append(v)
        want.append(token)
    return out, us, want


def _logits(z, f32):
    """(device bits, the values they hold)."""
    if f32:
        b = np.asarray(z, np.float32)
        return b, b.astype(np.float64)
    b = S.f32_to_bf16(z)
    return b, S.f64(b)


def _call(bits, vocab, stride, asked, u, offset=0, use=(1, 1, 1, 1)):
    rows = len(u)
    flat = to_dev(bits)[offset:]
    cols = list(zip(*asked))
    args = [to_dev(np.array(c, np.int32 if i == 1 else np.float32)) if use[i] else None for i, c in enumerate(cols)]
    tokens = to_dev(np.full(rows + 8, -7, np.int32))
    ws = A.sample_workspace(rows, vocab)
    if ws is not None:
        ws.fill_(float("nan"))
    A.dispatch_sample_tokens(flat, to_dev(np.array(u, np.float32)), tokens, ws, num_rows=rows, vocab=vocab, row_stride=stride,
                             temperature=args[0], top_k=args[1], top_p=args[2], min_p=args[3])
    got = from_dev(tokens, np.int32)
    assert np.all(got[rows:] == -7)
    return got[:rows]


def _check(z, asked, u, f32, pad=0, offset=0):
    z = np.atleast_2d(np.asarray(z, np.float64))
    rows, vocab = z.shape
    bits, held = _logits(z, f32)
    asked, u, want = _prepare(held, asked, u)
    buf = np.full(offset + rows * (vocab + pad), 0x7F01 if not f32 else 1e38, bits.dtype)  # large between the rows
    buf[offset:].reshape(rows, vocab + pad)[:, :vocab] = bits
    got = _call(buf, vocab, vocab + pad, asked, u, offset)
    assert np.array_equal(got, want), [(r, int(got[r]), want[r], asked[r], u[r]) for r in np.flatnonzero(got != want)[:5]]
    assert np.array_equal(_call(buf, vocab, vocab + pad, asked, u, offset), got)


MIX = [(0.8, 64, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 0.95, 0.0), (0.7, 20, 0.8, 0.02), (1.2, 0, 1.0, 0.05), (1.0, 1, 1.0, 0.0), OFF,
       (1.5, 500, 0.99, 0.0), (1.0, 0, 0.3, 0.1), (2.0, 3000, 0.999, 0.0), (1.0, 1025, 1.0, 0.0), (0.3, 0, 0.9999, 0.0), (1.0, 0, 0.0, 0.0),
       (1.0, 5, -1.0, 0.0), (1.0, 0, 1.0, 1.0), (1.0, 10 ** 6, 0.5, 0.0)]


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("kind", ["peaked", "flat", "gauss"])
@pytest.mark.parametrize("vocab,pad,offset", [(1, 0, 0), (2, 1, 1), (7, 0, 3), (63, 5, 0), (64, 0, 0), (65, 0, 1), (255, 3, 2), (256, 0, 0),
                                              (257, 0, 0), (1000, 7, 5), (4099, 0, 0), (32001, 1, 7), (262144, 0, 0), (262141, 3, 1)])
def test_the_token_of_the_definition(vocab, pad, offset, kind, f32):
    announce(f"sample vocab={vocab} pad={pad} offset={offset} {kind} f32={f32}")
    rng = np.random.default_rng(vocab + 7 * pad)
    rows = 2 * len(MIX) if vocab < 100000 else len(MIX)
    z = {"peaked": lambda: rng.exponential(1.6, (rows, vocab)) - 4, "gauss": lambda: rng.standard_normal((rows, vocab)) * 2.5,
         "flat": lambda: rng.standard_normal((rows, vocab)) * 0.01}[kind]()
    _check(z, [MIX[r % len(MIX)] for r in range(rows)], rng.random(rows), f32, pad, offset)


@pytest.mark.parametrize("f32", [False, True])
def test_ties_go_to_the_lowest_index(f32):
    """Few different values: the cuts of top-k and top-p fall among equal logits, a few and very many."""
    announce(f"sample ties f32={f32}")
    rng = np.random.default_rng(4)
    for vocab in (9, 300, 5000, 70000):
        z = rng.integers(0, 4, (32, vocab)).astype(np.float64)
        z[0], z[1] = 0, -3.0
        z[2] = np.where(np.arange(vocab) % 2, 0.0, -0.0)  # -0 is 0
        asked = [(1.0, 2, 1.0, 0.0), (1.0, 5, 1.0, 0.0), (1.0, vocab // 2 + 1, 1.0, 0.0), (1.0, 0, 0.37, 0.0), (1.0, 7, 0.61, 0.0),
                 (1.0, vocab - 1, 0.93, 0.0), (1.0, 0, 1.0, 0.5), (0.0, 0, 1.0, 0.0)]
        _check(z, [asked[r % 8] for r in range(32)], rng.random(32), f32)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("vocab", [70, 3000, 40000])
def test_masked_rows(vocab, f32):
    """-inf, NaN, the type's lowest value and +inf among the logits; rows that a mask leaves nothing of."""
    announce(f"sample masked vocab={vocab} f32={f32}")
    rng = np.random.default_rng(vocab)
    low = -3.4028234663852886e38 if f32 else -3.3895313892515355e38
    z = rng.standard_normal((20, vocab)) * 3
    hide = rng.random((20, vocab)) < 0.9
    z[0:4] = np.where(hide[0:4], -np.inf, z[0:4])
    z[4:8] = np.where(hide[4:8], low, z[4:8])
    z[8] = -np.inf
    z[9] = np.nan
    z[10] = low
    z[11] = np.where(hide[11], np.nan, z[11])
    z[12, [3, 50, 60]] = np.inf
    z[13] = np.inf
    z[14] = -np.inf
    z[14, 66] = low
    z[15] = np.where(np.arange(vocab) < 3, -1.0, -np.inf)  # fewer than top-k
    z[16] = np.where(np.arange(vocab) < 3, -1.0, low)
    z[17] = -np.inf
    z[17, vocab - 1] = np.inf
    z[18, 0] = 3e38
    z[19] = -3e38
    for asked in (OFF, (0.8, 64, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 0, 1.0, 0.2), (1e-30, 5, 1.0, 0.0),
                  (1e30, 0, 1.0, 0.0), (1e-45, 0, 0.5, 0.0), (float("inf"), 0, 1.0, 0.0), (float("inf"), 9, 1.0, 0.0)):
        with np.errstate(over="ignore"):
            _check(z, [asked] * 20, rng.random(20), f32)


def test_numbers_at_the_ends_and_outside():
    announce("sample ends")
    rng = np.random.default_rng(8)
    z = rng.standard_normal((1, 5000)) * 2
    u = [0.0, 1 - 2.0 ** -24, 1.0, 2.0, -1.0, float("nan"), float("inf"), -float("inf"), 1e-30, 0.5]
    for asked in (OFF, (1.0, 50, 1.0, 0.0), (1.0, 0, 0.9, 0.0)):
        _check(np.repeat(z, 10, 0), [asked] * 10, u, True)
    # Parameters that switch their part off.
    nan = float("nan")
    for off in ((1.0, -5, 1.0, 0.0), (1.0, 0, 2.0, 0.0), (1.0, 0, nan, 0.0), (1.0, 0, 1.0, -1.0), (1.0, 0, 1.0, nan)):
        _check(z, [off], [0.37], True)
    for greedy in ((-1.0, 0, 1.0, 0.0), (nan, 0, 1.0, 0.0), (-0.0, 9, 0.5, 0.1)):
        _check(z, [greedy], [0.37], True)


def test_numbers_that_are_not_passed():
    announce("sample without parameters")
    rng = np.random.default_rng(9)
    bits, held = _logits(rng.exponential(1.6, (6, 3000)), True)
    for use in ((0, 0, 0, 0), (1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1)):
        asked = [tuple(v if on else off for v, on, off in zip((0.7, 30, 0.8, 0.02), use, OFF))] * 6
        asked, u, want = _prepare(held, asked, rng.random(6))
        assert list(_call(bits.ravel(), 3000, 3000, asked, u, use=use)) == want


def test_rows_of_a_matrix_apart():
    """Without row_stride a matrix gives it, also as a view."""
    announce("sample strided view")
    rng = np.random.default_rng(10)
    full = rng.exponential(1.6, (9, 1100)).astype(np.float32)
    asked, u, want = _prepare(full[:, 50:1050].astype(np.float64), [(0.9, 40, 0.9, 0.0)] * 9, rng.random(9))
    view = to_dev(full)[:, 50:1050]
    tokens = empty_dev(9, np.int32)
    c = [to_dev(np.array(v, np.int32 if i == 1 else np.float32)) for i, v in enumerate(zip(*asked))]
    A.dispatch_sample_tokens(view, to_dev(np.array(u, np.float32)), tokens, A.sample_workspace(9, 1000), num_rows=9, vocab=1000,
                             temperature=c[0], top_k=c[1], top_p=c[2], min_p=c[3])
    assert list(from_dev(tokens, np.int32)) == want
    for bad in (dict(vocab=1001), dict(num_rows=10)):
        with pytest.raises(ValueError):
            A.dispatch_sample_tokens(view, to_dev(np.zeros(16, np.float32)), empty_dev(16, np.int32), A.sample_workspace(16, 1200),
                                     **{**dict(num_rows=9, vocab=1000), **bad})
    with pytest.raises(ValueError):
        A.dispatch_sample_tokens(view.t(), to_dev(np.zeros(1000, np.float32)), empty_dev(1000, np.int32), None, num_rows=9, vocab=9)


def test_the_largest_vocabulary():
    announce("sample vocab 2^20")
    rng = np.random.default_rng(12)
    z = rng.standard_normal((6, 1 << 20)) * 2
    _check(z, [OFF, (1.0, 64, 0.9, 0.0), (1.0, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.01), (1.0, 100000, 0.99, 0.0), (0.0, 0, 1.0, 0.0)], rng.random(6), True)


def test_captured_and_on_another_stream():
    import torch

    announce("sample graph")
    rng = np.random.default_rng(13)
    rows, vocab = 16, 50001
    sets = []
    for _ in range(3):
        bits, held = _logits(rng.exponential(1.6, (rows, vocab)), False)
        asked, u, want = _prepare(held, [MIX[r % len(MIX)] for r in range(rows)], rng.random(rows))
        sets.append((bits, asked, u, want))
    z, du = to_dev(sets[0][0]), to_dev(np.array(sets[0][2], np.float32))
    cols = [to_dev(np.array(c, np.int32 if i == 1 else np.float32)) for i, c in enumerate(zip(*sets[0][1]))]
    tokens, ws = empty_dev(rows, np.int32), A.sample_workspace(rows, vocab)

    def call():
        A.dispatch_sample_tokens(z, du, tokens, ws, num_rows=rows, vocab=vocab, row_stride=vocab, temperature=cols[0], top_k=cols[1],
                                 top_p=cols[2], min_p=cols[3])

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
    stream.synchronize()
    assert list(from_dev(tokens, np.int32)) == sets[0][3]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in (1, 2, 0, 1):
        bits, asked, u, want = sets[i]
        z.copy_(to_dev(bits))
        du.copy_(to_dev(np.array(u, np.float32)))
        for d, (j, c) in zip(cols, enumerate(zip(*asked))):
            d.copy_(to_dev(np.array(c, np.int32 if j == 1 else np.float32)))
        tokens.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert list(from_dev(tokens, np.int32)) == want, i
        assert list(_call(sets[0][0].ravel(), vocab, vocab, sets[0][1], sets[0][2])) == sets[0][3]
    del graph


def test_refusals():
    z, u, t = empty_dev(4 * 100, np.float32), empty_dev(4, np.float32), empty_dev(4, np.int32)
    ws = A.sample_workspace(4, 100)

    def call(z=z, u=u, t=t, ws=ws, **kw):
        A.dispatch_sample_tokens(z, u, t, ws, **{**dict(num_rows=4, vocab=100, row_stride=100), **kw})

    call()
    call(num_rows=0)
    for bad in (dict(num_rows=5), dict(u=u[:3]), dict(t=u), dict(u=t), dict(top_k=u), dict(temperature=t), dict(z=z.cpu()), dict(u=u.cpu()),
                dict(z=z.half()), dict(z=z.double())):
        with pytest.raises(ValueError):
            call(**bad)
    for bad in (dict(vocab=0), dict(row_stride=99), dict(num_rows=-1), dict(vocab=(1 << 20) + 1, num_rows=1, row_stride=1 << 21, z=empty_dev((1 << 20) + 1, np.float32))):
        with pytest.raises(InfernoHipError):
            call(**bad)


@pytest.mark.parametrize("f32", [False, True])
def test_rows_with_very_many_kept_tokens(f32):
    """Cuts among tens of thousands of tokens, equal ones among them, and thresholds that keep that many: the rows of the
    third launch, of odd lengths at odd addresses."""
    announce(f"sample wide rows f32={f32}")
    rng = np.random.default_rng(21)
    vocab = 150001
    z = rng.standard_normal((14, vocab)) * 2.5
    z[4:8] = rng.exponential(1.25, (4, vocab)) - 4
    z[8] = np.round(z[8] * 2) / 2          # some forty values
    z[9] = 1.0                             # one
    z[10] = np.where(rng.random(vocab) < 0.3, 2.0, 1.0)
    z[11, ::2] = -np.inf
    z[12] = np.linspace(5, -5, vocab)      # in order, which a sample of every n-th token sees well
    z[13] = np.where(np.arange(vocab) % 16 == 0, -20.0, z[13])  # and one that it sees badly
    asked = [(1.0, 0, p, floor) for p, floor in ((0.9, 0.0), (0.5, 0.0), (0.99, 1e-4), (0.05, 0.0))] * 3 + [(1.0, 0, 0.95, 0.0)] * 2
    _check(z, asked, rng.random(14), f32, pad=5, offset=3)
    _check(z, [(1.3, 0, 1.0, f) for f in (1e-3, 1e-2, 1e-4, 0.3, 1e-6, 1e-3, 0.05, 1e-5, 0.5, 0.9, 0.37, 0.01, 0.2, 1e-7)], rng.random(14), f32)
    _check(z, [(0.7, k, 0.97, 0.0) for k in (2000, 5000, 1024, 1025, 70000, 149999, 1500, 3000, 4000, 77777, 50000, 60000, 1100, 9000)],
           rng.random(14), f32, offset=1)


@pytest.mark.parametrize("f32", [False, True])
def test_candidates_among_equal_logits(f32):
    """Cuts of top-k and top-p that fall among hundreds of equal logits within the candidates."""
    announce(f"sample equal candidates f32={f32}")
    rng = np.random.default_rng(22)
    z = rng.standard_normal((8, 30000)) - 8
    for r in range(8):
        at = rng.permutation(30000)
        z[r, at[:5]] = 4.0
        z[r, at[5:5 + 150 * (r + 1)]] = 3.0
    _check(z, [(1.0, k, p, 0.0) for k, p in ((64, 1.0), (100, 0.9), (300, 0.5), (0, 0.8), (700, 0.999), (0, 0.5), (1000, 0.99), (1024, 0.7))],
           rng.random(8), f32)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("rows,vocab", [(1, 40003), (3, 8191), (5, 12289), (70, 40003), (128, 9000), (129, 9000)])
def test_rows_that_keep_many_among_few_and_many_rows(rows, vocab, f32):
    """The workgroups that share a row number from one to eight, by the rows and the vocabulary."""
    announce(f"sample parts rows={rows} vocab={vocab} f32={f32}")
    rng = np.random.default_rng(rows)
    z = rng.standard_normal((rows, vocab)) * 0.7
    z[1::4] = np.sort(z[1::4], axis=1)  # all that is kept in one part
    z[2::4, 5:] = -np.inf               # and in the first places
    asked = [[(1.0, 0, 0.9, 0.0), (1.0, 0, 1.0, 1e-3), (0.8, 0, 0.97, 1e-3), (1.0, 5000, 0.9, 0.0)][(r // 4) % 4] for r in range(rows)]
    _check(z, asked, rng.random(rows), f32, pad=3, offset=1)


@pytest.mark.parametrize("rows,every", [(300, 3), (300, 60), (40, 13)])
def test_a_few_rows_that_keep_many_in_a_batch(rows, every):
    """The rows that the third launch takes are dealt to its workgroups by how many there are."""
    announce(f"sample few left rows={rows} every={every}")
    rng = np.random.default_rng(every)
    vocab = 20001
    z = rng.standard_normal((rows, vocab)) * 0.7
    wide = [(1.0, 0, 0.9, 0.0), (1.0, 0, 1.0, 1e-3), (0.8, 0, 0.97, 1e-3), (1.0, 5000, 0.9, 0.0)]
    asked = [wide[(r // every) % 4] if r % every == every - 1 else (0.0, 0, 1.0, 0.0) if r % 2 else OFF for r in range(rows)]
    _check(z, asked, rng.random(rows), True)


def test_parts_of_a_row_meet_the_same_way_every_time():
    """Rows in eight parts each, call behind call into one workspace, the rows' order changing between them."""
    import torch

    announce("sample parts again")
    rng = np.random.default_rng(31)
    rows, vocab = 16, 100003
    bits, held = _logits(rng.standard_normal((rows, vocab)), True)
    asked, u, want = _prepare(held, [(1.0, 0, 0.9, 0.0), (1.0, 0, 1.0, 1e-3)] * (rows // 2), rng.random(rows))
    z, du = to_dev(bits), to_dev(np.array(u, np.float32))
    cols = [to_dev(np.array(c, np.int32 if i == 1 else np.float32)) for i, c in enumerate(zip(*asked))]
    tokens, ws = empty_dev(rows, np.int32), A.sample_workspace(rows, vocab)
    got = []
    for i in range(30):
        order = torch.from_numpy(np.roll(np.arange(rows), i)).to(z.device)
        one = [t[order].contiguous() for t in (z, du, *cols)]
        A.dispatch_sample_tokens(one[0], one[1], tokens, ws, num_rows=rows, vocab=vocab, temperature=one[2], top_k=one[3],
                                 top_p=one[4], min_p=one[5])
        got.append((i, tokens.clone()))
    for i, t in got:
        assert list(from_dev(t, np.int32)) == list(np.roll(want, i)), i


def test_calls_at_once_and_graphs_that_share_a_workspace():
    import torch

    announce("sample at once")
    rows, vocab = 24, 40000
    cases = []
    for s in (1, 2):
        rng = np.random.default_rng(s)
        bits, held = _logits(rng.exponential(1.3, (rows, vocab)) - 4, True)
        asked, u, want = _prepare(held, [MIX[r % len(MIX)] for r in range(rows)], rng.random(rows))
        cols = [to_dev(np.array(c, np.int32 if i == 1 else np.float32)) for i, c in enumerate(zip(*asked))]
        cases.append((to_dev(bits), to_dev(np.array(u, np.float32)), empty_dev(rows, np.int32), cols, want))
    spaces = [A.sample_workspace(rows, vocab) for _ in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()

    def call(i, ws):
        z, u, tokens, cols, _ = cases[i]
        A.dispatch_sample_tokens(z, u, tokens, ws, num_rows=rows, vocab=vocab, temperature=cols[0], top_k=cols[1], top_p=cols[2], min_p=cols[3])

    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                call(i, spaces[i])
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        assert list(from_dev(cases[i][2], np.int32)) == cases[i][4]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(i, spaces[0])
        graphs.append(g)
    for i in (0, 1, 1, 0, 1):
        cases[i][2].zero_()
        graphs[i].replay()
        torch.cuda.synchronize()
        assert list(from_dev(cases[i][2], np.int32)) == cases[i][4]
    del graphs
