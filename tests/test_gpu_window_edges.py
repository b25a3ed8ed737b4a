"""The window and 8-bit cache operators where their numbers are at an end (blocks that grow from a scale of 0, scales and values
at the top of f32's range, rows of weights of which one has nearly all), and in forms that take many sequences or certain lengths
to be planned.  Against the definition in 64 bits."""
import math

import numpy as np
import pytest
import torch

from tests.gpu_util import announce
from tests.test_gpu_kv8_write import Cache, make_plan, same_codes, tables, write
from tests.test_gpu_window import Step
from tests.window_util import bf16, code_values, make_case, round_code, to_codes

pytestmark = pytest.mark.gpu

KINDS = ["bf16", "e4m3", "int8"]
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


def values_of(step):
    """k and v of a Step as its codes and scales have them now (8 bits)."""
    out = []
    for raw, scales in zip(step.raw, step.scales):
        codes = code_values(raw[:, :step.nkv * step.d].cpu().numpy(), step.kv).reshape(-1, step.nkv, step.d)
        out.append(codes * np.repeat(scales.cpu().numpy(), step.block, 0)[:, :, None])
    return out


def faint_queries(step, seed):
    """Queries of a few values of 2^-126 and the next ones, of any sign, and for the first token all 0."""
    rng = np.random.default_rng(seed)
    q = rng.integers(-2, 3, step.q.shape) * (rng.random(step.q.shape) < 1 / 16) * 2.0 ** -126
    q[0] = 0.0
    step.q = q.astype(np.float32)
    step.q_dev = torch.from_numpy(step.q).to(torch.bfloat16).cuda()


@pytest.mark.parametrize("shape", [(2, 1, 128), (2, 1, 256), (4, 1, 512)])
def test_int8_prompts_under_the_largest_scales(shape):
    """Scales of 2^121 and 2^122 (the largest that the write makes), in v and in k."""
    announce(f"window int8 largest scales {shape}")
    n, d = 80, shape[2]
    rng = np.random.default_rng(4)
    for e, most in ((121, 127), (122, 63)):
        # One visible position: the result is the row.
        case = make_case(5, [(70, n)], window=1)
        step = Step(case, "int8", shape, 6)
        codes = rng.integers(-most, most + 1, (case.rows, shape[1] * d)).astype(np.int8)
        step.raw[1] = torch.from_numpy(codes).view(torch.uint8).cuda()
        step.scales[1][:] = 2.0 ** e
        got, plan = step.run()
        assert plan.info[14] > 0
        at = case.row(0, np.arange(70, 70 + n))
        want = (codes[at].astype(np.float64) * 2.0 ** e).reshape(n, 1, d)
        assert np.array_equal(got, np.broadcast_to(want, got.shape)), e
        # The same in k.
        step = Step(make_case(7, [(70, n)]), "int8", shape, 8)
        codes = rng.integers(-most, most + 1, (step.case.rows, shape[1] * d)).astype(np.int8)
        step.raw[0] = torch.from_numpy(codes).view(torch.uint8).cuda()
        step.scales[0][:] = 2.0 ** e
        step.k = values_of(step)[0]
        faint_queries(step, 9)
        step.check(f"k 2^{e}", scale=1.0 / 16)


TOP = float(np.float32(255 * 2.0 ** 120))  # the largest bf16


@pytest.mark.parametrize("kv", ["e4m3", "int8"])
def test_what_is_written_reads_as_finite_values(kv):
    """The largest bf16 values, and infinities beside them: where the nearest code times the scale is 2^128, the code below."""
    announce(f"kv8 top of the range {kv}")
    first = bf16(np.random.default_rng(10).standard_normal((2, 1, 128)))
    for dim, x in ((20, TOP), (21, -TOP), (22, 2.0 ** 127), (23, 248 * 2.0 ** 120), (24, -2.0 ** 126)):
        first[0, 0, dim] = x
    first[1, 0, 25], first[1, 0, 26] = np.inf, -np.inf
    want = {"e4m3": [240, -240, 128, 240, -64, 240, -240], "int8": [63, -63, 32, 62, -16, 63, -63]}[kv]
    scale = 2.0 ** (120 if kv == "e4m3" else 122)
    cos, sin = tables(make_case(1, [(0, 64)]), 8)
    cache = Cache(4 * 64, 1, 128, kv, 32, 11)
    whole = steps_of([(32, 2)], WRITE, kv, cache, cos, sin, (first, first))
    row = whole.row(0, np.arange(32, 35))
    for i in range(2):
        raw, scales = cache.got(i)
        assert scales[row[0] // 32, 0] == scale
        held = code_values(raw[row[:2]], kv)
        assert [*held[0, 20:25], *held[1, 25:27]] == want, held[:, 20:27]
        with np.errstate(over="ignore"):
            assert np.isfinite(held * np.float32(scale)).all()
    # A block of the next smaller scale and its largest code, which grows.
    old = np.zeros((1, 1, 128), dtype=np.float32)
    old[0, 0, 30] = 448 * 2.0 ** 119 if kv == "e4m3" else 127 * 2.0 ** 121
    old[0, 0, 31] = -old[0, 0, 30]
    cache = Cache(4 * 64, 1, 128, kv, 32, 12)
    steps_of([(32, 1), (33, 1)], WRITE, kv, cache, cos, sin, (old, old), (first[:1], first[:1]))
    for i in range(2):
        raw, scales = cache.got(i)
        assert scales[row[0] // 32, 0] == scale
        held = code_values(raw[row[:2]], kv)
        assert list(held[0, 30:32]) == ([224, -224] if kv == "e4m3" else [63, -63])
        assert list(held[1, 20:25]) == want[:5]


def shared_rounding64(case, q, k, v, scale, gqa, step):
    """(o, bound) where numerator and denominator take the same rounded weights, each off by `step` of itself at most.

    o' = sum p (1 + e) v / sum p (1 + e), |e| <= step:  o' - o = sum p e (v - o) / sum p (1 + e), at most
    step / (1 - step) sum p |v - o|, and 1 / (1 - step) < 1 + 2 step.  The rest as in attention64: 2^-8 |o|, the result's own
    rounding; (2 (ds + n 2^-24) + 2^-18) sum p |v|.  A prompt's largest weight is 2^-16 at least, and exp2, bf16 and the
    products take what is below 2^-126 to 0: less than 2^-110 (2 |v| + 1) for each position, and n 2^-108 (1 + max |v|) for all."""
    o, bound = (np.zeros(q.shape) for _ in range(2))
    t = 0
    for r, (c, n) in enumerate(case.lens):
        rows = case.row(r, np.arange(c + n))
        for h in range(q.shape[1]):
            kk, vv = k[rows, h // gqa].astype(np.float64), v[rows, h // gqa].astype(np.float64)
            for i in range(n):
                kp, vp, qq = kk[:c + i + 1], vv[:c + i + 1], q[t + i, h].astype(np.float64)
                s = kp @ qq * scale
                w = np.exp(s - s.max())
                w /= w.sum()
                x = w @ vp
                ds = (q.shape[2] + 4) * 2.0 ** -24 * scale * (np.abs(kp) @ np.abs(qq)).max()
                m = len(s)
                o[t + i, h] = x
                bound[t + i, h] = (2.0 ** -8 * np.abs(x) + step * (1 + 2 * step) * (w @ np.abs(vp - x))
                                   + (2 * (ds + m * 2.0 ** -24) + 2.0 ** -18) * (w @ np.abs(vp)) + m * 2.0 ** -108 * (1 + np.abs(vp).max()))
        t += n
    return o, bound


def one_sharp_position(step, at, lo, hi, seed, v_size=1.0):
    """Scores near 0 in powers of two, but for position `at` of each run, which is at lo to hi, another for each query; v times
    v_size."""
    rng = np.random.default_rng(seed)
    step.k, step.v = bf16(step.k * 2.0 ** -7), bf16(step.v * v_size)
    step.k[:, :, 0] = 0.0
    step.k[[int(step.case.row(r, at)) for r in range(len(step.case.lens))], :, 0] = 1.0
    step.q = bf16(step.q / 2.0)
    scale = 1 / math.sqrt(step.d)
    step.q[:, :, 0] = bf16(rng.uniform(lo, hi, step.q.shape[:2]) * math.log(2.0) / scale)
    step.q_dev = torch.from_numpy(step.q).to(torch.bfloat16).cuda()
    for i, x in enumerate((step.k, step.v)):
        if step.kv == "bf16":
            step.raw[i] = step.wide(torch.from_numpy(x).to(torch.bfloat16))
            continue
        s = 2.0 ** -6 if i == 0 else v_size * 2.0 ** -5
        step.raw[i] = step.wide(torch.from_numpy(to_codes(round_code(x.astype(np.float64) / s, step.kv).reshape(x.shape), step.kv)))
        step.scales[i][:] = s
    if step.kv != "bf16":
        step.k, step.v = values_of(step)


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("shape", [(4, 2, 128), (4, 2, 256), (4, 1, 512)])
def test_a_position_that_has_nearly_all_of_the_weight(shape, kv):
    """A prompt's scores pass the maximum of their first tile by 10 to 20 powers of two: such a weight's rounding is in the sum of
    weights too, so that next to nothing of it is left in the result."""
    announce(f"window sharp weights {shape} {kv}")
    case = make_case(13, [(100, 80), (40, 70)])
    step = Step(case, kv, shape, 14)
    one_sharp_position(step, 38, 10.0, 20.0, 15)
    got, plan = step.run()
    assert plan.info[14] > 0
    want, bound = shared_rounding64(case, step.q, step.k, step.v, 1 / math.sqrt(step.d), shape[0] // shape[1], 2.0 ** -8)
    far = np.abs(got - want)
    print(f"  {shape} {kv}: {float((far / bound).max()):.3f} of the bound, relative rms {float(np.sqrt((far ** 2).sum() / (want ** 2).sum())):.2e}",
          flush=True)
    assert (far <= bound).all()


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("shape", [(4, 2, 128), (4, 2, 256), (4, 1, 512)])
def test_large_values_under_scores_that_rise(shape, kv):
    """v of about 2^112, and scores that pass the maximum of their first tile by 17 to 23 powers of two: the sums are finite."""
    announce(f"window large values {shape} {kv}")
    case = make_case(16, [(100, 80), (40, 70)])
    step = Step(case, kv, shape, 17)
    one_sharp_position(step, 38, 17.0, 23.0, 18, v_size=2.0 ** 112)
    assert np.isfinite(step.v).all()
    got, plan = step.run()
    assert plan.info[14] > 0 and np.isfinite(got).all()
    want, bound = shared_rounding64(case, step.q, step.k, step.v, 1 / math.sqrt(step.d), shape[0] // shape[1], 2.0 ** -8)
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("kv,e,most", [("e4m3", 120, 15), ("int8", 122, 63)])
@pytest.mark.parametrize("shape", [(2, 1, 128), (2, 1, 256), (4, 1, 512)])
def test_a_scale_of_the_scores_times_the_largest_scale_of_k(shape, kv, e, most):
    """Their product passes f32's range, the scores do not (of queries of 0 they are 0)."""
    announce(f"window scale overflow {shape} {kv}")
    for lens in ([(70, 1), (33, 1)], [(70, 80)]):
        step = Step(make_case(19, lens), kv, shape, 20)
        rng = np.random.default_rng(21)
        codes = rng.integers(-1, 2, (step.case.rows, shape[1] * step.d)).astype(np.float32)
        codes[:, 1::2] *= most * (rng.random(codes[:, 1::2].shape) < 1 / 64)
        step.raw[0] = torch.from_numpy(to_codes(codes, kv)).cuda()
        step.scales[0][:] = 2.0 ** e
        step.k = values_of(step)[0]
        faint_queries(step, 22)
        step.check(f"{lens}", scale=512.0)


@pytest.mark.parametrize("shape", [(2, 1, 128), (2, 1, 256), (2, 1, 512)])
@pytest.mark.parametrize("kv", ["e4m3", "int8"])
def test_every_code_in_prompts(shape, kv):
    """Every code through the prompt kernel, whose conversion is its own: one visible position, so that the result is the row."""
    announce(f"window all codes in prompts {shape} {kv}")
    n, d = 80, shape[2]
    case = make_case(23, [(70, n)], window=1)
    step = Step(case, kv, shape, 24)
    raw = np.arange(256, dtype=np.uint8)
    if kv == "e4m3":
        raw = np.where((raw & 0x7F) == 0x7F, 0, raw).astype(np.uint8)
    rng = np.random.default_rng(25)
    rows = np.stack([rng.permutation(np.resize(np.roll(raw, 128 * i), d)) for i in range(n)])
    assert len(np.unique(rows)) == (254 if kv == "e4m3" else 256)
    step.raw[1][torch.from_numpy(case.row(0, np.arange(70, 70 + n))).cuda()] = torch.from_numpy(rows).cuda()
    step.scales[1][:] = 2.0 ** -5
    got, plan = step.run()
    assert plan.info[14] > 0 and plan.info[0] == 0
    want = code_values(rows, kv).reshape(n, 1, d) * 2.0 ** -5
    assert np.array_equal(got, np.broadcast_to(want, got.shape))


@pytest.mark.parametrize("kv", KINDS)
def test_replays_read_the_inputs_of_their_time(kv):
    """A captured step with other queries in every replay, between eager calls of another step on the same workspace."""
    announce(f"window replays {kv}")
    step = Step(make_case(26, [(1500, 1), (40, 1), (300, 90)]), kv, (8, 2, 128), 27)
    other = Step(make_case(28, [(1200, 1), (100, 70)]), kv, (8, 2, 128), 29)
    plan, plan2 = step.plan(), other.plan()
    assert plan.info[0] and plan.info[1] and plan.info[14] and plan2.info[1]
    ws = torch.empty(max(plan.workspace_bytes, plan2.workspace_bytes) // 4, device="cuda")
    scale = 1 / math.sqrt(128)
    queries = [step.q_dev, -step.q_dev, step.q_dev.flip(0).contiguous()]
    want = []
    for q in queries:
        out = torch.empty_like(q)
        step.attend(plan, out, ws, scale, q)
        want.append(out)
    torch.cuda.synchronize()
    assert not torch.equal(want[0], want[1])
    out, out2, q = torch.zeros_like(step.q_dev), torch.zeros_like(other.q_dev), step.q_dev.clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step.attend(plan, out, ws, scale, q)
    for r in (1, 0, 2, 1, 1, 2, 0):
        out.zero_()
        q.copy_(queries[r])
        other.attend(plan2, out2, ws, scale)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[r]), r
    del g


def shared_pages_case(lens, page=64, of=3):
    """Sequences that read the pages of the longest ones of `of` groups."""
    top = max(c + n for c, n in lens)
    pool = make_case(30, [(top - 1, 1)] * of, page=page)
    case = make_case(30, [(0, n) for _, n in lens], page=page)
    case.lens, case.rows = list(lens), pool.rows
    case.pages = [pool.pages[r % of][:(c + n - 1) // page + 1] for r, (c, n) in enumerate(lens)]
    case.table = type(case.table)()
    t = 0
    for (c, n), pages in zip(lens, case.pages):
        case.table.begin_run(t, c)
        for row in pages:
            case.table.add_base_row(row)
        t += n
    return case


# Single sequences, shortest and longest context, kv heads that a work item's waves take, and whether some tokens are split.
BUSY = [(300, 300, 310, 2, False), (180, 60, 900, 2, True), (256, 500, 520, 4, False), (130, 60, 2500, 4, True)]


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("shape", [(16, 8, 256), (8, 8, 128), (8, 4, 512)])
@pytest.mark.parametrize("busy", BUSY)
def test_busy_decode(busy, shape, kv):
    """Batches whose work items take two and four kv heads, whole and split, among them runs of a few tokens."""
    runs, lo, hi, heads, split = busy
    announce(f"window busy decode {busy} {shape} {kv}")
    lens = [(int(c), 3 if i % 31 == 7 else 1) for i, c in enumerate(np.linspace(lo, hi, runs))]
    case = shared_pages_case(lens)
    step = Step(case, kv, shape, 31)
    plan = step.plan()
    assert plan.info[25] == heads and plan.info[14] == 0
    assert (0 < plan.info[1] < case.seq) if split else plan.info[1] == 0
    step.check("busy", plan=plan)


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("shape", [(16, 8, 256), (8, 8, 128), (8, 4, 512)])
@pytest.mark.parametrize("busy", [BUSY[0], BUSY[3]])
def test_busy_decode_of_an_infinite_value(busy, shape, kv):
    """One dim of one position of v infinite, or NaN: the sequences on that page get it there, and no other value changes a bit."""
    runs, lo, hi, heads, _ = busy
    announce(f"window busy decode of infinities {busy} {shape} {kv}")
    lens = [(int(c), 1) for c in np.linspace(lo, hi, runs)]
    case = shared_pages_case(lens)
    step = Step(case, kv, shape, 32)
    want, plan = step.run()
    assert plan.info[25] == heads
    flat = step.raw[1][int(case.row(1, 37))]
    flat[shape[2] + 3] = float("-inf") if kv == "bf16" else 0x7F  # kv head 1, dim 3
    got, _ = step.run(plan=plan)
    gqa = shape[0] // shape[1]
    hit = np.zeros(got.shape, dtype=bool)
    hit[1::3, gqa:2 * gqa, 3] = True
    assert np.array_equal(got[~hit], want[~hit])
    assert (np.isneginf(got[hit]) if kv == "bf16" else np.isnan(got[hit])).all()
