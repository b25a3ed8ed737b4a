"""Attention with a window and sinks over bf16 and 8-bit caches against the 64-bit
oracle: head layouts, lengths, windows, pages, splits, what masked places hold, strides,
graphs, streams, far rows."""
import math

import numpy as np
import pytest
import torch

from inferno_amd import attention as A
from tests.gpu_util import announce
from tests.window_util import attention64, bf16, code_values, make_case, need_scale, round_code, to_codes

pytestmark = pytest.mark.gpu

STEP = {"rows": 2.0 ** -15, "prompts": 2.0 ** -8}  # a weight's rounding: two bf16 parts, one


class Step:
    """A case's buffers on the GPU and its values on the CPU."""

    def __init__(self, case, kv, shape, seed, *, block=32, gap=0, q_size=2.0):
        self.case, self.kv, self.block = case, kv, block
        self.nq, self.nkv, self.d = shape
        self.stride = self.nkv * self.d + gap
        rng = np.random.default_rng(seed)
        self.q = bf16(rng.standard_normal((case.seq, self.nq, self.d)) * q_size)
        kvs = [bf16(rng.standard_normal((case.rows, self.nkv, self.d))) for _ in range(2)]
        self.scales = [None, None]
        self.raw = []
        for i, x in enumerate(kvs):
            if kv == "bf16":
                self.raw.append(self.wide(torch.from_numpy(x).to(torch.bfloat16)))
                continue
            b = x.reshape(-1, block, self.nkv, self.d)
            s = np.array([[need_scale(a, kv) for a in row] for row in np.abs(b).max((1, 3))], dtype=np.float32)
            codes = round_code(b / s[:, None, :, None], kv)
            kvs[i] = (codes * s[:, None, :, None]).reshape(x.shape).astype(np.float32)
            self.raw.append(self.wide(torch.from_numpy(to_codes(codes.reshape(x.shape), kv))))
            self.scales[i] = torch.from_numpy(s).cuda()
        self.k, self.v = kvs
        self.q_dev = torch.from_numpy(self.q).to(torch.bfloat16).cuda()

    def wide(self, x):
        """Rows of `stride` elements on the GPU, what is past the heads filled with NaN or 0x7F."""
        out = torch.full((self.case.rows, self.stride), float("nan") if x.dtype == torch.bfloat16 else 0x7F,
                         dtype=x.dtype)
        out[:, :self.nkv * self.d] = x.reshape(self.case.rows, -1)
        return out.cuda()

    def plan(self):
        c = self.case
        return A.WindowPlan(c.table, c.seq, window=c.window, sinks=c.sinks, page_len=c.page, cache_rows=c.rows,
                            num_q=self.nq, num_kv=self.nkv, head_dim=self.d,
                            block_len=0 if self.kv == "bf16" else self.block)

    def attend(self, plan, out, workspace, scale, q=None):
        kw = dict(num_q=self.nq, num_kv=self.nkv, head_dim=self.d, kv_stride=self.stride, scale=scale)
        q = self.q_dev if q is None else q
        if self.kv == "bf16":
            A.window_attention_bf16(plan, q, *self.raw, out, workspace, **kw)
        else:
            A.kv8_attention(plan, q, self.raw[0], self.scales[0], self.raw[1], self.scales[1], out, workspace,
                            kv_format=self.kv, **kw)

    def run(self, scale=None, plan=None):
        scale = 1 / math.sqrt(self.d) if scale is None else scale
        plan = self.plan() if plan is None else plan
        ws = A.window_workspace(plan)
        if ws is not None:
            ws.fill_(float("nan"))
        out = torch.full((self.case.seq + 2, self.nq, self.d), 7.0, dtype=torch.bfloat16, device="cuda")
        self.attend(plan, out, ws, scale)
        torch.cuda.synchronize()
        assert (out[self.case.seq:] == 7.0).all(), "rows behind the last token were written"
        return out[:self.case.seq].float().cpu().numpy(), plan

    def check(self, label, scale=None, plan=None):
        scale = 1 / math.sqrt(self.d) if scale is None else scale
        got, plan = self.run(scale, plan)
        step = STEP["prompts"] if plan.info[14] else STEP["rows"]
        want, bound = attention64(self.case, self.q, self.k, self.v, scale, self.nq // self.nkv, step)
        far = np.abs(got - want)
        worst = float((far / np.maximum(bound, 1e-300)).max())  # 0 where both are
        print(f"  {label}: {worst:.3f} of the bound, max {far.max():.3g}", flush=True)
        assert bool(np.isfinite(got).all()), label
        assert worst <= 1.0, label
        return got


LAYOUTS = [(16, 8, 256), (16, 2, 512), (64, 4, 128), (8, 8, 256), (6, 2, 128), (5, 1, 256), (14, 2, 512)]
KINDS = ["bf16", "e4m3", "int8"]


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("shape", LAYOUTS)
def test_single_tokens(shape, kv):
    """Lengths around tiles and pages, one token to enough for splits, with and without a
    window; every sequence of a batch of its own length."""
    announce(f"window single {shape} {kv}")
    ctx = [0, 1, 14, 15, 16, 30, 31, 32, 62, 63, 64, 200]
    for window, sinks in [(0, 0), (1, 0), (17, 0), (32, 1), (50, 40), (1000, 4)]:
        case = make_case(11, [(c, 1) for c in ctx], window=window, sinks=sinks)
        Step(case, kv, shape, 12).check(f"batch w={window} s={sinks}")
    case = make_case(13, [(1500, 1)])
    step = Step(case, kv, shape, 14)
    plan = step.plan()
    assert plan.info[1] == 1  # split and merged
    step.check("one split sequence", plan=plan)
    case = make_case(15, [(1500, 1)], window=1100, sinks=37)
    Step(case, kv, shape, 16).check("one split sequence, window and sinks")


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("shape", LAYOUTS)
def test_short_runs(shape, kv):
    """Runs of a few tokens, whose queries see different positions."""
    announce(f"window short runs {shape} {kv}")
    lens = [(0, 2), (31, 2), (63, 3), (100, 1), (90, 2), (7, 4)]
    for window, sinks in [(0, 0), (3, 0), (40, 2), (64, 70)]:
        case = make_case(17, lens, window=window, sinks=sinks)
        Step(case, kv, shape, 18).check(f"w={window} s={sinks}")
    case = make_case(19, [(700, 5)], window=600, sinks=33)
    Step(case, kv, shape, 20).check("split")


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("shape", LAYOUTS)
def test_prompts(shape, kv):
    """Chunks past the row items: odd lengths, more than a block, contexts ahead, windows
    that start inside a block, sinks ahead of and inside the window."""
    announce(f"window prompts {shape} {kv}")
    gqa = shape[0] // shape[1]
    n = 128 // gqa + 1
    for lens, window, sinks in [([(0, n)], 0, 0), ([(45, n + 30), (3, n)], 0, 0), ([(130, n + 9)], 1, 0),
                                ([(130, n + 9)], 40, 5), ([(0, n + 90)], 37, 64), ([(200, n + 3)], 150, 50)]:
        case = make_case(21, lens, window=window, sinks=sinks)
        step = Step(case, kv, shape, 22)
        plan = step.plan()
        assert plan.info[14] > 0
        step.check(f"{lens} w={window} s={sinks}", plan=plan)


@pytest.mark.parametrize("kv", KINDS)
def test_prompt_blocks_and_splits(kv):
    """Several blocks of one run, and a chunk whose blocks are split over the context and
    merged; in one step with single tokens."""
    announce(f"window prompt splits {kv}")
    case = make_case(23, [(0, 150)])
    Step(case, kv, (8, 2, 128), 24).check("blocks")
    case = make_case(25, [(900, 70), (500, 1), (0, 1)])
    for shape in [(8, 2, 128), (8, 1, 256), (16, 1, 512)]:
        step = Step(case, kv, shape, 26)
        plan = step.plan()
        assert plan.info[14] > 1 and plan.info[0] > 0 and plan.info[1] > 70
        step.check(f"split {shape}", plan=plan)
    case = make_case(27, [(700, 70), (500, 1)], window=333, sinks=9)
    Step(case, kv, (8, 1, 256), 28).check("split, window")


@pytest.mark.parametrize("page,block", [(32, 16), (32, 32), (64, 16), (256, 128), (1024, 1024)])
@pytest.mark.parametrize("kv", KINDS)
def test_pages_and_blocks(kv, page, block):
    announce(f"window pages {kv} {page} {block}")
    case = make_case(29, [(95, 1), (31, 1), (320, 1), (64, 100)], page=page)
    Step(case, kv, (4, 2, 128), 30, block=block).check("full")
    case = make_case(31, [(95, 1), (31, 1), (320, 1), (64, 100)], page=page, window=70, sinks=33)
    Step(case, kv, (4, 2, 128), 32, block=block).check("window")


@pytest.mark.parametrize("kv", KINDS)
def test_rows_wider_than_their_heads(kv):
    announce(f"window stride {kv}")
    case = make_case(33, [(95, 1), (310, 2), (64, 100)])
    for shape in [(4, 2, 128), (4, 2, 256), (8, 1, 512)]:
        Step(case, kv, shape, 34, gap=48).check(f"{shape}")


@pytest.mark.parametrize("size,scale", [(2.0, 4.0), (40.0, 1.0), (1e-3, 1e-3)])
@pytest.mark.parametrize("kv", KINDS)
def test_score_ranges(kv, size, scale):
    """Scores of hundreds (one weight takes all) and of nothing (all weights alike), with
    maxima that move from tile to tile."""
    announce(f"window scores {kv} {size} {scale}")
    case = make_case(35, [(400, 1), (150, 100)])
    for shape in [(4, 2, 128), (2, 1, 256)]:
        Step(case, kv, shape, 36, q_size=size).check(f"{shape}", scale=scale)


def test_a_rising_and_a_falling_row():
    """Scores that rise (or fall) by more than 2^8 from tile to tile."""
    announce("window rising scores")
    case = make_case(37, [(300, 1), (200, 100)])
    for sign in (1.0, -1.0):
        step = Step(case, "bf16", (4, 2, 128), 38)
        for r, (c, n) in enumerate(case.lens):
            pos = np.arange(c + n)
            step.k[case.row(r, pos), :, 0] = bf16(sign * pos)[:, None]
        step.q[:, :, 0] = 1.0
        step.raw[0] = step.wide(torch.from_numpy(step.k).to(torch.bfloat16))
        step.q_dev = torch.from_numpy(step.q).to(torch.bfloat16).cuda()
        step.check(f"sign {sign}", scale=1.0)


BAD = {"bf16": [float("nan"), float("inf"), -float("inf")], "e4m3": [float("nan")], "int8": []}


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("shape", [(16, 8, 256), (16, 2, 512), (64, 4, 128)])
def test_unseen_positions_hold_anything(shape, kv):
    """Rows that no query sees (spare pages, behind the last token, between sinks and
    window) hold NaN, infinities or random bytes, scales too: not a bit changes."""
    announce(f"window unseen {shape} {kv}")
    for lens, window, sinks in [([(40, 1), (70, 1), (700, 1)], 0, 0), ([(40, 1), (200, 1)], 50, 5),
                                ([(37, 3), (200, 2)], 50, 5), ([(45, 70)], 0, 0), ([(250, 70)], 50, 5)]:
        case = make_case(39, lens, window=window, sinks=sinks)
        step = Step(case, kv, shape, 40)
        want, plan = step.run()
        seen = np.zeros(case.rows, dtype=bool)
        for r, (c, n) in enumerate(lens):
            pos = np.arange(c + n)
            if window:
                pos = pos[(pos > c - window) | (pos < sinks)]
            seen[case.row(r, pos)] = True
        hide = torch.from_numpy(~seen).cuda()
        fills = [0x7FC0, 0x7F80, 0xFF80 - 0x10000, 0x7F7F] if kv == "bf16" else [0x7F, 0x80, 0xFF]
        for fill in fills:
            for raw in step.raw:
                raw.view(torch.int16 if kv == "bf16" else torch.uint8)[hide] = fill
            if kv != "bf16":
                unused = torch.from_numpy(~seen.reshape(-1, step.block).any(1)).cuda()
                for s in step.scales:
                    s[unused] = float("nan")
            got, _ = step.run(plan=plan)
            assert np.array_equal(got, want), (lens, window, fill)


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("shape", [(16, 8, 256), (16, 2, 512), (64, 4, 128)])
def test_later_tokens_do_not_reach_earlier_ones(shape, kv):
    """NaN and infinities in k and v of a token of the step: the queries that see it get
    what the formula gives, the others the bits they had."""
    announce(f"window causal poison {shape} {kv}")
    for lens, window, sinks, at in [([(60, 2)], 0, 0, 61), ([(30, 70)], 0, 0, 70), ([(30, 70)], 20, 0, 40),
                                    ([(100, 70)], 40, 6, 4), ([(100, 70)], 40, 6, 75)]:
        case = make_case(41, lens, window=window, sinks=sinks)
        for bad in BAD[kv]:
            for which in (0, 1):
                step = Step(case, kv, shape, 42)
                want, plan = step.run()
                row = int(case.row(0, at))
                flat = step.raw[which][row]
                code = torch.tensor(bad, dtype=torch.bfloat16) if kv == "bf16" else torch.tensor(0x7F, dtype=torch.uint8)
                flat[3] = code.to(flat.dtype).cuda() if kv == "bf16" else code.cuda()
                got, _ = step.run(plan=plan)
                gqa = step.nq // step.nkv
                for i in range(case.seq):
                    p = lens[0][0] + i
                    sees = at <= p and (not window or at > p - window or at < sinks)
                    hit = np.zeros_like(got[i], dtype=bool)
                    if sees:  # kv head 0, dim 3
                        hit[:gqa] = which == 0
                        hit[:gqa, 3] = True
                    assert np.array_equal(got[i][~hit], want[i][~hit]), (lens, window, at, bad, which, i)
                    if sees and which == 1:
                        g = got[i][:gqa, 3]
                        assert (np.isnan(g) if np.isnan(bad) else g == bad).all()
                    if sees and which == 0 and np.isnan(bad):
                        assert np.isnan(got[i][:gqa]).all()


@pytest.mark.parametrize("kv", KINDS)
def test_rows_past_four_gigabytes(kv):
    """Pages at the end of a cache whose byte offsets pass 2^32."""
    announce(f"window far rows {kv}")
    nq, nkv, d, page = 4, 2, 128, 64
    stride = 1 << 14
    rows = (5 << 30) // (stride * (2 if kv == "bf16" else 1)) // page * page
    case = make_case(43, [(150, 1), (20, 80)])
    near = Step(case, kv, (nq, nkv, d), 44, gap=stride - nkv * d)
    want, _ = near.run()
    shift = rows - case.rows
    far = Step(case, kv, (nq, nkv, d), 44, gap=stride - nkv * d)
    for i in range(2):
        big = torch.empty(rows, stride, dtype=far.raw[i].dtype, device="cuda")
        big[shift:] = far.raw[i]
        far.raw[i] = big
        if kv != "bf16":
            s = torch.empty(rows // far.block, nkv, device="cuda")
            s[shift // far.block:] = far.scales[i]
            far.scales[i] = s
    case.table.base_rows = [b + shift for b in case.table.base_rows]
    case.rows = rows
    got, _ = far.run()
    assert np.array_equal(got, want)


@pytest.mark.parametrize("kv", KINDS)
def test_graph_replays_and_streams(kv):
    """A captured step, replayed between eager calls of another step on the same workspace;
    and two steps on two streams with a workspace each."""
    announce(f"window graph {kv}")
    case = make_case(45, [(1500, 1), (40, 1), (300, 50)])
    step = Step(case, kv, (8, 2, 128), 46)
    other = Step(make_case(47, [(1200, 1), (100, 40)]), kv, (8, 2, 128), 48)
    want, plan = step.run()
    want2, plan2 = other.run()
    n = max(plan.workspace_bytes, plan2.workspace_bytes) // 4
    assert plan.info[1] and plan2.info[1]
    ws = torch.empty(n, device="cuda")
    scale = 1 / math.sqrt(128)
    out = torch.zeros(case.seq, 8, 128, dtype=torch.bfloat16, device="cuda")
    out2 = torch.zeros(other.case.seq, 8, 128, dtype=torch.bfloat16, device="cuda")
    q = step.q_dev.clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step.attend(plan, out, ws, scale, q)
    for r in range(4):
        out.zero_()
        q.copy_(step.q_dev if r % 2 == 0 else -step.q_dev)
        other.attend(plan2, out2, ws, scale)
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(out2.float().cpu().numpy(), want2)
        if r % 2 == 0:
            assert np.array_equal(out.float().cpu().numpy(), want), f"replay {r}"
    del g
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    spaces = [torch.empty(n, device="cuda") for _ in streams]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, st, pl, o, w in zip(streams, (step, other), (plan, plan2), (out, out2), spaces):
            with torch.cuda.stream(s):
                o.zero_()
                st.attend(pl, o, w, scale)
        torch.cuda.synchronize()
        assert np.array_equal(out.float().cpu().numpy(), want)
        assert np.array_equal(out2.float().cpu().numpy(), want2)


def test_a_plan_of_another_device_is_refused():
    announce("window device")
    case = make_case(49, [(30, 1)])
    step = Step(case, "bf16", (4, 2, 128), 50)
    plan = step.plan()
    q = step.q_dev.cpu()
    with pytest.raises(ValueError, match="q is on cpu"):
        step.attend(plan, torch.empty_like(step.q_dev), None, 1.0, q)


def test_codes_read_as_their_values():
    """Every code of both formats through the attention: one visible position, so that the
    result is the row itself."""
    announce("window all codes")
    for kv in ("e4m3", "int8"):
        for shape, n in [((2, 1, 256), 1), ((2, 1, 512), 1), ((2, 1, 128), 1), ((2, 1, 256), 40), ((2, 1, 512), 40)]:
            case = make_case(51, [(70, n)], window=1)
            step = Step(case, kv, shape, 52)
            raw = np.tile(np.arange(256, dtype=np.uint8), 4)[:shape[2]]
            if kv == "e4m3":
                raw = np.where((raw & 0x7F) == 0x7F, 0, raw).astype(np.uint8)
            rng = np.random.default_rng(53)
            rows = np.stack([rng.permutation(raw) for _ in range(n)])
            at = case.row(0, np.arange(70, 70 + n))
            step.raw[1][torch.from_numpy(at).cuda()] = torch.from_numpy(rows).cuda()
            step.scales[1][:] = 2.0 ** -5
            got, _ = step.run()
            want = code_values(rows, kv).reshape(n, 1, -1) * 2.0 ** -5
            assert np.array_equal(got, np.broadcast_to(want, got.shape)), (kv, shape, n)
