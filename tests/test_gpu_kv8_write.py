"""RoPE and the quantising write into an 8-bit cache, against the definition in 64 bits:
codes and scales equal, bit for bit; special values; blocks that grow; what must not be
written; and the write together with the attention that reads it, with page copies, head
norm and o_proj, as a serving step runs them."""
import math

import numpy as np
import pytest
import torch

from inferno_amd import attention as A
from tests.gpu_util import announce
from tests.window_util import (attention64, bf16, code_values, make_case, need_scale, positions, rotate32,
                               round_code, to_codes, write64)

pytestmark = pytest.mark.gpu

SHAPES = {"256": (16, 8, 256, 128, 128), "512": (16, 2, 512, 64, 256), "128": (64, 4, 128, 64, 64),
          "partial": (6, 3, 128, 24, 40), "odd group": (5, 1, 256, 8, 128)}


class Cache:
    """An 8-bit cache of random codes and scales on both sides."""

    def __init__(self, rows, nkv, d, kv, block, seed, gap=0):
        rng = np.random.default_rng(seed)
        self.kv, self.block, self.nkv, self.d, self.stride = kv, block, nkv, d, nkv * d + gap
        raw = rng.integers(0, 256, (2, rows, self.stride), dtype=np.uint8)
        if kv == "e4m3":
            raw[(raw & 0x7F) == 0x7F] = 0x3C
        else:
            raw[raw == 0x80] = 0x81
        self.raw = raw
        self.scales = (2.0 ** rng.integers(-12, -5, (2, rows // block, nkv))).astype(np.float32)
        self.dev = [torch.from_numpy(x.copy()).cuda() for x in raw]
        self.dev_scales = [torch.from_numpy(x.copy()).cuda() for x in self.scales]

    def values(self, i):
        v = code_values(self.raw[i][:, :self.nkv * self.d], self.kv)
        return v.reshape(-1, self.nkv, self.d)

    def expect(self, case, i, x):
        """The step's tokens x in cache i, from the definition."""
        codes, scales = self.values(i), self.scales[i].astype(np.float64)
        write64(case, self.kv, self.block, codes, scales, x)
        raw = self.raw[i].copy()
        raw[:, :self.nkv * self.d] = to_codes(codes, self.kv).reshape(raw.shape[0], -1)
        # -0 and 0 are one value: the oracle's codes keep the bytes of what did not change
        return raw, scales.astype(np.float32)

    def got(self, i):
        return self.dev[i].cpu().numpy(), self.dev_scales[i].cpu().numpy()


def tables(case, half, seed=1):
    ang = np.random.default_rng(seed).uniform(-3, 3, (int(positions(case).max()) + 1, half))
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


def make_plan(case, shape, block):
    return A.WindowPlan(case.table, case.seq, window=case.window, sinks=case.sinks, page_len=case.page,
                        cache_rows=case.rows, num_q=shape[0], num_kv=shape[1], head_dim=shape[2], block_len=block)


def write(plan, cache, q, k, v, q_out, cos, sin, shape):
    dev = [torch.from_numpy(x).to(torch.bfloat16).cuda() if isinstance(x, np.ndarray) else x for x in (q, k, v)]
    A.dispatch_kv8_cache_write(plan, dev[0], dev[1], dev[2], dev[0] if q_out is None else q_out, cache.dev[0],
                               cache.dev_scales[0], cache.dev[1], cache.dev_scales[1], torch.from_numpy(cos).cuda(),
                               torch.from_numpy(sin).cuda(), num_q=shape[0], num_kv=shape[1], half=shape[3],
                               pair_stride=shape[4], head_dim=shape[2], kv_format=cache.kv, kv_stride=cache.stride)
    torch.cuda.synchronize()
    return dev[0]


def same_codes(got, want, kv, label):
    """Equal bytes, but for the sign of a zero."""
    zero = ((got & 0x7F) == 0) & ((want & 0x7F) == 0) if kv == "e4m3" else False
    bad = (got != want) & ~zero
    assert not bad.any(), (label, int(bad.sum()), np.argwhere(bad)[:4].tolist())


def check_step(case, shape, kv, block, seed, gap=0, size=1.0, in_place=False, edit=None):
    nq, nkv, d, half, pair = shape
    rng = np.random.default_rng(seed)
    q, k, v = (bf16(rng.standard_normal((case.seq, n, d)) * size) for n in (nq, nkv, nkv))
    if edit:
        edit(k, v)
    cos, sin = tables(case, half)
    cache = Cache(case.rows, nkv, d, kv, block, seed + 1, gap)
    at = positions(case)
    want = [cache.expect(case, 0, rotate32(k, cos[at], sin[at], half, pair)), cache.expect(case, 1, v)]
    q_out = None if in_place else torch.full((case.seq + 1, nq, d), 9.0, dtype=torch.bfloat16, device="cuda")
    out = write(make_plan(case, shape, block), cache, q, k, v, q_out, cos, sin, shape)
    if not in_place:
        assert np.array_equal(out.float().cpu().numpy(), q), "q_src was written"
        assert (q_out[case.seq:] == 9.0).all()
        out = q_out[:case.seq]
    assert np.array_equal(out.float().cpu().numpy(), bf16(rotate32(q, cos[at], sin[at], half, pair)))
    for i, name in enumerate("kv"):
        raw, scales = cache.got(i)
        assert np.array_equal(scales, want[i][1]), (name, "scales")
        same_codes(raw, want[i][0], kv, name)
    return cache


@pytest.mark.parametrize("kv", ["e4m3", "int8"])
@pytest.mark.parametrize("shape", SHAPES)
def test_write(shape, kv):
    """Single tokens at every kind of offset, chunks that begin and end inside blocks and
    cross pages, blocks of more rows than a pass holds."""
    announce(f"kv8 write {shape} {kv}")
    for page, block in [(64, 16), (64, 64), (256, 256)]:
        case = make_case(1, [(0, 1), (1, 1), (15, 1), (16, 1), (63, 1), (64, 1), (200, 1)], page=page)
        check_step(case, SHAPES[shape], kv, block, 2)
        case = make_case(3, [(0, 40), (7, 130), (63, 2), (250, 33), (100, 1)], page=page)
        check_step(case, SHAPES[shape], kv, block, 4, in_place=True)
    check_step(make_case(5, [(0, 300), (10, 3)], page=512), SHAPES[shape], kv, 512, 6, gap=32)


@pytest.mark.parametrize("kv", ["e4m3", "int8"])
@pytest.mark.parametrize("size", [1e-30, 3e-5, 300.0, 1e30])
def test_sizes(size, kv):
    """Values whose scales grow by far (older rows go to 0), stay, or lie at the end of the
    range."""
    announce(f"kv8 sizes {size} {kv}")
    case = make_case(7, [(5, 1), (16, 20), (70, 1)])
    check_step(case, SHAPES["partial"], kv, 32, 8, size=size)


@pytest.mark.parametrize("kv", ["e4m3", "int8"])
def test_scales_at_the_border(kv):
    """Largest values just at, below and above Q * 2^e, and rows of zeros."""
    announce(f"kv8 borders {kv}")
    top = 448.0 if kv == "e4m3" else 127.0
    shape = (2, 1, 128, 8, 64)
    for e in (-20, 0, 9):
        for x in (top, top * (1 - 2.0 ** -7), top * (1 + 2.0 ** -6), top / 2, 0.0):
            x = float(bf16(np.array([x * 2.0 ** e]))[0])

            def edit(k, v):
                v[:] = 0.0
                v[0, 0, 77] = -x
            cache = check_step(make_case(9, [(32, 1)]), shape, kv, 32, 10, edit=edit)
            _, scales = cache.got(1)
            assert need_scale(x, kv) in scales


@pytest.mark.parametrize("kv", ["e4m3", "int8"])
def test_special_values(kv):
    """Infinities saturate and do not count for the scale; NaN stays NaN in e4m3 and is 0 in
    int8."""
    announce(f"kv8 special {kv}")
    shape = (2, 1, 128, 8, 64)
    for rest in (1.0, 0.0):
        case = make_case(11, [(32, 3)])
        rng = np.random.default_rng(12)
        q, k, v = (bf16(rng.standard_normal((3, n, 128)) * rest) for n in (2, 1, 1))
        want_v = v.copy()
        v[1, 0, 5], v[1, 0, 6], v[2, 0, 7] = np.inf, -np.inf, np.nan
        want_v[1, 0, 5:7] = want_v[2, 0, 7] = 0.0
        cos, sin = tables(case, 8)
        cache = Cache(case.rows, 1, 128, kv, 32, 13)
        raw, scales = cache.expect(case, 1, want_v)
        write(make_plan(case, shape, 32), cache, q, k, v, None, cos, sin, shape)
        got, got_scales = cache.got(1)
        assert np.array_equal(got_scales, scales)
        row = case.row(0, np.arange(32, 35))
        big = 0x7E if kv == "e4m3" else 127
        assert got[row[1], 5] == big and got[row[1], 6] == (0xFE if kv == "e4m3" else 256 - 127)
        assert (got[row[2], 7] & 0x7F) == 0x7F if kv == "e4m3" else got[row[2], 7] == 0
        raw[row[1], 5:7], raw[row[2], 7] = got[row[1], 5:7], got[row[2], 7]
        same_codes(got, raw, kv, rest)


@pytest.mark.parametrize("kv", ["e4m3", "int8"])
def test_rounding_of_every_step(kv):
    """Every bf16 value of some octaves under scale 1: nearest even, as the format rounds."""
    announce(f"kv8 rounding {kv}")
    shape = (2, 1, 512, 8, 256)
    bits = np.arange(0, 0x8000, dtype=np.uint32) << 16
    vals = bits.view(np.float32)
    vals = vals[(vals >= 2.0 ** -11) & (vals <= (448.0 if kv == "e4m3" else 127.0))]
    n = -(-vals.size // 510)
    v = np.zeros((n, 1, 512), dtype=np.float32)
    v[:, 0, 0] = 448.0 if kv == "e4m3" else 127.0
    flat = np.zeros(n * 510, dtype=np.float32)
    flat[:vals.size] = np.where(np.arange(vals.size) % 2, vals, -vals)
    v[:, 0, 2:] = flat.reshape(n, 510)
    case = make_case(14, [(0, n)])
    rng = np.random.default_rng(15)
    q, k = (bf16(rng.standard_normal((n, h, 512))) for h in (2, 1))
    cos, sin = tables(case, 8)
    cache = Cache(case.rows, 1, 512, kv, 64, 16)
    write(make_plan(case, shape, 64), cache, q, k, v, None, cos, sin, shape)
    raw, scales = cache.got(1)
    row = case.row(0, np.arange(n))
    assert (scales[np.unique(row // 64)] == 1.0).all()
    assert np.array_equal(code_values(raw[row], kv), round_code(v[:, 0].astype(np.float64), kv).astype(np.float32))
    if kv == "e4m3":
        ref = torch.from_numpy(v[:, 0]).to(torch.float8_e4m3fn).float().numpy()
        assert np.array_equal(code_values(raw[row], kv), ref)


@pytest.mark.parametrize("kv", ["e4m3", "int8"])
def test_token_by_token(kv):
    """A sequence that is written token by token: the cache stays near what was written, by
    the steps that its blocks' growth allows."""
    announce(f"kv8 token by token {kv}")
    shape = SHAPES["partial"]
    nq, nkv, d, half, pair = shape
    n, block = 70, 32
    rng = np.random.default_rng(17)
    grow = np.exp2(np.arange(n) % block / 4.0)[:, None, None]
    k, v = (bf16(rng.standard_normal((n, nkv, d)) * grow) for _ in range(2))
    q = bf16(rng.standard_normal((n, nq, d)))
    whole = make_case(18, [(0, n)])
    cos, sin = tables(whole, half)
    cache = Cache(whole.rows, nkv, d, kv, block, 19)
    codes = [cache.values(i) for i in range(2)]
    scales = [cache.scales[i].astype(np.float64) for i in range(2)]
    for t in range(n):
        case = make_case(18, [(t, 1)])
        case.table, case.pages, case.rows = one_token(whole, t), whole.pages, whole.rows
        kk = rotate32(k[t:t + 1], cos[t:t + 1], sin[t:t + 1], half, pair)
        write64(case, kv, block, codes[0], scales[0], kk)
        write64(case, kv, block, codes[1], scales[1], v[t:t + 1])
        write(make_plan(case, shape, block), cache, q[t:t + 1], k[t:t + 1], v[t:t + 1], None, cos, sin, shape)
    row = whole.row(0, np.arange(n))
    at = positions(whole)
    for i, x in enumerate((rotate32(k, cos[at], sin[at], half, pair), v)):
        raw, got_scales = cache.got(i)
        assert np.array_equal(got_scales, scales[i].astype(np.float32))
        got = code_values(raw[row][:, :nkv * d], kv).reshape(n, nkv, d)
        assert np.array_equal(got, codes[i][row].astype(np.float32))
        s = got_scales[row // block][:, :, None]
        # int8: half a step now, and half, a quarter ... of what earlier, smaller scales were: one step;
        # e4m3: half a step of the value's own octave, and below 2^-6 * scale one of the subnormals.
        far = np.abs(got * s - x)
        room = s if kv == "int8" else np.maximum(np.abs(x) * 2.0 ** -4, s * 2.0 ** -9)
        assert (far <= room).all(), float((far / room).max())


def one_token(whole, t):
    from inferno_amd.kv import KVRunTable

    table = KVRunTable()
    table.begin_run(0, t)
    for row in whole.pages[0]:
        table.add_base_row(row)
    return table


@pytest.mark.parametrize("kv", ["e4m3", "int8"])
@pytest.mark.parametrize("shape", ["256", "512", "128"])
def test_a_serving_step(shape, kv):
    """Head norm, quantising write, attention and o_proj in one captured graph, replayed with
    other inputs: prompts, then single tokens, with a window and sinks, on pages copied from
    another sequence's (codes and scales alike)."""
    announce(f"kv8 serving step {shape} {kv}")
    nq, nkv, d, half, pair = SHAPES[shape]
    page, block, window, sinks, scale = 64, 32, 90, 5, 1 / math.sqrt(d)
    prompt = make_case(20, [(0, 100), (0, 100)], page=page, spare=4)
    cache = Cache(prompt.rows, nkv, d, kv, block, 21)
    cos, sin = tables(make_case(20, [(0, 200)]), half)
    cd, sd = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()
    rng = np.random.default_rng(22)
    rows_out = 256
    w = torch.from_numpy(bf16(rng.standard_normal((rows_out, nq * d)) / 32)).to(torch.bfloat16).cuda()
    qw, kw = (torch.from_numpy(bf16(1 + 0.1 * rng.standard_normal(d))).to(torch.bfloat16).cuda() for _ in range(2))

    def step(case, q, k, v, q_out, out, xs, plan, ws, gemm_ws):
        A.dispatch_rms_norm_qkv_heads(q, k, v, qw, kw, num_q=nq, num_kv=nkv, seq_len=case.seq, head_dim=d,
                                      sqrt_n=math.sqrt(d), n_eps=d * 1e-6)
        A.dispatch_kv8_cache_write(plan, q, k, v, q_out, cache.dev[0], cache.dev_scales[0], cache.dev[1],
                                   cache.dev_scales[1], cd, sd, num_q=nq, num_kv=nkv, half=half, pair_stride=pair,
                                   head_dim=d, kv_format=kv)
        A.kv8_attention(plan, q_out, cache.dev[0], cache.dev_scales[0], cache.dev[1], cache.dev_scales[1], out, ws,
                        num_q=nq, num_kv=nkv, head_dim=d, kv_stride=nkv * d, scale=scale, kv_format=kv)
        A.dispatch_gemm_cols(out, w, xs, rows=rows_out, cols=nq * d, seq_len=case.seq, workspace=gemm_ws)

    def buffers(case):
        new = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
        plan = A.WindowPlan(case.table, case.seq, window=window, sinks=sinks, page_len=page, cache_rows=cache.raw.shape[1],
                            num_q=nq, num_kv=nkv, head_dim=d, block_len=block)
        return (new(case.seq, nq, d), new(case.seq, nkv, d), new(case.seq, nkv, d), new(case.seq, nq, d),
                new(case.seq, nq, d), new(case.seq, rows_out), plan, A.window_workspace(plan),
                A.gemm_cols_workspace(rows_out, nq * d, case.seq))

    def fill(b, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        for t in b[:3]:
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))

    def look(case, b):
        """The attention against the oracle on what the cache holds now, and o_proj on it."""
        held = []
        for i in range(2):
            raw, scales = cache.got(i)
            held.append(code_values(raw, kv).reshape(-1, nkv, d) * np.repeat(scales, block, 0)[:, :, None])
        case.window, case.sinks = window, sinks
        step_w = 2.0 ** -8 if b[6].info[14] else 2.0 ** -15
        want, bound = attention64(case, b[3].float().cpu().numpy(), held[0], held[1], scale, nq // nkv, step_w)
        got = b[4].float().cpu().numpy()
        assert (np.abs(got - want) <= bound).all()
        xs = got.reshape(case.seq, -1).astype(np.float64) @ w.double().cpu().numpy().T
        room = 2.0 ** -8 * np.abs(xs) + nq * d * 2.0 ** -24 * (np.abs(got.reshape(case.seq, -1)) @ np.abs(w.double().cpu().numpy()).T)
        assert (np.abs(b[5].double().cpu().numpy() - xs) <= room).all()

    b = buffers(prompt)
    fill(b, 1)
    step(prompt, *b)
    torch.cuda.synchronize()
    look(prompt, b)
    # a third sequence shares the first one's tokens: its pages are copies of codes and scales
    spare = sorted(set(range(0, prompt.rows, page)) - {r for p in prompt.pages for r in p})[:2]
    for x in cache.dev + cache.dev_scales:
        row = x.numel() // (x.shape[0]) * x.element_size()
        per = page if x.dtype == torch.uint8 else page // block
        A.dispatch_copy_jobs(x, np.array([[s // page * per * row, t // page * per * row, per * row]
                                          for s, t in zip(prompt.pages[0], spare)]))
    torch.cuda.synchronize()
    pages = [prompt.pages[0], prompt.pages[1], spare]
    case = make_case(23, [(100, 1)] * 3, page=page)
    case.pages, case.rows = pages, prompt.rows
    case.table.base_rows = [r for p in pages for r in p]
    b = buffers(case)
    fill(b, 2)
    step(case, *b)
    torch.cuda.synchronize()
    look(case, b)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(case, *b)
    for seed in (3, 2, 4):
        fill(b, seed)
        g.replay()
        torch.cuda.synchronize()
        look(case, b)
        fill(b, seed)
        keep = [t.clone() for t in b[3:6]]
        step(case, *b)  # the same tokens again at the same positions
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(keep, b[3:6]))
    del g
