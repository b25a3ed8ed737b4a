"""CPU tests of the window plans: every visible tile of every token is in exactly one
work item, split tokens are merged over all their items, write blocks cover the step, and
what the planner and the entry points refuse.  No GPU is touched."""
import ctypes as C

import numpy as np
import pytest

from inferno_amd import _lib
from tests.window_util import make_case

lib = _lib.lib
TILE, ROW_COLS = 32, 16


def plan(case, *, nq=16, nkv=8, d=256, block=0, window=None, sinks=None, page=None, rows=None,
         seq=None, runs=None, base=None, short=0):
    r, b = case.table.arrays()
    r = r if runs is None else np.ascontiguousarray(runs, dtype=np.int32)
    b = b if base is None else np.ascontiguousarray(base, dtype=np.int32)
    seq = case.seq if seq is None else seq
    nbytes = lib().ifr_plan_window_bytes(r.shape[0], b.shape[0], max(seq, 0), max(block, 0))
    img = np.zeros(max(nbytes // 4 - short, 0), dtype=np.int32)
    info = (C.c_int64 * _lib.WINDOW_INFO_LEN)()
    st = lib().ifr_plan_window(
        img.ctypes.data, img.nbytes, r.ctypes.data_as(_lib.P_I32), r.shape[0],
        b.ctypes.data_as(_lib.P_I32), b.shape[0], seq, case.window if window is None else window,
        case.sinks if sinks is None else sinks, page or case.page,
        case.rows if rows is None else rows, nq, nkv, d, block, info)
    return st, img, info


def items_of(img, off, n):
    return img[off:off + 8 * n].reshape(n, 8)


def visible_tiles(case, p0, ntok):
    """Tile numbers (position / 32) that the planner's span holds for these queries."""
    lo = max(0, p0 - case.window + 1) // TILE if case.window else 0
    head = min(-(-case.sinks // TILE), lo) if case.window else 0
    return list(range(head)) + list(range(lo, (p0 + ntok - 1) // TILE + 1))


SHAPES = [(16, 8, 256), (16, 2, 512), (64, 4, 128), (12, 4, 128), (7, 1, 256)]
STEPS = [
    ([(0, 1)], 0, 0), ([(4096, 1)], 0, 0), ([(9000, 1)], 1024, 4), ([(70000, 1)], 0, 0),
    ([(c, 1) for c in (0, 5, 31, 32, 63, 64, 1000, 5000)], 100, 5),
    ([(500, 3), (0, 1), (77, 2)], 0, 0), ([(0, 2000)], 1024, 4), ([(7013, 500)], 0, 0),
    ([(3000, 512)] + [(100 * i, 1) for i in range(32)], 0, 0),
    ([(40, 33)], 1, 0), ([(40, 33)], 7, 200),
]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("step", range(len(STEPS)))
def test_items_cover_every_visible_tile_once(shape, step):
    nq, nkv, d = shape
    lens, window, sinks = STEPS[step]
    case = make_case(1, lens, window=window, sinks=sinks)
    st, img, info = plan(case, nq=nq, nkv=nkv, d=d)
    assert st == 0, _lib.last_error()
    gqa = nq // nkv
    assert info[2] == _lib.PLAN_WINDOW and info[4] <= img.nbytes
    run_of = np.repeat(np.arange(len(lens)), [n for _, n in lens])
    pos_of = np.concatenate([np.arange(c, c + n) for c, n in lens])
    covered = [[] for _ in range(case.seq)]
    columns = {}
    for off, n, most in ((16, info[0], ROW_COLS), (info[22], info[14], {128: 512, 256: 256, 512: 128}[d])):
        lengths = []
        for t0, ntok, rows_off, p0, lo, hi, col, _ in items_of(img, off, n):
            assert 0 < ntok and ntok * gqa <= most and p0 == pos_of[t0] and lo < hi
            run = run_of[t0]
            assert (run_of[t0:t0 + ntok] == run).all()
            assert rows_off == img[9] + case.table.runs[run][2]
            tiles = visible_tiles(case, p0, ntok)
            for t in range(ntok):
                covered[t0 + t] += [(tiles[x], col < 0) for x in range(lo, hi)]
                if col >= 0:
                    columns.setdefault(t0 + t, []).append((col + t * gqa, most))
            lengths.append(hi - lo)
        assert lengths == sorted(lengths, reverse=True)
    units = items_of(img, info[24], info[1])
    assert sorted(units[:, 0]) == sorted(columns)
    used = set()
    for token, n, col, step_, hstep, *_ in units:
        want = sorted(columns[token])
        assert 1 < n <= 64 and [c for c, _ in want] == [col + s * step_ for s in range(n)]
        assert hstep == want[0][1] if hstep == ROW_COLS else hstep >= ROW_COLS
        for s in range(n):
            for h in range(nkv):
                mine = set(range(col + s * step_ + h * hstep, col + s * step_ + h * hstep + gqa))
                assert not (mine & used) and max(mine) < info[3]
                used |= mine
    assert info[21] == info[3] * (d + 2) * 4
    for t in range(case.seq):
        mine = [x for x, _ in covered[t]]
        assert len(mine) == len(set(mine)), f"token {t} meets a tile twice"
        p = int(pos_of[t])
        must = {j // TILE for j in range(p + 1)
                if not window or j > p - window or j < sinks}
        assert must <= set(mine)
        direct = {x for _, x in covered[t]}
        assert len(direct) == 1  # all partial, or one item that writes the output
    assert list(img[img[10]:img[10] + case.seq]) == list(run_of)


@pytest.mark.parametrize("block", [16, 32, 64])
def test_write_blocks(block):
    lens = [(0, 1), (15, 1), (16, 1), (3, 130), (64, 64), (63, 2)]
    case = make_case(2, lens)
    st, img, info = plan(case, block=block)
    assert st == 0, _lib.last_error()
    assert info[20] == block and info[26] == 0
    got = img[info[23]:info[23] + 4 * info[15]].reshape(-1, 4)
    want, t = [], 0
    for r, (c, n) in enumerate(lens):
        p = c
        while p < c + n:
            end = min((p // block + 1) * block, c + n)
            want.append([t + p - c, end - p, int(case.row(r, p)), p])
            p = end
        t += n
    assert got.tolist() == want


def test_unseen_pages_may_be_anything_and_seen_ones_must_not():
    case = make_case(3, [(5000, 2)], window=100, sinks=70)
    assert -1 in case.pages[0]
    assert plan(case)[0] == 0
    _, base = case.table.arrays()
    for j, row in enumerate(case.pages[0]):
        for bad in (-1, case.rows - case.page + 1, 1 << 30):
            b = base.copy()
            b[j] = bad
            st, _, _ = plan(case, base=b)
            assert (st == 0) == (row == -1), (j, bad)
    # the window's first position lies at the end of a page: that page is seen
    edge = make_case(4, [(64 + 99, 1)], window=100)
    assert edge.pages[0][0] == -1 and edge.pages[0][1] >= 0 and plan(edge)[0] == 0
    edge = make_case(4, [(63 + 99, 1)], window=100)
    assert edge.pages[0][0] >= 0
    b = edge.table.arrays()[1].copy()
    b[0] = -1
    assert plan(edge, base=b)[0] == -1


def test_planner_refusals():
    case = make_case(5, [(100, 2), (30, 1)], window=64, sinks=4)
    ok = dict()
    assert plan(case, **ok)[0] == 0
    for bad, code in [
            (dict(page=48), -1), (dict(page=16), -1), (dict(window=-1), -1), (dict(sinks=-1), -1),
            (dict(window=0, sinks=4), -1), (dict(window=1 << 40), -1), (dict(rows=0), -1),
            (dict(rows=64), -1), (dict(nq=0), -1), (dict(nq=15), -1), (dict(nkv=0), -1),
            (dict(nq=136, nkv=8), -2), (dict(d=64), -2), (dict(d=192), -2), (dict(seq=0), -1),
            (dict(seq=-3), -1), (dict(seq=2), -1), (dict(block=8), -1), (dict(block=48), -1),
            (dict(block=128), -1), (dict(block=-16), -1)]:
        st, _, _ = plan(case, **bad)
        assert st == code, (bad, st, _lib.last_error())
        assert _lib.last_error()
    runs, base = case.table.arrays()
    for edit in [(0, 0, 1), (1, 0, 0), (1, 0, 3), (1, 1, -1), (1, 2, 99), (1, 3, 0), (0, 3, 1),
                 (1, 1, 1 << 30)]:
        r = runs.copy()
        r[edit[0], edit[1]] = edit[2]
        assert plan(case, runs=r)[0] == -1, edit
    assert plan(case, short=10 ** 6)[0] == -4
    assert lib().ifr_plan_window_bytes(-1, 1, 1, 0) == -1
    assert lib().ifr_plan_window_bytes(1, 1, 1, -1) == -1


def test_a_page_that_starts_inside_a_block_is_refused():
    case = make_case(6, [(10, 1)])
    _, base = case.table.arrays()
    b = base.copy()
    b[0] = 8
    assert plan(case, base=b)[0] == 0
    assert plan(case, base=b, block=16)[0] == -1 and "block" in _lib.last_error()
    b[0] = 16
    assert plan(case, base=b, block=16)[0] == 0


def _write(info, img, **kw):
    a = dict(nq=16, nkv=8, seq=3, half=128, pair=128, d=256, stride=2048, fmt=1, ptr=4096)
    a.update(kw)
    p = a["ptr"]
    return lib().ifr_kv8_cache_write(
        img.ctypes.data, info, p, p, p, a.get("q_out", p), p, p, p, p, p, p, a["nq"], a["nkv"],
        a["seq"], a["half"], a["pair"], a["d"], a["stride"], a["fmt"], 0)


def test_cache_write_refusals():
    """The addresses passed are no memory: a call that got past the checks would return
    an error of the runtime here, where there is no GPU, and not the one expected."""
    case = make_case(7, [(100, 2), (30, 1)])
    _, img, info = plan(case, block=64)
    for bad, code in [(dict(fmt=0), -1), (dict(fmt=3), -1), (dict(ptr=None), -1),
                      (dict(ptr=4096 + 8), -1), (dict(q_out=4096 + 2), -1), (dict(nq=8), -1),
                      (dict(nkv=16), -1), (dict(d=128), -1), (dict(seq=2), -1), (dict(half=0), -1),
                      (dict(half=129), -1), (dict(pair=64), -1), (dict(half=4), -2),
                      (dict(half=100, pair=100), -2), (dict(stride=2047), -1),
                      (dict(stride=2056), -1), (dict(stride=1 << 25), -2)]:
        assert _write(info, img, **bad) == code, (bad, _lib.last_error())
    _, img, info = plan(case)
    assert _write(info, img) == -1 and "block_len" in _lib.last_error()
    # two runs that write to one page, and pages that overlap by half
    runs, base = case.table.arrays()
    for other in (case.pages[0][1], case.pages[0][1] + 32):
        b = base.copy()
        b[runs[1, 2]] = other
        st, img, info = plan(case, base=b, block=32)
        assert st == 0 and info[26] == 1
        assert _write(info, img) == -1 and "share" in _lib.last_error()


def _attend(info, img, kv8=False, **kw):
    a = dict(nq=16, nkv=8, d=256, stride=2048, scale=0.1, ws=4096, ws_bytes=1 << 40, ptr=4096, fmt=1)
    a.update(kw)
    p = a["ptr"]
    if kv8:
        return lib().ifr_kv8_attention(img.ctypes.data, info, p, p, a.get("ks", p), p, p, p, a["ws"],
                                       a["ws_bytes"], a["nq"], a["nkv"], a["d"], a["stride"],
                                       a["scale"], a["fmt"], 0)
    return lib().ifr_window_attention_bf16(img.ctypes.data, info, p, p, p, p, a["ws"], a["ws_bytes"],
                                           a["nq"], a["nkv"], a["d"], a["stride"], a["scale"], 0)


@pytest.mark.parametrize("kv8", [False, True])
def test_attention_refusals(kv8):
    case = make_case(8, [(6000, 1)])
    _, img, info = plan(case, block=64 if kv8 else 0)
    assert info[1] == 1 and info[21] > 0
    bad = [(dict(ptr=None), -1), (dict(ptr=4096 + 8), -1), (dict(nq=8), -1), (dict(nkv=16), -1),
           (dict(d=128), -1), (dict(stride=2040), -1), (dict(stride=2049), -1),
           (dict(scale=0.0), -1), (dict(scale=-1.0), -1), (dict(scale=float("nan")), -1),
           (dict(scale=float("inf")), -1), (dict(ws=None), -4), (dict(ws_bytes=info[21] - 1), -4),
           (dict(ws=4096 + 4), -1)]
    if kv8:
        bad += [(dict(fmt=0), -1), (dict(fmt=4), -1), (dict(ks=None), -1)]
    for kw, code in bad:
        assert _attend(info, img, kv8, **kw) == code, (kw, _lib.last_error())
    if kv8:
        _, img, info = plan(case)
        assert _attend(info, img, True) == -1 and "block_len" in _lib.last_error()


def test_plans_are_not_taken_for_each_other():
    case = make_case(9, [(100, 1), (30, 1)])
    _, img, info = plan(case)
    p = 4096
    st = lib().ifr_attention_bf16(img.ctypes.data, info, p, p, p, p, p, 1 << 40, 16, 8, 256, 4128,
                                  2048, 64, -1, 0)
    assert st == -1 and "describe a plan" in _lib.last_error()
    st = lib().ifr_merge_flash_partials(img.ctypes.data, info, p, 1 << 40, p, 16, 256, 4128, 0)
    assert st == -1
    st = lib().ifr_bq_attn_prep(img.ctypes.data, info, *[p] * 14, 16, 8, 6, 63, -1, 2, 256, 128,
                                128, 16.0, 0.0, 0)
    assert st == -1 and "describe a plan" in _lib.last_error()
    # an attention plan is no window plan
    r, b = case.table.arrays()
    big = np.zeros(1 << 16, dtype=np.int32)
    other = (C.c_int64 * _lib.WINDOW_INFO_LEN)()
    assert lib().ifr_plan_attention(big.ctypes.data, big.nbytes, r.ctypes.data_as(_lib.P_I32), 2,
                                    b.ctypes.data_as(_lib.P_I32), b.shape[0], 2, 1, 0, 64, 64,
                                    case.rows, 16, 4096, other) == 0
    assert _attend(other, big) == -1 and "window plan" in _lib.last_error()
    # the bf16 appends take a window plan: what they refuse here is the null pointer
    st = lib().ifr_rope_cache_write(img.ctypes.data, info, None, p, p, p, p, p, p, 16, 8, 6, 63, -1,
                                    2, 128, 128, 256, 0)
    assert st == -1 and "null pointer" in _lib.last_error()
    st = lib().ifr_rope_cache_write(img.ctypes.data, info, p, p, p, p, p, p, p, 16, 8, 5, 31, -1, 2,
                                    128, 128, 256, 0)
    assert st == -1 and "page geometry" in _lib.last_error()


def test_wrappers_check_their_buffers():
    """On a plan that lies on the CPU: every buffer that does not fit is refused by name
    ahead of the library."""
    import torch

    from inferno_amd import attention as A

    case = make_case(10, [(100, 2), (30, 1)])
    plan_ = A.WindowPlan(case.table, case.seq, page_len=case.page, cache_rows=case.rows, num_q=16,
                         num_kv=8, head_dim=256, block_len=64, device="cpu")
    kw = dict(num_q=16, num_kv=8, head_dim=256, kv_stride=2048, scale=0.1)
    q = torch.zeros(3, 16, 256, dtype=torch.bfloat16)
    kv = torch.zeros(case.rows, 2048, dtype=torch.bfloat16)
    for bad in [dict(q=q[:2]), dict(q=q.float()), dict(q=torch.zeros(3, 16, 512, dtype=torch.bfloat16)[..., ::2]),
                dict(k=kv[:-1]), dict(v=kv.to(torch.int8)), dict(o=q[:1]), dict(ws=torch.zeros(4).double())]:
        a = dict(q=q, k=kv, v=kv, o=torch.empty_like(q), ws=None)
        a.update(bad)
        with pytest.raises(ValueError, match="must be contiguous"):
            A.window_attention_bf16(plan_, a["q"], a["k"], a["v"], a["o"], a["ws"], **kw)
    codes = torch.zeros(case.rows, 2048, dtype=torch.int8)
    scales = torch.zeros(case.rows // 64, 8)
    with pytest.raises(ValueError, match="k_scale"):
        A.kv8_attention(plan_, q, codes, scales[:-1], codes, scales, q, None, kv_format="int8", **kw)
    with pytest.raises(ValueError, match="kv_format"):
        A.kv8_attention(plan_, q, codes, scales, codes, scales, q, None, kv_format="e5m2", **kw)
    table = torch.zeros(102, 128)
    src = torch.zeros(3, 8, 256, dtype=torch.bfloat16)
    for bad, name in [(dict(cos=table[:101]), "cos_table"), (dict(k=src[:2]), "k_src"),
                      (dict(kc=kv), "k_cache"), (dict(vs=scales.double()), "v_scale")]:
        a = dict(k=src, cos=table, kc=codes, vs=scales)
        a.update(bad)
        with pytest.raises(ValueError, match=name):
            A.dispatch_kv8_cache_write(plan_, q, a["k"], src, q, a["kc"], scales, codes, a["vs"], a["cos"],
                                       table, num_q=16, num_kv=8, half=128, pair_stride=128,
                                       head_dim=256, kv_format="e4m3")


def test_splits_fit_the_image_that_was_asked_for():
    # One kv head: the rounds of row items and the pieces of a prompt block, at their most.
    for tokens in (1, 5, 33, 65):
        for ctx in (40, 3000, 30000):
            case = make_case(11, [(ctx + 17 * i, 1) for i in range(tokens)] + [(ctx, 3), (ctx, 40)])
            for nq, d in ((16, 128), (16, 512), (1, 256)):
                st, img, info = plan(case, nq=nq, nkv=1, d=d)
                assert st == 0, _lib.last_error()


@pytest.mark.parametrize("kv8", [False, True])
def test_a_scale_that_overflows_with_log2_e_is_refused(kv8):
    case = make_case(12, [(100, 1)])
    _, img, info = plan(case, block=64 if kv8 else 0)
    assert _attend(info, img, kv8, scale=3.0e38) == -1
