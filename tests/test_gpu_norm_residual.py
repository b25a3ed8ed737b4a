"""Norms around a block with gate and residual scale against 64 bits."""
import numpy as np
import pytest

from inferno_amd import attention as A
from inferno_amd._lib import InfernoHipError
from tests import step_util as S
from tests.gpu_util import announce, empty_dev, from_dev, to_dev

pytestmark = pytest.mark.gpu

GUARD = 64


def _case(seed, rows, hidden, f32, gate, post=True, pre=True):
    rng = np.random.default_rng(seed)
    y = S.f32_to_bf16(rng.standard_normal((rows, hidden)) * 3)
    r = (rng.standard_normal((rows, hidden)) * 8).astype(np.float32)
    c = {"y": y, "r": r if f32 else S.f32_to_bf16(r), "f32": f32, "post": None, "gate": None, "pre": None}
    if post:
        c["post"] = S.f32_to_bf16(1 + 0.3 * rng.standard_normal(hidden))
    if gate:
        c["gate"] = S.f32_to_bf16(rng.standard_normal(hidden if gate == "row" else (rows, hidden)))
    if pre:
        c["pre"] = S.f32_to_bf16(1 + 0.3 * rng.standard_normal(hidden))
    return c


def _opt(c, name):
    return None if c[name] is None else to_dev(c[name])


def _run(c, *, post_norm=True, x=True, a=0.75, b=0.5, eps=1e-6, in_place=False):
    rows, hidden = c["y"].shape
    dt = np.float32 if c["f32"] else np.uint16
    dy, dr = to_dev(c["y"]), to_dev(c["r"])
    if in_place:
        r_out, x_out = dr, dy
    else:
        r_out = to_dev(np.full(rows * hidden + GUARD, 7, dt))
        x_out = to_dev(np.full(rows * hidden + GUARD, 0x4242, np.uint16))
    A.dispatch_norm_residual(dy, dr, r_out, x_out if x else None, hidden=hidden, seq_len=rows, eps=eps, post_norm=post_norm,
                             post_weight=_opt(c, "post"), gate=_opt(c, "gate"), residual_scale=a, block_scale=b, pre_weight=_opt(c, "pre"))
    gr, gx = from_dev(r_out, dt).ravel(), from_dev(x_out, np.uint16).ravel()
    n = rows * hidden
    if not in_place:
        assert np.all(gr[n:] == 7) and np.all(gx[n if x else 0:] == 0x4242)
    return gr[:n].reshape(rows, hidden), gx[:n].reshape(rows, hidden)


def _check(c, **kw):
    got_r, got_x = _run(c, **kw)
    one = np.ones(1)
    r = c["r"].astype(np.float64) if c["f32"] else S.f64(c["r"])
    want_r, want_x, br, bx = S.norm_residual(
        S.f64(c["y"]), r, eps=kw.get("eps", 1e-6), post_norm=kw.get("post_norm", True),
        post=one if c["post"] is None else S.f64(c["post"]), gate=one if c["gate"] is None else S.f64(c["gate"]),
        pre=one if c["pre"] is None else S.f64(c["pre"]), a=np.float64(np.float32(kw.get("a", 0.75))),
        b=np.float64(np.float32(kw.get("b", 0.5))), r_eps=2.0 ** -24 if c["f32"] else 2.0 ** -8)
    gr = got_r.astype(np.float64) if c["f32"] else S.f64(got_r)
    assert np.all(np.abs(gr - want_r) <= br + 1e-38), float(np.max(np.abs(gr - want_r) - br))
    if kw.get("x", True):
        assert np.all(np.abs(S.f64(got_x) - want_x) <= bx + 1e-38), float(np.max(np.abs(S.f64(got_x) - want_x) - bx))
    return got_r, got_x


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("gate", [None, "row", "token"])
@pytest.mark.parametrize("rows,hidden", [(1, 8), (1, 2816), (2, 504), (3, 512), (5, 520), (33, 2816), (64, 2816), (7, 4096), (4, 8192),
                                         (3, 16384), (2, 16392), (1, 65536), (1031, 64), (2050, 2816), (300, 5376)])
def test_against_64_bits(rows, hidden, gate, f32):
    announce(f"norm_residual rows={rows} hidden={hidden} gate={gate} f32={f32}")
    _check(_case(rows + hidden, rows, hidden, f32, gate))


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("hidden", [1016, 1024, 1032, 2040, 2048, 2056, 4104, 8184, 8200, 16376, 32768, 32776])
def test_lengths_on_both_sides_of_each_variant(hidden, f32):
    announce(f"norm_residual hidden={hidden} f32={f32}")
    _check(_case(hidden, 6, hidden, f32, "token"))


@pytest.mark.parametrize("rows", [1, 70, 1500])
@pytest.mark.parametrize("post,pre,x,post_norm", [(False, False, True, True), (False, True, True, False), (False, False, False, False),
                                                  (True, False, False, True), (True, False, True, True)])
def test_parts_left_out(rows, post, pre, x, post_norm):
    announce(f"norm_residual parts rows={rows} {post} {pre} {x} {post_norm}")
    _check(_case(rows, rows, 1024, False, None, post, pre), x=x, post_norm=post_norm, a=1.0, b=1.0)


@pytest.mark.parametrize("rows,hidden", [(1, 2816), (1200, 2816), (5, 9000 // 8 * 8)])
@pytest.mark.parametrize("f32", [False, True])
def test_in_place_gives_the_same_bits(rows, hidden, f32):
    announce(f"norm_residual in place rows={rows} hidden={hidden}")
    c = _case(3, rows, hidden, f32, "token")
    want, got = _run(c), _run(c, in_place=True)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_rows_of_zeros_and_special_values():
    """A row of zeros stays finite under eps; a NaN or infinity stays in its row."""
    announce("norm_residual special rows")
    c = _case(9, 40, 2816, False, "row")
    clean = _run(c)
    c["y"][3], c["r"][3] = 0, 0
    c["y"][5, 100], c["r"][7, 9] = 0x7F80, 0x7FC0
    got = _run(c)
    assert np.all(S.f64(got[0])[3] == 0) and np.all(S.f64(got[1])[3] == 0)
    # y = inf: mean inf, 1 / sqrt(inf) = 0, inf * 0 = NaN there and 0 elsewhere, so x is NaN all over.
    assert np.isnan(S.f64(got[0])[5, 100]) and np.all(np.isnan(S.f64(got[1])[5]))
    assert np.all(np.isnan(S.f64(got[1])[7])) and np.isnan(S.f64(got[0])[7]).sum() == 1
    rest = np.delete(np.arange(40), [3, 5, 7])
    assert np.array_equal(got[0][rest], clean[0][rest]) and np.array_equal(got[1][rest], clean[1][rest])


def test_a_token_by_itself_and_in_a_batch_agree():
    """Within the bound of both (their sums are cut differently)."""
    announce("norm_residual single against batch")
    c = _case(11, 1300, 2816, True, "token")
    _check(c)
    one = {k: (v[700:701] if isinstance(v, np.ndarray) and v.ndim == 2 else v) for k, v in c.items()}
    _check(one)


@pytest.mark.parametrize("rows", [1, 64, 2000])
def test_captured_and_on_another_stream(rows):
    import torch

    announce(f"norm_residual graph rows={rows}")
    c = _case(21, rows, 2816, False, "row")
    want = _run(c)
    other = dict(c, y=np.roll(c["y"], 1, axis=1))
    want2 = _run(other)
    dy, dr, post, gate, pre = to_dev(c["y"]), to_dev(c["r"]), to_dev(c["post"]), to_dev(c["gate"]), to_dev(c["pre"])
    r_out, x_out = torch.zeros_like(dr), torch.zeros_like(dy)

    def call():
        A.dispatch_norm_residual(dy, dr, r_out, x_out, hidden=2816, seq_len=rows, eps=1e-6, post_weight=post, gate=gate,
                                 residual_scale=0.75, block_scale=0.5, pre_weight=pre)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
    stream.synchronize()
    assert np.array_equal(from_dev(r_out, np.uint16).reshape(want[0].shape), want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for src, w in ((other, want2), (c, want), (other, want2)):
        dy.copy_(to_dev(src["y"]))
        r_out.zero_()
        x_out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(from_dev(r_out, np.uint16).reshape(w[0].shape), w[0])
        assert np.array_equal(from_dev(x_out, np.uint16).reshape(w[1].shape), w[1])
        assert np.array_equal(_run(c)[1], want[1])
    del graph


def test_refusals():
    y, r, w = empty_dev(4 * 64, np.uint16), empty_dev(4 * 64, np.uint16), empty_dev(64, np.uint16)
    r_out, x_out = empty_dev(4 * 64, np.uint16), empty_dev(4 * 64, np.uint16)

    def call(y=y, r=r, r_out=r_out, x_out=x_out, **kw):
        A.dispatch_norm_residual(y, r, r_out, x_out, **{**dict(hidden=64, seq_len=4, eps=1e-6), **kw})

    call(post_weight=w, pre_weight=w, gate=w)
    call(seq_len=0)
    for bad in (dict(seq_len=5), dict(r_out=empty_dev(256, np.float32)), dict(post_norm=False, post_weight=w),
                dict(x_out=None, pre_weight=w), dict(gate=empty_dev(100, np.uint16)), dict(y=y.cpu()), dict(y=y.half()),
                dict(y=y.view(64, 4).t())):
        with pytest.raises(ValueError):
            call(**bad)
    for bad in (dict(hidden=60), dict(eps=0.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(x_out=r), dict(x_out=r_out), dict(r_out=y),
                dict(y=y[1:], seq_len=3), dict(seq_len=-1)):
        with pytest.raises(InfernoHipError):
            call(**bad)
