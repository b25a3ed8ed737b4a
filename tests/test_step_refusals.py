"""What the entry points behind the attention refuse, and the sizes of their workspaces, without a GPU: every call here
ends in an argument check or has nothing to do."""

import pytest

from inferno_amd import _lib

EINVAL, ESPACE = -1, -4
P = 1 << 40  # addresses that are 16-byte aligned, far apart and never read


def at(i):
    return P * (i + 1)


def w4(**kw):
    a = dict(x=P, codes=at(1), scales=at(2), output=at(3), rows=64, cols=256, seq_len=4, group=32, w_format=1, workspace=None,
             workspace_bytes=0)
    a.update(kw)
    return _lib.lib().ifr_dispatch_w4_gemm_cols(*a.values(), 0)


@pytest.mark.parametrize("bad", [dict(rows=0), dict(rows=-1), dict(rows=(1 << 24) + 1), dict(cols=0), dict(cols=192), dict(cols=1 << 21),
                                 dict(seq_len=-1), dict(seq_len=(1 << 19) + 1), dict(group=16), dict(group=0), dict(group=256),
                                 dict(w_format=0), dict(w_format=3), dict(x=None), dict(codes=None), dict(scales=None), dict(output=None),
                                 dict(x=P + 2), dict(codes=P + 8), dict(scales=P + 4), dict(output=P + 2),
                                 dict(output=P), dict(output=P + 2032), dict(output=P - 496), dict(output=at(1) + 8176), dict(output=at(2) + 16),
                                 dict(rows=2816, cols=4096, seq_len=64, workspace=at(3) + 16, workspace_bytes=1 << 40),
                                 dict(rows=2816, cols=4096, seq_len=64, workspace=at(1) + 16, workspace_bytes=1 << 40)])
def test_w4_refuses(bad):
    assert w4(**bad) == EINVAL, _lib.last_error()


def test_w4_nothing_to_do():
    assert w4(seq_len=0, x=None, codes=None, scales=None, output=None) == 0
    size = _lib.lib().ifr_w4_gemm_workspace_bytes
    assert size(64, 256, 0) == 0
    assert [size(0, 256, 1), size(64, 100, 1), size(64, 256, -1), size(64, 256, 1 << 20)] == [-1] * 4


def test_a_workspace_does_for_fewer_tokens_and_rows():
    size = _lib.lib().ifr_w4_gemm_workspace_bytes
    for rows, cols in ((2816, 4096), (2816, 8192), (64, 65536), (33000, 4096), (262144, 2816), (512, 1024), (100, 128)):
        sizes = [size(rows, cols, m) for m in [*range(0, 1300), *range(1300, 20000, 61)]]
        assert sizes == sorted(sizes)
        assert sizes[-1] <= 64 << 20
    size = _lib.lib().ifr_sample_workspace_bytes
    for vocab in (1, 8191, 8192, 262144, 1 << 20):
        sizes = [size(rows, vocab) for rows in range(0, 600)]
        assert sizes == sorted(sizes)


def test_w4_workspace_too_small():
    size = _lib.lib().ifr_w4_gemm_workspace_bytes
    for rows, cols in ((2816, 8192), (64, 65536), (272, 4096)):
        for m in (1, 4, 16, 17, 61, 64, 65, 100, 200, 500, 4099):
            need = size(rows, cols, m)
            assert 0 <= need <= 64 * rows * m * 4 and need % 4 == 0
            if need:
                assert w4(rows=rows, cols=cols, seq_len=m, workspace=at(4), workspace_bytes=need - 1) == ESPACE
                assert w4(rows=rows, cols=cols, seq_len=m, workspace=None, workspace_bytes=need) == ESPACE
                assert w4(rows=rows, cols=cols, seq_len=m, workspace=at(4) + 4, workspace_bytes=need) == ESPACE


def norm(**kw):
    a = dict(y=P, residual=2 * P, residual_out=3 * P, x_out=4 * P, post=None, gate=None, pre=None, hidden=64, seq_len=4, kind=0, post_norm=1,
             gate_stride=0, a=1.0, b=1.0, eps=1e-6)
    a.update(kw)
    return _lib.lib().ifr_norm_residual(*a.values(), 0)


@pytest.mark.parametrize("bad", [dict(hidden=0), dict(hidden=12), dict(hidden=65544), dict(seq_len=-1), dict(seq_len=(1 << 24) + 1), dict(kind=2),
                                 dict(kind=-1), dict(post_norm=2), dict(post_norm=0, post=P), dict(x_out=None, pre=P), dict(eps=0.0), dict(eps=-1.0),
                                 dict(eps=float("nan")), dict(eps=float("inf")), dict(gate=P, gate_stride=8), dict(gate=P, gate_stride=68),
                                 dict(gate=P, gate_stride=-64), dict(y=None), dict(residual=None), dict(residual_out=None), dict(y=P + 2),
                                 dict(residual=P + 8), dict(gate=P + 4), dict(post=P + 2), dict(pre=P + 2), dict(x_out=2 * P), dict(x_out=3 * P),
                                 dict(residual_out=P), dict(residual_out=2 * P + 16), dict(x_out=P + 16), dict(x_out=P - 16),
                                 dict(gate=3 * P), dict(post=4 * P + 16), dict(pre=3 * P + 496), dict(residual_out=P + 496),
                                 dict(gate=5 * P, gate_stride=P, seq_len=2, residual_out=6 * P + 112)])
def test_norm_refuses(bad):
    assert norm(**bad) == EINVAL, _lib.last_error()


def test_norm_nothing_to_do():
    assert norm(seq_len=0, y=None, residual=None, residual_out=None, x_out=None) == 0


def sample(**kw):
    a = dict(logits=P, uniform=at(1), tokens=at(2), temperature=None, top_k=None, top_p=None, min_p=None, rows=4, vocab=100, stride=100, kind=1,
             workspace=at(3), workspace_bytes=1 << 40)
    a.update(kw)
    return _lib.lib().ifr_dispatch_sample_tokens(*a.values(), 0)


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(rows=(1 << 20) + 1), dict(vocab=0), dict(vocab=(1 << 20) + 1, stride=1 << 21), dict(stride=99),
                                 dict(stride=(1 << 32) + 1), dict(kind=2), dict(logits=None), dict(uniform=None), dict(tokens=None), dict(logits=P + 2),
                                 dict(logits=P + 1, kind=0), dict(uniform=P + 1), dict(top_k=P + 2), dict(min_p=P + 2), dict(tokens=P + 1584), dict(tokens=at(1) + 8),
                                 dict(min_p=at(2)), dict(workspace=P + 16), dict(workspace=at(2)), dict(top_k=at(3) + 16)])
def test_sample_refuses(bad):
    assert sample(**bad) == EINVAL, _lib.last_error()


def test_sample_workspace():
    size = _lib.lib().ifr_sample_workspace_bytes
    assert size(0, 100) == 0 and sample(rows=0, logits=None, uniform=None, tokens=None) == 0
    assert [size(-1, 10), size(1, 0), size(1, (1 << 20) + 1)] == [-1] * 3
    for rows, vocab in ((1, 1), (3, 1000), (256, 262144), (1 << 20, 1 << 20)):
        need = size(rows, vocab)
        assert need >= 0 and need % 4 == 0
        if need:
            for bad in (dict(workspace_bytes=need - 1), dict(workspace=None, workspace_bytes=need), dict(workspace=P + 8, workspace_bytes=need)):
                assert sample(rows=rows, vocab=vocab, stride=vocab, **bad) == ESPACE


def test_last_error_names_the_argument():
    assert w4(group=16) == EINVAL and "group" in _lib.last_error()
    assert norm(eps=0.0) == EINVAL and "eps" in _lib.last_error()
    assert sample(stride=7) == EINVAL and "row_stride" in _lib.last_error()
