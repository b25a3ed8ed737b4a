"""A serving loop from token to token: the scheduler's steps run gathered embeddings, 4-bit projections, the append,
window attention, a 4-bit o_proj, the norms around the block, a 4-bit head and the sampling, whose tokens the scheduler
takes back.  Each of the operators behind the attention is checked on what it was really given, in 64 bits."""
import math

import numpy as np
import pytest

from inferno_amd import attention as A
from inferno_amd import host as P
from tests import step_util as S
from tests.gpu_util import announce, empty_dev, from_dev, to_dev

pytestmark = pytest.mark.gpu

HIDDEN, NQ, NKV, D, VOCAB, PAGE, EPS = 512, 4, 2, 128, 1501, 64, 1e-6
ASKED = {0: (0.8, 40, 0.95, 0.0), 1: (0.0, 0, 1.0, 0.0), 2: (1.2, 0, 0.9, 0.02)}  # by request


class Linear:
    def __init__(self, rng, rows, cols, group, fmt):
        self.rows, self.cols, self.group, self.fmt = rows, cols, group, fmt
        self.codes = rng.integers(0, 256, (rows, cols // 2), dtype=np.uint8)
        size = {"int4": 4.6, "e2m1": 2.8}[fmt] * math.sqrt(cols)  # outputs about as large as inputs
        self.scales = S.f32_to_bf16(np.exp(0.3 * rng.standard_normal((rows, cols // group))) / size)
        self.dev = to_dev(self.codes), to_dev(self.scales)
        self.weight = S.w4_weight(self.codes, self.scales, group, fmt)

    def __call__(self, x, n):
        out = empty_dev(n * self.rows, np.uint16)
        A.dispatch_w4_gemm_cols(x, *self.dev, out, rows=self.rows, cols=self.cols, seq_len=n, group=self.group,
                                w_format=self.fmt, workspace=A.w4_gemm_workspace(self.rows, self.cols, n))
        xf = S.f64(from_dev(x, np.uint16)[:n * self.cols].reshape(n, -1))
        exact = xf @ self.weight.T
        got = S.f64(from_dev(out, np.uint16).reshape(n, -1))
        assert np.all(np.abs(got - exact) <= S.w4_bound(xf, self.weight, exact, self.group)), (n, self.rows)
        return out


class Model:
    """One layer over a growing pool."""

    def __init__(self, seed, mirror, rows):
        rng = np.random.default_rng(seed)
        self.rng, self.mirror, self.rows = rng, mirror, rows
        self.embed = to_dev(S.f32_to_bf16(rng.standard_normal((VOCAB, HIDDEN))))
        self.q, self.k, self.v = (Linear(rng, h * D, HIDDEN, g, f) for h, g, f in ((NQ, 64, "int4"), (NKV, 32, "e2m1"), (NKV, 128, "int4")))
        self.o = Linear(rng, HIDDEN, NQ * D, 32, "int4")
        self.head = Linear(rng, VOCAB, HIDDEN, 64, "e2m1")
        self.norms = [S.f32_to_bf16(1 + 0.2 * rng.standard_normal(HIDDEN)) for _ in range(3)]
        self.gate = S.f32_to_bf16(rng.standard_normal(HIDDEN))
        self.cache = [empty_dev(rows * NKV * D, np.uint16) for _ in range(2)]
        ang = rng.uniform(-3, 3, 4096 * 64)
        self.cos, self.sin = to_dev(np.cos(ang).astype(np.float32)), to_dev(np.sin(ang).astype(np.float32))
        self.sizes, self.sampled = set(), 0

    def norm(self, y, r, n, post, gate, pre):
        r_out, x = empty_dev(n * HIDDEN, np.float32), empty_dev(n * HIDDEN, np.uint16)
        dev = [None if v is None else to_dev(v) for v in (post, gate, pre)]
        A.dispatch_norm_residual(y, r, r_out, x, hidden=HIDDEN, seq_len=n, eps=EPS, post_norm=post is not None, post_weight=dev[0],
                                 gate=dev[1], residual_scale=0.5, block_scale=0.75, pre_weight=dev[2])
        one = np.ones(1)
        want_r, want_x, br, bx = S.norm_residual(
            S.f64(from_dev(y, np.uint16).reshape(n, -1)), from_dev(r, np.float32).reshape(n, -1).astype(np.float64), eps=EPS,
            post_norm=post is not None, post=one if post is None else S.f64(post), gate=one if gate is None else S.f64(gate),
            pre=S.f64(pre), a=0.5, b=0.75, r_eps=2.0 ** -24)
        assert np.all(np.abs(from_dev(r_out, np.float32).reshape(n, -1) - want_r) <= br + 1e-38)
        assert np.all(np.abs(S.f64(from_dev(x, np.uint16).reshape(n, -1)) - want_x) <= bx + 1e-38)
        return r_out, x

    def execute(self, scheduler, sched, pages):
        n = len(sched.tokens)
        self.sizes.add(n)
        table = P.bind_pool_run_table(scheduler, 0, self.mirror)
        plan = A.WindowPlan(table, n, page_len=PAGE, cache_rows=self.rows, num_q=NQ, num_kv=NKV, head_dim=D)
        e = empty_dev(n * HIDDEN, np.uint16)
        A.dispatch_gather_rows(self.embed, e, to_dev(np.array(sched.tokens, np.int32)), n, HIDDEN)
        r = to_dev(S.f64(from_dev(e, np.uint16)).astype(np.float32))
        r, x = self.norm(empty_dev(n * HIDDEN, np.uint16), r, n, None, None, self.norms[0])
        q, k, v = self.q(x, n), self.k(x, n), self.v(x, n)
        A.dispatch_rope_cache_write(plan, q, k, v, *self.cache, self.cos, self.sin, num_q=NQ, num_kv=NKV, half=64, pair_stride=64, head_dim=D)
        attn = empty_dev(n * NQ * D, np.uint16)
        A.window_attention_bf16(plan, q, *self.cache, attn, A.window_workspace(plan), num_q=NQ, num_kv=NKV, head_dim=D, kv_stride=NKV * D,
                                scale=1 / math.sqrt(D))
        _, x = self.norm(self.o(attn, n), r, n, self.norms[1], self.gate, self.norms[2])
        # The last token of each sequence that emits.
        ends = np.cumsum([s.n_tokens for s in sched.slots]) - 1
        emit = [(int(end), s.request_id) for end, s in zip(ends, sched.slots) if s.emit]
        if not emit:
            return []
        m = len(emit)
        last = empty_dev(m * HIDDEN, np.uint16)
        A.dispatch_gather_rows(x, last, to_dev(np.array([i for i, _ in emit], np.int32)), m, HIDDEN)
        logits = self.head(last, m)
        asked = [ASKED[rid % 3] for _, rid in emit]
        u = self.rng.random(m).astype(np.float32)
        tokens = empty_dev(m, np.int32)
        cols = [to_dev(np.array(c, np.int32 if i == 1 else np.float32)) for i, c in enumerate(zip(*asked))]
        A.dispatch_sample_tokens(logits, to_dev(u), tokens, A.sample_workspace(m, VOCAB), num_rows=m, vocab=VOCAB, row_stride=VOCAB,
                                 temperature=cols[0], top_k=cols[1], top_p=cols[2], min_p=cols[3])
        got = from_dev(tokens, np.int32)
        z = S.f64(from_dev(logits, np.uint16).reshape(m, VOCAB))
        for i in range(m):
            t, k_, p, floor = (float(np.float32(a)) for a in asked[i])
            want, gap = S.sample_token(S.sample_weights(z[i], t, int(k_), p, floor), float(u[i]))
            assert got[i] == want and gap > 1e-9, (i, got[i], want, gap)
        self.sampled += m
        return [int(t) for t in got]


def test_tokens_from_tokens():
    announce("step: scheduler, projections, attention, norms, head, sampling")
    pages = 40
    spec = P.PagePoolSpec(pages, 0, 16)
    sched = P.ContinuousBatchScheduler(PAGE, P.BatchGeometry(4, 4, 160, [spec]), 160, [-1])
    mirror = P.KVPoolMirror(PAGE, 1, 0, 0, 1, [(0, NKV * D * 2)], spec)
    model = Model(3, mirror, pages * PAGE)
    rng = np.random.default_rng(5)
    ids = [sched.submit([int(t) for t in rng.integers(0, VOCAB, n)], 9) for n in (70, 131, 9)]
    clock = iter(range(1000, 10 ** 6, 1000))
    steps = 0
    while sched.pending_work() and steps < 60:
        assert sched.step(model, lambda: next(clock)) > 0
        steps += 1
    assert not sched.pending_work()
    for rid in ids:
        made = sched.request(rid).generated
        assert len(made) == 9 and all(0 <= t < VOCAB for t in made)
    assert model.sampled == 27 and max(model.sizes) > 64 and min(model.sizes) <= 3  # prompts and single tokens
