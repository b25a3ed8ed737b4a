"""From the attention's output to the next tokens without the host in between: o_proj, norms, head and sampling behind each
other over one workspace, eager, on another stream, and captured and replayed with other inputs."""
import numpy as np
import pytest

from inferno_amd import attention as A
from tests import step_util as S
from tests.gpu_util import announce, empty_dev, from_dev, to_dev

pytestmark = pytest.mark.gpu

COLS, HIDDEN, VOCAB, EPS = 4096, 1280, 40003, 1e-6
ASKED = [(0.8, 64, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.2, 0, 1.0, 0.05), (1.0, 0, 1.0, 0.0), (1.0, 3000, 0.99, 0.0)]


class Tail:
    """The operators' buffers for n tokens; every call of step() reads attn, residual and u and leaves tokens."""

    def __init__(self, rng, n):
        import torch

        self.n = n
        self.weights = [S.random_w4(rng, 1, rows, cols, group)[1:] for rows, cols, group in ((HIDDEN, COLS, 64), (VOCAB, HIDDEN, 32))]
        self.dev = [[to_dev(t) for t in w] for w in self.weights]
        self.norms = [to_dev(S.f32_to_bf16(1 + 0.2 * rng.standard_normal(HIDDEN))) for _ in range(3)]
        self.attn, self.residual, self.u = empty_dev(n * COLS, np.uint16), empty_dev(n * HIDDEN, np.float32), empty_dev(n, np.float32)
        self.y, self.r, self.x, self.logits = (empty_dev(n * c, t) for c, t in ((HIDDEN, np.uint16), (HIDDEN, np.float32), (HIDDEN, np.uint16), (VOCAB, np.uint16)))
        self.tokens = empty_dev(n, np.int32)
        self.asked = [ASKED[i % len(ASKED)] for i in range(n)]
        self.params = [to_dev(np.array(c, np.int32 if i == 1 else np.float32)) for i, c in enumerate(zip(*self.asked))]
        sizes = [A.w4_gemm_workspace(HIDDEN, COLS, n), A.w4_gemm_workspace(VOCAB, HIDDEN, n), A.sample_workspace(n, VOCAB)]
        self.ws = torch.empty(max(0 if w is None else w.numel() for w in sizes), dtype=torch.float32, device="cuda")

    def load(self, inputs):
        for t, v in zip((self.attn, self.residual, self.u), inputs):
            t.copy_(to_dev(v).view(-1))

    def step(self):
        n = self.n
        A.dispatch_w4_gemm_cols(self.attn, *self.dev[0], self.y, rows=HIDDEN, cols=COLS, seq_len=n, group=64, w_format="int4", workspace=self.ws)
        A.dispatch_norm_residual(self.y, self.residual, self.r, self.x, hidden=HIDDEN, seq_len=n, eps=EPS, post_weight=self.norms[0],
                                 gate=self.norms[1], residual_scale=0.5, block_scale=0.75, pre_weight=self.norms[2])
        A.dispatch_w4_gemm_cols(self.x, *self.dev[1], self.logits, rows=VOCAB, cols=HIDDEN, seq_len=n, group=32, w_format="e2m1", workspace=self.ws)
        A.dispatch_sample_tokens(self.logits, self.u, self.tokens, self.ws, num_rows=n, vocab=VOCAB, row_stride=VOCAB, temperature=self.params[0],
                                 top_k=self.params[1], top_p=self.params[2], min_p=self.params[3])

    def results(self):
        return [from_dev(t, d) for t, d in ((self.r, np.float32), (self.logits, np.uint16), (self.tokens, np.int32))]


@pytest.mark.parametrize("n", [1, 7, 20, 61, 130])
def test_captured_and_replayed(n):
    import torch

    announce(f"step graph n={n}")
    rng = np.random.default_rng(n)
    tail, other = Tail(rng, n), Tail(rng, 9)
    inputs = [(S.f32_to_bf16(rng.standard_normal((n, COLS))), rng.standard_normal((n, HIDDEN)).astype(np.float32), rng.random(n).astype(np.float32))
              for _ in range(3)]
    want = []
    for one in inputs:
        tail.load(one)
        tail.step()
        want.append(tail.results())
    # The eager step itself: the head and the tokens against 64 bits, on what each was given last.
    x, logits = S.f64(from_dev(tail.x, np.uint16).reshape(n, HIDDEN)), S.f64(want[-1][1].reshape(n, VOCAB))
    w = S.w4_weight(*tail.weights[1], 32, "e2m1")
    exact = x @ w.T
    assert np.all(np.abs(logits - exact) <= S.w4_bound(x, w, exact, 32))
    for i, (t, k, p, floor) in enumerate(tail.asked):
        t, p, floor = (float(np.float32(v)) for v in (t, p, floor))
        kept = S.sample_weights(logits[i], t, k, p, floor)
        token, gap = S.sample_token(kept, float(inputs[-1][2][i]))
        assert token == want[-1][2][i] or gap < 1e-9, (i, token, want[-1][2][i], gap)
    stream = torch.cuda.Stream()
    tail.load(inputs[0])
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        tail.step()
    stream.synchronize()
    assert all(np.array_equal(a, b) for a, b in zip(tail.results(), want[0]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tail.step()
    for i in (1, 2, 0, 0, 2):
        tail.load(inputs[i])
        for t in (tail.y, tail.r, tail.x, tail.logits, tail.tokens, tail.ws):
            t.fill_(77)
        graph.replay()
        other.step()  # the program's own work behind it
        assert all(np.array_equal(a, b) for a, b in zip(tail.results(), want[i])), i
    del graph
