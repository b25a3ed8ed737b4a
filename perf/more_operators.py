"""From the attention's output to the next token, as a serving loop calls it: 4-bit projections, norms around a block, sampling.

Each case is one call of one operator:
  "w4"      out = x . W^T for bf16 x and a weight of 4-bit codes with a scale for each
            `group` columns of a row: int4 (two's complement) or e2m1
  "norm"    r' = a r + b g norm(y) w_post and x = norm(r') w_pre: the norm behind a block, its
            gate and residual scale, and the norm ahead of the next block
  "sample"  a token a row from its logits and a given random number, with temperature,
            top-k, top-p and min-p
Widths are those of this repository's benchmark and tests (2,816 wide tokens, projections from 4,096
and 8,192), and a generic vocabulary of 2^18.

Fields of a case:
  w4      m tokens, n rows and k columns of the weight, group, fmt "int4" or "e2m1"
  norm    t tokens of `hidden`, res "bf16" or "f32" (the residual stream), post and pre (the norms
          that there are), gate "none", "row" (one for all tokens) or "token" (one each)
  sample  rows, vocab, dtype "bf16" or "f32" of the logits, pad (elements between rows), mode: "chat"
          (temperature 0.8, top-k 64, top-p 0.95), "nucleus" (top-p alone), "minp" (min-p alone),
          "plain" (temperature alone), "mixed" (every row its own, greedy ones among them)
"""
import math

import numpy as np
import torch

own = False


def _w4(name, m, n, k, group, fmt):
    return _named(name, {"op": "w4", "m": m, "n": n, "k": k, "group": group, "fmt": fmt})


def _norm(name, t, hidden, res="bf16", post=True, gate="none", pre=True):
    return _named(name, {"op": "norm", "t": t, "hidden": hidden, "res": res, "post": post, "gate": gate, "pre": pre})


def _sample(name, rows, vocab, dtype, mode, pad=0):
    return _named(name, {"op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "mode": mode, "pad": pad})


def _named(name, case):
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # One user's next token through the projection behind the attention.
        _w4("w4_proj_one", 1, 2816, 4096, 128, "int4"),
        # Sixteen users', from the wide layers' 8,192 columns, fine groups.
        _w4("w4_proj_few", 16, 2816, 8192, 32, "e2m1"),
        # A full decode batch and a draft's tokens with it: an odd count.
        _w4("w4_proj_batch", 61, 2816, 4096, 64, "int4"),
        # Prompt chunks: the most arithmetic for its bytes.
        _w4("w4_proj_prompt", 4099, 2816, 4096, 128, "int4"),
        # The output head for one user: a stream of weights.
        _w4("w4_head_one", 1, 262144, 2816, 128, "int4"),
        # The output head for a batch, on an odd vocabulary.
        _w4("w4_head_batch", 64, 262143, 2816, 32, "e2m1"),
        # One user's token between two blocks.
        _norm("norm_one", 1, 2816),
        # A decode batch with a gate for each token and a 32-bit residual stream.
        _norm("norm_batch", 64, 2816, "f32", gate="token"),
        # Eight prompts of 2,048 tokens, a gate of the layer.
        _norm("norm_prompt", 16384, 2816, gate="row"),
        # One user's logits, as a chat samples them.
        _sample("sample_one", 1, 262144, "f32", "chat"),
        # A batch whose users each ask for something else.
        _sample("sample_mixed", 64, 262144, "bf16", "mixed"),
        # A large batch that keeps the most likely 95 %, padded rows of an odd vocabulary.
        _sample("sample_nucleus", 256, 262141, "f32", "nucleus", pad=3),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["w4", "w4", "w4", "norm", "sample", "sample"])
    if kind == "w4":
        k = 128 * _log(rng, 1, 64)
        n = _log(rng, 64, min(262144, 262143 * 2816 // k))
        m = _log(rng, 1, max(1, min(4099, 64 * 262143 * 2816 // (n * k))))
        return _w4(None, m, n, k, rng.choice([32, 64, 128]), rng.choice(["int4", "e2m1"]))
    if kind == "norm":
        hidden = 8 * _log(rng, 16, 1024)
        t = _log(rng, 1, 16384 * 2816 // max(hidden, 2816))
        return _norm(None, t, hidden, rng.choice(["bf16", "bf16", "f32"]), rng.random() < 0.8, rng.choice(["none", "row", "token"]), rng.random() < 0.8)
    vocab = _log(rng, 1000, 262144)
    return _sample(None, _log(rng, 1, 256), vocab, rng.choice(["bf16", "f32"]), rng.choice(["chat", "nucleus", "minp", "plain", "mixed", "mixed"]), rng.choice([0, 0, rng.randrange(1, 100)]))


# ---- inputs -----------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 2 + 1)
    return {"w4": _prepare_w4, "norm": _prepare_norm, "sample": _prepare_sample}[case["op"]](case, gen)


def _normal(gen, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)


def _prepare_w4(case, gen):
    m, n, k, group = case["m"], case["n"], case["k"], case["group"]
    # Activations have channels of different size, weights groups of different scale.
    x = _normal(gen, m, k) * torch.exp(0.7 * _normal(gen, k, dtype=torch.float32)).to(torch.bfloat16)
    codes = torch.randint(0, 256, (n, k // 2), generator=gen, device="cuda", dtype=torch.uint8)
    scales = (0.004 * torch.exp(0.4 * _normal(gen, n, k // group))).to(torch.bfloat16)
    st = {"case": case, "x": x, "codes": codes, "scales": scales, "out": torch.empty(m, n, device="cuda", dtype=torch.bfloat16)}
    if own:
        from inferno_amd import attention as A

        st["workspace"] = A.w4_gemm_workspace(n, k, m)
    return st


def _prepare_norm(case, gen):
    t, h = case["t"], case["hidden"]
    rdt = torch.bfloat16 if case["res"] == "bf16" else torch.float32
    st = {"case": case, "y": _normal(gen, t, h) * 3, "r": _normal(gen, t, h, dtype=rdt) * 8, "r_out": torch.empty(t, h, device="cuda", dtype=rdt),
          "post": None, "gate": None, "pre": None, "x_out": None}
    if case["post"]:
        st["post"] = (1 + 0.3 * _normal(gen, h)).to(torch.bfloat16)
    if case["gate"] != "none":
        st["gate"] = _normal(gen, *((h,) if case["gate"] == "row" else (t, h)))
    if case["pre"]:
        st["pre"] = (1 + 0.3 * _normal(gen, h)).to(torch.bfloat16)
        st["x_out"] = torch.empty(t, h, device="cuda", dtype=torch.bfloat16)
    return st


EPS, RES_SCALE, BLOCK_SCALE = 1e-6, 0.75, 0.5


def _asked(mode, row):
    """(temperature, top-k, top-p, min-p) of a row; 0, 0, 1 and 0 switch each off (temperature 0: greedy)."""
    every = {"chat": (0.8, 64, 0.95, 0.0), "nucleus": (1.0, 0, 0.95, 0.0), "minp": (1.2, 0, 1.0, 0.05), "plain": (1.0, 0, 1.0, 0.0)}
    if mode != "mixed":
        return every[mode]
    return [every["chat"], (0.0, 0, 1.0, 0.0), every["nucleus"], (0.7, 20, 0.8, 0.02), every["minp"], (1.0, 1, 1.0, 0.0), every["plain"], (1.5, 500, 0.99, 0.0)][row % 8]


def _prepare_sample(case, gen):
    rows, vocab = case["rows"], case["vocab"]
    # Logits whose ordered values fall as -a ln(rank): token probabilities follow a power law, as a language model's do.
    a = 1.2 + 0.8 * torch.rand(rows, 1, generator=gen, device="cuda")
    z = torch.empty(rows, vocab + case["pad"], device="cuda").exponential_(1.0, generator=gen) * a - 4
    asked = [_asked(case["mode"], r) for r in range(rows)]
    cols = [torch.tensor(c, device="cuda", dtype=torch.int32 if i == 1 else torch.float32) for i, c in enumerate(zip(*asked))]
    st = {"case": case, "logits": z.to(torch.bfloat16) if case["dtype"] == "bf16" else z, "u": torch.rand(rows, generator=gen, device="cuda"),
          "temperature": cols[0], "top_k": cols[1], "top_p": cols[2], "min_p": cols[3], "tokens": torch.empty(rows, device="cuda", dtype=torch.int32)}
    if own:
        from inferno_amd import attention as A

        st["workspace"] = A.sample_workspace(rows, vocab)
    return st


# ---- the operators ------------------------------------------------------------

def run(state):
    return {"w4": _run_w4, "norm": _run_norm, "sample": _run_sample}[state["case"]["op"]](state)


def _run_w4(st):
    case = st["case"]
    if own:
        from inferno_amd import attention as A

        A.dispatch_w4_gemm_cols(st["x"], st["codes"], st["scales"], st["out"], rows=case["n"], cols=case["k"], seq_len=case["m"],
                                group=case["group"], w_format=case["fmt"], workspace=st["workspace"])
    else:
        w = _values(st["codes"], case["fmt"]).view(case["n"], -1, case["group"]) * st["scales"].float()[..., None]
        st["out"].copy_(torch.matmul(st["x"].float(), w.view(case["n"], case["k"]).t()))
    return st["out"]


def _values(codes, fmt):
    """codes [n, k / 2], the lower four bits first -> their values [n, k] in 32 bits."""
    c = torch.stack([codes & 15, codes >> 4], -1).view(codes.shape[0], -1)
    if fmt == "int4":
        return (c ^ 8).float() - 8
    mag = (c & 7).float()
    mag = torch.where(mag < 4, mag * 0.5, torch.where(mag < 6, mag - 2, mag * 2 - 8))
    return torch.where(c >= 8, -mag, mag)


def _run_norm(st):
    case = st["case"]
    if own:
        from inferno_amd import attention as A

        A.dispatch_norm_residual(st["y"], st["r"], st["r_out"], st["x_out"], hidden=case["hidden"], seq_len=case["t"], eps=EPS,
                                 post_norm=case["post"], post_weight=st["post"], gate=st["gate"], residual_scale=RES_SCALE,
                                 block_scale=BLOCK_SCALE, pre_weight=st["pre"])
    else:
        y = st["y"].float()
        if case["post"]:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * st["post"].float()
        if st["gate"] is not None:
            y = y * st["gate"].float()
        r = RES_SCALE * st["r"].float() + BLOCK_SCALE * y
        st["r_out"].copy_(r)
        if case["pre"]:
            st["x_out"].copy_(r * torch.rsqrt((r * r).mean(-1, keepdim=True) + EPS) * st["pre"].float())
    return [st["r_out"], st["x_out"]] if case["pre"] else [st["r_out"]]


def _run_sample(st):
    case = st["case"]
    if own:
        from inferno_amd import attention as A

        A.dispatch_sample_tokens(st["logits"], st["u"], st["tokens"], st["workspace"], num_rows=case["rows"], vocab=case["vocab"],
                                 row_stride=case["vocab"] + case["pad"], temperature=st["temperature"], top_k=st["top_k"], top_p=st["top_p"], min_p=st["min_p"])
        return st["tokens"]
    vocab = case["vocab"]
    # In 64 bits: a draw lies next to the border between two tokens as often as their sums are off.
    z, order = torch.sort(st["logits"][:, :vocab].float(), dim=1, descending=True, stable=True)  # ties: the lowest index first
    rank = torch.arange(vocab, device=z.device)
    t = st["temperature"].double()[:, None]
    greedy = t <= 0
    w = torch.exp((z.double() - z[:, :1].double()) / torch.where(greedy, torch.ones_like(t), t))
    k = st["top_k"][:, None]
    keep = (k <= 0) | (rank < k)
    keep &= ~greedy | (rank == 0)
    w = w * keep
    total = w.sum(1, keepdim=True)
    before = torch.cumsum(w, 1) - w
    top_p = st["top_p"].double()[:, None]
    keep &= (top_p >= 1) | (rank == 0) | (before < top_p * total)
    keep &= w >= st["min_p"].double()[:, None]
    w = w * keep
    w = torch.zeros_like(w).scatter_(1, order, w)  # by index
    c = torch.cumsum(w, 1)
    pick = (c <= st["u"].double()[:, None] * c[:, -1:]).sum(1)
    last = vocab - 1 - (w.flip(1) > 0).int().argmax(1)
    st["tokens"].copy_(torch.minimum(pick, last))
    return st["tokens"]


# ---- what a pass cannot do without, and the results in 64 bits -----------------

def work(case):
    if case["op"] == "w4":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * k // 2 + 2 * n * k // case["group"] + 2 * m * (n + k), "flops": 2 * m * n * k}
    if case["op"] == "norm":
        t, h = case["t"], case["hidden"]
        res = 2 if case["res"] == "bf16" else 4
        gate = {"none": 0, "row": 2 * h, "token": 2 * t * h}[case["gate"]]
        return {"bytes": t * h * (2 + 2 * res + 2 * case["pre"]) + gate + 2 * h * (case["post"] + case["pre"]),
                "flops": t * h * (3 + 4 * case["post"] + (case["gate"] != "none") + 4 * case["pre"])}
    # A maximum, an exponential and a sum for each logit: about one operation each.
    return {"bytes": case["rows"] * (case["vocab"] * (2 if case["dtype"] == "bf16" else 4) + 24), "flops": 3 * case["rows"] * case["vocab"]}


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = kept
    return {"w4": _exact_w4, "norm": _exact_norm, "sample": _exact_sample}[case["op"]](st)


E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _exact_w4(st):
    """A slice of the weight's rows at a time: the codes from a table of their 16 values."""
    case = st["case"]
    n, k, group = case["n"], case["k"], case["group"]
    table = [float(c - 16 * (c > 7)) for c in range(16)] if case["fmt"] == "int4" else E2M1 + [-v for v in E2M1]
    table = torch.tensor(table, dtype=torch.float64, device="cuda")
    x = st["x"].double()
    out = torch.empty(case["m"], n, dtype=torch.float64, device="cuda")
    step = max(1, (1 << 27) // k)
    for n0 in range(0, n, step):
        c = st["codes"][n0:n0 + step].long()
        w = torch.empty(c.shape[0], k, dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = table[c % 16], table[c // 16]
        w *= st["scales"][n0:n0 + step].double().repeat_interleave(group, 1)
        out[:, n0:n0 + step] = x @ w.t()
    return out


def _exact_norm(st):
    case = st["case"]

    def normed(v, weight):
        return v / torch.sqrt(v.square().sum(-1, keepdim=True) / case["hidden"] + EPS) * weight.double()

    y, r = st["y"].double(), st["r"].double()
    if case["post"]:
        y = normed(y, st["post"])
    if case["gate"] != "none":
        y = y * st["gate"].double()
    r = RES_SCALE * r + BLOCK_SCALE * y
    return [r, normed(r, st["pre"])] if case["pre"] else [r]


def _exact_sample(st):
    """Row by row on the host, from the definition."""
    case = st["case"]
    out = np.empty(case["rows"], np.int32)
    u = st["u"].cpu().numpy().astype(np.float64)
    # The numbers that the caller passes are 32-bit ones.
    asked = [[float(np.float32(v)) for v in _asked(case["mode"], r)] for r in range(case["rows"])]
    for r, (t, k, p, floor) in enumerate(asked):
        z = st["logits"][r, :case["vocab"]].double().cpu().numpy()
        best = int(np.argmax(z))
        if t <= 0:
            out[r] = best
            continue
        w = np.exp((z - z[best]) / t)
        kept = np.lexsort((np.arange(z.size), -z))
        if k > 0:
            kept = kept[:int(k)]
        if p < 1:
            sums = np.cumsum(w[kept])
            kept = kept[:int(np.searchsorted(sums, p * sums[-1], side="left")) + 1]
        kept = np.sort(kept[w[kept] >= floor])
        sums = np.cumsum(w[kept])
        out[r] = kept[min(int(np.searchsorted(sums, u[r] * sums[-1], side="right")), kept.size - 1)]
    return torch.from_numpy(out).cuda()
