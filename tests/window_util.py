"""Cases, the 64-bit oracle and the error bounds of the window and 8-bit cache
operators.  Everything here runs on the CPU."""
from __future__ import annotations

import math
from dataclasses import dataclass, field

import numpy as np
import torch

from inferno_amd.kv import KVRunTable

QMAX = {"e4m3": 448.0, "int8": 127.0}


@dataclass
class Case:
    """lens: (context before the step, new tokens) of each run; rows: of the caches."""
    lens: list
    page: int
    window: int
    sinks: int
    table: KVRunTable
    pages: list = field(default_factory=list)  # of each run: first row of each page, -1 unseen
    rows: int = 0

    @property
    def seq(self):
        return sum(n for _, n in self.lens)

    def row(self, r, pos):
        pos = np.asarray(pos)
        return np.asarray(self.pages[r])[pos // self.page] + pos % self.page


def make_case(seed, lens, *, page=64, window=0, sinks=0, spare=3):
    """Run tables over shuffled pages; pages that no query sees have base row -1."""
    rng = np.random.default_rng(seed)
    need = []
    for c, n in lens:
        last = c + n - 1
        lo = max(0, c - window + 1) if window else 0
        seen = set(range(lo // page, last // page + 1))
        if window and sinks:
            seen |= set(range(0, min(sinks - 1, last) // page + 1))
        need.append(seen)
    pool = sum(map(len, need)) + spare
    free = list(rng.permutation(pool))
    table, pages, t = KVRunTable(), [], 0
    for (c, n), seen in zip(lens, need):
        table.begin_run(t, c)
        mine = [int(free.pop()) * page if j in seen else -1 for j in range((c + n - 1) // page + 1)]
        for row in mine:
            table.add_base_row(row)
        pages.append(mine)
        t += n
    return Case(list(lens), page, window, sinks, table, pages, pool * page)


def seen_by(case, p):
    j = np.arange(p + 1)
    return j if not case.window else j[(j > p - case.window) | (j < case.sinks)]


def bf16(x):
    """Rounded to bf16, as f32."""
    return torch.from_numpy(np.asarray(x, dtype=np.float32)).to(torch.bfloat16).float().numpy()


def attention64(case, q, k, v, scale, gqa, weight_step):
    """(o, bound): the attention in 64 bits and how far a kernel may be off, q [seq, nq,
    d], k and v [rows, nkv, d] as f32 arrays of the values themselves.

    bound = 2^-8 |o|                         o rounded to bf16 (half a step)
          + (weight_step                     each weight's rounding ahead of the sum over v
             + 2 (ds + n 2^-24) + 2^-18)     numerator and sum of weights: scores off by ds,
            * sum p |v|                      n additions, and exp2, log2 e and 1 / l
          + n 2^-116 (1 + max |v|)           what f32 and bf16 cannot hold
    with ds = (d + 4) 2^-24 scale sum |q k|: d products and sums in f32, the scale.

    The last term: exp2, and MFMA on bf16, take values below 2^-126 to 0.  A weight
    relative to the largest (which is 1, so that the sum of weights is at least 1) loses
    less than 2^-126 so, and each of its bf16 parts, times the block's scale in an 8-bit
    cache, again less than 2^-126 of what it multiplies: |v| in a bf16 cache, a code of
    at most 448 in an 8-bit one.  Per position that is at most 2^-126 (3 |v| + 2 * 448)
    < 2^-116 (1 + |v|)."""
    seq, nq, d = q.shape
    o, bound = np.zeros((seq, nq, d)), np.zeros((seq, nq, d))
    t = 0
    for r, (c, n) in enumerate(case.lens):
        for i in range(n):
            pos = seen_by(case, c + i)
            rows = case.row(r, pos)
            for h in range(nq):
                kk, vv = k[rows, h // gqa].astype(np.float64), v[rows, h // gqa].astype(np.float64)
                qq = q[t, h].astype(np.float64)
                s = kk @ qq * scale
                w = np.exp(s - s.max())
                w /= w.sum()
                o[t, h] = w @ vv
                ds = (d + 4) * 2.0 ** -24 * scale * (np.abs(kk) @ np.abs(qq)).max()
                rel = weight_step + 2 * (ds + len(pos) * 2.0 ** -24) + 2.0 ** -18
                bound[t, h] = 2.0 ** -8 * np.abs(o[t, h]) + rel * (w @ np.abs(vv)) + len(pos) * 2.0 ** -116 * (
                    1 + np.abs(vv).max())
            t += 1
    return o, bound


def round_code(y, kv):
    """Nearest even among the codes' values, saturating, in 64 bits; y finite."""
    if kv == "int8":
        return np.clip(np.rint(y), -127, 127)
    mag = np.minimum(np.abs(y), 448.0)
    step = 2.0 ** (np.floor(np.log2(np.maximum(mag, 2.0 ** -6))) - 3)
    return np.sign(y) * np.rint(mag / step) * step


def need_scale(amax, kv):
    """The smallest power of two s >= 2^-126 with amax <= Q s; 0 for 0."""
    if amax == 0:
        return 0.0
    e = math.ceil(math.log2(amax / QMAX[kv])) - 1
    while QMAX[kv] * 2.0 ** e < amax:
        e += 1
    return 2.0 ** max(e, -126)


def write64(case, kv, block, codes, scales, x):
    """The step's tokens x [seq, nkv, d] (finite) into codes [rows, nkv, d] (values of the
    codes) and scales, in place, from the definition."""
    t = 0
    for r, (c, n) in enumerate(case.lens):
        p = c
        while p < c + n:
            end = min((p // block + 1) * block, c + n)
            row = int(case.row(r, p))
            b, off = row // block, row % block
            for h in range(x.shape[1]):
                y = x[t + p - c:t + end - c, h].astype(np.float64)
                s = need_scale(np.abs(y).max(), kv)
                if off:
                    s = max(s, float(scales[b, h]))
                    if s > scales[b, h]:
                        old = codes[row - off:row, h]
                        codes[row - off:row, h] = round_code(old * (float(scales[b, h]) / s), kv)
                codes[row:row + end - p, h] = round_code(y / s, kv) if s else 0.0
                scales[b, h] = s
            p = end
        t += n


def rotate32(x, cos, sin, half, pair):
    """RoPE with f32 products and sums, each rounded once: x [seq, heads, d]; cos, sin
    [seq, half]."""
    y = x.astype(np.float32).copy()
    lo, hi = y[..., :half].copy(), y[..., pair:pair + half].copy()
    c, s = cos[:, None].astype(np.float32), sin[:, None].astype(np.float32)
    y[..., :half] = lo * c - hi * s
    y[..., pair:pair + half] = hi * c + lo * s
    return y


def positions(case):
    return np.concatenate([np.arange(c, c + n) for c, n in case.lens])


def code_values(raw, kv):
    """uint8 codes as the values they stand for, f32."""
    t = torch.from_numpy(np.ascontiguousarray(raw).view(np.uint8))
    t = t.view(torch.float8_e4m3fn if kv == "e4m3" else torch.int8)
    return t.float().numpy()


def to_codes(values, kv):
    """Values that are codes exactly, as uint8."""
    t = torch.from_numpy(np.ascontiguousarray(values, dtype=np.float32))
    return t.to(torch.float8_e4m3fn if kv == "e4m3" else torch.int8).view(torch.uint8).numpy()
