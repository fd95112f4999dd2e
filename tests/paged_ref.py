"""Plain 64-bit evaluation of the paged-cache and packed-batch operators, and how far a
result rounded the way the kernels round may be from it (tests only)."""
from __future__ import annotations

import math

import numpy as np
import torch

# half a step of a rounding, relative to the value
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def quantise(x):
    """Q8 codes and scales of f32 rows [..][d], in numpy so that every step is one f32
    rounding: scale = amax * (1/127), code = round(x * (127 * (1/amax)))."""
    x = x.detach().float().cpu().numpy()
    one, top = np.float32(1), np.float32(127)
    amax = np.abs(x).max(-1, keepdims=True)
    amax = np.where(amax < np.float32(2.0 ** -100), np.float32(0), amax)
    scale = np.where(amax == 0, one, amax * (one / top)).astype(np.float32)
    inv = np.where(amax == 0, np.float32(0), one / np.where(amax == 0, one, amax) * top)
    y = (x * inv.astype(np.float32)).astype(np.float32)
    whole = np.trunc(y)
    y = whole + np.where(np.abs(y - whole) >= 0.5, np.sign(y), 0)
    codes = np.clip(y, -127, 127).astype(np.int8)
    return torch.from_numpy(codes), torch.from_numpy(scale[..., 0])


def attention(q, k, v, pos0, window, scale, absent=None):
    """One sequence: q [n][Hq][d] at positions pos0 .., k / v [len][Hkv][d] (float64); absent:
    bool [len], keys that are not there.  Returns the result and the largest error of a
    kernel that sums in f32 and rounds the weights and the result to f16 / bf16, as a
    function of that type."""
    n, h, d = q.shape
    length, g, _ = k.shape
    out = torch.zeros((n, h, d), dtype=torch.float64)
    spread, drift, sub = torch.zeros_like(out), torch.zeros(n, h, 1, dtype=torch.float64), torch.zeros(n, h, 1, dtype=torch.float64)
    pos = torch.arange(pos0, pos0 + n).unsqueeze(1)
    key = torch.arange(length).unsqueeze(0)
    seen = (key <= pos) & (key > pos - window) if window else key <= pos
    if absent is not None:
        seen = seen & ~absent.unsqueeze(0)
    some = seen.any(1)
    for i in range(h):
        ki, vi = k[:, i // (h // g)], v[:, i // (h // g)]
        # keys that no row sees do not enter, whatever they hold
        use = seen.any(0)
        ki, vi = ki[use], vi[use]
        if not use.any():
            continue
        s = (q[:, i] @ ki.T) * scale
        s = s.masked_fill(~seen[:, use], -math.inf)
        p = torch.softmax(s, -1)
        p[~some] = 0.0
        out[:, i] = p @ vi
        spread[:, i] = p @ vi.abs()
        big = (q[:, i].abs() @ ki.abs().T) * scale            # sum |q k| of every score
        big = big + q[:, i].abs().amax(1, keepdim=True) * ki.abs().sum(1).unsqueeze(0) * scale
        big = torch.where(seen[:, use], big, 0.0)
        drift[:, i, 0] = big.amax(1)
        sub[:, i, 0] = seen.sum(1) * p.amax(1) * vi.abs().max()

    def bound(dtype):
        u = HALF_STEP[dtype]
        # a score's f32 sum of d products and its exponential, relative to the weight; it
        # enters the numerator and the sum
        w = 2 * (d + 16) * 2.0 ** -24 * (drift + 1)
        tol = u * out.abs() + spread * (1 + u) * (2 * u + w)
        if dtype == torch.float16:
            tol = tol + sub * 2.0 ** -25 + 2.0 ** -25  # weights and results below f16's normal range
        return tol

    return out, bound


class Batch:
    """A ragged batch over a paged cache, on the CPU: rows per sequence, lengths, a page
    table of random pages (entries past a sequence's last page: -1)."""

    def __init__(self, rows, lens, page, seed, *, lead=0, tail=0, spare=2, table_extra=1):
        rng = np.random.default_rng(seed)
        self.rows, self.lens, self.page = list(rows), list(lens), page
        self.start = np.concatenate([[lead], lead + np.cumsum(rows)]).astype(np.int32)
        self.n_rows = int(self.start[-1]) + tail
        per = [-(-n // page) for n in lens]
        self.n_pages = sum(per) + spare
        order = rng.permutation(self.n_pages)
        self.table = np.full((len(lens), max(per + [1]) + table_extra), -1, np.int32)
        at = 0
        for i, n in enumerate(per):
            self.table[i, :n] = order[at:at + n]
            at += n

    def places(self, s):
        """(page, row) of every position of sequence s."""
        pos = np.arange(self.lens[s])
        return self.table[s][pos // self.page].astype(np.int64), pos % self.page

    def device(self, ops, **kw):
        return ops.PagedBatch(torch.from_numpy(self.start).cuda(), torch.tensor(self.lens, dtype=torch.int32).cuda(),
                              torch.from_numpy(self.table).cuda(), n_rows=self.n_rows,
                              max_rows=max(self.rows + [1]), max_len=max(list(self.lens) + [1]), **kw)
