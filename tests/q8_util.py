"""Pages in 8 bits and the attention over them from their formulas in 64 bits, for the tests of the kernels."""
import math
import random

import numpy as np
import torch

TINY = 2.0 ** -100


def quantise(x):
    """(codes, scales) of rows of the last axis, in 64 bits."""
    x = x.double()
    a = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    scale = torch.where(a < TINY, 0.0, a / 127.0)
    codes = torch.round(torch.where(scale[..., None] > 0, x / torch.where(scale > 0, scale, 1.0)[..., None], 0.0))
    return torch.where(bad[..., None], 0.0, codes), torch.where(bad, math.nan, scale)


class Step:
    """The step as the parts see it (what `StepBatch` holds of it)."""

    def __init__(self, counts, starts, slots, device, padding=0):
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
        self.n_seqs, self.n_rows = len(counts), sum(counts) + padding
        self.positions = ints([s + i for s, c in zip(starts, counts) for i in range(c)] + [0] * padding)
        self.seq_of_row = ints([s for s, c in zip(slots, counts) for _ in range(c)] + [-1] * padding)
        row0 = np.concatenate([[0], np.cumsum(counts)[:-1]]).astype(int).tolist() if counts else []
        if padding:  # rows of no request, a request of one row each
            self.n_seqs += padding
            row0 += [sum(counts) + i for i in range(padding)]
        self.req_row0, self.req_count = ints(row0), ints(list(counts) + [1] * padding)
        self.req_start = ints(list(starts) + [0] * padding)
        self.host = {"counts": list(counts) + [1] * padding, "starts": list(starts) + [0] * padding}
        self.static_max_len, self.plans = None, {}


class Case:
    """Requests with `starts` cached positions that bring `counts` rows each, their pages filled with random rows in a random
    order; places of the pages that no request holds are NaN scales and arbitrary codes."""

    def __init__(self, heads, kv, dim, page, counts, starts, dtype, device="cuda:0", seed=0, spread=0.5, level=1.3, padding=0,
                 fill=True):
        self.heads, self.kv, self.dim, self.page, self.dtype = heads, kv, dim, page, dtype
        self.counts, self.starts = list(counts), list(starts)
        g = torch.Generator(device=device).manual_seed(seed)
        r = random.Random(seed)
        self.g, self.device = g, device
        n = len(counts)
        self.slots = r.sample(range(n + 2), n)
        totals = [a + b for a, b in zip(counts, starts)]
        self.totals = totals
        need = [-(-t // page) for t in totals]
        n_pages = sum(need) + 2
        ids = r.sample(range(n_pages), n_pages)
        width = max(need, default=1) + 1
        tables = torch.full((n + 2, width), -1, dtype=torch.int32)
        at = 0
        for s, m in zip(self.slots, need):
            tables[s, :m] = torch.tensor(ids[at:at + m], dtype=torch.int32)
            at += m
        self.tables = tables.to(device)
        shape = (n_pages, kv, page, dim)
        self.k = torch.randint(-127, 128, shape, dtype=torch.int8, device=device, generator=g)
        self.v = torch.randint(-127, 128, shape, dtype=torch.int8, device=device, generator=g)
        self.k_scale = torch.full(shape[:3], math.nan, device=device)
        self.v_scale = torch.full(shape[:3], math.nan, device=device)
        channel = torch.exp(spread * torch.randn(kv, dim, device=device, generator=g))
        for s, t in zip(self.slots, totals if fill else []):
            p = torch.arange(t, device=device)
            where = (self.tables[s].long()[p // page], slice(None), p % page)
            for pool, scales, x in ((self.k, self.k_scale, torch.randn(t, kv, dim, device=device, generator=g) * channel),
                                    (self.v, self.v_scale, torch.randn(t, kv, dim, device=device, generator=g))):
                codes, scale = quantise(x)
                pool[where], scales[where] = codes.to(torch.int8), scale.float()
        self.step = Step(counts, starts, self.slots, device, padding)
        self.q = (level * torch.randn(self.step.n_rows, heads * dim, device=device, generator=g)).to(dtype)
        self.err = torch.zeros(1, dtype=torch.int32, device=device)

    def pages(self):
        from cuca_b200.kernels import ops
        return ops.QuantizedPages(self.k, self.v, self.k_scale, self.v_scale)

    def rows(self, slot, total):
        """A request's keys and values in 64 bits, [positions, kv heads, dim]."""
        p = torch.arange(total, device=self.device)
        at = self.tables[slot].long()[p // self.page]
        return tuple(c[at, :, p % self.page].double() * s[at, :, p % self.page].double()[..., None]
                     for c, s in ((self.k, self.k_scale), (self.v, self.v_scale)))

    def attend(self, scale, window=None, keep_first=0, softcap=0.0, sink=False, sink_values=None, slopes=None):
        """(results, sums of weight times |value|, largest sum of |q_i k_i| of a row, number of keys times the largest weight times
        the key's largest value) in 64 bits, [rows, heads, dim] (the last two: [rows, heads])."""
        out = torch.zeros(self.step.n_rows, self.heads, self.dim, dtype=torch.float64, device=self.device)
        size, work, most = torch.zeros_like(out), torch.zeros_like(out[..., 0]), torch.zeros_like(out[..., 0])
        row0 = 0
        for slot, count, start in zip(self.slots, self.counts, self.starts):
            k, v = self.rows(slot, start + count)
            p = torch.arange(start, start + count, device=self.device)[:, None]
            j = torch.arange(start + count, device=self.device)[None]
            see = j <= p
            if window:
                see = see & ((p - j < window) | (j < keep_first))
            rows = slice(row0, row0 + count)
            for h in range(self.heads):
                kh, vh = k[:, h * self.kv // self.heads], v[:, h * self.kv // self.heads]
                q = self.q[rows, h * self.dim:(h + 1) * self.dim].double()
                s = (q @ kh.T) * scale
                if softcap:
                    s = softcap * torch.tanh(s / softcap)
                if slopes is not None:
                    s = s - slopes[h].double() * (p - j)
                s = s.masked_fill(~see, -math.inf)
                e = torch.exp(s - s.amax(-1, keepdim=True))
                den = e.sum(-1, keepdim=True)
                if sink:
                    den = den + torch.exp((sink_values[h].double() if sink_values is not None else 0.0) - s.amax(-1, keepdim=True))
                w = e / den
                out[rows, h], size[rows, h] = w @ vh, w @ vh.abs()
                most[rows, h] = (w * vh.abs().amax(-1).clamp_min(127 * 2.0 ** -60)).amax(-1) * see.sum(-1)
                work[rows, h] = ((q.abs() @ kh.abs().T) * abs(scale)).masked_fill(~see, 0.0).amax(-1)
            row0 += count
        return out, size, work, most

    def bound(self, out, size, work, most):
        """How far a result may be: its own rounding; the weights' (11 bits, in 32-bit mode 22; the exponent of 2 and the value
        scale's logarithm are good to 2^-21); the scores' 32-bit sums of d products in steps of 16 in each of two parts, whose
        error e changes a weight by a factor of e^e above and below the line. A 16-bit float has no steps under 2^-24, and the
        largest weight is 2^7 or more: each key's weight may be off by 2^-32 of that (a value
        scale counts as 2^-60 at least there)."""
        f32 = self.dtype == torch.float32
        steps = (2 if f32 else 1) * self.dim / 16 + 4
        score = steps * 2.0 ** -23 * work[..., None]
        return (2.0 ** -23 if f32 else 2.0 ** -8) * out.abs() + size * ((2.0 ** -19 if f32 else 2.0 ** -10) + 2 * score) + 2.0 ** -32 * most[..., None]
