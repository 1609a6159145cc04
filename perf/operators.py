"""The key/value cache in 8 bits and the attention that reads it, measured operator by operator.

A cached row (the d keys or values of one position and key head) is d signed 8-bit codes and a 32-bit scale:
a = max |x|, scale = a / 127, code = round(x * (127 / a)); it stands for code * scale. Pages hold `page` positions of every key
head: codes [pages, key heads, page, d], scales [pages, key heads, page]; a request finds its pages through its row of the
page tables.

* "write": rows of q | k | v at their positions; q and k are rotated, k and v quantised into the pages. The pass reads the rows
  back too: what is held in 8 bits is returned as the values it stands for.
* "read": positions of some requests, brought back from their pages as dense rows.
* "attend": causal grouped-query attention of a step's rows over the pages: `requests` requests that bring up to `tokens` new
  tokens each on top of up to `cached` ones (whose pages hold the new ones already, as in a step of the engine). One token
  each: decoding.

Shapes: 32 query heads over 8 key heads of 128 or 64 and 40 heads over 40 of 128 (the benchmark's), eight to a key head, and
small ones as in the tests.
"""
from __future__ import annotations

import math
import random
from types import SimpleNamespace

import torch

own = False

TINY = 2.0 ** -100  # rows whose largest value is below are kept as zeros


# ------------------------------------------------------------------------------------------------------- cases
def _case(name, op, dtype, heads, kv, dim, page, requests, tokens, cached, ragged, window=0, keep=0, sink=False, softcap=0.0):
    c = {"op": op, "dtype": dtype, "heads": heads, "kv": kv, "dim": dim, "page": page, "requests": requests, "tokens": tokens,
         "cached": cached, "ragged": ragged, "window": window, "keep": keep, "sink": sink, "softcap": softcap}
    return {"name": name, **c} if name else c


def listed():
    return [
        # the new tokens of one decode step of eight requests: latency
        _case("write-decode-8", "write", "bfloat16", 32, 8, 128, 16, 8, 1, 1280, 1),
        # one portion of a long prompt
        _case("write-portion-2048", "write", "bfloat16", 32, 8, 128, 16, 1, 2048, 512, 0),
        # ragged portions of five requests in the 32-bit mode, heads of 64
        _case("write-ragged-f32", "write", "float32", 32, 8, 64, 16, 5, 211, 700, 2),
        # whole contexts of a batch taken out of the cache (moved to another pool, looked at)
        _case("read-contexts", "read", "bfloat16", 32, 8, 128, 16, 8, 1, 8191, 3),
        # a few short requests in 32 bits, heads of 64, larger pages
        _case("read-short-f32", "read", "float32", 32, 8, 64, 32, 3, 1, 333, 4),
        # one request decoding early in its reply: latency
        _case("decode-1-short", "attend", "bfloat16", 32, 8, 128, 16, 1, 1, 76, 0),
        # the benchmark's decode: eight requests of some 1,100 positions
        _case("decode-8", "attend", "bfloat16", 32, 8, 128, 16, 8, 1, 1151, 0),
        # a full batch of long and short requests
        _case("decode-64-ragged", "attend", "bfloat16", 32, 8, 128, 16, 64, 1, 8191, 5),
        # 32-bit decode with a window, kept first positions and learned sinks
        _case("decode-f32-window-sink", "attend", "float32", 32, 8, 64, 16, 5, 1, 3000, 6, window=1024, keep=4, sink=True),
        # portions of a few tokens beside single ones: prompts' tails, drafts to be checked
        _case("portions-short", "attend", "bfloat16", 32, 8, 128, 16, 12, 9, 2500, 7),
        # a portion of a long document on top of what is cached
        _case("portion-512-on-8192", "attend", "bfloat16", 32, 8, 128, 16, 1, 512, 8192, 0),
        # the benchmark's prompt in one step
        _case("prompt-2048", "attend", "bfloat16", 32, 8, 128, 16, 1, 2048, 0, 0),
    ]


_HEADS = [(32, 8, 128), (32, 8, 64), (40, 40, 128), (16, 2, 128), (8, 8, 64), (24, 4, 80), (4, 2, 16), (12, 12, 96), (6, 1, 256)]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = [work(c) for c in listed()]
    bytes_, flops = max(w["bytes"] for w in most), max(w["flops"] for w in most)
    while True:
        heads, kv, dim = rng.choice(_HEADS)
        dtype = "float32" if rng.random() < 0.3 else "bfloat16"
        page = rng.choice([8, 16, 16, 24, 32, 64])
        kind = rng.choice(["write", "read", "decode", "decode", "portion", "portion"])
        mix = rng.randrange(1, 1 << 20)
        options = {}
        if kind == "write":
            c = _case("", "write", dtype, heads, kv, dim, page, rng.randint(1, 16), _spread(rng, 1, 2048), _spread(rng, 1, 4096) - 1, mix)
        elif kind == "read":
            c = _case("", "read", dtype, heads, kv, dim, page, rng.randint(1, 8), 1, _spread(rng, 1, 8192) - 1, mix)
        else:
            if rng.random() < 0.35:
                options = {"window": _spread(rng, 1, 4096), "keep": rng.choice([0, 0, 4, 100])}
            if rng.random() < 0.25:
                options["sink"] = True
            if rng.random() < 0.2:
                options["softcap"] = rng.choice([15.0, 30.0, 50.0])
            if kind == "decode":
                c = _case("", "attend", dtype, heads, kv, dim, page, _spread(rng, 1, 64), 1, _spread(rng, 1, 8192) - 1, mix, **options)
            else:
                c = _case("", "attend", dtype, heads, kv, dim, page, _spread(rng, 1, 12), _spread(rng, 2, 2048), _spread(rng, 1, 8192) - 1,
                          mix, **options)
        w = work(c)
        if w["bytes"] <= bytes_ and w["flops"] <= flops and _padded(c) <= 2 ** 30:
            return c


# ------------------------------------------------------------------------------------------------------- layout
def _layout(c):
    """(counts, starts): how many tokens each request brings, how many it had. `ragged` 0: all alike; else a seed, and the
    first request has the most."""
    n, t, s = c["requests"], c["tokens"], c["cached"]
    if not c["ragged"]:
        return [t] * n, [s] * n
    r = random.Random(c["ragged"])
    return [t] + [r.randint(1, t) for _ in range(n - 1)], [s] + [r.randint(0, s) for _ in range(n - 1)]


def _seen(first, count, window, keep):
    """(pairs of a query and a key that it sees, keys that some query sees), queries at first .. first + count - 1."""
    if not window:
        return sum(range(first + 1, first + count + 1)), first + count
    pairs = sum(min(p + 1, window) + max(0, min(keep, p + 1 - window)) for p in range(first, first + count))
    low = max(0, first + 1 - window)
    return pairs, first + count - low + min(keep, low)


def _padded(c):
    """Values of the padded score matrix of the plain form."""
    counts, starts = _layout(c)
    if c["op"] != "attend":
        return 0
    return len(counts) * c["heads"] * max(counts) * max(a + b for a, b in zip(counts, starts))


def work(c):
    counts, starts = _layout(c)
    e = 2 if c["dtype"] == "bfloat16" else 4
    nh, nkv, d = c["heads"], c["kv"], c["dim"]
    if c["op"] == "write":  # rows in, rotated queries, codes and scales out, and those in and their values out again
        rows = sum(counts)
        return {"bytes": rows * (e * (nh + 2 * nkv) * d + e * nh * d + 2 * 2 * nkv * (d + 4) + e * 2 * nkv * d),
                "flops": rows * (3 * (nh + nkv) * d + 4 * 2 * nkv * d)}
    if c["op"] == "read":
        rows = sum(a + b for a, b in zip(counts, starts))
        return {"bytes": rows * 2 * nkv * (d + 4 + e * d), "flops": rows * 2 * nkv * d}
    seen = [_seen(s, t, c["window"], c["keep"]) for t, s in zip(counts, starts)]
    return {"bytes": 2 * e * sum(counts) * nh * d + sum(k for _, k in seen) * 2 * nkv * (d + 4),
            "flops": 4 * d * nh * sum(p for p, _ in seen)}


# ------------------------------------------------------------------------------------------------------- inputs
def _codes(x):
    """Rows of the last axis as codes (whole numbers in 32 bits) and scales."""
    a = x.abs().amax(-1, keepdim=True)
    zero = a < TINY
    most = torch.full_like(a, 127.0)  # (a division by or of a Python number would go by its reciprocal)
    inv = torch.where(zero, 0.0, most / torch.where(zero, 1.0, a))
    return torch.round(x * inv), torch.where(zero, 0.0, a / most).squeeze(-1)


def prepare(c, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = getattr(torch, c["dtype"])
    nh, nkv, d, page = c["heads"], c["kv"], c["dim"], c["page"]
    counts, starts = _layout(c)
    n, rows = len(counts), sum(counts)
    totals = [a + b for a, b in zip(counts, starts)]
    width = max(-(-t // page) for t in totals) + 1
    n_pages = sum(-(-t // page) for t in totals) + 3
    order = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32).cpu()
    slots = torch.randperm(n, generator=g, device=dev).cpu().tolist()  # a request's row of the tables
    tables, at = torch.full((n, width), -1, dtype=torch.int32), 0
    for s, t in zip(slots, totals):
        m = -(-t // page)
        tables[s, :m] = order[at:at + m]
        at += m
    channel = torch.exp(0.5 * torch.randn(nkv, 1, d, generator=g, device=dev))  # keys have channels larger than others
    channel = channel / channel.square().mean(-1, keepdim=True).sqrt()
    shape = (n_pages, nkv, page, d)
    filled = c["op"] != "write"

    def pool(factor):
        if not filled:
            return torch.zeros(shape, dtype=torch.int8, device=dev), torch.zeros(shape[:3], device=dev)
        k = torch.empty(shape, dtype=torch.int8, device=dev)
        s = torch.empty(shape[:3], device=dev)
        for i in range(0, n_pages, 4096):
            x = torch.randn(shape, generator=g, device=dev) if n_pages <= 4096 else \
                torch.randn((min(4096, n_pages - i), *shape[1:]), generator=g, device=dev)
            q, s[i:i + 4096] = _codes(x * factor)
            k[i:i + 4096] = q.to(torch.int8)
        return k, s

    k, k_scale = pool(channel)
    v, v_scale = pool(0.8)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    state = SimpleNamespace(c=c, k=k, v=v, k_scale=k_scale, v_scale=v_scale, tables=tables.to(dev),
                            err=torch.zeros(1, dtype=torch.int32, device=dev))
    if c["op"] == "read":  # every position of every request
        state.positions = ints([p for t in totals for p in range(t)])
        state.seq_of_row = ints([s for s, t in zip(slots, totals) for _ in range(t)])
        state.k_out = torch.empty(sum(totals), nkv, d, dtype=dtype, device=dev)
        state.v_out = torch.empty_like(state.k_out)
    else:
        positions = [a + i for a, t in zip(starts, counts) for i in range(t)]
        state.positions = ints(positions)
        state.seq_of_row = ints([s for s, t in zip(slots, counts) for _ in range(t)])
        row0 = [sum(counts[:i]) for i in range(n)]
        # the step as the engine's parts see it
        state.step = SimpleNamespace(n_rows=rows, n_seqs=n, positions=state.positions, seq_of_row=state.seq_of_row,
                                     req_row0=ints(row0), req_count=ints(counts), req_start=ints(starts),
                                     host={"counts": counts, "starts": starts}, static_max_len=None, plans={})
    if c["op"] == "write":
        x = torch.randn(rows, nh + 2 * nkv, d, generator=g, device=dev)
        x[:, nh:nh + nkv] *= channel.squeeze(1)
        state.qkv = x.reshape(rows, -1).to(dtype)
        freq = 500000.0 ** (-torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d)
        angle = torch.arange(max(totals), device=dev, dtype=torch.float64)[:, None] * freq
        state.cos, state.sin = angle.cos().float(), angle.sin().float()
        state.q_out = torch.empty(rows, nh * d, dtype=dtype, device=dev)
        state.k_out = torch.empty(rows, nkv, d, dtype=dtype, device=dev)
        state.v_out = torch.empty_like(state.k_out)
    if c["op"] == "attend":
        # the queries stand at the head of the rows that the stacked projection made
        qkv = (1.3 * torch.randn(rows, (nh + 2 * nkv) * d, generator=g, device=dev)).to(dtype)
        state.q = qkv[:, :nh * d]
        state.out = torch.empty(rows, nh * d, dtype=dtype, device=dev)
        state.sinks = torch.randn(nh, generator=g, device=dev) if c["sink"] else None
    return state


# ------------------------------------------------------------------------------------------------------- a pass
def run(s):
    c = s.c
    if own:
        from cuca_b200.kernels import ops
        pages = ops.QuantizedPages(s.k, s.v, s.k_scale, s.v_scale)
        if c["op"] == "write":
            ops.rope_store_q8(s.qkv, s.q_out, s.positions, s.seq_of_row, s.tables, s.cos, s.sin, c["dim"], pages, c["heads"],
                              c["kv"], c["dim"], s.err)
            ops.read_q8(pages, s.positions, s.seq_of_row, s.tables, s.k_out, s.v_out, s.err)
            return {"q": s.q_out, "k": s.k_out, "v": s.v_out}
        if c["op"] == "read":
            ops.read_q8(pages, s.positions, s.seq_of_row, s.tables, s.k_out, s.v_out, s.err)
            return {"k": s.k_out, "v": s.v_out}
        ops.attention_q8(s.q, s.out, pages, s.tables, s.step, c["heads"], c["kv"], c["dim"], c["dim"] ** -0.5,
                         c["window"] or None, s.err, keep_first=c["keep"], softcap=c["softcap"], sink=c["sink"],
                         sink_values=s.sinks)
        return {"out": s.out}
    return {"write": _plain_write, "read": _plain_read, "attend": _plain_attend}[c["op"]](s)


def _places(s, positions, seqs):
    """(pages, places in them) of positions of requests."""
    return s.tables[seqs, positions // s.c["page"]].clamp_min(0), positions % s.c["page"]


def _plain_read(s):
    page, off = _places(s, s.positions.long(), s.seq_of_row.long())
    dtype = getattr(torch, s.c["dtype"])
    return {"k": (s.k[page, :, off].float() * s.k_scale[page, :, off][..., None]).to(dtype),
            "v": (s.v[page, :, off].float() * s.v_scale[page, :, off][..., None]).to(dtype)}


def _plain_write(s):
    c = s.c
    nh, nkv, d = c["heads"], c["kv"], c["dim"]
    x = s.qkv.float().view(-1, nh + 2 * nkv, d)
    cos, sin = s.cos[s.positions.long()][:, None], s.sin[s.positions.long()][:, None]
    a, b = x[:, :nh + nkv, :d // 2], x[:, :nh + nkv, d // 2:]
    qk = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    page, off = _places(s, s.positions.long(), s.seq_of_row.long())
    codes, scale = _codes(qk[:, nh:])
    s.k[page, :, off], s.k_scale[page, :, off] = codes.to(torch.int8), scale
    codes, scale = _codes(x[:, nh + nkv:])
    s.v[page, :, off], s.v_scale[page, :, off] = codes.to(torch.int8), scale
    return {"q": qk[:, :nh].to(s.qkv.dtype).reshape(-1, nh * d), **_plain_read(s)}


def _plain_attend(s):
    c, step = s.c, s.step
    nh, nkv, d = c["heads"], c["kv"], c["dim"]
    group = nh // nkv
    # requests padded to the most tokens and the most positions
    tokens, keys = max(step.host["counts"]), max(a + b for a, b in zip(step.host["counts"], step.host["starts"]))
    t = torch.arange(tokens, device=s.q.device)
    live = t < step.req_count[:, None]
    row = (step.req_row0[:, None] + t).clamp_max(step.n_rows - 1).long()
    pos = torch.where(live, s.positions[row], -1)  # [requests, tokens]
    j = torch.arange(keys, device=s.q.device)
    held = j < (step.req_start + step.req_count)[:, None]
    page, off = _places(s, j[None], s.seq_of_row[step.req_row0.long()].long()[:, None])
    off = off.expand_as(page)
    k = torch.where(held[..., None, None], s.k[page, :, off].float() * s.k_scale[page, :, off][..., None], 0.0)
    v = torch.where(held[..., None, None], s.v[page, :, off].float() * s.v_scale[page, :, off][..., None], 0.0)
    q = s.q.float()[row].view(-1, tokens, nkv, group, d)
    score = torch.matmul(q.permute(0, 2, 3, 1, 4).reshape(-1, nkv, group * tokens, d), k.permute(0, 2, 3, 1)) * d ** -0.5
    score = score.view(-1, nkv, group, tokens, keys)
    if c["softcap"]:
        score = c["softcap"] * torch.tanh(score / c["softcap"])
    far = pos[..., None] - j
    see = far >= 0
    if c["window"]:
        see = see & ((far < c["window"]) | (j < c["keep"]))
    score = torch.where(see[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    sink = s.sinks.view(1, nkv, group, 1, 1) if s.sinks is not None else None
    if sink is not None:
        top = torch.maximum(top, sink)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink - top)
    o = torch.matmul(p.view(-1, nkv, group * tokens, keys), v.permute(0, 2, 1, 3)).view(-1, nkv, group, tokens, d)
    o = (o / torch.where(total > 0, total, 1.0)).permute(0, 3, 1, 2, 4).reshape(-1, tokens, nh * d)
    return {"out": o[live].to(s.q.dtype)}


# ------------------------------------------------------------------------------------------------------- in 64 bits
def exact(c, seed):
    s = prepare(c, seed)
    nh, nkv, d, page = c["heads"], c["kv"], c["dim"], c["page"]
    tables = s.tables.long()

    def cached(codes, scales, slot, length):
        p = torch.arange(length, device=codes.device)
        at = tables[slot, p // page]
        return codes[at, :, p % page].double() * scales[at, :, p % page].double()[..., None]  # [length, kv, d]

    if c["op"] == "read":
        counts, starts = _layout(c)
        slots, at = s.seq_of_row.tolist(), 0
        k, v = [], []
        for total in (a + b for a, b in zip(counts, starts)):
            k.append(cached(s.k, s.k_scale, slots[at], total))
            v.append(cached(s.v, s.v_scale, slots[at], total))
            at += total
        return {"k": torch.cat(k), "v": torch.cat(v)}
    if c["op"] == "write":
        x = s.qkv.double().view(-1, nh + 2 * nkv, d)
        # the rotation as a product of complex numbers, with the tables' cosines and sines
        turn = torch.complex(s.cos.double(), s.sin.double())[s.positions.long()][:, None]
        turned = torch.complex(x[:, :nh + nkv, :d // 2], x[:, :nh + nkv, d // 2:]) * turn
        turned = torch.cat((turned.real, turned.imag), -1)

        def held(rows):
            most = rows.abs().max(-1, keepdim=True).values
            step = torch.where(most < TINY, torch.ones_like(most), most / 127)
            return torch.round(rows / step) * step

        return {"q": turned[:, :nh].reshape(-1, nh * d), "k": held(turned[:, nh:]), "v": held(x[:, nh + nkv:])}
    out = torch.zeros(s.q.shape[0], nh, d, dtype=torch.float64, device=s.q.device)
    for row0, count, start in zip(s.step.req_row0.tolist(), *(s.step.host[x] for x in ("counts", "starts"))):
        slot = int(s.seq_of_row[row0])
        k, v = cached(s.k, s.k_scale, slot, start + count), cached(s.v, s.v_scale, slot, start + count)
        p = torch.arange(start, start + count, device=s.q.device)[:, None]
        j = torch.arange(start + count, device=s.q.device)[None]
        hidden = j > p
        if c["window"]:
            hidden |= (p - j >= c["window"]) & (j >= c["keep"])
        for h in range(nh):
            q = s.q[row0:row0 + count, h * d:(h + 1) * d].double()
            z = q @ k[:, h * nkv // nh].T / math.sqrt(d)
            if c["softcap"]:
                z = c["softcap"] * torch.tanh(z / c["softcap"])
            z = z.masked_fill(hidden, -math.inf)
            if s.sinks is not None:  # one more term, whose value is zero
                z = torch.cat((z, s.sinks[h].double().expand(count, 1)), 1)
                out[row0:row0 + count, h] = torch.softmax(z, -1)[:, :-1] @ v[:, h * nkv // nh]
            else:
                out[row0:row0 + count, h] = torch.softmax(z, -1) @ v[:, h * nkv // nh]
    return {"out": out.view(-1, nh * d)}
