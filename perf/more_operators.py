"""Weights and activations in microscaled 4-bit floating point, measured operator by operator.

A row is cut into blocks of 32 values. A block is a power of two (one byte e, it stands for 2^(e - 127); 255 for NaN) and 32 codes of
4 bits: a sign and one of 0, 1/2, 1, 3/2, 2, 3, 4, 6. With a = max |x| of the block the power is 2^(floor(log2 a) - 2), not below
2^-127, and a code stands for x over that power, rounded to the nearest (ties to the even code) and to 6 at most.
The last block of a row may be short.

* "quantise": rows to 4 bits. The pass reads them back too: what is held in 4 bits is returned as the values it stands for.
* "wide": x W^T with x as it is (16 or 32 bits) and the weight in 4 bits: a projection of a model that keeps its weights small.
* "narrow": the same with x quantised first, both operands in 4 bits: the projection where activations are small too.

`epilogue` "store" leaves the sums (plus a bias) in the compute type or, with `sums`, in 32 bits for the residual stream; "swiglu" makes
silu(g) u of the stacked gate and up rows of the weight. Shapes: the projections of the benchmark's models and ragged small ones.
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

BLOCK = 32


# ------------------------------------------------------------------------------------------------------- cases
def _case(name, op, dtype, rows, k, n=0, epilogue="store", sums=False, bias=False):
    c = {"op": op, "dtype": dtype, "rows": rows, "k": k, "n": n, "epilogue": epilogue, "sums": sums, "bias": bias}
    return {"name": name, **c} if name else c


def listed():
    return [
        # what enters a projection of a decode step of eight requests: latency
        _case("quantise-decode-8", "quantise", "bfloat16", 8, 4096),
        # what a feed-forward's inner layer of a prompt makes, before its last projection
        _case("quantise-prompt-2048", "quantise", "bfloat16", 2048, 14336),
        # a weight of 32-bit numbers with rows of an odd size, as it is loaded
        _case("quantise-ragged-f32", "quantise", "float32", 1003, 2050),
        # one request's output projection: latency
        _case("wide-decode-1", "wide", "bfloat16", 1, 4096, 4096, sums=True),
        # the benchmark's decode of eight requests: gate, up and their unit
        _case("wide-decode-8-swiglu", "wide", "bfloat16", 8, 4096, 14336, epilogue="swiglu"),
        # a full batch of single tokens: the feed-forward's last projection, into the stream
        _case("wide-decode-64", "wide", "bfloat16", 64, 14336, 4096, sums=True),
        # a few tokens in the 32-bit mode, odd sizes, with a bias
        _case("wide-ragged-f32", "wide", "float32", 5, 1010, 2050, bias=True),
        # a prompt in one step: gate, up and their unit
        _case("wide-prompt-2048-swiglu", "wide", "bfloat16", 2048, 4096, 14336, epilogue="swiglu"),
        # eight requests: the stacked query, key and value projection
        _case("narrow-decode-8", "narrow", "bfloat16", 8, 4096, 6144),
        # an odd portion of tokens at odd sizes, with a bias
        _case("narrow-ragged-77", "narrow", "bfloat16", 77, 1010, 2050, bias=True),
        # a prompt in one step: gate, up and their unit
        _case("narrow-prompt-2048-swiglu", "narrow", "bfloat16", 2048, 4096, 14336, epilogue="swiglu"),
        # the same prompt: the feed-forward's last projection, into the stream
        _case("narrow-prompt-2048", "narrow", "bfloat16", 2048, 14336, 4096, sums=True),
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """A layer's size: mostly a multiple of 64, at times any number."""
    n = _spread(rng, lo, hi)
    return n if rng.random() < 0.3 or n < 64 else n // 64 * 64


def draw(rng):
    most = [work(c) for c in listed()]
    bytes_, flops = max(w["bytes"] for w in most), max(w["flops"] for w in most)
    while True:
        op = rng.choice(["quantise", "wide", "wide", "narrow", "narrow"])
        k = _size(rng, 20, 14336)
        if op == "quantise":
            c = _case("", op, "float32" if rng.random() < 0.3 else "bfloat16", _spread(rng, 1, 16384), k)
        else:
            # the 32-bit mode: up to a default portion of a prompt
            f32 = op == "wide" and rng.random() < 0.25
            rows = _spread(rng, 1, 256 if f32 else 2048)
            swiglu = rng.random() < 0.3
            n = _size(rng, 8, 14336 if swiglu else 16384)
            c = _case("", op, "float32" if f32 else "bfloat16", rows, k, n, "swiglu" if swiglu else "store",
                      not swiglu and rng.random() < 0.4, not swiglu and rng.random() < 0.3)
        w = work(c)
        if w["bytes"] <= bytes_ and w["flops"] <= flops:
            return c


def work(c):
    e = 2 if c["dtype"] == "bfloat16" else 4
    m, k = c["rows"], c["k"]
    if c["op"] == "quantise":  # x in, codes and scales out, and the values that they stand for
        return {"bytes": m * (k * e + (k + 1) // 2 + -(-k // BLOCK) + k * e), "flops": 4 * m * k}
    n = c["n"] * (2 if c["epilogue"] == "swiglu" else 1)
    return {"bytes": m * k * e + n * ((k + 1) // 2 + -(-k // BLOCK)) + m * c["n"] * (4 if c["sums"] else e) + (n * e if c["bias"] else 0),
            "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------------------------------- inputs
def prepare(c, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = getattr(torch, c["dtype"])
    m, k = c["rows"], c["k"]
    # activations have channels larger than others
    channel = torch.exp(0.7 * torch.randn(k, generator=g, device=dev))
    x = (torch.randn(m, k, generator=g, device=dev) * channel).to(dtype)
    s = SimpleNamespace(c=c, x=x, err=torch.zeros(1, dtype=torch.int32, device=dev))
    if c["op"] == "quantise":
        s.out = torch.empty_like(x)
        return s
    n = c["n"] * (2 if c["epilogue"] == "swiglu" else 1)
    w = torch.randn(n, k, generator=g, device=dev) * (1.0 / math.sqrt(k))
    s.bias = (0.1 * torch.randn(n, generator=g, device=dev)).to(dtype) if c["bias"] else None
    s.out = torch.empty(m, c["n"], dtype=torch.float32 if c["sums"] else dtype, device=dev)
    if own:  # the weight as the framework keeps it
        from cuca_b200.kernels import ops
        s.w = ops.mx4_quantise(w)
    else:
        s.codes, s.scales = _quantise(w)
    return s


# ------------------------------------------------------------------------------------------------------- a pass
def run(s):
    c = s.c
    if own:
        from cuca_b200.kernels import ops
        if c["op"] == "quantise":
            ops.mx4_values(ops.mx4_quantise(s.x), s.out)
            return {"values": s.out}
        a = ops.mx4_quantise(s.x) if c["op"] == "narrow" else s.x
        ops.gemm_mx4(a, s.w, s.out, ops.EPI_SWIGLU if c["epilogue"] == "swiglu" else ops.EPI_STORE, s.bias, s.err)
        return {"out": s.out}
    if c["op"] == "quantise":
        return {"values": _values(*_quantise(s.x), c["k"]).to(s.x.dtype)}
    x = _values(*_quantise(s.x), c["k"]) if c["op"] == "narrow" else s.x.float()
    y = torch.matmul(x, _values(s.codes, s.scales, c["k"]).T)
    if c["epilogue"] == "swiglu":
        gate, up = y[:, :c["n"]], y[:, c["n"]:]
        y = gate / (1.0 + torch.exp(-gate)) * up
    if s.bias is not None:
        y = y + s.bias.float()
    return {"out": y.to(s.out.dtype)}


def _quantise(x):
    """Rows in 4 bits: two codes to a byte [rows, blocks, 16], the first in the low half, and a byte per block [rows, blocks]."""
    m, k = x.shape
    blocks = -(-k // BLOCK)
    v = torch.zeros(m, blocks * BLOCK, device=x.device)
    v[:, :k] = x
    v = v.view(m, blocks, BLOCK)
    most = v.abs().amax(-1)
    exponent = torch.where(most > 0, torch.frexp(most)[1] - 3, -127).clamp_min(-127)  # frexp: a = f 2^e with f from 1/2 on
    scales = (exponent + 127).to(torch.uint8)
    v = v / _powers(scales)[..., None]
    a = v.abs()
    a = torch.where(a < 2, torch.round(a * 2) / 2, torch.where(a < 4, torch.round(a), torch.round(a / 2) * 2)).clamp_max(6)
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = code + 8 * (v < 0).to(torch.uint8)
    return code[..., ::2] + 16 * code[..., 1::2], scales


def _powers(scales):
    """2^(e - 127) of bytes e, by the bits of 32-bit numbers (a power function is not exact on the device)."""
    e = scales.int()
    return torch.where(e > 0, e << 23, 1 << 22).view(torch.float32)


def _values(codes, scales, k):
    """The values that codes and scales stand for, in 32 bits."""
    code = torch.stack((codes % 16, codes // 16), -1).flatten(-2).float()
    sign = torch.where(code >= 8, -1.0, 1.0)
    a = code % 8
    a = torch.where(a < 4, a / 2, torch.where(a < 6, a - 2, 2 * a - 8))
    return (sign * a * _powers(scales)[..., None]).flatten(1)[:, :k]


# ------------------------------------------------------------------------------------------------------- in 64 bits
_BORDERS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)  # between the magnitudes that codes stand for


def _power(exponent):
    """Powers of two in 64 bits, by their bits."""
    return ((exponent.long() + 1023) << 52).view(torch.float64)


def _nearest(x):
    """What rows in 4 bits stand for, in 64 bits, by the borders between magnitudes."""
    m, k = x.shape
    magnitudes = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    out = torch.empty(m, k, dtype=torch.float64, device=x.device)
    for at in range(0, k, BLOCK):
        v = x[:, at:at + BLOCK].double()
        most = v.abs().max(1, keepdim=True).values
        exponent = torch.floor(torch.log2(most)).clamp_min(-125)
        exponent = exponent + (most >= _power(exponent + 1)).double() - (most < _power(exponent)).double()  # (log2 may be a bit off)
        power = _power(exponent.clamp_min(-125) - 2)
        a = v.abs() / power
        index = torch.zeros_like(a, dtype=torch.long)
        for i, border in enumerate(_BORDERS):  # a value on a border takes the even code
            index += (a > border) if i % 2 == 0 else (a >= border)
        out[:, at:at + BLOCK] = torch.sign(v) * magnitudes[index] * power
    return out


def exact(c, seed):
    global own
    mine, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = mine
    if c["op"] == "quantise":
        return {"values": _nearest(s.x)}
    x = _nearest(s.x) if c["op"] == "narrow" else s.x.double()
    # the weight's values, from its bytes
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64, device=x.device)
    n = s.codes.shape[0]
    y = torch.empty(c["rows"], n, dtype=torch.float64, device=x.device)
    for at in range(0, n, 4096):
        codes = s.codes[at:at + 4096].long()
        w = torch.stack((table[codes & 15], table[codes >> 4]), -1).flatten(-2) * _power(s.scales[at:at + 4096].long() - 127)[..., None]
        y[:, at:at + 4096] = x @ w.flatten(1)[:, :c["k"]].T
    if s.bias is not None:
        y += s.bias.double()
    if c["epilogue"] == "swiglu":
        y = y[:, :c["n"]] * torch.sigmoid(y[:, :c["n"]]) * y[:, c["n"]:]
    return {"out": y}
