"""Microscaled 4-bit rows and their products from the formulas in 64 bits, for the tests of the kernels."""
import torch

MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BORDERS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)  # between two magnitudes: a value on one takes the even code


def quantise(x):
    """(codes [rows, blocks, 32], bytes [rows, blocks]) of rows, in 64 bits; what a last block has beyond its row is zeros."""
    m, k = x.shape
    blocks = -(-k // 32)
    v = torch.zeros(m, blocks * 32, dtype=torch.float64, device=x.device)
    v[:, :k] = x.double()
    v = v.view(m, blocks, 32)
    bad = ~torch.isfinite(v).all(-1)
    v = torch.where(bad[..., None], 0.0, v)
    most = v.abs().amax(-1)
    power = torch.where(most > 0, torch.frexp(most)[1].long() - 3, -127).clamp_min(-127)
    a = v.abs() * torch.ldexp(torch.ones_like(most).cpu(), -power.cpu()).to(x.device)[..., None]
    code = torch.zeros_like(a, dtype=torch.long)
    for i, border in enumerate(BORDERS):
        code += (a > border) if i % 2 == 0 else (a >= border)
    code += 8 * ((v < 0) & (code > 0))
    return code, torch.where(bad, 255, power + 127)


def values(code, byte, k):
    """The values of codes and bytes in 64 bits."""
    table = torch.tensor(MAGNITUDES + tuple(-v for v in MAGNITUDES), dtype=torch.float64, device=code.device)
    power = torch.ldexp(torch.ones(byte.shape, dtype=torch.float64), byte.cpu().long() - 127).to(code.device)
    power = torch.where(byte == 255, torch.nan, power)
    return (table[code] * power[..., None]).flatten(1)[:, :k]


def unpack(matrix):
    """(codes [rows, blocks, 32], bytes [rows, blocks]) that a `Mx4Matrix` holds, without its padding."""
    rows, cols = matrix.shape
    blocks = -(-cols // 32)
    c = matrix.codes.long()
    code = torch.stack((c & 15, c >> 4), -1).view(rows, -1, 2, 4).transpose(2, 3).reshape(rows, -1, 32)  # 0 2 4 6 1 3 5 7
    tail = code[:, blocks:]
    assert not tail.any(), "what lies beyond a row in its last step is zeros"
    s = matrix.scales.long()  # [tiles, steps, 32, 4, 4]
    byte = s.permute(0, 3, 2, 1, 4).reshape(s.shape[0] * 128, -1)[:rows, :blocks]
    return code[:, :blocks], byte


def held(x):
    """What rows in 4 bits stand for, in 64 bits."""
    return values(*quantise(x), x.shape[1])


def chain_bound(x, w, additions):
    """How far a sum of exact products may be off: each of so many additions in a row cuts off at most 2^-23 of what has been
    summed, which is at most the sum of the products' magnitudes."""
    return additions * 2.0 ** -23 * (x.abs() @ w.abs().T)


def digits_bound(x, w):
    """How far a product may be off whose rows go as eight digits in 4 bits: what is left of a value is at most 2^-23 of the largest
    magnitude among its 32."""
    m, k = x.shape
    most = torch.zeros(m, -(-k // 32) * 32, dtype=torch.float64, device=x.device)
    most[:, :k] = x.abs()
    most = most.view(m, -1, 32).amax(-1, keepdim=True).expand(-1, -1, 32).flatten(1)[:, :k]
    return 2.0 ** -23 * (most @ w.abs().T)


def product(x, w, epilogue, out_dtype, additions, bias=None, stream=None, digits=False):
    """(result, bound on the error) of epilogue(x w^T) over 64-bit rows. `digits`: the rows go as digits in 4 bits; a value's digits, the
    first of which may be twice it and the others an eighth of it in all, come to 2.5 of its magnitude at most."""
    y, b = x @ w.T, chain_bound(x, w, additions)
    if digits:
        b = 2.5 * b + digits_bound(x, w)
    if epilogue == "swiglu":
        n = y.shape[1] // 2
        g, u, bg, bu = y[:, :n], y[:, n:], b[:, :n], b[:, n:]
        s = g * torch.sigmoid(g)
        y = s * u
        # silu's slope is below 1.1; exponential and quotient are good to 2^-20 of the result and an ulp of the exponent
        b = 1.1 * bg * (u.abs() + bu) + s.abs() * bu + y.abs() * (2.0 ** -20 + g.abs() * 2.0 ** -22)
    if bias is not None:
        y = y + bias.double()
        b = b + y.abs() * 2.0 ** -24
    if stream is not None:
        y = y + stream.double()
    step = torch.finfo(out_dtype).eps / 2
    least = 2.0 ** -133 if out_dtype == torch.bfloat16 else 2.0 ** -149
    return y, b + step * (y.abs() + b) + least
