"""Products with 4-bit weights where bits are easily lost or places mixed up, against the formulas in 64 bits (`mx4_util`)."""
import math

import pytest
import torch

import mx4_util as mx

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def lib():
    from cuca_b200.kernels import library
    return library.load()


def _normal(rows, cols, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(rows, cols, generator=g, device="cuda").to(dtype)


def _multiply(kind, x, w, epilogue="store", out_dtype=F32, bias=None, stream=None):
    """(what the kernels make of it, the rows' values and the weight's in 64 bits)"""
    from cuca_b200.kernels import ops
    q = ops.mx4_quantise(w)
    a, xv = (ops.mx4_quantise(x), mx.held(x)) if kind == "codes" else (x, x.double())
    n = w.shape[0] // (2 if epilogue == "swiglu" else 1)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full((x.shape[0], n), 7.0, dtype=out_dtype, device="cuda") if stream is None else stream.clone()
    code = {"store": ops.EPI_STORE, "swiglu": ops.EPI_SWIGLU, "residual": ops.EPI_RESIDUAL}[epilogue]
    ops.gemm_mx4(a, q, out, code, bias, err)
    assert err.item() == 0
    return out, xv, mx.held(w)


def _within(out, want, bound):
    off = (out.double() - want).abs()
    assert torch.isfinite(out).all() and (off <= bound).all(), f"{(off / bound).max().item()} of the bound"


@pytest.mark.parametrize("kind", ["bf16", "f32", "codes"])
@pytest.mark.parametrize("m", [1, 3, 9, 20, 41, 70])
@pytest.mark.parametrize("n", [5, 77, 130, 201])
def test_ragged_tiles_that_share_a_long_sum(kind, m, n):
    """Blocks of a cluster add up sums of ragged tiles: lanes of a warp leave that with different numbers of rows."""
    k = 2050
    x, w = _normal(m, k, F32 if kind == "f32" else BF16, m), _normal(2 * n, k, F32, n) / math.sqrt(k)
    for epilogue in ("store", "swiglu"):
        out, xv, wv = _multiply(kind, x, w, epilogue)
        _within(out, *mx.product(xv, wv, epilogue, F32, k / 16 + 24, digits=kind != "codes"))


def _drift(values, one_sign=False):
    """How far (2-norm over that of the result) a 32-bit sum of so many exact products may be off. The tensor cores take 16 at a time and cut
    off at most 2^-23 of what has been summed. Cut off evenly up to that, with signs that vary over sums that grow as a square root,
    n times come to sqrt(n / 6) of it; where everything has one sign half of it each time, over sums that are half the last in
    the mean. One more for the rounding of what is left and joined."""
    n = values / 16
    return 2.0 ** -23 * ((n / 4 if one_sign else math.sqrt(n / 6)) + 1)


@pytest.mark.parametrize("one_sign", [False, True])
@pytest.mark.parametrize("m,k,n,epilogue", [
    (200, 40_000, 8192, "store"), (20, 40_000, 9000, "residual"), (250, 36_000, 8192, "store"),
    (200, 20_000, 9500, "swiglu"), (300, 20_000, 2050, "swiglu"), (40, 36_000, 4600, "swiglu"), (300, 17_000, 19_200, "store")])
def test_long_sums_in_32_bits_leave_after_8192_values(m, k, n, epilogue, one_sign):
    """Alone, in a cluster's shares and in a gated unit alike."""
    gated = epilogue == "swiglu"
    x, w = _normal(m, k, BF16, 1), _normal(2 * n if gated else n, k, BF16, 2) / math.sqrt(k)
    if one_sign:
        x, w = x.abs(), w.abs()
    stream = _normal(m, n, F32, 3) if epilogue == "residual" else None
    from cuca_b200.kernels import ops
    some = torch.arange(0, n, 257, device="cuda")
    held = mx.held(w[torch.cat((some, n + some)) if gated else some])
    q = ops.mx4_quantise(w)
    del w
    out = torch.empty(m, n, device="cuda") if stream is None else stream.clone()
    ops.gemm_mx4(x, q, out, {"store": ops.EPI_STORE, "swiglu": ops.EPI_SWIGLU, "residual": ops.EPI_RESIDUAL}[epilogue])
    want = x.double() @ held.T
    limit = _drift(8192, one_sign)
    if gated:  # silu's slope is below 1.1, both factors are off
        g, u = want.chunk(2, 1)
        want, limit = g * torch.sigmoid(g) * u, 2.1 * limit
    elif stream is not None:
        want = want + stream[:, some].double()
    assert (out[:, some].double() - want).norm() < limit * want.norm()
