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
