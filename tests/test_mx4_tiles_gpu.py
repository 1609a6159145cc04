"""Products with 4-bit weights whose blocks take several tiles in turn: every result against the formula in 64 bits (`mx4_util`)."""
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


# More tiles than an SM's blocks, of 128 features (256 over many rows that are not gated) by up to 192 rows (256); an odd number of steps of
# 128 values; more stages of 256 values than shared memory holds (three of the largest tiles, eight of the smallest); features off 128, so
# that the up rows' scales are read word by word; a last tile of few rows or features.
CASES = [
    ("codes", 2048, 320, 2176, "swiglu"), ("codes", 2048, 320, 2050, "swiglu"), ("codes", 2000, 1300, 2100, "swiglu"), ("codes", 1999, 1300, 2176, "swiglu"),
    ("codes", 2048, 320, 4100, "store"), ("codes", 2048, 1300, 4100, "residual"), ("codes", 2017, 2500, 4230, "store"), ("codes", 3000, 100, 3000, "residual"),
    ("codes", 40, 2400, 40_000, "store"), ("codes", 200, 700, 20_000, "residual"), ("codes", 30, 1300, 20_001, "swiglu"), ("codes", 150, 1300, 20_096, "swiglu"),
    ("bf16", 3, 2500, 40_003, "store"), ("bf16", 10, 600, 50_000, "residual"), ("bf16", 16, 700, 40_000, "store"),
    ("bf16", 1, 2500, 40_010, "swiglu"), ("bf16", 9, 600, 20_096, "swiglu"), ("bf16", 16, 1300, 20_001, "swiglu"),
    ("bf16", 600, 700, 9000, "store"), ("bf16", 513, 700, 5000, "swiglu"), ("f32", 512, 300, 2304, "swiglu"), ("f32", 512, 2300, 2304, "store"), ("f32", 512, 700, 4700, "residual")]


@pytest.mark.parametrize("kind,m,k,n,epilogue", CASES)
def test_every_result_of_many_tiles(kind, m, k, n, epilogue):
    from cuca_b200.kernels import ops
    gated = epilogue == "swiglu"
    x, w = _normal(m, k, F32 if kind == "f32" else BF16, m), _normal(2 * n if gated else n, k, F32, n) / math.sqrt(k)
    q = ops.mx4_quantise(w)
    a, xv, wv = (ops.mx4_quantise(x), mx.held(x), mx.held(w)) if kind == "codes" else (x, x.double(), mx.held(w))
    bias = None if gated else _normal(1, n, F32, 5)[0].contiguous()
    for out_dtype in (BF16, F32):
        if out_dtype == BF16 and (kind == "f32" or epilogue == "residual"):
            continue
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        stream = _normal(m, n, F32, 6) if epilogue == "residual" else None
        out = torch.full((m, n), 7.0, dtype=out_dtype, device="cuda") if stream is None else stream.clone()
        ops.gemm_mx4(a, q, out, {"store": ops.EPI_STORE, "swiglu": ops.EPI_SWIGLU, "residual": ops.EPI_RESIDUAL}[epilogue], bias, err)
        assert err.item() == 0
        want, bound = mx.product(xv, wv, epilogue, out_dtype, k / 16 + 24, bias, stream, digits=kind == "bf16" and m <= 16)
        off = (out.double() - want).abs()
        assert torch.isfinite(out).all() and (off <= bound).all(), f"{(off / bound).max().item()} of the bound"
        # a place that another tile's sums reached, or one that was passed over, is off by as much as results are large
        assert (out.double() - want).norm() < (2.0 ** -8 if out_dtype == BF16 else 1e-6) * want.norm()
