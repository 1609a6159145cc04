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
@pytest.mark.parametrize("k,n", [(2050, 5), (2050, 77), (2050, 130), (2050, 201), (14_337, 1201)])
def test_ragged_tiles_that_share_a_long_sum(kind, m, k, n):
    """Blocks of a cluster add up sums of ragged tiles: lanes of a warp leave that with different numbers of rows."""
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


def _plain(xv, wv):
    """The same product summed in 32 bits by PyTorch, in 64 bits."""
    return (xv.float() @ wv.float().T).double()


@pytest.mark.parametrize("k", [256, 4096])
@pytest.mark.parametrize("larger", [1e3, 1e4, 1e9])
@pytest.mark.parametrize("m", [1, 5, 64, 256, 300])
def test_32_bit_rows_keep_their_bits_beside_larger_values(m, larger, k):
    """Rows of 24 significant bits with one value of every 32 much larger, where the weight is zero: what counts is the others, and all of
    their bits."""
    n = 300
    x, w = _normal(m, k, F32, m), _normal(n, k, F32, 2)
    x[:, 5::32] *= larger
    w[:, 5::32] = 0
    out, xv, wv = _multiply("f32", x, w)
    want = xv @ wv.T
    assert (out.double() - want).norm() < _drift(min(k, 2048)) * want.norm()
    rest = xv.clone()
    rest[:, 5::32] = 0
    _within(out, want, mx.chain_bound(rest, wv, k / 16 + 24) + 2.0 ** -24 * want.abs())


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("m,k,n", [(1, 33, 300), (3, 130, 257), (5, 1010, 2050), (8, 4096, 512), (16, 14_336, 300), (24, 640, 200), (2, 14_336, 77),
                                   (40, 4096, 320), (100, 2048, 130), (256, 4096, 512), (300, 14_336, 256), (1, 4096, 4100), (8, 14_336, 1300), (16, 2050, 9000)])
def test_products_in_32_bits_by_their_2_norm(kind, m, k, n):
    """As near to 64 bits as sums in 32 bits are, channels larger than others among the rows."""
    g = torch.Generator(device="cuda").manual_seed(k)
    x = (_normal(m, k, F32, m) * torch.exp(0.7 * torch.randn(k, generator=g, device="cuda"))).to(F32 if kind == "f32" else BF16)
    out, xv, wv = _multiply(kind, x, _normal(n, k, F32, 2) / math.sqrt(k))
    want = xv @ wv.T
    assert (out.double() - want).norm() < _drift(min(k, 2048 if kind == "f32" else 8192)) * want.norm()


def test_32_bit_rows_of_all_sizes():
    """Numbers from the smallest on whose parts bfloat16 holds, up to the largest, times powers of two that bring them near one."""
    k, n = 64, 40
    for power in (-109, -60, 0, 100, 126):
        x = _normal(7, k, F32, power % 97).clamp(-1.9, 1.9)
        x = torch.where(x.abs() < 1, x.sign() + x, x) * 2.0 ** power  # 1 to 2 and their negatives
        w = _normal(n, k, F32, 3) * 2.0 ** (-power / 2)
        if power > 100:
            w /= 1024  # (sums in range)
        out, xv, wv = _multiply("f32", x, w)
        _within(out, *mx.product(xv, wv, "store", F32, k / 16 + 24))


def test_32_bit_rows_that_are_not_finite():
    x, w = _normal(9, 96, F32, 1), _normal(33, 96, F32, 2)
    x[2, 40], x[4, 3] = math.inf, -math.inf
    x.view(torch.int32)[6, 70] = 0x7F800001  # a NaN of the lowest bits
    out, xv, wv = _multiply("f32", x, w)
    assert out[6].isnan().all() and not out[[2, 4]].isfinite().any()
    good = [0, 1, 3, 5, 7, 8]
    _within(out[good], *mx.product(xv[good], wv, "store", F32, 30))


@pytest.mark.parametrize("epilogue", ["store", "residual", "swiglu"])
@pytest.mark.parametrize("m,k,n", [(1, 2049, 200), (8, 4096, 1100), (17, 6100, 77), (85, 2500, 130), (86, 4100, 9500), (171, 9000, 96), (256, 2300, 640)])
def test_32_bit_rows_whose_sums_leave_several_times(m, k, n, epilogue):
    """Alone, shared and gated, tiles of 85 rows and of few; a bias and a stream are rounded into a result once."""
    gated = epilogue == "swiglu"
    x, w = _normal(m, k, F32, m), _normal(2 * n if gated else n, k, F32, n) / math.sqrt(k)
    bias, stream = (None if gated else _normal(1, n, F32, 5)[0].contiguous()), (_normal(m, n, F32, 6) if epilogue == "residual" else None)
    out, xv, wv = _multiply("f32", x, w, epilogue, F32, bias, stream)
    _within(out, *mx.product(xv, wv, epilogue, F32, k / 16 + 24, bias, stream))


def _small_beside_large(m, k, dtype, seed):
    """Rows whose blocks hold values of four sizes, 2^40, 2^25, 2^12 and about one; the weights to go with them are zero for all but the last."""
    x = _normal(m, k, F32, seed)
    counts = torch.ones(k, dtype=torch.bool, device="cuda")
    for at, power in ((3, 40), (4, 25), (17, 12), (30, 40), (31, 25)):
        x[:, at::32] *= 2.0 ** power
        counts[at::32] = False
    return x.to(dtype), counts


@pytest.mark.parametrize("epilogue", ["store", "swiglu"])
@pytest.mark.parametrize("k,n", [(200, 130), (4096, 300), (2050, 201), (512, 9600), (4096, 4100), (2050, 9001), (200, 84_000), (14_337, 1201)])
@pytest.mark.parametrize("m", [1, 3, 8, 9, 11, 16, 17, 24])
def test_few_rows_keep_their_bits_beside_larger_values(m, k, n, epilogue):
    """The products of few rows are exact too: a value's bits are all there, however much larger its block's others are."""
    x, counts = _small_beside_large(m, k, BF16, m)
    w = _normal(2 * n if epilogue == "swiglu" else n, k, F32, 2) / math.sqrt(k)
    w[:, ~counts] = 0
    out, xv, wv = _multiply("bf16", x, w, epilogue)
    xv[:, ~counts] = 0
    _within(out, *mx.product(xv, wv, epilogue, F32, 2.5 * k / 16 + 24))


@pytest.mark.parametrize("m", [1, 5, 16])
def test_few_rows_of_every_size_in_a_block(m):
    """A block whose values go from 2^70 down to 2^-120 in steps of 2^6, in any order; the weight reads one of them at a time."""
    k = 96
    g = torch.Generator(device="cuda").manual_seed(m)
    x = _normal(m, k, F32, m)
    x = (x.sign() * (1 + x.abs() % 1)).to(BF16).float()
    for b in range(3):
        x[:, 32 * b:32 * b + 32] *= torch.exp2(70.0 - 6 * torch.randperm(32, generator=g, device="cuda"))
    x = x.to(BF16)
    for n in (96, 180_000):
        w = torch.zeros(n, k, device="cuda")
        w[torch.arange(n), torch.arange(n) % k] = 1
        out, xv, wv = _multiply("bf16", x, w)
        assert torch.equal(out.double(), xv @ wv.T)


def test_few_rows_of_the_smallest_numbers():
    """Numbers below 2^-126, times weights that bring them up."""
    x = (_normal(4, 64, F32, 1) * 2.0 ** -128).to(BF16)
    for n in (70, 270_000):
        out, xv, wv = _multiply("bf16", x, _normal(n, 64, F32, 2) * 2.0 ** 100)
        _within(out, *mx.product(xv, wv, "store", F32, 30))


@pytest.mark.parametrize("m", [1, 4, 10, 11, 16])
def test_few_rows_of_a_large_weight_every_way(m):
    """Rows with gaps and off 16 bytes, results into columns of a wider matrix, every epilogue and result type, a bias of either type, values
    and weights that are not finite, and a graph replayed on other rows."""
    from cuca_b200.kernels import ops
    k, n = 2056, 8200
    w = _normal(n, k, F32, 2) / math.sqrt(k)
    w[5] = 0
    w[7, 100] = math.inf
    q, held = ops.mx4_quantise(w), mx.held(w)
    fine = [i for i in range(n) if i != 7]
    for gap, shift in ((0, 0), (8, 0), (3, 1)):
        memory = torch.zeros(m * (k + gap) + shift, dtype=BF16, device="cuda")
        x = memory[shift:].view(m, k + gap)[:, :k]
        x.copy_(_normal(m, k, BF16, m))
        for out_dtype, bias_dtype in ((BF16, BF16), (F32, F32), (F32, BF16)):
            bias = _normal(1, n, bias_dtype, 3)[0].contiguous()
            wide = torch.full((m, n + 9), 7.0, dtype=out_dtype, device="cuda")
            ops.gemm_mx4(x, q, wide[:, 3:3 + n], bias=bias)
            assert (wide[:, :3] == 7).all() and (wide[:, 3 + n:] == 7).all() and wide[:, 10].isnan().all()
            _within(wide[:, 3:3 + n][:, fine], *mx.product(x.double(), held[fine], "store", out_dtype, 2.5 * k / 16 + 24, bias[fine]))
        gated = torch.empty(m, n // 2, dtype=BF16, device="cuda")
        ops.gemm_mx4(x, q, gated, ops.EPI_SWIGLU)
        assert gated[:, 7].isnan().all()
        pair = [i for i in range(n // 2) if i != 7]
        both = held[pair + [n // 2 + i for i in pair]]
        _within(gated[:, pair], *mx.product(x.double(), both, "swiglu", BF16, 2.5 * k / 16 + 24))
    stream = _normal(m, n, F32, 4)
    out = stream.clone()
    ops.gemm_mx4(x, q, out, ops.EPI_RESIDUAL, bias)
    _within(out[:, fine], *mx.product(x.double(), held[fine], "store", F32, 2.5 * k / 16 + 24, bias[fine], stream[:, fine]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.gemm_mx4(x, q, out)
        ops.gemm_mx4(x, q, gated, ops.EPI_SWIGLU)
    for seed in (8, 9):
        x.copy_(_normal(m, k, BF16, seed))
        x[0, 40] = math.nan
        x[0, 70] *= 2.0 ** 90  # what these digits leave is multiplied too
        x[-1, 1000] = 0.5 if m == 1 else math.inf
        graph.replay()
        torch.cuda.synchronize()
        assert out[0].isnan().all() and (m == 1 or not out[-1].isfinite().any())
        if m > 2:
            _within(out[1:-1][:, fine], *mx.product(x[1:-1].double(), held[fine], "store", F32, 2.5 * k / 16 + 24))


@pytest.mark.parametrize("m", [1, 7, 16, 20])
def test_few_rows_of_the_largest_numbers(m):
    """The type's largest and lowest values come through weights of one: no part of them is past the range."""
    k, n = 96, 180_000
    x = _normal(m, k, BF16, m)
    x[0, 3], x[0, 40], x[-1, 70] = torch.finfo(BF16).max, torch.finfo(BF16).min, 1.75 * 2.0 ** 127
    w = torch.zeros(n, k, device="cuda")
    w[torch.arange(n), torch.arange(n) % k] = 1
    out, xv, wv = _multiply("bf16", x, w)
    assert torch.equal(out.double(), xv @ wv.T)


@pytest.mark.parametrize("out_dtype", [BF16, F32])
@pytest.mark.parametrize("kind,m,n", [("bf16", 97, 40), ("bf16", 10, 131_072), ("f32", 50, 24), ("codes", 30, 24)])
def test_gated_unit_over_the_whole_range(kind, m, n, out_dtype):
    """silu(g) u for g from -120 to 120. 32-bit results are good to 2^-20 of themselves, but for the exponential's own last place where that lies
    under 2^-126; bfloat16 ones to |g| 2^-23 more, and a sigmoid under 2^-126 may be taken as zero."""
    if kind == "f32" and out_dtype == BF16:
        pytest.skip("32-bit rows have 32-bit results")
    k = 64
    x = torch.zeros(m, k, device="cuda")
    x[:, 0] = torch.linspace(-120, 120, m, device="cuda") if kind != "codes" else torch.tensor([-96.0, -64, -3, 0.5, 48, 96], device="cuda").repeat(5)
    x[:, 32] = 1
    w = torch.zeros(2 * n, k, device="cuda")
    w[:n, 0] = 1
    w[n:, 32] = torch.tensor([1.0, 2.0 ** 20, -1.5, 2.0 ** 60], device="cuda").repeat(n // 4)
    out, xv, wv = _multiply(kind, x if kind == "f32" else x.to(BF16), w, "swiglu", out_dtype)
    g, u = (xv @ wv.T).chunk(2, 1)
    want = g * torch.sigmoid(g) * u
    if out_dtype == BF16:
        bound = want.abs() * (2.0 ** -8 + 2.0 ** -20 + g.abs() * 2.0 ** -23) + (g * u).abs() * 2.0 ** -126 + 2.0 ** -134
    else:
        bound = want.abs() * (2.0 ** -24 + 2.0 ** -20) + (g * u).abs() * 2.0 ** -148 + 2.0 ** -150
    _within(out, want, bound)
