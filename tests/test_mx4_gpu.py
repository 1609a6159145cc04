"""Rows in microscaled 4-bit floating point: quantising, reading back, and products with them, each against its formula in 64 bits
(`mx4_util`)."""
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


def _rows(rows, cols, dtype, seed, spread=0.7):
    g = torch.Generator(device="cuda").manual_seed(seed)
    channel = torch.exp(spread * torch.randn(cols, generator=g, device="cuda"))
    return (torch.randn(rows, cols, generator=g, device="cuda") * channel).to(dtype)


def _strided(x, gap, shift):
    """The same rows with `gap` values between them, `shift` values into their memory."""
    rows, cols = x.shape
    memory = torch.full((rows * (cols + gap) + shift,), 7.0, dtype=x.dtype, device=x.device)
    out = memory[shift:].view(rows, cols + gap)[:, :cols]
    out.copy_(x)
    return out


# ------------------------------------------------------------------ quantising and reading back
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,cols,gap,shift", [
    (1, 1, 0, 0), (1, 31, 0, 0), (3, 32, 0, 0), (5, 33, 0, 1), (129, 128, 0, 0), (128, 256, 8, 0), (300, 70, 2, 8), (17, 1000, 0, 0),
    (260, 4096, 0, 0), (7, 14336, 16, 0), (2, 5001, 3, 5), (1000, 130, 0, 0)])
def test_codes_and_values(dtype, rows, cols, gap, shift):
    from cuca_b200.kernels import ops
    x = _strided(_rows(rows, cols, dtype, rows + cols), gap, shift)
    q = ops.mx4_quantise(x)
    code, byte = mx.unpack(q)
    want, want_byte = mx.quantise(x)
    assert torch.equal(byte, want_byte)
    assert torch.equal(torch.where(code == 8, 0, code), want)  # (a negative value that becomes zero keeps its sign)
    for out_dtype in (BF16, F32):
        out = _strided(torch.zeros(rows, cols, dtype=out_dtype, device="cuda"), gap, shift)
        ops.mx4_values(q, out)
        assert torch.equal(out.double(), mx.values(want, want_byte, cols))


def test_borders_and_extremes():
    from cuca_b200.kernels import ops
    x = torch.zeros(16, 64, device="cuda")
    ties = torch.tensor([4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.96875, 0.2490234375, 0.25390625, 4.96875, 5.03125],
                        device="cuda")
    x[0, :15], x[0, 32:47] = ties, -ties
    x[1, 3], x[2, 5] = 2.0 ** -126, 2.0 ** -149  # the smallest normal number, the smallest of all
    x[3, :] = torch.finfo(F32).max
    x[4, 7], x[4, 40] = math.inf, 1.0
    x[5, 31], x[5, 32] = math.nan, 3.0
    x[6, 0], x[6, 33] = -math.inf, -1.0
    x[7, 0] = -0.0
    x[8, :32] = torch.linspace(-2.0 ** -125, 2.0 ** -125, 32)
    x[9, :32] = torch.linspace(-2.0 ** -127, 2.0 ** -127, 32)
    x[10, 0], x[10, 1] = 3.0e38, 1.0e-30
    for dtype in (F32, BF16):
        y = x.to(dtype)
        y[3] = torch.finfo(dtype).max
        q = ops.mx4_quantise(y)
        code, byte = mx.unpack(q)
        want, want_byte = mx.quantise(y)
        assert torch.equal(byte, want_byte) and torch.equal(torch.where(code == 8, 0, code), want)
        out = torch.empty_like(y)
        ops.mx4_values(q, out)
        assert torch.equal(torch.nan_to_num(out.double(), nan=-1e300), torch.nan_to_num(mx.values(want, want_byte, 64), nan=-1e300))
        assert out[4, :32].isnan().all() and out[4, 40] == 1 and out[5, :32].isnan().all() and out[5, 32] == 3


def test_given_memory_is_used_and_rows_beyond_are_left():
    from cuca_b200.kernels import ops
    x = _rows(100, 200, BF16, 1)
    q = ops.Mx4Matrix.empty(100, 200, "cuda")
    q.codes.fill_(255)
    q.scales.fill_(77)
    assert ops.mx4_quantise(x, q) is q
    other = ops.mx4_quantise(x)
    assert torch.equal(q.codes, other.codes)
    s = q.scales.permute(0, 3, 2, 1, 4).reshape(128, -1)
    assert (s[100:] == 77).all()


def test_no_rows():
    from cuca_b200.kernels import ops
    q = ops.mx4_quantise(torch.empty(0, 64, device="cuda"))
    ops.mx4_values(q, torch.empty(0, 64, device="cuda"))
    w = ops.mx4_quantise(_rows(8, 64, F32, 1))
    ops.gemm_mx4(torch.empty(0, 64, dtype=BF16, device="cuda"), w, torch.empty(0, 8, dtype=BF16, device="cuda"))
    ops.gemm_mx4(q, w, torch.empty(0, 8, dtype=BF16, device="cuda"))
    ops.gemm_mx4(_rows(3, 64, BF16, 1), q, torch.empty(3, 0, dtype=BF16, device="cuda"))


# ------------------------------------------------------------------ products
KINDS = ["bf16", "f32", "codes"]


def _operands(kind, m, k, n, seed, x=None, w=None):
    """(rows as they go into a call, their values in 64 bits, weight, its values)."""
    from cuca_b200.kernels import ops
    x = _rows(m, k, F32 if kind == "f32" else BF16, seed) if x is None else x
    w = _rows(n, k, F32, seed + 1, 0.0) / math.sqrt(k) if w is None else w
    q = ops.mx4_quantise(w)
    if kind == "codes":
        return ops.mx4_quantise(x), mx.held(x), q, mx.held(w)
    return x, x.double(), q, mx.held(w)


def _additions(k):
    """Additions in a row of one output: the matrix instructions of 16 products and more, then shares and digits."""
    return k / 16 + 24


def _product(kind, x, w, epilogue, out_dtype, bias=None, stream=None):
    """(result, bound): rows that are not in 4 bits may go as digits."""
    return mx.product(x, w, epilogue, out_dtype, _additions(x.shape[1]), bias, stream, digits=kind != "codes")


def _check(out, want, bound):
    off = (out.double() - want).abs()
    worst = (off / bound).max().item()
    assert torch.isfinite(out).all() and worst <= 1, f"{worst} of the bound, off by {off.max().item()}"


SIZES = [(1, 1, 1), (1, 32, 1), (1, 128, 130), (2, 100, 64), (3, 33, 129), (5, 1010, 2050), (8, 4096, 512), (9, 256, 96), (16, 640, 200),
         (17, 512, 384), (33, 1024, 136), (64, 2048, 256), (65, 96, 77), (100, 4000, 300), (128, 512, 128), (129, 520, 257), (200, 1280, 640),
         (256, 384, 512), (257, 130, 100), (400, 2048, 1024), (1025, 320, 264)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,k,n", SIZES)
def test_products(kind, m, k, n):
    from cuca_b200.kernels import ops
    a, x, q, w = _operands(kind, m, k, n, m + k + n)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    for out_dtype in ((F32,) if kind == "f32" else (BF16, F32)):
        out = torch.full((m, n), 7.0, dtype=out_dtype, device="cuda")
        ops.gemm_mx4(a, q, out, err=err)
        _check(out, *_product(kind, x, w, "store", out_dtype))
    bias = _rows(1, n, F32 if (kind == "f32") == (n % 2 == 0) else BF16, 5)[0].contiguous()
    out = torch.full((m, n), 7.0, dtype=F32 if kind == "f32" else BF16, device="cuda")
    ops.gemm_mx4(a, q, out, bias=bias, err=err)
    _check(out, *_product(kind, x, w, "store", out.dtype, bias=bias))
    stream = _rows(m, n, F32, 6)
    out = stream.clone()
    ops.gemm_mx4(a, q, out, ops.EPI_RESIDUAL, bias, err)
    want, bound = _product(kind, x, w, "store", F32, bias=bias, stream=stream)
    _check(out, want, bound)
    assert err.item() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,k,n", [(1, 64, 1), (1, 4096, 256), (3, 100, 70), (8, 512, 192), (15, 257, 65), (16, 1024, 128), (40, 384, 100),
                                   (64, 512, 320), (130, 640, 129), (300, 512, 256), (600, 130, 200)])
def test_gated_unit(kind, m, k, n):
    from cuca_b200.kernels import ops
    a, x, q, w = _operands(kind, m, k, 2 * n, m + k + n)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full((m, n), 7.0, dtype=F32 if kind == "f32" else BF16, device="cuda")
    ops.gemm_mx4(a, q, out, ops.EPI_SWIGLU, err=err)
    _check(out, *_product(kind, x, w, "swiglu", out.dtype))
    assert err.item() == 0


@pytest.mark.parametrize("kind", ["bf16", "codes"])
@pytest.mark.parametrize("m,k,n", [(4, 300, 100), (40, 300, 192), (300, 700, 130)])
def test_gated_unit_in_32_bits(kind, m, k, n):
    from cuca_b200.kernels import ops
    a, x, q, w = _operands(kind, m, k, 2 * n, m)
    out = torch.full((m, n), 7.0, device="cuda")
    ops.gemm_mx4(a, q, out, ops.EPI_SWIGLU)
    _check(out, *_product(kind, x, w, "swiglu", F32))


@pytest.mark.parametrize("kind", KINDS)
def test_one_shape_with_every_epilogue_in_turn(kind):
    """What a call needs of memory depends on its epilogue too: the same rows and sizes, one after the other, from a fresh memory of it."""
    from cuca_b200.kernels import ops
    m, k, n = 20, 128, 64
    a, x, q, w = _operands(kind, m, k, n, 1)
    for order in ((ops.EPI_STORE, ops.EPI_SWIGLU, ops.EPI_RESIDUAL), (ops.EPI_SWIGLU, ops.EPI_STORE)):
        ops._mx4_scratch.clear()
        for epilogue in order:
            gated = epilogue == ops.EPI_SWIGLU
            out = torch.zeros(m, n // 2 if gated else n, device="cuda")
            ops.gemm_mx4(a, q, out, epilogue)
            _check(out, *_product(kind, x, w, "swiglu" if gated else "store", F32))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [2, 40, 300])
def test_strides(kind, m):
    """Rows with gaps, off 16 bytes, results into columns of a wider matrix whose rest stays."""
    from cuca_b200.kernels import ops
    k, n = 328, 200
    a, x, q, w = _operands(kind, m, k, n, m)
    for gap, shift in ((8, 0), (3, 0), (0, 1), (5, 3)):
        if kind != "codes":
            a = _strided(a, gap, shift)
        wide = torch.full((m, n + gap + 9), 7.0, device="cuda")
        out = wide[:, 3 + shift:3 + shift + n]
        ops.gemm_mx4(a, q, out)
        _check(out, *_product(kind, x, w, "store", F32))
        assert (wide[:, :3 + shift] == 7).all() and (wide[:, 3 + shift + n:] == 7).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [3, 50, 300])
def test_powers_far_apart(kind, m):
    """Blocks of weights and rows from 2^-60 to 2^60: what is large does not take the bits of what is small."""
    k, n = 256, 140
    g = torch.Generator(device="cuda").manual_seed(m)
    scale = lambda r: torch.exp2(torch.randint(-60, 61, (r, k // 32), generator=g, device="cuda").float()).repeat_interleave(32, 1)  # noqa: E731
    x = (_rows(m, k, F32, 1, 0.0) * scale(m)).to(F32 if kind == "f32" else BF16)
    w = _rows(n, k, F32, 2, 0.0) * scale(n)
    a, x, q, w = _operands(kind, m, k, n, 1, x, w)
    from cuca_b200.kernels import ops
    out = torch.empty(m, n, device="cuda")
    ops.gemm_mx4(a, q, out)
    _check(out, *_product(kind, x, w, "store", F32))


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_a_large_value_of_no_weight_beside_small_ones(kind):
    """Few rows go as eight digits: a value of 2^30 that meets weights of zero leaves the others digits of their own. It has eight
    significant bits, which three digits hold, four where a digit carries; four are left, and after a digit at most an eighth is."""
    from cuca_b200.kernels import ops
    m, k, n = 4, 256, 64
    x, w = _rows(m, k, BF16, 1, 0.0).float(), _rows(n, k, F32, 2, 0.0)
    x[:, ::32] = (x[:, ::32] * 2.0 ** 30).to(BF16).float()
    w[:, ::32] = 0
    a, xv, q, wv = _operands(kind, m, k, n, 1, x.to(F32 if kind == "f32" else BF16), w)
    out = torch.empty(m, n, device="cuda")
    ops.gemm_mx4(a, q, out)
    rest = xv.clone()
    rest[:, ::32] = 0
    most = rest.view(m, -1, 32).abs().amax(-1, keepdim=True).expand(-1, -1, 32).flatten(1)
    bound = 2.0 ** -11 * (most @ wv.abs().T) + mx.chain_bound(rest, wv, 2.5 * _additions(k))
    _check(out, xv @ wv.T, bound)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [3, 50, 300])
def test_weights_of_no_size_and_not_finite(kind, m):
    """A weight row of zeros gives zeros, one with an infinity NaN, and neither touches the rows beside it; so with rows."""
    from cuca_b200.kernels import ops
    k, n = 192, 150
    x = _rows(m, k, F32 if kind == "f32" else BF16, 1)
    w = _rows(n, k, F32, 2, 0.0)
    w[5] = 0
    w[7, 100] = math.inf
    w[140, 3] = math.nan
    x[1, 64] = math.nan
    x[2] = 0
    a, xv, q, wv = _operands(kind, m, k, n, 1, x, w)
    out = torch.empty(m, n, device="cuda")
    ops.gemm_mx4(a, q, out)
    bad = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    bad[1], bad[:, 7], bad[:, 140] = True, True, True
    assert torch.equal(out.isnan(), bad)
    good_n = [i for i in range(n) if i not in (7, 140)]
    good_m = [i for i in range(m) if i != 1]
    want, bound = _product(kind, xv[good_m], wv[good_n], "store", F32)
    _check(out[good_m][:, good_n], want, bound)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,k,n", [(1, 4096, 512), (8, 2048, 300), (64, 4096, 256), (300, 1024, 512)])
def test_equal_bits_in_every_run_and_on_another_stream(kind, m, k, n):
    from cuca_b200.kernels import ops
    a, _, q, _ = _operands(kind, m, k, n, 3)
    outs = [torch.empty(m, n, device="cuda") for _ in range(4)]
    for o in outs[:3]:
        ops.gemm_mx4(a, q, o)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.gemm_mx4(a, q, outs[3])
    side.synchronize()
    assert all(torch.equal(outs[0], o) for o in outs[1:])


@pytest.mark.parametrize("m", [1, 7, 70, 300])
def test_a_chain_in_a_graph(m):
    """Quantise a weight and rows, multiply, unit, quantise, multiply into the stream: one graph, replayed on other inputs, each
    launch reading what the one just before it wrote."""
    from cuca_b200.kernels import ops
    e, f = 160, 224
    w1, w2 = _rows(2 * f, e, F32, 1, 0.0) / math.sqrt(e), _rows(e, f, F32, 2, 0.0) / math.sqrt(f)
    x, stream = _rows(m, e, BF16, 3), _rows(m, e, F32, 4)
    q1, q2 = ops.Mx4Matrix.empty(2 * f, e, "cuda"), ops.Mx4Matrix.empty(e, f, "cuda")

    def chain():
        ops.mx4_quantise(w1, q1)
        ops.mx4_quantise(w2, q2)
        act = torch.empty(m, f, dtype=BF16, device="cuda")
        ops.gemm_mx4(ops.mx4_quantise(x), q1, act, ops.EPI_SWIGLU)
        ops.gemm_mx4(ops.mx4_quantise(act), q2, stream, ops.EPI_RESIDUAL)
        wide = torch.empty(m, f, dtype=BF16, device="cuda")
        ops.gemm_mx4(x, q1, wide, ops.EPI_SWIGLU)
        ops.gemm_mx4(wide, q2, stream, ops.EPI_RESIDUAL)
        return act, wide

    kept = stream.clone()
    chain()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        act, wide = chain()
    for seed in (10, 11):
        x.copy_(_rows(m, e, BF16, seed))
        w1.copy_(_rows(2 * f, e, F32, seed + 5, 0.0) / math.sqrt(e))
        stream.copy_(kept)
        graph.replay()
        torch.cuda.synchronize()
        v1, v2 = mx.held(w1), mx.held(w2)
        _check(act, *_product("codes", mx.held(x), v1, "swiglu", BF16))
        _check(wide, *_product("bf16", x.double(), v1, "swiglu", BF16))
        y1, b1 = _product("codes", mx.held(act), v2, "store", F32, stream=kept)
        y2, b2 = _product("bf16", wide.double(), v2, "store", F32, stream=y1)
        _check(stream, y2, b1 + b2)


@pytest.mark.parametrize("m", [2, 20, 90])
def test_two_graphs_at_once(m):
    """Two captured graphs replayed on two streams at once keep what they make for themselves apart."""
    from cuca_b200.kernels import ops
    k, n = 2048, 512
    cases, graphs = [_operands("bf16", m, k, n, s) for s in (1, 2)], []
    outs = [torch.zeros(m, n, device="cuda") for _ in cases]
    for (a, _, q, _), out in zip(cases, outs):
        ops.gemm_mx4(a, q, out)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(20):
                ops.gemm_mx4(a, q, out)
        graphs.append(g)
        out.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for (_, x, _, w), out in zip(cases, outs):
        _check(out, *_product("bf16", x, w, "store", F32))


@pytest.mark.parametrize("sign", [False, True])
def test_long_sums_in_32_bits(sign):
    """Of 17,000 values 32-bit sums run over 8,192 at most: 512 contractions in a row cut off at most 2^-23 of the sum each, in the mean
    a quarter of that over a sum that grows from nothing."""
    from cuca_b200.kernels import ops
    m, k, n = 300, 17_000, 19_200
    x, w = _rows(m, k, BF16, 1, 0.0), _rows(n, k, BF16, 2, 0.0)
    if sign:
        x, w = x.abs(), w.abs()
    q = ops.mx4_quantise(w)
    bias, stream = _rows(1, n, F32, 3)[0].contiguous(), _rows(m, n, F32, 4)
    out = stream.clone()
    ops.gemm_mx4(x, q, out, ops.EPI_RESIDUAL, bias)
    some = torch.arange(0, n, 257, device="cuda")
    want = x.double() @ mx.held(w[some]).T + bias[some].double() + stream[:, some].double()
    assert (out[:, some].double() - want).norm() < 512 * 2.0 ** -25 * want.norm()


@pytest.mark.parametrize("epilogue", [0, 1])
def test_parts_of_a_long_sum_beside_a_large_stream(epilogue):
    """Of 17,000 values three parts are added to the bias and the stream, each with one rounding, at most 2^-24 of what has been added;
    a bias is added to the first part with one more."""
    from cuca_b200.kernels import ops
    m, k, n = 300, 17_000, 19_200
    x, w = _rows(m, k, BF16, 1, 0.0) / 4096, _rows(n, k, BF16, 2, 0.0)
    q = ops.mx4_quantise(w)
    bias, out = _rows(1, n, F32, 3)[0].contiguous(), _rows(m, n, F32, 4)
    some = torch.arange(0, n, 257, device="cuda")
    rows, held = x.double(), mx.held(w[some])
    want = rows @ held.T + bias[some].double() + epilogue * out[:, some].double()
    most = rows.abs() @ held.abs().T + bias[some].double().abs() + epilogue * out[:, some].double().abs()
    bound = 4 * 2.0 ** -24 * most + mx.chain_bound(rows, held, 512)
    ops.gemm_mx4(x, q, out, epilogue, bias)
    assert ((out[:, some].double() - want).abs() <= bound).all()


def test_codes_past_2_to_the_31_bytes():
    """A weight and rows whose codes reach past 2^31 bytes: their ends are where they should be."""
    from cuca_b200.kernels import ops
    n, k = 140_001, 32_768
    w = _rows(2048, k, BF16, 1, 0.0)
    big = torch.empty(n, k, dtype=BF16, device="cuda")
    for at in range(0, n, 2048):
        big[at:at + 2048] = w[:min(2048, n - at)]
    big[-3:] = _rows(3, k, BF16, 2, 0.0)
    q = ops.mx4_quantise(big)
    assert q.codes.numel() > 2 ** 31
    tail = mx.held(big[-200:])
    back = torch.empty(n, k, dtype=BF16, device="cuda")
    ops.mx4_values(q, back)
    assert torch.equal(back[-200:].double(), tail)
    del back
    for m in (2, 33):
        x = _rows(m, k, BF16, 3, 0.0)
        out = torch.empty(m, n, dtype=BF16, device="cuda")
        ops.gemm_mx4(x, q, out)
        _check(out[:, -200:], *_product("bf16", x.double(), tail, "store", BF16))
    few = ops.mx4_quantise(big[:70].contiguous())
    out = torch.empty(n, 70, dtype=BF16, device="cuda")
    ops.gemm_mx4(q, few, out)
    _check(out[-200:], *_product("codes", tail, mx.held(big[:70]), "store", BF16))


# ------------------------------------------------------------------ refusals
def test_refusals():
    from cuca_b200.kernels import library, ops
    x, w = _rows(4, 64, BF16, 1), ops.mx4_quantise(_rows(10, 64, F32, 2))
    out = torch.empty(4, 10, dtype=BF16, device="cuda")
    refuse = lambda *a, **k: pytest.raises(library.KernelError, ops.gemm_mx4, *a, **k)  # noqa: E731
    refuse(_rows(4, 65, BF16, 1), w, out)
    refuse(x, w, out[:, :9])
    refuse(x, w, out[:3])
    refuse(x.t().contiguous().t(), w, out)
    refuse(x.half(), w, out)
    refuse(x, w, out.half())
    refuse(x.float(), w, out)
    refuse(x, w, out, ops.EPI_RESIDUAL)
    refuse(x, w, torch.empty(4, 5, dtype=BF16, device="cuda"), ops.EPI_SWIGLU, torch.zeros(5, dtype=BF16, device="cuda"))
    refuse(x, w, out, bias=torch.zeros(10, dtype=torch.half, device="cuda"))
    refuse(x, w, out, bias=torch.zeros(10, device="cuda").cpu())
    refuse(x, w, out, bias=torch.zeros(9, dtype=BF16, device="cuda"))
    refuse(x, w, out, 7)
    refuse(x, w, out, err=torch.zeros(1, device="cuda"))
    refuse(x, w, out, err=torch.zeros(1, dtype=torch.int32))
    off = ops.Mx4Matrix(10, 64, torch.zeros(10 * 64 + 8, dtype=torch.uint8, device="cuda")[8:].view(10, 64), w.scales)
    refuse(x, off, out)  # codes off 16 bytes
    refuse(ops.mx4_quantise(x), off, out)
    refuse(x.cpu(), w, out)
    refuse(x, ops.mx4_quantise(_rows(9, 64, F32, 2)), torch.empty(4, 4, dtype=BF16, device="cuda"), ops.EPI_SWIGLU)
    refuse(x, w, torch.empty(1, 10, dtype=BF16, device="cuda").expand(4, 10))
    for bad in (x.half(), x[0], torch.empty(3, 0, device="cuda"), x.cpu()):
        pytest.raises(library.KernelError, ops.mx4_quantise, bad)
    pytest.raises(library.KernelError, ops.mx4_quantise, x, ops.Mx4Matrix.empty(4, 96, "cuda"))
    pytest.raises(library.KernelError, ops.mx4_values, w, torch.empty(10, 63, device="cuda"))
    pytest.raises(library.KernelError, ops.mx4_values, w, torch.empty(10, 64, dtype=torch.half, device="cuda"))
    torch.cuda.synchronize()
