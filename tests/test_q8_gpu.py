"""The cache in 8 bits: quantising rows as they are written, reading them back, and the attention over them, each alone against
its formulas in 64 bits (`q8_util`)."""
import math

import pytest
import torch

from q8_util import TINY, Case, Step, quantise

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def lib():
    from cuca_b200.kernels import library
    return library.load()


def _tables(positions, rot, dev):
    freq = 10000.0 ** (-torch.arange(0, rot, 2, device=dev, dtype=torch.float64) / rot)
    a = torch.arange(positions, device=dev, dtype=torch.float64)[:, None] * freq
    return a.cos().float(), a.sin().float()


def _rotated(x, cos, sin, positions, rot, adjacent):
    """Heads [rows, heads, dim] rotated in 64 bits."""
    x = x.double().clone()
    if rot == 0:
        return x
    c, s = cos[positions.long()].double()[:, None], sin[positions.long()].double()[:, None]
    a, b = (x[..., 0:rot:2].clone(), x[..., 1:rot:2].clone()) if adjacent else (x[..., :rot // 2].clone(), x[..., rot // 2:rot].clone())
    ra, rb = a * c - b * s, a * s + b * c
    if adjacent:
        x[..., 0:rot:2], x[..., 1:rot:2] = ra, rb
    else:
        x[..., :rot // 2], x[..., rot // 2:rot] = ra, rb
    return x


def _write(c, qkv, q_out, cos, sin, rot, adjacent=False):
    from cuca_b200.kernels import ops
    ops.rope_store_q8(qkv, q_out, c.step.positions, c.step.seq_of_row, c.tables, cos, sin, rot, c.pages(), c.heads, c.kv, c.dim,
                      c.err, adjacent=adjacent)


def _read(c, dtype, positions=None, seqs=None):
    from cuca_b200.kernels import ops
    positions = c.step.positions if positions is None else positions
    seqs = c.step.seq_of_row if seqs is None else seqs
    k = torch.full((positions.shape[0], c.kv, c.dim), 7.0, dtype=dtype, device=c.device)
    v = torch.full_like(k, 7.0)
    ops.read_q8(c.pages(), positions, seqs, c.tables, k, v, c.err)
    return k, v


# ------------------------------------------------------------------ writing and reading back
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,dim,rot,adjacent,page", [
    (32, 8, 128, 128, False, 16), (8, 8, 64, 64, False, 8), (4, 2, 16, 16, False, 16), (3, 1, 80, 80, False, 24),
    (6, 2, 96, 96, True, 32), (4, 1, 256, 256, False, 64), (5, 5, 48, 32, False, 7), (4, 2, 64, 32, True, 16),
    (2, 2, 112, 0, False, 16), (4, 4, 32, 2, False, 1)])
def test_rows_are_rotated_quantised_and_read_back(dtype, heads, kv, dim, rot, adjacent, page):
    c = Case(heads, kv, dim, page, [1, 7, 40, 1], [0, 13, 5, 90], dtype, seed=dim + rot, fill=False, padding=2)
    rows = c.step.n_rows
    wide = torch.randn(rows, (heads + 2 * kv) * dim + 8, device=c.device, generator=c.g).to(dtype)
    qkv = wide[:, :(heads + 2 * kv) * dim]
    before = qkv.clone()
    cos, sin = _tables(100, rot, c.device) if rot else (None, None)
    q_out = torch.full((rows, heads * dim), 3.0, dtype=dtype, device=c.device)
    _write(c, qkv, q_out, cos, sin, rot, adjacent)
    assert int(c.err) == 0 and torch.equal(qkv, before)
    live = c.step.seq_of_row >= 0
    x = before.view(rows, heads + 2 * kv, dim) if not before.stride(0) != before.shape[1] else before.reshape(rows, heads + 2 * kv, dim)
    turned = _rotated(x[:, :heads + kv], cos, sin, c.step.positions, rot, adjacent)
    q = q_out.view(rows, heads, dim).double()
    size = x[:, :heads].double().abs().amax(-1, keepdim=True) * 1.5
    near = (2.0 ** -8 * turned[:, :heads].abs() if dtype == torch.bfloat16 else 0) + 2.0 ** -22 * size
    assert ((q - turned[:, :heads]).abs() <= near)[live].all()
    assert (q[~live] == 3.0).all()  # rows of no request are left alone
    for got, want in zip(_read(c, torch.float32), (turned[:, heads:], x[:, heads + kv:].double())):
        a = want.abs().amax(-1, keepdim=True)
        # half a 127th of the row's largest, and the 32-bit roundings of rotation, quotients and product
        assert ((got.double() - want).abs() <= a / 254 * (1 + 1e-4) + 2.0 ** -20 * a)[live].all()
        assert (got[~live] == 0).all()
        steps = got.double() / (a / 127)
        assert ((steps - torch.round(steps)).abs() < 1e-3)[live].all()
        assert (got.abs().amax(-1, keepdim=True).double() - a).abs().le(2.0 ** -20 * a)[live].all()  # the largest is kept
    # in place
    _write(c, qkv, qkv[:, :heads * dim], cos, sin, rot, adjacent)
    assert torch.equal(qkv[live][:, :heads * dim], q_out[live]) and torch.equal(qkv[:, heads * dim:], before[:, heads * dim:])


def test_codes_of_the_vectorised_and_the_plain_form_are_the_same():
    """Rows off their alignment take the plain form: same codes, same scales, same queries."""
    c = Case(4, 2, 64, 16, [33, 1], [0, 20], torch.bfloat16, seed=3, fill=False)
    cos, sin = _tables(64, 64, c.device)
    flat = torch.randn(34 * 512 + 8, device=c.device, generator=c.g).to(torch.bfloat16)
    qkv = flat[:34 * 512].view(34, 512)
    off = torch.empty(34 * 514 + 8, dtype=torch.bfloat16, device=c.device)[1:34 * 514 + 1].view(34, 514)[:, :512]
    off.copy_(qkv)
    results = []
    for x in (qkv, off):
        c.k.zero_(), c.v.zero_(), c.k_scale.zero_(), c.v_scale.zero_()
        q = torch.empty(34, 256, dtype=torch.bfloat16, device=c.device)
        _write(c, x, q, cos, sin, 64)
        results.append([t.clone() for t in (q, c.k, c.v, c.k_scale, c.v_scale)])
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("slices,dim,rot,rows", [(1, 128, 128, 3), (5, 64, 64, 40), (16, 80, 80, 1), (3, 96, 32, 9), (2, 32, 0, 7)])
def test_k_slices_are_added_before_they_are_rotated_and_quantised(slices, dim, rot, rows, with_bias):
    """The same codes, bit for bit, as from the 32-bit rows that the slices, added in order, make; the same queries, rounded."""
    from cuca_b200.kernels import ops
    heads, kv = 4, 2
    c = Case(heads, kv, dim, 16, [rows], [5], torch.bfloat16, seed=slices, fill=False, padding=1)
    n, width = rows + 1, (heads + 2 * kv) * dim
    data = torch.randn(slices, n + 3, width, device=c.device, generator=c.g)[:, :n]
    bias = torch.randn(width, device=c.device, generator=c.g).to(torch.bfloat16) if with_bias else None
    total = torch.zeros(n, width, device=c.device)
    for s in range(slices):
        total = total + data[s]
    if with_bias:
        total = total + bias.float()
    cos, sin = _tables(64, rot, c.device) if rot else (None, None)
    results = []
    for source, dtype in ((ops.PartialSums(data, slices), torch.bfloat16), (total, torch.float32)):
        c.k.zero_(), c.v.zero_(), c.k_scale.zero_(), c.v_scale.zero_()
        q = torch.zeros(n, heads * dim, dtype=dtype, device=c.device)
        ops.rope_store_q8(source, q, c.step.positions, c.step.seq_of_row, c.tables, cos, sin, rot, c.pages(), heads, kv, dim, c.err,
                          bias=bias if dtype == torch.bfloat16 else None)
        results.append([t.clone() for t in (q.to(torch.bfloat16), c.k, c.v, c.k_scale, c.v_scale)])
    assert all(torch.equal(a, b) for a, b in zip(*results)) and int(c.err) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_of_zeros_of_tiny_values_and_rows_that_are_not_finite(dtype):
    c = Case(2, 1, 32, 16, [8], [3], dtype, seed=9, fill=False)
    qkv = torch.randn(8, 4 * 32, device=c.device, generator=c.g).to(dtype)
    k, v = qkv[:, 64:96], qkv[:, 96:]
    k[0] = 0
    v[1] = 0
    k[2] = TINY / 4
    k[3] = 1e30
    v[4, 5] = math.inf
    v[5, 31] = -math.inf
    k[6, 0] = math.nan
    v[7] = 1e-20
    _write(c, qkv, torch.empty(8, 64, dtype=dtype, device=c.device), None, None, 0)
    gk, gv = _read(c, torch.float32)
    assert (gk[0] == 0).all() and (gv[1] == 0).all() and (gk[2] == 0).all()
    for got, want in ((gk[3], k[3]), (gv[7], v[7])):
        assert ((got.double() - want.double().view(1, -1)).abs() <= want.double().abs().max() / 254 * (1 + 1e-4)).all()
    assert gv[4].isnan().all() and gv[5].isnan().all() and gk[6].isnan().all()
    assert gk[4].isfinite().all() and gv[6].isfinite().all()


@pytest.mark.parametrize("what", [0.0, TINY / 4, math.inf, -math.inf, math.nan])
def test_a_row_that_keeps_nothing_has_codes_of_zero(what):
    c = Case(2, 1, 32, 16, [8], [0], torch.float32, seed=2, fill=False)
    qkv = torch.randn(8, 4 * 32, device=c.device, generator=c.g)
    qkv[:, 64:] *= 0 if abs(what) < 1 else 1
    qkv[:, 64::7] = what
    c.k.fill_(5), c.v.fill_(5)
    _write(c, qkv, torch.empty(8, 64, device=c.device), None, None, 0)
    page = c.tables[c.slots[0], 0].long()
    assert (c.k[page, :, :8] == 0).all() and (c.v[page, :, :8] == 0).all() and (c.k[page, :, 8:] == 5).all()
    scales = torch.cat([c.k_scale[page, :, :8], c.v_scale[page, :, :8]])
    assert (scales == 0).all() if abs(what) < 1 else scales.isnan().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kv,dim,page,totals", [(8, 128, 16, [300, 1, 77]), (1, 16, 8, [9]), (3, 80, 24, [50, 49]), (2, 256, 1, [5])])
def test_reading_back_is_exact(dtype, kv, dim, page, totals):
    from cuca_b200.kernels import ops
    c = Case(kv, kv, dim, page, [1] * len(totals), [t - 1 for t in totals], dtype, seed=dim)
    positions = torch.cat([torch.randperm(t, device=c.device, generator=c.g) for t in totals] + [torch.zeros(2, device=c.device)]).int()
    seqs = torch.tensor([s for s, t in zip(c.slots, totals) for _ in range(t)] + [-1, -1], dtype=torch.int32, device=c.device)
    k, v = _read(c, dtype, positions, seqs)
    at, page_of = positions.long() % page, c.tables[seqs.long().clamp_min(0), positions.long() // page].long()
    for got, codes, scales in ((k, c.k, c.k_scale), (v, c.v, c.v_scale)):
        want = (codes[page_of, :, at].float() * scales[page_of, :, at][..., None]).to(dtype)
        want[seqs < 0] = 0
        assert torch.equal(got, want)
    only = torch.empty_like(k)
    ops.read_q8(c.pages(), positions, seqs, c.tables, None, only, c.err)
    assert torch.equal(only, v) and int(c.err) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kv,dim,page,totals", [(2, 64, 16, [4003, 1500, 1]), (9, 256, 24, [2051, 333]), (1, 16, 64, [9001])])
def test_reading_many_rows_back_is_exact(kv, dim, page, totals, dtype):
    test_reading_back_is_exact(dtype=dtype, kv=kv, dim=dim, page=page, totals=totals)


def test_no_rows_write_and_read_nothing():
    c = Case(2, 1, 32, 16, [4], [0], torch.float32, fill=False)
    empty = torch.empty(0, dtype=torch.int32, device=c.device)
    from cuca_b200.kernels import ops
    before = c.k.clone()
    ops.rope_store_q8(torch.empty(0, 128, device=c.device), torch.empty(0, 64, device=c.device), empty, empty, c.tables, None, None, 0,
                      c.pages(), 2, 1, 32, c.err)
    ops.read_q8(c.pages(), empty, empty, c.tables, torch.empty(0, 1, 32, device=c.device), None, c.err)
    assert torch.equal(before, c.k)


# ------------------------------------------------------------------ attention
SHAPES = [(32, 8, 128), (8, 8, 64), (16, 2, 128), (24, 4, 80), (4, 2, 16), (6, 1, 256), (40, 2, 64), (12, 12, 96), (3, 1, 48)]
BATCHES = {"one": ([1], [0]), "singles": ([1] * 5, [0, 15, 16, 333, 1027]), "portion": ([70], [45]),
           "mixed": ([1, 5, 1, 37, 2, 130], [40, 100, 0, 0, 700, 1])}


def _attend(c, q=None, **options):
    from cuca_b200.kernels import ops
    q = c.q if q is None else q
    out = torch.full((c.step.n_rows, c.heads * c.dim), 5.0, dtype=c.dtype, device=c.device)
    window = options.pop("window", None)
    ops.attention_q8(q, out, c.pages(), c.tables, c.step, c.heads, c.kv, c.dim, options.pop("scale", c.dim ** -0.5), window,
                     c.err, **options)
    assert int(c.err) == 0
    return out.view(-1, c.heads, c.dim)


def _check(c, **options):
    got = _attend(c, **options)
    scale = options.pop("scale", c.dim ** -0.5)
    want, *sizes = c.attend(scale, **options)
    off = (got.double() - want).abs() - c.bound(want, *sizes)
    assert (off <= 0).all(), (float(off.max()), float((got.double() - want).abs().max()))
    return got


@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,dim", SHAPES)
def test_attention(heads, kv, dim, dtype, batch):
    c = Case(heads, kv, dim, 16, *BATCHES[batch], dtype, seed=dim + heads)
    _check(c)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page", [1, 8, 24, 32, 64, 128])
def test_attention_over_pages_of_any_size(page, dtype):
    _check(Case(8, 2, 64, page, *BATCHES["mixed"], dtype, seed=page))
    _check(Case(8, 2, 128, page, *BATCHES["singles"], dtype, seed=page))


OPTIONS = [dict(window=1), dict(window=17), dict(window=64, keep_first=4), dict(window=100, keep_first=33), dict(window=5000, keep_first=3),
           dict(softcap=5.0), dict(softcap=30.0, window=40), dict(sink=True), dict(sink=True, sink_values=True, window=30),
           dict(slopes=True), dict(slopes=True, window=77, keep_first=16, sink=True, softcap=20.0), dict(scale=1.7)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,dim", [(32, 8, 128), (6, 2, 64), (9, 3, 80)])
@pytest.mark.parametrize("number", range(len(OPTIONS)))
def test_attention_options(number, heads, kv, dim, dtype):
    c = Case(heads, kv, dim, 16, *BATCHES["mixed"], dtype, seed=number)
    o = dict(OPTIONS[number])
    if o.get("sink_values"):
        o["sink_values"] = 2 * torch.randn(heads, device=c.device, generator=c.g)
    if o.get("slopes"):
        o["slopes"] = torch.rand(heads, device=c.device, generator=c.g) * 0.1
    _check(c, **o)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,dim,counts,starts", [(8, 2, 128, [64, 1, 20], [3000, 5000, 2]), (4, 4, 64, [1, 300], [40, 2500]),
                                                         (8, 2, 128, [1], [4000]), (8, 2, 64, [2, 1], [4000, 700])])
def test_sinks_that_weigh_as_much_as_the_keys_where_keys_are_shared_out(heads, kv, dim, counts, starts, dtype):
    c = Case(heads, kv, dim, 16, counts, starts, dtype, seed=5)
    _check(c, sink=True, sink_values=8 + torch.randn(heads, device=c.device, generator=c.g))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,dim,counts,starts", [
    (8, 2, 128, [1, 1], [9000, 30]), (2, 1, 64, [3], [20000]), (32, 8, 128, [300], [2000]), (4, 4, 128, [1], [40000])])
def test_attention_over_many_keys(heads, kv, dim, counts, starts, dtype):
    _check(Case(heads, kv, dim, 32, counts, starts, dtype, seed=1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("counts", [[1, 1], [40, 1], [200]])
def test_value_scales_far_apart_and_large_scores(counts, dtype):
    """Value rows from 1e-12 to 1e12, zeros among them, and scores that leave all but one key no weight."""
    c = Case(8, 2, 64, 16, counts, [100 * (i + 1) for i in range(len(counts))], dtype, seed=4, level=30.0)
    c.v_scale *= 10.0 ** torch.randint(-12, 13, c.v_scale.shape, device=c.device, generator=c.g).float()
    nothing = torch.rand(c.v_scale.shape, device=c.device, generator=c.g) < 0.2
    c.v_scale[nothing & c.v_scale.isfinite()] = 0.0
    _check(c)
    c.q.zero_()  # every key alike
    _check(c)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_queries_of_any_magnitude(dtype):
    c = Case(8, 2, 64, 16, [1, 20], [100, 50], dtype, seed=6)
    c.q.copy_((c.q.float() * 10.0 ** torch.randint(-30, 3, (c.step.n_rows, 8), device=c.device, generator=c.g).float().repeat_interleave(64, 1)).to(dtype))
    _check(c)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("counts,starts", [([1, 1], [50, 200]), ([30, 150], [50, 20])])
def test_what_is_not_finite_reaches_those_who_see_it_alone(counts, starts, dtype):
    c = Case(4, 2, 64, 16, counts, starts, dtype, seed=8)
    clean = _attend(c)
    places = c.tables[c.slots[0]].long()
    first, last = c.starts[0], c.starts[0] + counts[0] - 1
    c.v_scale[places[last // 16], 1, last % 16] = math.nan  # the last position, key head 1: only its own row sees it
    got = _attend(c)
    assert got[counts[0] - 1, 2:].isnan().all() and torch.equal(got[counts[0] - 1, :2], clean[counts[0] - 1, :2])
    rest = [i for i in range(c.step.n_rows) if i != counts[0] - 1]
    assert torch.equal(got[rest], clean[rest])
    c.k_scale[places[0], 0, 0] = math.nan  # the first position, key head 0: every row of the request without a window
    got = _attend(c)
    assert got[:counts[0], :2].isnan().all() and torch.equal(got[counts[0]:], clean[counts[0]:])
    windowed = _attend(c, window=first - 16)
    assert windowed[:, :2].isfinite().all()
    c.q[0, 64] = math.inf
    got = _attend(c, window=first - 16)
    assert got[0, 1].isnan().all() and got[0, 0].isfinite().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("counts", [[1, 1, 1], [1, 40, 1]])
def test_rows_of_no_request_get_zeros(counts, dtype):
    c = Case(4, 2, 64, 16, counts, [3, 40, 7], dtype, seed=2, padding=3)
    got = _attend(c)
    n = sum(counts)
    assert (got[n:] == 0).all()
    want, *sizes = c.attend(64 ** -0.5)
    assert ((got.double() - want).abs() <= c.bound(want, *sizes)).all()


def test_a_row_does_not_depend_on_its_batch_order_or_run():
    c = Case(32, 8, 128, 16, *BATCHES["mixed"], torch.bfloat16, seed=5)
    first = _attend(c)
    for _ in range(3):
        assert torch.equal(first, _attend(c))


def test_strided_rows_and_another_stream():
    c = Case(8, 2, 64, 16, *BATCHES["mixed"], torch.bfloat16, seed=5)
    want = _attend(c)
    wide = torch.zeros(c.step.n_rows, 12 * 64 + 2, dtype=c.dtype, device=c.device)
    wide[:, :512] = c.q
    assert torch.equal(want, _attend(c, q=wide[:, :512]))
    shifted = torch.empty(c.step.n_rows * 512 + 1, dtype=c.dtype, device=c.device)[1:].view(-1, 512)
    shifted.copy_(c.q)
    assert torch.equal(want, _attend(c, q=shifted))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [_attend(c) for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(want, g) for g in got)


def test_pages_beyond_two_gigabytes():
    """Codes and scales of pages whose offset passes 2^31 and 2^32 bytes."""
    dev = torch.device("cuda:0")
    pages = (1 << 32) // (8 * 16 * 128) + 40
    c = Case(32, 8, 128, 16, [1, 9], [200, 55], torch.bfloat16, seed=7)
    big = [torch.zeros(pages, *t.shape[1:], dtype=t.dtype, device=dev) for t in (c.k, c.v, c.k_scale, c.v_scale)]
    n = c.k.shape[0]
    want = _attend(c)
    for b, t in zip(big, (c.k, c.v, c.k_scale, c.v_scale)):
        b[pages - n:] = t
    c.tables = torch.where(c.tables >= 0, c.tables + pages - n, -1)
    c.k, c.v, c.k_scale, c.v_scale = big
    assert torch.equal(want, _attend(c))
    k, v = _read(c, torch.bfloat16)
    assert k.isfinite().all() and float(k.float().abs().sum()) > 0
    qkv = torch.randn(c.step.n_rows, 48 * 128, device=dev).to(torch.bfloat16)
    _write(c, qkv, torch.empty(c.step.n_rows, 32 * 128, dtype=torch.bfloat16, device=dev), None, None, 0)
    k, _ = _read(c, torch.float32)
    x = qkv[:, 32 * 128:40 * 128].float().view(-1, 8, 128)
    assert ((k - x).abs() <= x.abs().amax(-1, keepdim=True) / 250).all()


# ------------------------------------------------------------------ refusals
def test_refusals():
    from cuca_b200.kernels import library, ops
    c = Case(4, 2, 64, 16, [3], [10], torch.bfloat16, seed=1)
    out = torch.empty(3, 256, dtype=torch.bfloat16, device=c.device)
    args = lambda **k: dict(q=c.q, out=out, pages=c.pages(), tables=c.tables, step=c.step, n_heads=4, n_kv_heads=2, head_dim=64,  # noqa: E731
                            scale=0.1, window=None, err=c.err) | k
    half = ops.QuantizedPages(c.k, c.v, c.k_scale.half(), c.v_scale)
    for bad in (dict(q=c.q.half()), dict(out=out.float()), dict(q=c.q[:2]), dict(out=out[:, :100]), dict(n_heads=3, n_kv_heads=2),
                dict(head_dim=32), dict(pages=half), dict(tables=c.tables.long()), dict(window=-1), dict(keep_first=-1, window=3),
                dict(softcap=-1.0), dict(sink=True, sink_values=torch.zeros(3, device=c.device)), dict(q=c.q.cpu()),
                dict(pages=ops.QuantizedPages(c.k[:, :, ::2], c.v[:, :, ::2], c.k_scale[:, :, ::2], c.v_scale[:, :, ::2])),
                dict(slopes=torch.zeros(4, dtype=torch.float64, device=c.device))):
        with pytest.raises(library.KernelError):
            ops.attention_q8(**args(**bad))
    odd = Case(4, 2, 48, 16, [3], [10], torch.bfloat16)
    wrong = ops.QuantizedPages(odd.k[..., :40].contiguous(), odd.v[..., :40].contiguous(), odd.k_scale, odd.v_scale)
    with pytest.raises(library.KernelError):
        ops.attention_q8(**args(pages=wrong, head_dim=40))
    qkv = torch.zeros(3, 8 * 64, dtype=torch.bfloat16, device=c.device)
    cos, sin = _tables(32, 64, c.device)
    store = lambda **k: dict(qkv=qkv, q_out=out, positions=c.step.positions, seq_of_row=c.step.seq_of_row, tables=c.tables, cos=cos,  # noqa: E731
                             sin=sin, rotary_dim=64, pages=c.pages(), n_heads=4, n_kv_heads=2, head_dim=64, err=c.err) | k
    before = c.k.clone()
    for bad in (dict(qkv=qkv[:, :400]), dict(q_out=out.float()), dict(rotary_dim=32), dict(sin=None), dict(cos=cos.double()),
                dict(positions=c.step.positions.long()), dict(positions=c.step.positions[:2]), dict(n_kv_heads=1), dict(qkv=qkv.cpu()),
                dict(bias=qkv[0]), dict(qkv=ops.PartialSums(qkv[None], 1)),
                dict(qkv=ops.PartialSums(qkv[None].float(), 1), bias=qkv[0].float())):
        with pytest.raises(library.KernelError):
            ops.rope_store_q8(**store(**bad))
    assert torch.equal(before, c.k)
    k = torch.empty(3, 2, 64, dtype=torch.bfloat16, device=c.device)
    for bad in (k.half(), k[:, :1], torch.empty(3, 2, 128, dtype=torch.bfloat16, device=c.device)[..., ::2]):
        with pytest.raises(library.KernelError):
            ops.read_q8(c.pages(), c.step.positions, c.step.seq_of_row, c.tables, bad, None, c.err)


def test_a_page_that_is_not_there_is_recorded():
    """A position without a page: the error word says so, nothing is read or written outside."""
    from cuca_b200.kernels import ops
    c = Case(4, 2, 64, 16, [3], [10], torch.bfloat16, seed=1)
    for bad in (-1, c.k.shape[0], 1 << 30):
        c.tables[c.slots[0], 0] = bad
        for call in (lambda: ops.attention_q8(c.q, torch.empty_like(c.q), c.pages(), c.tables, c.step, 4, 2, 64, 0.1, None, c.err),
                     lambda: _read(c, torch.bfloat16),
                     lambda: _write(c, torch.zeros(3, 512, dtype=torch.bfloat16, device=c.device), torch.empty_like(c.q), None, None, 0)):
            before = c.k.clone()
            call()
            assert int(c.err) == 2 and torch.equal(before, c.k)
            c.err.zero_()


@pytest.mark.parametrize("heads,kv,dim,counts,starts", [(32, 8, 128, [300], [2000]), (32, 8, 128, [700], [3000]), (8, 2, 64, [200, 90], [700, 1]),
                                                         (6, 1, 96, [256, 3], [1500, 900])])
def test_portions_give_the_same_bits_in_every_run(heads, kv, dim, counts, starts):
    """Warps of a block run apart from one another; what they hand over does not depend on by how much."""
    c = Case(heads, kv, dim, 16, counts, starts, torch.bfloat16, seed=dim, level=4.0)
    first = _check(c)
    for _ in range(60):
        assert torch.equal(first, _attend(c))


def test_no_rows_attend_to_nothing():
    c = Case(4, 2, 64, 16, [], [], torch.bfloat16)
    assert _attend(c).numel() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cluster", [True, False])
@pytest.mark.parametrize("starts", [[600], [700, 3], [1500, 0, 40], [2500]])
def test_shares_join_through_a_cluster_and_through_memory(monkeypatch, starts, cluster, dtype):
    from cuca_b200.kernels import ops
    monkeypatch.setattr(ops, "CLUSTER_MERGE", cluster)
    c = Case(8, 2, 128, 16, [1] * len(starts), starts, dtype, seed=len(starts))
    *_, share, shares, memory = ops.attention_q8_plan(c.step).launches(8, 2, 128, dtype, None, 0)[0]
    assert shares > 1
    assert memory == (not cluster) and (memory or shares in (2, 4, 8))
    got = _check(c, sink=True)
    assert torch.equal(got, _attend(c, sink=True))
    _check(c, window=300, keep_first=5, softcap=20.0)


@pytest.mark.parametrize("few,along", [(0, 0.0), (0, 10.0), (24, 0.0), (10 ** 6, 0.0)])
def test_a_mixed_step_in_every_form(monkeypatch, few, along):
    """Portions through blocks of few rows or through tcgen05, single tokens apart or with them."""
    from cuca_b200.kernels import ops
    monkeypatch.setattr(ops, "Q8_FEW_ROWS", few)
    monkeypatch.setattr(ops, "Q8_SINGLES_ALONG", along)
    for heads, kv, dim in ((8, 2, 64), (5, 1, 112)):
        c = Case(heads, kv, dim, 16, *BATCHES["mixed"], torch.bfloat16, seed=few % 7)
        _check(c)
        _check(c, window=33, keep_first=2, sink=True)


@pytest.fixture
def through_tcgen05(monkeypatch):
    """32-bit portions of any size through tcgen05, and that they went there."""
    from cuca_b200.kernels import ops
    monkeypatch.setattr(ops, "Q8_FEW_ROWS", 0)
    monkeypatch.setattr(ops, "Q8_LEAST_F32", 0)
    seen, launches = [], ops.QuantizedPlan.launches

    def watched(self, *a, **k):
        plan = launches(self, *a, **k)
        seen.extend(n[0] for n in plan if n[2] > 1)
        return plan
    monkeypatch.setattr(ops.QuantizedPlan, "launches", watched)
    return seen


@pytest.mark.parametrize("heads,kv,dim", [s for s in SHAPES if s[2] <= 128])
def test_32_bit_portions_of_every_shape_through_tcgen05(through_tcgen05, heads, kv, dim):
    c = Case(heads, kv, dim, 16, *BATCHES["mixed"], torch.float32, seed=dim)
    _check(c)
    _check(c, window=33, keep_first=2, sink=True, sink_values=4 * torch.randn(heads, device=c.device, generator=c.g))
    _check(Case(heads, kv, dim, 24, [3, 2, 130], [0, 1000, 600], torch.float32, seed=dim + 1), scale=0.4)
    assert set(through_tcgen05) == {1}
    _check(c, softcap=9.0)  # (this form does not take it)
    assert set(through_tcgen05) == {0, 1}


def test_32_bit_portions_through_tcgen05_where_it_can_go_wrong(through_tcgen05):
    f32 = torch.float32
    for page in (1, 8, 24, 128):
        _check(Case(8, 2, 64, page, *BATCHES["mixed"], f32, seed=page))
    test_value_scales_far_apart_and_large_scores([200], f32)
    test_value_scales_far_apart_and_large_scores([40, 1], f32)
    test_queries_of_any_magnitude(f32)
    test_what_is_not_finite_reaches_those_who_see_it_alone([30, 150], [50, 20], f32)
    test_rows_of_no_request_get_zeros([1, 40], f32)
    test_sinks_that_weigh_as_much_as_the_keys_where_keys_are_shared_out(8, 2, 128, [64, 1, 20], [3000, 5000, 2], f32)
    assert 1 in through_tcgen05


@pytest.mark.parametrize("skew", [0, 1, 2])
def test_32_bit_portions_through_tcgen05_anywhere_in_memory(through_tcgen05, skew):
    """Rows that do not begin on 16 bytes, further apart than they are long; the same bits from each, and in every run."""
    from cuca_b200.kernels import ops
    c = Case(6, 2, 80, 16, [33, 70], [700, 0], torch.float32, seed=3)
    want = _attend(c).flatten(1)
    wide = torch.zeros(c.step.n_rows, 480 + 16 + skew, device=c.device)
    q, out = wide[:, skew:skew + 480], torch.full_like(wide, 3.0)
    q.copy_(c.q)
    for _ in range(3):
        ops.attention_q8(q, out[:, skew:skew + 480], c.pages(), c.tables, c.step, 6, 2, 80, 80 ** -0.5, None, c.err)
        assert torch.equal(out[:, skew:skew + 480], want) and int(c.err) == 0
    assert (out[:, :skew] == 3).all() and (out[:, skew + 480:] == 3).all() and set(through_tcgen05) == {1}
