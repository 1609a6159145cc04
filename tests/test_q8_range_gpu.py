"""The attention over 8-bit pages where magnitudes, masks, page tables and sizes lie far apart, against its formulas in 64 bits
(`q8_util`); writing many rows; what a call leaves behind."""
import itertools
import math

import numpy as np
import pytest
import torch

from q8_util import Case

pytestmark = pytest.mark.gpu
DTYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])


@pytest.fixture(scope="module", autouse=True)
def lib():
    from cuca_b200.kernels import library
    return library.load()


@pytest.fixture
def through_tcgen05(monkeypatch):
    """Portions of any size through tcgen05."""
    from cuca_b200.kernels import ops
    monkeypatch.setattr(ops, "Q8_FEW_ROWS", 0)
    monkeypatch.setattr(ops, "Q8_LEAST_F32", 0)


def _call(c, window=None, scale=None, **options):
    from cuca_b200.kernels import ops
    out = torch.full((c.step.n_rows, c.heads * c.dim), 5.0, dtype=c.dtype, device=c.device)
    ops.attention_q8(c.q, out, c.pages(), c.tables, c.step, c.heads, c.kv, c.dim, scale or c.dim ** -0.5, window, c.err, **options)
    return out.view(-1, c.heads, c.dim)


def _check(c, scale=None, most_work=math.inf, **options):
    got = _call(c, scale=scale, **options)
    assert int(c.err) == 0
    want, size, work, most = c.attend(scale or c.dim ** -0.5, **options)
    off = (got.double() - want).abs() - c.bound(want, size, work.clamp_max(most_work), most)
    assert (off <= 0).all(), (float(off.max()), float((got.double() - want).abs().max()))
    return got


def _at(c, positions, request=0):
    """Where positions of a request stand in the pools, for all key heads."""
    p = torch.as_tensor(positions, device=c.device)
    return c.tables[c.slots[request]].long()[p // c.page], slice(None), p % c.page


# ------------------------------------------------------------------ magnitudes
def _one_axis(counts, starts, dtype, positions, scores, values, value_scales):
    """The first request's queries are 1 along the first dimension alone: its scores (in log2 units, with a scale of ln 2, whose
    product with log2 e is 1 in 32 bits) are what its keys say, and `values` codes times `value_scales` its values."""
    c = Case(8, 2, 64, 16, counts, starts, dtype, seed=1)
    c.q.zero_()
    c.q.view(-1, 8, 64)[..., 0] = 1
    where = _at(c, positions)
    k = torch.zeros(len(positions), 64, dtype=torch.int8, device=c.device)
    k[:, 0] = -1
    c.k[where] = k[:, None].expand(-1, 2, -1)
    c.k_scale[where] = -torch.as_tensor(scores, device=c.device).float()[:, None].expand(-1, 2)
    c.v[where] = torch.as_tensor(values, device=c.device).to(torch.int8)[:, None, None].expand(-1, 2, 64)
    c.v_scale[where] = torch.as_tensor(value_scales, device=c.device).float()[:, None].expand(-1, 2)
    return c


@DTYPES
@pytest.mark.parametrize("count", [1, 2, 40])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("power", [3, 16, 20, 23, 24, 25, 26, 27, 28, 30, 40, 60, 90])
def test_scores_with_steps_of_one_and_more(through_tcgen05, power, sign, count, dtype):
    """Scores of 2^power and the next few 32-bit numbers above, over all the rest: the larger comes 64 keys later each time. Where
    steps are smaller than one the weights are the formula's; else results lie between the values of the largest three."""
    n = 400
    for odd in (0, 1):
        step = max(1.0, 2.0 ** (power - 23))
        scores = np.full(n, min(0.0, 2 * sign * 2.0 ** power) - 1000.0)
        largest = [3, 67, 131]
        scores[largest] = sign * 2.0 ** power + step * (odd + np.array([1, 2, 4]))
        codes = np.arange(n) % 100 + 20
        c = _one_axis([count], [n - count], dtype, range(n), scores, codes, np.full(n, 2.0 ** -3))
        if power <= 23:  # (the scores are exact: what a form's 32-bit sums cost shows between keys less than some 2^8 apart)
            _check(c, scale=math.log(2), most_work=2.0 ** 8)
            continue
        got, near = _call(c, scale=math.log(2)), 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -19
        assert int(c.err) == 0
        assert (got >= codes[largest].min() / 8 * (1 - near)).all() and (got <= codes[largest].max() / 8 * (1 + near)).all()


@DTYPES
@pytest.mark.parametrize("counts", [[40, 1], [3, 1]])
@pytest.mark.parametrize("power", [8, 16, 24, 30, 40, 60])
def test_rows_beside_much_larger_queries(through_tcgen05, power, counts, dtype):
    """Other tokens' and other heads' queries are 2^power larger, or as much smaller."""
    c = Case(8, 2, 64, 16, counts, [200, 100], dtype, seed=power)
    q = c.q.view(-1, 8, 64)
    q[1, 1] *= 2.0 ** power
    q[-1, 6] *= 2.0 ** power
    q[2, :4] *= 2.0 ** -power
    q[0] *= 2.0 ** power
    _check(c)
    _check(c, window=50, keep_first=3, sink=True)


@DTYPES
@pytest.mark.parametrize("power", [3, 5, 8, 12, 16, 18, 20, 21, 30])
@pytest.mark.parametrize("where", [1, 100, 3000])
def test_a_large_value_without_weight_leaves_a_flat_tail_its_weight(through_tcgen05, where, power, dtype):
    """One key of weight 2^-14.5 of the first for each of four thousand: together they weigh six times what the first does.
    A key of no weight has a value scale 2^power above the others."""
    n = 4140
    scores, scales = np.full(n, -14.5), np.full(n, 2.0 ** -6)
    scores[0], scores[where], scales[where] = 0.0, -60.0, 2.0 ** (power - 6)
    got = _check(_one_axis([40], [n - 40], dtype, range(n), scores, np.full(n, 64), scales), scale=math.log(2))
    assert (got.float() - 1).abs().max() < 2.0 ** -7


def _rounded_twice(up):
    """(scale, code) whose product, the scale rounded to 11 bits and then the product, is furthest up or down in units of 2^-11."""
    best = None
    for a, code in itertools.product(range(64), range(64, 80)):
        x = 1 + (a + (0.51 if up else 0.49)) * 2.0 ** -10
        off = (float(np.float16(code * float(np.float16(x)))) / (code * x) - 1) * 2048
        if best is None or (off > best[0] if up else off < best[0]):
            best = off, x, code
    return best


@DTYPES
def test_results_that_rest_on_two_keys_of_opposite_sign(through_tcgen05, dtype):
    """Weights and values that lie between two 16-bit floats, so that what is rounded away of the one is not made up by the other."""
    (far, x, cx), (near, y, cy) = _rounded_twice(True), _rounded_twice(False)
    assert far > 1.8 and near < -1.8
    n = 140
    scores, scales, codes = np.full(n, -200.0), np.full(n, 2.0 ** -3), np.full(n, 64)
    scores[:3] = 0.0, np.log2(1 + 1.02 * 2.0 ** -11) - 1, np.log2(1 + 0.98 * 2.0 ** -11) - 1
    scales[:3], codes[:3] = (0.0, x, y), (0, cx, -cy)
    c = _one_axis([40], [n - 40], dtype, range(n), scores, codes, scales)
    _check(c, scale=math.log(2))


@DTYPES
@pytest.mark.parametrize("depth", [10, 20, 30, 60])
def test_what_is_left_beside_a_value_of_zeros(through_tcgen05, depth, dtype):
    """The key that has nearly all the weight has a value of zeros: the result is what the others' 2^-depth make, to its own bits."""
    n = 340
    scores, scales = np.full(n, -float(depth)), np.full(n, 2.0 ** -6)
    scores[5], scales[5] = 0.0, 0.0
    _check(_one_axis([40], [n - 40], dtype, range(n), scores, np.arange(n) % 50 + 50, scales), scale=math.log(2))


@DTYPES
@pytest.mark.parametrize("few", [10 ** 6, 0])
def test_weights_of_values_of_any_size(monkeypatch, few, dtype):
    """Rows that see five keys of about the same weight, whose values are up to 2^70 apart."""
    from cuca_b200.kernels import ops
    monkeypatch.setattr(ops, "Q8_FEW_ROWS", few)
    monkeypatch.setattr(ops, "Q8_LEAST_F32", 0)
    for seed in range(6):
        c = Case(12, 12, 96, 32, [322], [12], dtype, seed=seed, level=1e-3)
        c.v_scale *= 2.0 ** torch.randint(0, 71, c.v_scale.shape, device=c.device, generator=c.g).float()
        _check(c, window=1, keep_first=4)


# ------------------------------------------------------------------ masks and tables
@DTYPES
@pytest.mark.parametrize("keep", [0, 20])
@pytest.mark.parametrize("page", [4, 16, 24])
def test_pages_behind_a_window_may_be_gone(through_tcgen05, page, keep, dtype):
    """Without them, and whatever the pool's first page holds, the same bits."""
    c = Case(8, 2, 64, page, [50, 1, 2], [400, 300, 155], dtype, seed=page)
    for name in ("k", "v", "k_scale", "v_scale"):
        x = getattr(c, name)
        first = torch.randint(-127, 128, x[:1].shape, device=c.device, generator=c.g).to(x.dtype) if x.dtype == torch.int8 else \
            torch.full_like(x[:1], 3.0)
        setattr(c, name, torch.cat([first, x]))
    c.tables = torch.where(c.tables >= 0, c.tables + 1, -1)
    whole = _check(c, window=100, keep_first=keep)
    for slot, start in zip(c.slots, c.starts):
        behind = [p for p in range((start - 99) // page) if p * page >= keep]
        assert behind
        c.tables[slot, behind] = -1
    for scale in (3.0, 1e9, 0.0):
        c.k_scale[0], c.v_scale[0] = scale, scale
        assert torch.equal(whole, _call(c, window=100, keep_first=keep)) and int(c.err) == 0


@DTYPES
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("counts", [[40], [1], [3, 1]])
def test_positions_without_a_page_are_recorded(through_tcgen05, counts, page, dtype):
    """In every form: entries that are no page, and tables that end before the positions do."""
    c = Case(8, 2, 64, page, counts, [100] * len(counts), dtype, seed=1)
    whole = c.tables.clone()
    for entry, bad in itertools.product((0, 3), (-1, c.k.shape[0], 1 << 30)):
        c.tables[c.slots[0], entry] = bad
        _call(c)
        assert int(c.err) == 2
        c.err.zero_()
        c.tables.copy_(whole)
    _check(c)
    c.tables = whole[:, :3].contiguous()
    _call(c)
    assert int(c.err) == 2


@DTYPES
@pytest.mark.parametrize("counts", [[40], [1], [3, 1]])
def test_first_keys_that_stay_without_end(through_tcgen05, counts, dtype):
    """As many as a 32-bit number holds: every key is seen."""
    c = Case(8, 2, 64, 16, counts, [300] * len(counts), dtype, seed=2)
    assert torch.equal(_call(c, window=5, keep_first=2 ** 31 - 1), _check(c)) and int(c.err) == 0


@DTYPES
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 64), (6, 1, 96)])
def test_every_option_with_every_other(through_tcgen05, heads, kv, dim, dtype):
    c = Case(heads, kv, dim, 16, [1, 37, 2], [150, 70, 0], dtype, seed=dim)
    sinks = 3 * torch.randn(heads, device=c.device, generator=c.g)
    slopes = 0.1 * torch.rand(heads, device=c.device, generator=c.g)
    for window, keep, cap, sink, slope in itertools.product((None, 40), (0, 5), (0.0, 8.0), (None, True, sinks), (None, slopes)):
        _check(c, window=window, keep_first=keep, softcap=cap, sink=sink is not None, sink_values=sink if sink is sinks else None,
               slopes=slope)


@DTYPES
def test_a_request_alone_first_and_last(dtype):
    """Within the bound of the formula whatever else the step brings."""
    mine, others = (37, 100), [(1, 900), (150, 30), (5, 2000)]
    for order in ([mine], [mine] + others, others + [mine], others[:1] + [mine] + others[1:]):
        _check(Case(8, 2, 64, 16, [n for n, _ in order], [s for _, s in order], dtype, seed=3))


# ------------------------------------------------------------------ memory
@pytest.mark.parametrize("counts,starts,dtype", [([8192], [0], torch.float32), ([512, 64], [30000, 100], torch.float32),
                                                 ([1] * 256, [60000] + [50] * 255, torch.bfloat16)])
def test_what_a_call_needs_of_memory_is_bounded(counts, starts, dtype):
    c = Case(32, 8, 128, 64, counts, starts, dtype, seed=1, fill=False)
    c.k_scale.fill_(0.01), c.v_scale.fill_(0.01)
    out = torch.empty_like(c.q)
    from cuca_b200.kernels import ops
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    ops.attention_q8(c.q, out, c.pages(), c.tables, c.step, 32, 8, 128, 0.01, None, c.err)
    torch.cuda.synchronize()
    assert int(c.err) == 0 and out.isfinite().all()
    assert torch.cuda.max_memory_allocated() - before <= 300 * 2 ** 20


@DTYPES
@pytest.mark.parametrize("counts,starts", [([300, 40], [2000, 1500]), ([1, 1, 1], [4000, 3, 2500]), ([5, 2], [3000, 2000])])
def test_launches_in_parts_give_the_same_bits(monkeypatch, counts, starts, dtype):
    from cuca_b200.kernels import ops
    monkeypatch.setattr(ops, "CLUSTER_MERGE", False)
    c = Case(8, 2, 128, 16, counts, starts, dtype, seed=4)
    want = _check(c, sink=True)
    for limit in (0, 1 << 21):
        monkeypatch.setattr(ops, "Q8_SCRATCH", limit)
        assert torch.equal(want, _call(c, sink=True))


# ------------------------------------------------------------------ many rows
@DTYPES
@pytest.mark.parametrize("adjacent,rot,slices", [(True, 16, 0), (False, 8, 0), (False, 16, 2), (True, 16, 2)])
def test_more_rows_than_a_grid_has_along_its_second_axis(adjacent, rot, slices, dtype):
    """As in two calls of fewer rows."""
    from cuca_b200.kernels import ops
    if slices and dtype == torch.float32:
        pytest.skip("K slices give bfloat16 queries")
    n, cut = 70_000, 40_000
    c = Case(2, 1, 16, 64, [n], [0], dtype, seed=1, fill=False)
    angle = torch.arange(n, device=c.device, dtype=torch.float64)[:, None] * 0.1 ** torch.arange(rot // 2, device=c.device)
    cos, sin = angle.cos().float(), angle.sin().float()
    x = torch.randn(max(slices, 1), n, 64, device=c.device, generator=c.g)

    def write(lo, hi, q):
        rows = ops.PartialSums(x[:, lo:hi], slices) if slices else x[0, lo:hi].to(dtype)
        ops.rope_store_q8(rows, q[lo:hi], c.step.positions[lo:hi], c.step.seq_of_row[lo:hi], c.tables, cos, sin, rot, c.pages(), 2, 1,
                          16, c.err, adjacent=adjacent)
        assert int(c.err) == 0
    results = []
    for parts in ([(0, n)], [(0, cut), (cut, n)]):
        for t in (c.k, c.v, c.k_scale, c.v_scale):
            t.zero_()
        q = torch.zeros(n, 32, dtype=dtype, device=c.device)
        for lo, hi in parts:
            write(lo, hi, q)
        results.append([t.clone() for t in (q, c.k, c.v, c.k_scale, c.v_scale)])
    assert all(torch.equal(a, b) for a, b in zip(*results)) and (results[0][3][c.tables[c.slots[0], :n // 64].long()] > 0).all()
