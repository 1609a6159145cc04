"""The option that keeps keys and values in 8 bits, on the host."""
import pytest

from cuca_b200.config.engine_config import EngineConfigError, LocalModelConfig


def test_kv_cache_dtype_is_int8_or_absent():
    assert LocalModelConfig.from_json({"source": "x"}).kv_cache_dtype is None
    config = LocalModelConfig.from_json({"source": "x", "kv_cache_dtype": "int8"})
    config.validate()
    config.kv_cache_dtype = "int4"
    with pytest.raises(EngineConfigError, match="kv_cache_dtype"):
        config.validate()


def test_shares_of_the_keys_cover_the_longest_tile():
    """However a batch's keys are cut, the shares reach its longest tile, and no share is empty of work by more than rounding."""
    from cuca_b200.kernels.ops import _q8_shares
    for blocks, keys, longest, dim, nt in ((8, 8 * 77, 77, 128, 1), (64, 64 * 1152, 1152, 128, 1), (512, 512 * 4000, 8192, 128, 1),
                                           (40, 40 * 100000, 100000, 64, 2), (1, 5, 5, 16, 4), (8, 8 * 1000000, 1000000, 128, 1)):
        share, shares = _q8_shares(blocks, keys, longest, dim, nt, sms=148)
        if shares == 1:
            assert share == 0
        else:
            assert share % 64 == 0 and 2 <= shares <= 64 and (shares - 1) * share < longest + 32


def test_every_request_of_a_step_is_in_one_launch_exactly():
    from types import SimpleNamespace

    import torch

    from cuca_b200.kernels import ops
    saved, ops.sm_count = ops.sm_count, lambda: 148
    try:
        for counts in ([1], [1, 1, 1], [2], [5, 1, 9, 40], [300, 1], [4, 4], [17]):
            step = SimpleNamespace(static_max_len=None, n_rows=sum(counts), host={"counts": counts, "starts": [7] * len(counts)})
            for heads, kv, dim in ((32, 8, 128), (40, 2, 64), (6, 1, 256), (3, 3, 16), (260, 2, 64)):
                for dtype in (torch.bfloat16, torch.float32):
                    plan = ops.QuantizedPlan(step).launches(heads, kv, dim, dtype, None, 0)
                    for c in counts:
                        assert sum(lo <= c <= hi for _, lo, hi, *_ in plan) == 1
                    for form, lo, hi, tokens, tiles, group, nt, share, shares, _ in plan:
                        assert tiles == sum(-(-c // tokens) for c in counts if lo <= c <= hi)
                        if form == 0:
                            assert tokens * group * (2 if dtype == torch.float32 else 1) <= 8 * nt
    finally:
        ops.sm_count = saved
