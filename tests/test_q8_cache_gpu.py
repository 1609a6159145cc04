"""Reading a request's 8-bit pages back where some are not there."""
import pytest
import torch

import tiny

pytestmark = pytest.mark.gpu


def test_positions_without_a_page_are_refused_and_the_next_step_is_not(tmp_path):
    from cuca_b200.engine.core import EngineCore
    from cuca_b200.engine.step import StepEntry
    tiny.write_tiny(tmp_path, "D")
    core = EngineCore.from_folder(tmp_path, dtype="float32", kv_tokens=512, max_sequences=4, kv_cache_dtype="int8")
    blocks, slot = core.pools.new_seq(), core.slots.alloc()
    tokens = tiny.random_tokens(41, core.spec.vocab_size, seed=1)

    def step(part):
        core.pools.reserve(blocks, blocks.length + len(part))
        logits = core.stepper.step([StepEntry(blocks, slot, part, [len(part) - 1])])
        core.rt.check_device_errors()
        return logits
    step(tokens[:40])
    k, v = core.cache.read(0, slot, 40)
    assert k.abs().sum() > 0 and v.abs().sum() > 0
    with pytest.raises(IndexError, match="no page"):
        core.cache.read(0, slot, 400)
    with pytest.raises(IndexError, match="no page"):
        core.cache.read(0, (slot + 1) % 4, 1)
    core.rt.check_device_errors()
    assert step(tokens[40:]).isfinite().all()
    assert torch.equal(core.cache.read(0, slot, 41)[0][:40], k)
