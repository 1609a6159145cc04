"""The engine with keys and values kept in 8 bits: logits, graphs, prefix reuse, reading back, refusals."""
import numpy as np
import pytest
import torch

import plain_llama
import tiny
from q8_util import quantise

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    made = {}

    def get(which):
        if which not in made:
            made[which] = tmp_path_factory.mktemp("q8_" + which)
            tiny.write_tiny(made[which], which)
        return made[which]
    return get


def _plain(folder, tokens, kept=None):
    """Logits of the plain implementation, in 64 bits, whose attention reads keys and values through codes and scales."""
    cfg, weights = plain_llama.load_model_dir(folder)
    whole = plain_llama.causal_attention

    def attention(q, k, v, scale, window=None):
        rows = []
        for x in (k, v):
            codes, scales = quantise(x)
            rows.append(codes * scales[..., None])
        if kept is not None:
            kept.append(rows)
        return whole(q, rows[0].to(q.dtype), rows[1].to(q.dtype), scale, window)
    plain_llama.causal_attention = attention
    try:
        return plain_llama.forward(cfg, weights, tokens, dtype=torch.float64)
    finally:
        plain_llama.causal_attention = whole


def _core(folder, dtype, **kw):
    from cuca_b200.engine.core import EngineCore
    return EngineCore.from_folder(folder, dtype=dtype, kv_tokens=512, max_sequences=4, kv_cache_dtype="int8", max_step_tokens=256, **kw)


def _run(core, requests, cuts):
    """Each request's tokens in portions of the given sizes, the requests together; logits of every token."""
    from cuca_b200.engine.step import StepEntry
    n = len(requests)
    blocks = [core.pools.new_seq() for _ in range(n)]
    slots = [core.slots.alloc() for _ in range(n)]
    at, out = [0] * n, [[] for _ in range(n)]
    turn = 0
    while any(a < len(r) for a, r in zip(at, requests)):
        entries, who = [], []
        for i, r in enumerate(requests):
            size = min(cuts[(turn + i) % len(cuts)], len(r) - at[i])
            if size:
                core.pools.reserve(blocks[i], at[i] + size)
                entries.append(StepEntry(blocks[i], slots[i], r[at[i]:at[i] + size], list(range(size))))
                who.append((i, size))
        logits = core.stepper.step(entries)
        core.rt.check_device_errors()
        row = 0
        for i, size in who:
            out[i].append(logits[row:row + size].double().cpu())
            row += size
            at[i] += size
        turn += 1
    return [torch.cat(o) for o in out], slots


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("which", ["A", "B", "C", "D", "E"])
def test_logits_match_the_plain_model_over_codes(folders, which, dtype):
    core = _core(folders(which), dtype, block_size=16)
    vocab = core.spec.vocab_size
    requests = [tiny.random_tokens(n, vocab, seed=n) for n in (90, 1, 47)]
    got, _ = _run(core, requests, (1, 40, 3, 1, 17, 5))
    for tokens, logits in zip(requests, got):
        want = _plain(folders(which), tokens)
        # 32-bit: a value on the edge between two codes may fall to the other side, 1/127 of its row's largest; bfloat16: as the
        # other replays in bfloat16
        far = (5e-3 if dtype == "float32" else 3e-2) * want.abs().max()
        assert (logits - want).abs().max() < far


def test_pages_take_about_half_the_memory(folders):
    from cuca_b200.engine.core import EngineCore
    kw = dict(dtype="bfloat16", kv_tokens=512, max_sequences=4)
    whole, codes = EngineCore.from_folder(folders("D"), **kw), EngineCore.from_folder(folders("D"), kv_cache_dtype="int8", **kw)
    assert codes.cache.bytes_per_token() * 2 * 128 == whole.cache.bytes_per_token() * (128 + 4)
    assert codes.cache.bytes() / whole.cache.bytes() == (128 + 4) / 256


def test_what_is_cached_reads_back(folders):
    core = _core(folders("D"), "float32")
    tokens = tiny.random_tokens(70, core.spec.vocab_size, seed=3)
    _, slots = _run(core, [tokens], (33, 1, 20))
    kept = []
    _plain(folders("D"), tokens, kept)
    for layer, (k, v) in enumerate(kept):
        got = core.cache.read(layer, slots[0], len(tokens))
        assert int(core.rt.err) == 0
        for g, want in zip(got, (k, v)):
            step = want.abs().amax(-1, keepdim=True) / 127
            off = (g.double().cpu() - want).abs() / step
            assert off.max() < 1.01 and (off > 0.01).float().mean() < 1e-3  # the same codes but for values between two
    with pytest.raises(IndexError):
        core.cache.read(0, 4, 1)
    with pytest.raises(ValueError, match="8 bits"):
        from cuca_b200.engine.core import EngineCore
        EngineCore.from_folder(folders("D"), dtype="float32", kv_tokens=64).cache.read(0, 0, 1)


@pytest.mark.parametrize("which,dtype", [("B", "float32"), ("D", "bfloat16"), ("E", "bfloat16")])
def test_generation_through_graphs_and_eagerly(folders, which, dtype):
    from cuca_b200 import BatchingConfig, LocalModel, LocalModelConfig
    folder = folders(which)
    prompts = [tiny.random_tokens(n, tiny.CONFIGS[which]["vocab_size"], seed=n) for n in (3, 20, 47)]
    config = LocalModelConfig(source=str(folder), dtype=dtype, kv_cache_dtype="int8", batching=BatchingConfig(max_sequences=4))
    graphs, eager = LocalModel.load(config), LocalModel.load(config)
    eager.backend.use_graphs = False
    outs = [m.generate(prompts, max_tokens=24, temperature=0.0) for m in (graphs, eager)]
    assert graphs.backend.graph_steps >= 23 and eager.backend.graph_steps == 0
    for results in outs:
        for prompt, out in zip(prompts, results):
            ref = _plain(folder, prompt + out.tokens)
            for i, tok in enumerate(out.tokens):
                row = ref[len(prompt) - 1 + i]
                assert float(row.max() - row[tok]) < (5e-3 if dtype == "float32" else 0.03) * float(row.abs().max())


def test_a_shared_prefix_is_read_from_the_pages_of_the_first(folders):
    from cuca_b200 import BatchingConfig, LocalModel, LocalModelConfig
    folder = folders("D")
    head = tiny.random_tokens(64, 1000, seed=1)
    prompts = [head + tiny.random_tokens(9, 1000, seed=s) for s in (2, 3)]
    tokens = []
    for cached in (False, True):
        model = LocalModel.load(LocalModelConfig(source=str(folder), dtype="float32", kv_cache_dtype="int8",
                                                 batching=BatchingConfig(max_sequences=2, prefix_cache=cached)))
        tokens.append([model.generate(p, max_tokens=8, temperature=0.0).tokens for p in prompts])
    assert tokens[0] == tokens[1]


def test_models_whose_layers_do_not_take_codes_are_refused(tmp_path):
    import pafutar_util
    from cuca_b200 import LocalModel, LocalModelConfig
    cfg = pafutar_util.CONFIGS["wide"]
    pafutar_util.write_model(tmp_path, cfg, pafutar_util.make_weights(cfg, seed=1))
    with pytest.raises(ValueError, match="8 bits"):
        LocalModel.load(LocalModelConfig(source=str(tmp_path), dtype="float32", kv_cache_dtype="int8"))
