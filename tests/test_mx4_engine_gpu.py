"""The engine with projections whose weights, or weights and rows, are kept in 4 bits: logits, graphs, memory, refusals."""
import pytest
import torch

import mx4_util as mx
import plain_llama
import tiny
from q8_util import quantise

pytestmark = pytest.mark.gpu


class _SmallRows:
    """A projection of the plain model whose rows are brought to 4 bits before the product."""

    def __init__(self, w):
        self.w = w

    def to(self, dtype):
        return _SmallRows(self.w.to(dtype))

    @property
    def T(self):
        return self

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        x, w = args
        return mx.held(x).to(w.w.dtype) @ w.w.T


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    made = {}

    def get(which):
        if which not in made:
            made[which] = tmp_path_factory.mktemp("mx4_" + which)
            tiny.write_tiny(made[which], which)
        return made[which]
    return get


def _plain(folder, tokens, small_rows=False, kv=None):
    """Logits of the plain implementation, in 64 bits, whose projections have the values that 4 bits hold; with `kv` the attention reads
    keys and values through 8-bit codes."""
    cfg, weights = plain_llama.load_model_dir(folder)
    for name, w in weights.items():
        if "_proj.weight" in name:
            w = mx.held(w.to(torch.bfloat16))
            weights[name] = _SmallRows(w) if small_rows else w
    whole = plain_llama.causal_attention

    def attention(q, k, v, scale, window=None):
        k, v = ((c * s[..., None]).to(q.dtype) for c, s in (quantise(k), quantise(v)))
        return whole(q, k, v, scale, window)
    if kv:
        plain_llama.causal_attention = attention
    try:
        return plain_llama.forward(cfg, weights, tokens, dtype=torch.float64)
    finally:
        plain_llama.causal_attention = whole


def _core(folder, dtype, **kw):
    from cuca_b200.engine.core import EngineCore
    return EngineCore.from_folder(folder, dtype=dtype, kv_tokens=512, max_sequences=4, weight_dtype="mxfp4", max_step_tokens=256, **kw)


def _run(core, requests, cuts):
    """Each request's tokens in portions of the given sizes, the requests together; logits of every token."""
    from cuca_b200.engine.step import StepEntry
    n = len(requests)
    blocks = [core.pools.new_seq() for _ in range(n)]
    slots = [core.slots.alloc() for _ in range(n)]
    at, out, turn = [0] * n, [[] for _ in range(n)], 0
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
    return [torch.cat(o) for o in out]


@pytest.mark.parametrize("kv", [None, "int8"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("which", ["A", "B", "C", "D", "E"])
def test_logits_match_the_plain_model_over_held_weights(folders, which, dtype, kv):
    if kv and dtype == "float32":
        pytest.skip("a value between two 8-bit codes may fall to either side")
    core = _core(folders(which), dtype, kv_cache_dtype=kv)
    requests = [tiny.random_tokens(n, core.spec.vocab_size, seed=n) for n in (90, 1, 47)]
    got = _run(core, requests, (1, 40, 3, 1, 17, 5))
    for tokens, logits in zip(requests, got):
        want = _plain(folders(which), tokens, kv=kv)
        # as the other replays: 32-bit sums and rows to 2^-23 of a block's largest; bfloat16 activations
        far = (1e-4 if dtype == "float32" else 3e-2) * want.abs().max()
        assert (logits - want).abs().max() < far


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("which", ["A", "B", "C", "D", "E"])
def test_logits_with_rows_in_4_bits(folders, which, dtype):
    core = _core(folders(which), dtype, activation_dtype="mxfp4")
    requests = [tiny.random_tokens(n, core.spec.vocab_size, seed=n) for n in (90, 1, 47)]
    got = _run(core, requests, (1, 40, 3, 1, 17, 5))
    off = noise = size = 0.0
    for tokens, logits in zip(requests, got):
        want, wide = (_plain(folders(which), tokens, small_rows=small) for small in (True, False))
        off += (logits - want).square().sum().item()
        noise += (wide - want).square().sum().item()
        size += want.square().sum().item()
    if dtype == "float32":  # a value within 2^-20 of a border takes the next code: hardly one does
        assert (off / size) ** 0.5 < 1e-2
    else:
        # A value that bfloat16 puts on a border's other side is a step s off where rounding to codes is off by s / sqrt(12) in the
        # mean. Codes are a third of their value apart, so with values e off a share e / (1/3) of them is, and rows differ by
        # sqrt(12 * 3 e) of what rounding them does: by less than that as long as e < 1/36. bfloat16 rows are 2^-8 off, and what
        # earlier layers add goes with the noise of their own rounding.
        assert off < noise


def test_weights_take_a_quarter_of_the_memory(folders):
    from cuca_b200.engine.core import EngineCore
    kw = dict(dtype="bfloat16", kv_tokens=512, max_sequences=4)
    whole, small = EngineCore.from_folder(folders("D"), **kw), EngineCore.from_folder(folders("D"), weight_dtype="mxfp4", **kw)
    a, b = ([sum(p.weight_bytes() for p in (x.mixer, x.feed_forward)) for x in core.model.blocks] for core in (whole, small))
    assert all(y * 32 == x * 8.5 for x, y in zip(a, b))  # sizes of whole tiles: 17 bytes for 32 numbers of 16 bits


@pytest.mark.parametrize("rows", [None, "mxfp4"])
@pytest.mark.parametrize("which,dtype", [("B", "float32"), ("D", "bfloat16"), ("E", "bfloat16")])
def test_generation_through_graphs_and_eagerly(folders, which, dtype, rows):
    from cuca_b200 import BatchingConfig, LocalModel, LocalModelConfig
    folder = folders(which)
    prompts = [tiny.random_tokens(n, tiny.CONFIGS[which]["vocab_size"], seed=n) for n in (3, 20, 47)]
    config = LocalModelConfig(source=str(folder), dtype=dtype, weight_dtype="mxfp4", activation_dtype=rows,
                              batching=BatchingConfig(max_sequences=4))
    graphs, eager = LocalModel.load(config), LocalModel.load(config)
    eager.backend.use_graphs = False
    outs = [m.generate(prompts, max_tokens=24, temperature=0.0) for m in (graphs, eager)]
    assert graphs.backend.graph_steps >= 23 and eager.backend.graph_steps == 0
    for results in outs:
        for prompt, out in zip(prompts, results):
            ref = _plain(folder, prompt + out.tokens, small_rows=rows is not None)
            for i, tok in enumerate(out.tokens):
                row = ref[len(prompt) - 1 + i]
                far = (2e-4 if dtype == "float32" else 0.03) if rows is None else 0.3
                assert float(row.max() - row[tok]) < far * float(row.abs().max())


def test_random_weights(folders):
    from cuca_b200 import LocalModel, LocalModelConfig
    from cuca_b200.config.engine_config import RandomWeights
    config = LocalModelConfig(model_config=tiny.CONFIGS["D"], random_weights=RandomWeights(seed=3), weight_dtype="mxfp4")
    assert len(LocalModel.load(config).generate([5, 6, 7], max_tokens=5, temperature=0.0).tokens) == 5


def test_refusals(folders, tmp_path):
    import pafutar_util
    from cuca_b200 import LocalModel, LocalModelConfig
    from cuca_b200.engine.core import EngineCore
    cfg = pafutar_util.CONFIGS["wide"]
    pafutar_util.write_model(tmp_path, cfg, pafutar_util.make_weights(cfg, seed=1))
    with pytest.raises(ValueError, match="4 bits"):
        LocalModel.load(LocalModelConfig(source=str(tmp_path), dtype="float32", weight_dtype="mxfp4"))
    with pytest.raises(ValueError, match="mxfp4"):
        EngineCore.from_folder(folders("D"), weight_dtype="int4")
    with pytest.raises(ValueError, match="mxfp4"):
        EngineCore.from_folder(folders("D"), activation_dtype="mxfp4")
