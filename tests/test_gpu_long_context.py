"""Sliding windows, sinks and quantised caches as they are used together: forwards of the runner
(prompts in chunks, then decoding) against the same model computed by torch, in one batch, in a
graph, with blocks outside the window freed, and over forks and exports."""

import numpy as np
import pytest
import torch

from tests._util import cosine, f64
from tests.toy_lm import GEOMETRY, _draw, toy_lm

pytestmark = pytest.mark.gpu
DEV = "cuda"
BS = 16
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


class Engine:
    """Sequences of one runner over one cache; a step appends rows and returns their logits."""

    def __init__(self, model, dtype, fmt=None, blocks=96, **kw):
        from dispec_amd.engine.model_runner import ModelRunner
        from dispec_amd.kv.paged_cache import PagedKVCache
        from dispec_amd.kv.quant_cache import QuantPagedKVCache
        self.runner = ModelRunner(model, **kw)
        self.cache = (QuantPagedKVCache.for_model(model.config, blocks, BS, dtype, DEV, format=fmt)
                      if fmt else PagedKVCache.for_model(model.config, blocks, BS, dtype, DEV))
        perm = torch.randperm(blocks, generator=torch.Generator().manual_seed(1)).tolist()
        self.tables = [perm[i * 16:(i + 1) * 16] for i in range(4)]
        self.cur = [0] * 4
        self.gone = [0] * 4          # leading blocks behind the sinks' that are freed

    def rows(self, batch):
        from dispec_amd.engine.model_runner import SeqMeta
        toks, pos, slots, meta = [], [], [], []
        for s, ids in batch:
            t, n = self.tables[s], self.cur[s]
            toks += ids
            pos += range(n, n + len(ids))
            slots += [t[p // BS] * BS + p % BS for p in range(n, n + len(ids))]
            table = [t[0]] + [-1] * self.gone[s] + t[1 + self.gone[s]:]
            self.cur[s] = n + len(ids)
            meta.append(SeqMeta(table, len(ids), self.cur[s]))
        return toks, pos, slots, meta

    def step(self, batch):
        toks, pos, slots, meta = self.rows(batch)
        put = lambda x: torch.tensor(x, device=DEV)  # noqa: E731
        h = self.runner.forward(put(toks), put(pos), put(slots), meta, self.cache)
        return f64(self.runner.logits(h))


def _plan(seed=0):
    """Prompts in chunks of all sizes beside decodes, then decoding."""
    rng = np.random.default_rng(seed)
    ids = lambda n: rng.integers(0, GEOMETRY["vocab_size"], n).tolist()  # noqa: E731
    steps = [[(0, ids(70)), (1, ids(1)), (2, ids(33))], [(0, ids(50)), (1, ids(64)), (2, ids(1))],
             [(2, ids(90)), (0, ids(5)), (3, ids(7))]]
    return steps + [[(s, ids(1)) for s in range(4)] for _ in range(6)]


def _agree(a, b, dtype):
    """fp32: the same sums in another order; 16 bits: a cosine, as for the other backends."""
    if dtype == F32:
        np.testing.assert_allclose(a, b, rtol=0, atol=2e-4 * max(1.0, np.abs(b).max()))
    else:
        assert cosine(a, b) >= 0.999


@pytest.mark.parametrize("family", ["qwen2", "qwen3"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("fmt", [None, "fp8", "fp4"])
@pytest.mark.parametrize("window,sinks", [(24, 4), (0, 0)])
def test_against_the_native_backend(hip, family, dtype, fmt, window, sinks):
    if fmt is None and not window:
        pytest.skip("the runner's other paths")
    # (fp32 over a quantised cache: one layer, whose rows are the same bits in both.  A second layer's
    # differ in the last ones, and where such a difference lies across the border between two codes
    # they are a whole step apart: 2^-3 of a number, however near the borders' two sides are)
    model = toy_lm(family, 1 if fmt and dtype == F32 else 2).to(dtype).to(DEV)
    kw = dict(window=window, sinks=sinks)
    hip_, native = (Engine(model, dtype, fmt, attn_backend=b, **kw) for b in ("hip", "native"))
    for batch in _plan():
        _agree(hip_.step(batch), native.step(batch), dtype)
    hip_.cache.check_errors()
    if window:   # the window counts
        wide = Engine(model, dtype, fmt, attn_backend="native")
        for batch in _plan():
            far = wide.step(batch)
        assert cosine(far, native.step(_plan(1)[-1])) < 0.99


@pytest.mark.parametrize("backend", ["hip", "native"])
def test_a_model_with_sliding_layers(hip, backend):
    """Layers that the config calls sliding, beside full ones: against the model's own forward."""
    import transformers
    cfg = transformers.Qwen2Config(num_hidden_layers=4, use_sliding_window=True, sliding_window=20,
                                   layer_types=["sliding_attention", "full_attention"] * 2,
                                   attn_implementation="eager", **GEOMETRY)
    model = _draw(transformers.Qwen2ForCausalLM(cfg), 3)
    ids = np.random.default_rng(2).integers(0, 128, 100).tolist()
    with torch.no_grad():
        want = f64(model(torch.tensor([ids])).logits[0])
    e = Engine(model.to(DEV), F32, attn_backend=backend)
    assert e.runner.windows == [(20, 0), (0, 0)] * 2
    got = np.concatenate([e.step([(0, ids[a:b])]) for a, b in ((0, 61), (61, 62), (62, 99), (99, 100))])
    _agree(got, want, F32)


@pytest.mark.parametrize("fmt", [None, "fp8"])
def test_freed_blocks(hip, fmt):
    """Blocks between the sinks' and the window's may go: their entries and rows are not read."""
    model = toy_lm("qwen3").to(BF16).to(DEV)
    kept, freed = (Engine(model, BF16, fmt, window=24, sinks=4) for _ in range(2))
    for batch in _plan():
        want = kept.step(batch)
        for s, _ in batch:
            # a step's first query sees from its position - 23 on
            gone = max(0, (freed.cur[s] - 23) // BS - 1)
            for b in range(freed.gone[s], gone):
                slot = freed.tables[s][1 + b] * BS
                for t in (freed.cache.key, freed.cache.value):
                    t[:, slot:slot + BS] = 255 if fmt else float("nan")
            freed.gone[s] = max(freed.gone[s], gone)
        np.testing.assert_array_equal(freed.step(batch), want)
    assert max(freed.gone) > 3


@pytest.mark.parametrize("fmt,window,sinks", [("fp8", 0, 0), ("fp4", 24, 4), (None, 24, 4)])
def test_graph_decoder(hip, fmt, window, sinks):
    """Captured steps over 40 tokens, each against an eager one over a cache of its own."""
    from dispec_amd.engine.hip_graph import HipGraphDecoder
    model = toy_lm("qwen3").to(BF16).to(DEV)
    eager, graph = (Engine(model, BF16, fmt, window=window, sinks=sinks) for _ in range(2))
    for batch in _plan()[:3]:
        eager.step(batch)
        graph.step(batch)
    dec = HipGraphDecoder(graph.runner, graph.cache, buckets=(256,))
    rng = np.random.default_rng(4)
    for _ in range(40):
        batch = [(s, rng.integers(0, 128, 1).tolist()) for s in range(4)]
        toks, pos, slots, meta = graph.rows(batch)
        got = f64(dec.decode_batch(toks, pos, slots, meta))
        torch.cuda.synchronize()
        want = eager.step(batch)
        assert cosine(got, want) >= 0.9999
    graph.cache.check_errors()


def test_quantised_blocks_fork_and_export(hip):
    """A fork's copied block, and an export into a second cache, carry on as the original does."""
    model = toy_lm("qwen3").to(BF16).to(DEV)
    a, b = (Engine(model, BF16, "fp8") for _ in range(2))
    prompt = _plan()[0][0][1]
    a.step([(0, prompt)])
    # sequence 1 forks sequence 0: shared full blocks, its own copy of the last
    full = len(prompt) // BS
    a.cache.copy_blocks([(a.tables[0][full], a.tables[1][full])])
    a.tables[1][:full] = a.tables[0][:full]
    a.cur[1] = a.cur[0]
    # the second cache takes what the first exports
    k, v = a.cache.export_contiguous(a.tables[0], len(prompt))
    b.cache.import_contiguous(b.tables[0], k, v)
    b.cur[0] = len(prompt)
    x, y = a.step([(0, [5]), (1, [5])]), b.step([(0, [5])])
    _agree(x[0], x[1], BF16)
    _agree(y[0], x[0], BF16)


def test_refused(hip):
    from dispec_amd.engine.model_runner import SeqMeta
    model = toy_lm("qwen3").to(BF16).to(DEV)
    for e in (Engine(model, BF16, "fp8"), Engine(model, BF16, window=8)):
        with pytest.raises(ValueError, match="drafted trees"):
            e.runner._batch([SeqMeta(e.tables[0], 3, 30, parents=[-1, 0, 0])], e.cache)
    Engine(model, BF16, window=4096).runner._batch(
        [SeqMeta(list(range(16)), 3, 30, parents=[-1, 0, 0])], e.cache)   # wider than the context
