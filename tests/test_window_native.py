"""attn_backend="native" under a window: blocks without a visible token may be freed."""

import types

import numpy as np
import pytest
import torch

from tests._util import f64

BS = 16


@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 3), (40, 0), (33, 20), (64, 70), (500, 4)])
@pytest.mark.parametrize("seqs", [[(1, 200)], [(5, 5), (17, 160), (1, 47)], [(30, 130), (1, 1)]])
def test_keys_that_no_query_sees_are_not_read(window, sinks, seqs):
    """Against the attention in float64; the table has -1 where no query sees a key of the block, and
    the pool NaN where none sees the row."""
    from dispec_amd.engine.model_runner import ModelRunner, SeqMeta
    from dispec_amd.kv.paged_cache import PagedKVCache
    from tests.toy_lm import toy_lm
    runner = ModelRunner(toy_lm("qwen3"), attn_backend="native")
    g = torch.Generator().manual_seed(1)
    blocks = sum(-(-c // BS) for _, c in seqs)
    perm = torch.randperm(blocks, generator=g).tolist()
    k, v = (torch.randn(blocks * BS, 2, 64, generator=g) for _ in range(2))
    q = torch.randn(sum(n for n, _ in seqs), 4, 64, generator=g)
    held = torch.zeros(blocks * BS, dtype=torch.bool)
    meta, want, at = [], [], 0
    for n, ctx in seqs:
        ids = [perm.pop() for _ in range(-(-ctx // BS))]
        key = np.arange(ctx)
        pos = key[ctx - n:, None]
        see = (key <= pos) & ((key > pos - window) | (key < sinks))
        slots = torch.tensor([ids[j // BS] * BS + j % BS for j in key])
        some = torch.from_numpy(see.any(0))
        held[slots[some]] = True
        for h in range(4):
            s = np.where(see, f64(q[at:at + n, h]) @ f64(k[slots, h // 2]).T / 8.0, -np.inf)
            p = np.exp(s - s.max(1, keepdims=True))
            want.append(p / p.sum(1, keepdims=True) @ f64(v[slots, h // 2]))
        at += n
        live = [i for i in range(len(ids)) if some[i * BS:(i + 1) * BS].any()]
        meta.append(SeqMeta([b if i in live else -1 for i, b in enumerate(ids)], n, ctx))
    k[~held], v[~held] = float("nan"), float("nan")

    def gather(layer, slots):
        assert layer == 1 and bool((slots >= 0).all())
        return k[slots], v[slots]

    cache = types.SimpleNamespace(block_size=BS, gather=gather)
    cache.slots_for_positions = lambda ids, p: PagedKVCache.slots_for_positions(cache, ids, p)
    cache.context_slots = lambda ids, n: cache.slots_for_positions(ids, torch.arange(n))
    got = f64(runner._torch_attention(q, cache, 1, meta, window, sinks))
    at = 0
    for i, (n, _) in enumerate(seqs):
        for h in range(4):
            # fp32: a score, |q| |k| / 8 <= 18 here, is a sum of 64 products, off by 66 2^-24 of that;
            # a probability follows twice (its own and the row's sum), sum p |v| <= 4
            np.testing.assert_allclose(got[at:at + n, h], want[4 * i + h], rtol=0, atol=6e-4)
        at += n


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [None, "fp8"])
def test_freed_blocks(hip, fmt):
    """Forwards over a cache whose unseen blocks are gone, NaN in their rows and -1 in the table."""
    from tests.test_gpu_long_context import BF16, Engine, _plan
    from tests.toy_lm import toy_lm
    model = toy_lm("qwen3").to(BF16).to("cuda")
    kept, freed = (Engine(model, BF16, fmt, attn_backend="native", window=24, sinks=4)
                   for _ in range(2))
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
    freed.cache.check_errors()
