"""Blocks are copied as bytes: between caches of one format only."""

import pytest
import torch

from dispec_amd import _lib
from dispec_amd.kv.paged_cache import PagedKVCache
from dispec_amd.kv.prefix_cache import PrefixCache
from dispec_amd.kv.quant_cache import QuantPagedKVCache


@pytest.fixture()
def caches(monkeypatch):
    """Pools whose blocks have as many bytes: in bf16, in 8 bits with heads twice as wide, in 4 bits
    with four times as wide ones."""
    monkeypatch.setattr(_lib, "require_gpu", lambda *t: None)
    monkeypatch.setattr(_lib, "stream_of", lambda t: 0)

    class Reached(Exception):
        pass

    class Library:
        def __getattr__(self, name):
            def call(*a):
                raise Reached(name)
            return call

    monkeypatch.setattr(_lib, "lib", lambda: Library())
    monkeypatch.setattr(_lib, "calls", lambda: Library())
    made = (PagedKVCache(2, 4, 16, 2, 64, torch.bfloat16, "cpu"),
            QuantPagedKVCache(2, 4, 16, 2, 128, torch.bfloat16, "cpu", format="fp8"),
            QuantPagedKVCache(2, 4, 16, 2, 256, torch.bfloat16, "cpu", format="fp4"))
    assert len({c.block_bytes for c in made}) == 1
    return Reached, made


def test_other_formats_are_refused(caches):
    Reached, made = caches
    ids = torch.zeros(1, dtype=torch.int32)
    for dst in made:
        for src in made:
            for copy in (lambda: dst.copy_blocks_from(src, [1], [2]),
                         lambda: dst.copy_blocks_from(src, [1, 1], [2, 3]),
                         lambda: dst.copy_blocks_device(src, ids, ids + 1),
                         lambda: dst.copy_block_fanout_device(src, 0, ids + 1)):
                if dst is src:
                    with pytest.raises(Reached):
                        copy()
                else:
                    with pytest.raises(ValueError, match="cache into a"):
                        copy()


def test_a_spill_into_another_format(caches):
    _, (plain, fp8, _) = caches
    prefixes = PrefixCache(fp8.manager, 16)
    prefixes.bind(fp8)
    table = fp8.manager.allocate(1, 16)
    prefixes.insert(list(range(16)), table.block_ids)
    fp8.manager.free(1)
    with pytest.raises(ValueError, match="fp8 cache into a plain one"):
        prefixes.evict(1, spill_to=plain)
