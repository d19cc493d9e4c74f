"""commit_path against a copy row by row, bit for bit."""

import random

import pytest
import torch

from tests._util import gen

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class Pool:
    """A pool of random bytes, trees of q_lens nodes behind `bases` tokens, and rising paths."""

    def __init__(self, q_lens, bases, paths, L, KVH, D, dtype, seed=0, bs=16, wide=False):
        need = [-(-(a + n) // bs) for a, n in zip(bases, q_lens)]
        blocks = sum(need) + 2
        perm = torch.randperm(blocks, generator=gen(seed)).tolist()
        self.bs, self.q_lens, self.bases, self.paths = bs, q_lens, bases, paths
        self.bt = torch.zeros((len(need), max(need + [1])), dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.bt[b, :n] = torch.tensor(perm[at:at + n], dtype=torch.int32)
            at += n
        shape = (L, blocks * bs, KVH + wide, D)
        self.key, self.value = (torch.randn(shape, generator=gen(seed + i)).to(dtype).to(DEV)
                                for i in (1, 2))
        if wide:                                    # rows at a stride, off 16 bytes for odd ones
            self.key, self.value = self.key[:, :, :KVH], self.value[:, :, :KVH]
        self.cu = _i32([sum(q_lens[:i]) for i in range(len(q_lens) + 1)])
        self.lens = _i32([a + n for a, n in zip(bases, q_lens)])
        width = max([len(p) for p in paths] + [1]) + 1
        self.path = _i32([list(p) + [-1] * (width - len(p)) for p in paths])
        self.num = _i32([max(0, len(p) - 1) for p in paths])
        self.blocks = self.bt.to(DEV)

    def slot(self, b, pos):
        return int(self.bt[b, pos // self.bs]) * self.bs + pos % self.bs

    def expected(self):
        out = []
        for pool in (self.key, self.value):
            new = pool.clone()
            for b, p in enumerate(self.paths):
                for j in range(1, len(p)):
                    new[:, self.slot(b, self.bases[b] + j)] = pool[:, self.slot(b, self.bases[b] + p[j])]
            out.append(new)
        return out

    def call(self, **kw):
        from dispec_amd.kv.paged_cache import commit_path
        args = dict(block_size=self.bs)
        args.update(kw)
        commit_path(self.key, self.value, self.blocks, self.cu, self.lens, self.path, self.num, **args)

    def check(self):
        want = self.expected()
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        self.call(err=err)
        assert int(err) == 0
        assert torch.equal(self.key, want[0]) and torch.equal(self.value, want[1])


def _random(seed, B, n_max, bs, **kw):
    rng = random.Random(seed)
    q_lens = [rng.randint(0, n_max) for _ in range(B)]
    paths = []
    for n in q_lens:
        m = rng.randint(0, max(0, n - 1))
        paths.append([0] + sorted(rng.sample(range(1, n), m)) if n else [])
    return Pool(q_lens, [rng.randint(0, 3 * bs) for _ in range(B)], paths, seed=seed, bs=bs, **kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("L,KVH,D", [(1, 2, 64), (5, 1, 8), (3, 8, 128), (2, 3, 36), (2, 1, 1)])
@pytest.mark.parametrize("bs", [1, 16, 64])
def test_random_paths(hip, dtype, L, KVH, D, bs):
    for seed in range(4):
        _random(seed, 5, 40, bs, L=L, KVH=KVH, D=D, dtype=dtype).check()


def test_sources_that_are_destinations(hip):
    """Rows that are written after they were read, over more rows than a thread holds at once."""
    for path in ([0, 1, 2, 3], [0, 2, 3, 4], list(range(0, 2)) + list(range(3, 60)),
                 [0] + list(range(40, 99)), list(range(0, 100, 3)), [0, 99]):
        Pool([100], [7], [path], L=3, KVH=2, D=64, dtype=torch.float16, seed=len(path)).check()


@pytest.mark.parametrize("D", [64, 3])
def test_rows_at_a_stride(hip, D):
    _random(3, 4, 30, 16, L=3, KVH=2, D=D, dtype=torch.bfloat16, wide=True).check()


def test_a_cache_method_and_its_errors(hip):
    from dispec_amd.kv.paged_cache import PagedKVCache
    cache = PagedKVCache(2, 8, 16, 2, 64, dtype=torch.bfloat16)
    cache.key.normal_()
    cache.value.normal_()
    table = cache.block_table([[5, 2, 7], [1, 0]])
    cu, lens = _i32([0, 6, 9]), _i32([40, 20])
    old = cache.key.clone()
    cache.commit_path(table, cu, lens, _i32([[0, 3, 5], [0, 2, -1]]), _i32([2, 1]))
    cache.check_errors()
    s = [7 * 16 + 2 + i for i in range(6)]          # positions 34 .. 39
    want = old.clone()
    want[:, s[1]], want[:, s[2]] = old[:, s[3]], old[:, s[5]]
    want[:, 0 * 16 + 2] = old[:, 0 * 16 + 3]        # positions 17 .. 19 of the second
    assert torch.equal(cache.key, want)
    # an id outside the pool: its rows stay, and are counted
    old = cache.key.clone()
    table[0, 2] = 8
    cache.commit_path(table, cu, lens, _i32([[0, 3, 5], [0, -1, -1]]), _i32([2, 0]))
    assert torch.equal(cache.key, old)
    with pytest.raises(IndexError):
        cache.check_errors()


def test_bad_paths(hip):
    """Nothing is moved from an entry on that does not rise, or is no node; a count past the width
    is the width's; lengths that do not fit move nothing."""
    rows = [([0, 2, 1, 4], 3, 1), ([0, 3, 9, 4], 3, 1), ([0, 2, 2, 4], 3, 1), ([-1, 2, 3, 4], 3, 0),
            ([0, 2, 4, 5], 9, 3), ([0, -1, 3, 4], 3, 0), ([0, 2, 3, 4], 0, 0), ([0, 2, 3, 4], -5, 0)]
    for path, num, moved in rows:
        p = Pool([6], [10], [[0] + path[1:moved + 1]], L=2, KVH=2, D=64, dtype=torch.bfloat16)
        want = p.expected()
        p.path, p.num = _i32([path]), _i32([num])
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        p.call(err=err)
        assert torch.equal(p.key, want[0]) and torch.equal(p.value, want[1]), path
        assert int(err) == (1 if 0 < num <= 3 and moved < num else 0), path
    p = Pool([6], [10], [[0, 2, 3]], L=2, KVH=2, D=64, dtype=torch.bfloat16)
    old = p.key.clone()
    p.lens = _i32([4])                              # fewer tokens than nodes
    p.call()
    assert torch.equal(p.key, old)


def test_graph_and_stream(hip):
    p = _random(11, 6, 50, 16, L=4, KVH=2, D=64, dtype=torch.bfloat16)
    k0, v0 = p.key.clone(), p.value.clone()
    want = p.expected()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        p.call()
    side.synchronize()
    assert torch.equal(p.key, want[0]) and torch.equal(p.value, want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p.call()
    for _ in range(3):
        p.key.copy_(k0)
        p.value.copy_(v0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(p.key, want[0]) and torch.equal(p.value, want[1])


def test_offsets_past_32_bits(hip):
    """Layers more than 2^32 bytes apart."""
    L, slots, KVH, D = 3, 1 << 22, 4, 128
    key = torch.zeros((L, slots, KVH, D), dtype=torch.bfloat16, device=DEV)
    value = torch.zeros_like(key)
    from dispec_amd.kv.paged_cache import commit_path
    last = slots // 16 - 1
    for t, x in ((key, 1.0), (value, 2.0)):
        t[:, last * 16 + 9] = x
    commit_path(key, value, _i32([[last]]), _i32([0, 10]), _i32([10]), _i32([[0, 9]]), _i32([1]))
    for t, x in ((key, 1.0), (value, 2.0)):
        assert bool((t[:, last * 16 + 1] == x).all()) and float(t.sum(dtype=torch.float64)) == \
            2 * x * L * KVH * D
