"""Speculative decoding with drafted trees, the operators as they are used together: a forward of
the runner over the trees (SeqMeta.parents -> tree_mask, paged_tree_attention), the verdict on the
device (match_draft, verify_draft), the kept path moved behind its context (commit_path), and the
next step over what it left."""

import random

import numpy as np
import pytest
import torch

from tests._tree import random_parents
from tests.toy_lm import toy_lm

pytestmark = pytest.mark.gpu
DEV = "cuda"
VOCAB = 128


class Engine:
    """Sequences of one runner; a step appends rows and returns their logits."""

    def __init__(self, model, dtype, backend="hip", blocks=96, bs=16):
        from dispec_amd.engine.model_runner import ModelRunner
        from dispec_amd.kv.paged_cache import PagedKVCache
        self.runner = ModelRunner(model, attn_backend=backend)
        self.cache = PagedKVCache.for_model(model.config, blocks, bs, dtype, DEV)
        self.bs = bs

    def forward(self, rows):
        """rows: (sequence, token ids, parents or None); the logits of all of them."""
        from dispec_amd.engine.model_runner import SeqMeta
        mgr = self.cache.manager
        tokens, positions, slots, meta = [], [], [], []
        for sid, ids, parents in rows:
            if not mgr.has_table(sid):
                mgr.allocate(sid, 0)
            table = mgr.block_table(sid)
            start = table.num_tokens
            mgr.reserve(sid, len(ids))
            table.num_tokens = start + len(ids)
            depth = list(range(len(ids)))
            if parents is not None:
                for i, p in enumerate(parents):
                    depth[i] = 0 if p < 0 else depth[p] + 1
            tokens += ids
            positions += [start + d for d in depth]
            slots += [table.block_ids[p // self.bs] * self.bs + p % self.bs
                      for p in range(start, start + len(ids))]
            meta.append(SeqMeta(list(table.block_ids), len(ids), start + len(ids), parents))
        put = lambda x: torch.tensor(x).to(DEV)  # noqa: E731
        hidden = self.runner.forward(put(tokens), put(positions), put(slots), meta, self.cache)
        return self.runner.logits(hidden).float()

    def batch(self, rows):
        """(block_table, cu_q, ctx_lens, parents, max_q_len) of the rows just run, on the GPU."""
        mgr = self.cache.manager
        tables = [mgr.block_table(sid) for sid, _, _ in rows]
        cu = np.cumsum([0] + [len(ids) for _, ids, _ in rows])
        parents = [p for _, ids, par in rows
                   for p in (range(-1, len(ids) - 1) if par is None else par)]
        put = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
        return (self.cache.block_table([t.block_ids for t in tables]), put(cu.tolist()),
                put([t.num_tokens for t in tables]), put(parents),
                max(len(ids) for _, ids, _ in rows))

    def keep(self, rows, verdict):
        """The kept paths committed; the host's tables follow.  Returns the new tokens."""
        table, cu, ctx, _, _ = self.batch(rows)
        self.cache.commit_path(table, cu, ctx, verdict.path, verdict.num_accepted)
        kept = verdict.num_accepted.tolist()
        for (sid, ids, _), k in zip(rows, kept):
            before = self.cache.manager.block_table(sid).num_tokens - len(ids)
            self.cache.manager.truncate(sid, before + 1 + k)
        self.cache.check_errors()
        return [t[:k + 1] for t, k in zip(verdict.tokens.tolist(), kept)]


def prompts(n, seed):
    rng = random.Random(seed)
    return [[rng.randrange(VOCAB) for _ in range(rng.choice((5, 16, 33, 47)))] for _ in range(n)]


def drafted(ahead, n, rng):
    """A tree of n nodes (its root's token left open) that holds some of the tokens that follow,
    others beside them."""
    parents = random_parents(n, rng)
    ids, right = [0] * n, [0] + [None] * (n - 1)       # right: how many tokens the node's path has
    taken = set()
    for i in range(1, n):
        p = parents[i]
        d = right[p]
        if d is not None and p not in taken and d < len(ahead) and rng.random() < 0.7:
            ids[i], right[i] = ahead[d], d + 1
            taken.add(p)
        else:
            ids[i], right[i] = rng.randrange(VOCAB), None
    return ids, parents


@pytest.mark.parametrize("family,backend", [("qwen3", "hip"), ("qwen2", "hip"), ("qwen2", "native")])
def test_greedy_trees_give_the_tokens_of_plain_decoding(family, backend):
    """fp32: each step drafts trees (some of the tokens that follow among others), the kept ones
    and the next are those of token-by-token decoding."""
    from dispec_amd.engine.hip_verify import match_draft
    model = toy_lm(family).to(DEV)
    steps, B = 40, 3
    plain, tree = Engine(model, torch.float32), Engine(model, torch.float32, backend)
    first = [(b, ids, None) for b, ids in enumerate(prompts(B, 3))]
    ends = np.cumsum([len(ids) for _, ids, _ in first]) - 1
    logits = plain.forward(first)
    want = [[t] for t in logits[ends.tolist()].argmax(-1).tolist()]
    for _ in range(steps):
        nxt = plain.forward([(b, [want[b][-1]], None) for b in range(B)]).argmax(-1).tolist()
        for b in range(B):
            want[b].append(nxt[b])
    rng = random.Random(5)
    got = [[t] for t in tree.forward(first)[ends.tolist()].argmax(-1).tolist()]
    kept_most = 0
    while min(len(g) for g in got) <= steps:
        rows = []
        for b in range(B):
            ids, parents = drafted(want[b][len(got[b]):], rng.choice((1, 2, 7, 40)), rng)
            ids[0] = got[b][-1]
            rows.append((b, ids, parents))
        choice = tree.forward(rows).argmax(-1)
        _, cu, _, parents, most = tree.batch(rows)
        tokens = torch.tensor([t for _, ids, _ in rows for t in ids], device=DEV)
        verdict = match_draft(tokens, choice, cu, parents=parents, max_q_len=most)
        for b, new in enumerate(tree.keep(rows, verdict)):
            got[b] += new
            kept_most = max(kept_most, len(new) - 1)
    assert kept_most >= 2
    for b in range(B):
        n = min(len(got[b]), len(want[b]))
        assert got[b][:n] == want[b][:n], b


@pytest.mark.parametrize("family,dtype,least", [("qwen3", torch.bfloat16, 0.999),
                                                ("qwen2", torch.float16, 0.999),
                                                ("qwen3", torch.float32, 0.99999)])
def test_a_node_s_logits_are_its_path_s(family, dtype, least):
    """The logits of every node are those of its path run as a chain behind the same context, in a
    batch with a single token and a chunk of a prompt."""
    model = toy_lm(family).to(dtype).to(DEV)
    rng = random.Random(11)
    first = [(b, ids, None) for b, ids in enumerate(prompts(3, 12))]
    e = Engine(model, dtype)
    e.forward(first)
    n = 37
    parents = random_parents(n, rng)
    ids = [rng.randrange(VOCAB) for _ in range(n)]
    one, chunk = [rng.randrange(VOCAB)], [rng.randrange(VOCAB) for _ in range(21)]
    got = e.forward([(0, one, None), (1, ids, parents), (2, chunk, None)])
    chains = Engine(model, dtype, blocks=400)
    for i in range(n):
        path = [i]
        while parents[path[0]] >= 0:
            path.insert(0, parents[path[0]])
        chains.forward([(i, first[1][1], None)])
        want = chains.forward([(i, [ids[j] for j in path], None)])[-1]
        cos = torch.nn.functional.cosine_similarity(got[1 + i], want, dim=0)
        assert cos >= least, (i, float(cos))
        chains.cache.manager.free(i)
    plain = Engine(model, dtype)
    plain.forward(first)
    want = plain.forward([(0, one, None), (2, chunk, None)])
    cos = torch.nn.functional.cosine_similarity(torch.cat((got[:1], got[1 + n:])), want, dim=-1)
    assert cos.min() >= least


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("with_draft", [False, True])
def test_sampled_step_keeps_what_the_verdict_says(dtype, with_draft):
    """Sampling: the verdict on given random numbers is the formula's, and the cache behind it
    holds the kept path's rows: the next step's logits are those of the kept tokens run plainly."""
    from dispec_amd.engine.hip_verify import verify_draft
    model = toy_lm("qwen3").to(dtype).to(DEV)
    rng = random.Random(23)
    g = torch.Generator().manual_seed(24)
    first = [(b, ids, None) for b, ids in enumerate(prompts(4, 25))]
    e = Engine(model, dtype)
    e.forward(first)
    rows = []
    for b in range(4):
        n = (1, 6, 12, 9)[b]
        parents = None if with_draft else random_parents(n, rng)
        rows.append((b, [rng.randrange(VOCAB) for _ in range(n)], parents))
    # (a sharp target: that some drafted tokens are kept)
    probs = torch.softmax(12 * e.forward(rows), -1)
    _, cu, _, parents, most = e.batch(rows)
    T = probs.shape[0]
    tokens = [t for _, ids, _ in rows for t in ids]
    # every other sequence drafts what the target finds likeliest
    at = 0
    for b, (_, ids, par) in enumerate(rows):
        for i in range(1, len(ids)):
            if b % 2:
                tokens[at + i] = int(probs[at + (i - 1 if par is None else par[i])].argmax())
        at += len(ids)
    u, u_last = torch.rand(T, generator=g), torch.rand(4, generator=g)
    draft = torch.softmax(torch.randn(T - 4, VOCAB, generator=g), -1) if with_draft else None
    verdict = verify_draft(torch.tensor(tokens, device=DEV), probs, u.to(DEV), u_last.to(DEV), cu,
                           parents=None if with_draft else parents,
                           draft_probs=None if draft is None else draft.to(DEV), max_q_len=most)
    # the formula, in 64 bits on the host
    p64, at, row = probs.double().cpu().numpy(), 0, 0
    u64, want = u.double().numpy(), []
    for b, (_, ids, par) in enumerate(rows):
        cur, path, new = 0, [0], []
        while True:
            if with_draft:
                kids = [cur + 1] if cur + 1 < len(ids) else []
            else:
                kids = [i for i in range(1, len(ids)) if par[i] == cur]
            rest, total, keep = p64[at + cur].copy(), 0.0, None
            seen = set()
            for i in kids:
                x = tokens[at + i]
                if with_draft:
                    q = draft[row + cur].double().numpy()
                    if u64[at + cur] * q[x] < rest[x]:
                        keep = i
                    rest = np.maximum(rest - q, 0)
                    break
                if x in seen:
                    continue
                seen.add(x)
                total += p64[at + cur][x]
                rest[x] = 0
                if u64[at + cur] < total:
                    keep = i
                    break
            if keep is None:
                break
            cur = keep
            path.append(cur)
            new.append(tokens[at + cur])
        upto = np.cumsum(rest)
        new.append(int(np.argmax(upto > float(u_last[b]) * upto[-1])))
        want.append((path, new))
        at += len(ids)
        row += len(ids) - 1
    assert [t[:k + 1] for t, k in zip(verdict.path.tolist(), verdict.num_accepted.tolist())] \
        == [p for p, _ in want]
    new = e.keep(rows, verdict)
    assert new == [n for _, n in want]
    assert max(len(x) for x in new) >= 3
    # the forward above ran other tokens where the likeliest replaced them: run the step again with
    # the tokens that were taken, so that the cache holds theirs
    e2, plain = Engine(model, dtype), Engine(model, dtype)
    e2.forward(first)
    at, taken = 0, []
    for b, ids, par in rows:
        taken.append((b, tokens[at:at + len(ids)], par))
        at += len(ids)
    e2.forward(taken)
    e2.keep(taken, verdict)
    plain.forward(first)
    plain.forward([(b, [tok[i] for i in path], None)
                   for (b, tok, _), (path, _) in zip(taken, want)])
    step = [(b, [n[-1]], None) for b, (_, n) in enumerate(want)]
    got, ref = e2.forward(step), plain.forward(step)
    cos = torch.nn.functional.cosine_similarity(got, ref, dim=-1)
    assert cos.min() >= (0.99999 if dtype == torch.float32 else 0.999), cos
