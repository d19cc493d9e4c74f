"""Speculative decoding with drafted trees, as cases that can be timed and checked.

Three operators, each through the calls that a speculative engine makes of this package:

* ``attend``: one layer's attention of the drafted tokens over the paged cache.  A sequence's
  last tokens are the nodes of a tree (node 0: the last token that was kept); a node sees the
  whole context before the tree and, of the tree, itself and its ancestors.
* ``verify``: which path of each tree the target keeps, and the token that follows it.
  "sample": a drafted chain against the target's and the draft's probabilities (rejection
  sampling); "tree": a tree of proposed tokens against the target's probabilities; "match":
  a tree against the tokens that the target chose.  The random numbers are inputs.
* ``commit``: the K and V rows of the kept path, over all layers, move to the places right
  behind the context.

Head shapes are (query heads, KV heads, head_dim) of the Qwen2.5 / Qwen3 configurations that
the benchmark and the tests use, plus 256-wide heads; the vocabulary is Qwen2.5's.

Where `own` is false the operators are computed in elementary torch operations, batched over
sequences padded to the longest; where it is true, by the package's kernels.
"""

import functools
import math
from types import SimpleNamespace

import torch

own = False

BS = 16              # tokens per block
VOCAB = 151936
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SHAPES = ((14, 2, 64), (12, 2, 128), (16, 8, 128), (28, 4, 128), (32, 8, 128))
PAIRS = 4 * 64 * 32 * 32768   # sequences x nodes x heads x keys of the largest attention case


# ------------------------------------------------------------------------------- the cases
def _attend(name, shape, seqs, ctx, nodes, dtype="bf16", lengths=0):
    """seqs sequences of ctx[0]..ctx[1] tokens, the nodes[0]..nodes[1] tree nodes included;
    the lengths follow from the number `lengths`."""
    case = {"kind": "attend", "heads": shape[0], "kv_heads": shape[1], "dim": shape[2],
            "dtype": dtype, "seqs": seqs, "ctx_lo": ctx[0], "ctx_hi": ctx[1],
            "n_lo": nodes[0], "n_hi": nodes[1], "lengths": lengths}
    return {"name": name, **case} if name else case


def _verify(name, mode, seqs, nodes, vocab=VOCAB, dtype="fp32", lengths=0):
    case = {"kind": "verify", "mode": mode, "seqs": seqs, "n_lo": nodes[0], "n_hi": nodes[1],
            "vocab": vocab, "dtype": dtype, "lengths": lengths}
    return {"name": name, **case} if name else case


def _commit(name, layers, kv_heads, dim, seqs, nodes, kept, dtype="bf16", lengths=0):
    """kept: 0..kept drafted tokens of each tree are kept."""
    case = {"kind": "commit", "layers": layers, "kv_heads": kv_heads, "dim": dim, "seqs": seqs,
            "n_lo": nodes[0], "n_hi": nodes[1], "kept": kept, "dtype": dtype, "lengths": lengths}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one request's small tree early in its answer: the smallest call, where launches count
        _attend("draft_tree", (14, 2, 64), 1, (300, 300), (8, 8)),
        # a serving batch, the same tree size for all
        _attend("batch_tree", (16, 8, 128), 32, (500, 4000), (16, 16)),
        # trees of all sizes beside sequences that decode a single token
        _attend("ragged_tree", (12, 2, 128), 24, (40, 3001), (1, 33)),
        # large trees over middling contexts, seven query heads to a KV head
        _attend("large_tree_fp16", (28, 4, 128), 8, (1000, 8000), (64, 64), dtype="fp16"),
        # long documents: the largest
        _attend("long_tree", (32, 8, 128), 4, (32768, 32768), (64, 64)),
        # an fp32 model (reference-precision runs)
        _attend("fp32_tree", (14, 2, 64), 4, (200, 2000), (26, 26), dtype="fp32"),
        # a few requests, five tokens drafted for each and sampled by a draft model
        _verify("sample_chain", "sample", 8, (6, 6)),
        # trees of the draft's likeliest tokens
        _verify("sample_tree", "tree", 16, (26, 26)),
        # a full batch with chains of all lengths
        _verify("sample_batch", "sample", 64, (1, 9)),
        # greedy decoding: the target's tokens are known, and only integers are compared
        _verify("match_tree", "match", 32, (1, 61)),
        # one request of a small model
        _commit("commit_one", 24, 2, 64, 1, (8, 8), 3),
        # a serving batch, every layer's rows
        _commit("commit_batch", 36, 8, 128, 32, (33, 64), 8),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    case = _draw(rng)
    case["lengths"] = rng.randrange(1 << 30)
    return case


def _draw(rng):
    what = rng.choice(["attend", "attend", "wide", "fp32", "verify", "verify", "commit"])
    if what == "verify":
        mode = rng.choice(["sample", "tree", "match"])
        hi = _log_int(rng, 1, 12 if mode == "sample" else 100)
        return _verify(None, mode, _log_int(rng, 1, min(64, 600 // hi)),
                       (rng.choice([hi, rng.randint(1, hi)]), hi),
                       vocab=rng.choice([VOCAB, _log_int(rng, 1000, 160000)]),
                       dtype=rng.choice(["fp32", "fp32", "bf16", "fp16"]))
    if what == "commit":
        hi = _log_int(rng, 4, 100)
        kv_heads, dim = rng.choice([(2, 64), (2, 128), (4, 128), (8, 128)])
        return _commit(None, rng.randint(4, 36), kv_heads, dim, _log_int(rng, 1, 32),
                       (rng.randint(2, hi), hi), rng.randint(1, 10),
                       dtype=rng.choice(["bf16", "fp16", "fp32"]))
    dtype = "fp32" if what == "fp32" else rng.choice(["bf16", "bf16", "fp16"])
    shape = (rng.choice([8, 16]), 8, 256) if what == "wide" else rng.choice(SHAPES)
    most = 64 if what == "attend" else 12
    n_hi = _log_int(rng, 1, 128 if what == "attend" else 64)
    ctx_hi = max(n_hi, _log_int(rng, 20, 32768 if what == "attend" else 4000))
    seqs = max(1, min(_log_int(rng, 1, most), PAIRS // (n_hi * shape[0] * ctx_hi)))
    n_hi = max(1, min(n_hi, PAIRS // (seqs * shape[0] * ctx_hi)))
    return _attend(None, shape, seqs, (rng.randint(1, ctx_hi), ctx_hi),
                   (rng.choice([n_hi, rng.randint(1, n_hi)]), n_hi), dtype=dtype)


# ----------------------------------------------------------------------------- the inputs
def _between(lo, hi, n, g):
    return torch.randint(lo, max(lo, hi) + 1, (n,), generator=g).tolist()


def _lengths(case):
    """Tree sizes of a case's sequences, and their context lengths (attend) or the numbers of
    drafted tokens that are kept (commit)."""
    g = torch.Generator().manual_seed(case["lengths"])
    nodes = _between(case["n_lo"], case["n_hi"], case["seqs"], g)
    nodes[-1] = case["n_hi"]
    if case["kind"] == "attend":
        ctx = _between(case["ctx_lo"], case["ctx_hi"], case["seqs"], g)
        return nodes, [max(c, n) for c, n in zip(ctx, nodes)]
    if case["kind"] == "commit":
        return nodes, [int(torch.randint(0, 1 + min(case["kept"], (n - 1) // 2), (1,),
                                         generator=g)) if i else min(case["kept"], (n - 1) // 2)
                       for i, n in enumerate(nodes)]
    return nodes, None


def _parents(n, g):
    """Parents of a tree's nodes, two or three children to a node (-1: the root)."""
    return [-1] + [int(torch.randint((i - 1) // 3, (i - 1) // 2 + 1, (1,), generator=g))
                   for i in range(1, n)]


def _cu(lengths):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return cu


def _i32(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _tables(lengths, g):
    """A block table of blocks in random places, and the pool's number of blocks."""
    need = [-(-n // BS) for n in lengths]
    perm = torch.randperm(sum(need) + 4, generator=g).to(torch.int32)
    table = torch.zeros((len(need), max(need)), dtype=torch.int32)
    for i, (n, at) in enumerate(zip(need, _cu(need))):
        table[i, :n] = perm[at:at + n]
    return table.cuda(), sum(need) + 4


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    g = torch.Generator().manual_seed(seed + 1)
    s = SimpleNamespace(case=case)
    nodes, second = _lengths(case)
    s.nodes, s.max_q = nodes, max(nodes)
    s.cu_q = _i32(_cu(nodes))
    s.T = sum(nodes)
    return {"attend": _prepare_attend, "verify": _prepare_verify,
            "commit": _prepare_commit}[case["kind"]](case, s, second, gen, g)


def _prepare_attend(case, s, ctx, gen, g):
    dtype, D = DTYPES[case["dtype"]], case["dim"]
    words = -(-s.max_q // 32)
    mask = torch.zeros((s.T, words), dtype=torch.int64)
    for n, at in zip(s.nodes, s.cu_q.tolist()):
        bits = []
        for i, p in enumerate(_parents(n, g)):
            bits.append((bits[p] if p >= 0 else 0) | 1 << i)
            for w in range(words):
                mask[at + i, w] = bits[i] >> 32 * w & 0xffffffff
    s.mask = mask.to(torch.int32).cuda()   # bit a of row i: node i sees node a
    s.ctx, s.ctx_lens = ctx, _i32(ctx)
    s.block_table, blocks = _tables(ctx, g)
    s.max_ctx = s.block_table.shape[1] * BS
    s.G = case["heads"] // case["kv_heads"]

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)

    s.q = randn(s.T, case["heads"], D)
    s.key = randn(blocks * BS, case["kv_heads"], D)
    s.value = randn(blocks * BS, case["kv_heads"], D)
    return s


def _prepare_verify(case, s, _, gen, g):
    dtype, V, T, B = DTYPES[case["dtype"]], case["vocab"], s.T, case["seqs"]
    parents = [p for n in s.nodes
               for p in (list(range(-1, n - 1)) if case["mode"] == "sample" else _parents(n, g))]
    s.parents = _i32(parents)
    # the target's row of each node's parent (a root's: its own)
    first = torch.tensor(_cu(s.nodes)[:-1]).repeat_interleave(torch.tensor(s.nodes))
    prow = (first + torch.tensor(parents).clamp(min=0)).cuda()
    s.u = torch.rand(T, generator=gen, device="cuda")
    s.u_last = torch.rand(B, generator=gen, device="cuda")
    # logits with a few likely tokens, and a draft that is nearly right
    logits = torch.randn((T, V), generator=gen, device="cuda").mul_(4.0)
    s.target = logits.softmax(-1).to(dtype)
    s.draft = None
    noise = torch.randn((T, V), generator=gen, device="cuda")
    if case["mode"] == "sample":
        draft = logits.add_(noise.mul_(0.8)).softmax(-1).to(dtype)
        pick = torch.multinomial(draft[prow].float(), 1, generator=gen)[:, 0]
        keep = torch.ones(T, dtype=torch.bool)
        keep[(s.cu_q[1:].long() - 1).cpu()] = False   # nothing was drafted after a last node
        s.draft = draft[keep.cuda()]
        s.tokens = pick
    else:
        # the children of a node: its likeliest tokens, in order
        rank = torch.zeros(T, dtype=torch.long)
        seen = {}
        for i, p in enumerate(prow.tolist()):
            if parents[i] >= 0:
                rank[i] = seen.get(p, 0)
                seen[p] = seen.get(p, 0) + 1
        k = min(V, 1 + max(list(seen.values()) + [0]))
        likely = logits.add_(noise.mul_(0.4)).topk(k, -1).indices
        s.tokens = likely[prow, rank.cuda().clamp(max=k - 1)]
    # a greedy target: the same likely tokens, right now and then
    s.choice = None
    if case["mode"] == "match":
        other = torch.randint(0, V, (T,), generator=gen, device="cuda")
        hit = torch.rand(T, generator=gen, device="cuda") < 0.7
        s.choice = torch.where(hit, likely[:, min(1, k - 1)], other)
        s.target = None
    return s


def _prepare_commit(case, s, kept, gen, g):
    path = torch.full((case["seqs"], s.max_q), -1, dtype=torch.int32)
    for i, (n, m) in enumerate(zip(s.nodes, kept)):
        far = torch.randperm(n - 1 - m, generator=g)[:m].sort().values + m + 1
        stay = i % 4 == 3           # every fourth path is in its place already
        path[i, 0] = 0
        path[i, 1:m + 1] = torch.arange(1, m + 1) if stay else far
    s.path, s.kept = path.cuda(), _i32(kept)
    base = _between(1, 60, case["seqs"], torch.Generator().manual_seed(case["lengths"] + 1))
    ctx = [b + n for b, n in zip(base, s.nodes)]
    s.ctx_lens = _i32(ctx)
    s.block_table, blocks = _tables(ctx, g)
    shape = (case["layers"], blocks * BS, case["kv_heads"], case["dim"])
    s.key = torch.empty(shape, dtype=DTYPES[case["dtype"]], device="cuda").normal_(generator=gen)
    s.value = torch.empty_like(s.key).normal_(generator=gen)
    return s


# -------------------------------------------------------------------------------- the pass
def run(s):
    kind = s.case["kind"]
    if own:
        from dispec_amd.engine.hip_attn import paged_tree_attention
        from dispec_amd.engine.hip_verify import match_draft, verify_draft
        from dispec_amd.kv.paged_cache import commit_path
        if kind == "attend":
            return paged_tree_attention(s.q, s.key, s.value, s.block_table, s.cu_q, s.ctx_lens,
                                        s.mask, s.G, block_size=BS, max_q_len=s.max_q,
                                        max_ctx=s.max_ctx)
        if kind == "commit":
            commit_path(s.key, s.value, s.block_table, s.cu_q, s.ctx_lens, s.path, s.kept,
                        block_size=BS)
            return {"key": s.key, "value": s.value}
        if s.choice is not None:
            return tuple(match_draft(s.tokens, s.choice, s.cu_q, parents=s.parents,
                                     max_q_len=s.max_q))
        if s.draft is not None:
            return tuple(verify_draft(s.tokens, s.target, s.u, s.u_last, s.cu_q,
                                      draft_probs=s.draft, max_q_len=s.max_q))
        return tuple(verify_draft(s.tokens, s.target, s.u, s.u_last, s.cu_q, parents=s.parents,
                                  max_q_len=s.max_q))
    if kind == "attend":
        return _plain_attend(s)
    if kind == "verify":
        return _plain_verify(s)
    return _plain_commit(s)


def _slots(table, pos):
    """Pool slots of the positions pos (B, n)."""
    return torch.gather(table.long(), 1, pos // BS) * BS + pos % BS


def _plain_attend(s):
    B, (T, Hq, D), KVH, dev = len(s.nodes), s.q.shape, s.key.shape[1], s.q.device
    n, C = s.max_q, s.max_ctx
    cu, ctx = s.cu_q.long(), s.ctx_lens.long()
    base = ctx - (cu[1:] - cu[:-1])
    node = torch.arange(n, device=dev)
    row = (cu[:-1, None] + node).clamp(max=T - 1)                      # (B, n)
    key = torch.arange(C, device=dev)
    slots = _slots(s.block_table, key.expand(B, C))
    # (B, KVH, C, D) keys and values, (B, KVH, G n, D) queries
    k = s.key[slots].float().transpose(1, 2)
    v = s.value[slots].float().transpose(1, 2).contiguous()
    q = s.q[row].float().view(B, n, KVH, s.G, D).permute(0, 2, 3, 1, 4)
    q = q.reshape(B, KVH, s.G * n, D)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(D ** -0.5)
    # a node sees the context before the tree, and the nodes of its bits
    at = key - base[:, None]                                           # (B, C)
    word = (at.clamp(min=0) // 32).clamp(max=s.mask.shape[1] - 1)
    bits = torch.gather(s.mask[row], 2, word[:, None].expand(B, n, C))
    seen = (bits >> (at % 32)[:, None]) & 1 != 0
    seen = (seen | (at < 0)[:, None]) & (key < ctx[:, None])[:, None]  # (B, n, C)
    scores = scores.view(B, KVH, s.G, n, C).masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, KVH, s.G * n, C), v).view(B, KVH, s.G, n, D)
    o = o / total.masked_fill(total == 0, 1.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(B * n, Hq, D)
    seq = torch.repeat_interleave(torch.arange(B, device=dev), cu[1:] - cu[:-1], output_size=T)
    return o[seq * n + torch.arange(T, device=dev) - cu[seq]].to(s.q.dtype)


def _plain_verify(s):
    B, n, T, dev = len(s.nodes), s.max_q, s.T, s.tokens.device
    cu = s.cu_q.long()
    node = torch.arange(n, device=dev)
    row = (cu[:-1, None] + node).clamp(max=T - 1)
    drafted = (node < (cu[1:] - cu[:-1])[:, None]) & (node > 0)
    par = s.parents[row].long().clamp(min=0)
    prow, tok = cu[:-1, None] + par, s.tokens[row]
    prow = prow.clamp(max=T - 1)
    # earlier siblings, (B, i, j); a token that one of them has already counts no second time
    older = (par[:, :, None] == par[:, None, :]) & (node[:, None] > node) & drafted[:, None]
    again = (older & (tok[:, :, None] == tok[:, None, :])).any(-1)
    fresh = drafted & ~again
    first_q = cu[:-1] - torch.arange(B, device=dev)     # rows of the draft's probabilities
    if s.choice is not None:
        chosen = fresh & (tok == s.choice[prow])
    elif s.draft is not None:
        qrow = (first_q[:, None] + par).clamp(max=max(0, s.draft.shape[0] - 1))
        q = s.draft[qrow, tok].double() if s.draft.shape[0] else torch.zeros_like(tok).double()
        chosen = fresh & (s.u[prow].double() * q < s.target[prow, tok].double())
    else:
        p = s.target[prow, tok].double().masked_fill(~fresh, 0.0)
        before = torch.matmul(older.double(), p[:, :, None])[:, :, 0]
        u = s.u[prow].double()
        chosen = fresh & (u < before + p) & ~(u < before)
    # the kept path: nodes whose chosen edges lead up to the root
    up = (chosen[:, :, None] & (par[:, :, None] == node)).float() + torch.eye(n, device=dev)
    up = functools.reduce(lambda a, _: (torch.matmul(a, a) > 0).float(),
                          range(max(1, (n - 1).bit_length())), up)
    kept = (up[:, :, 0] > 0) & (drafted | (node == 0))
    num = kept.sum(1) - 1
    last = torch.where(kept, node, 0).amax(1)
    path = torch.where(kept, node, n).sort(1).values
    tokens = torch.gather(tok, 1, path.clamp(max=n - 1)).roll(-1, 1)
    end = (cu[:-1] + last).clamp(max=T - 1)
    if s.choice is not None:
        final = s.choice[end]
    else:
        whole = s.target[end].double()
        if s.draft is not None and s.draft.shape[0]:
            more = last + 1 < cu[1:] - cu[:-1]
            q = s.draft[(first_q + last).clamp(max=s.draft.shape[0] - 1)].double()
            rest = (whole - q * more[:, None]).clamp(min=0.0)
        else:
            child = drafted & (par == last[:, None])
            V = whole.shape[1]
            rest = torch.cat([whole, whole[:, :1]], 1)
            rest = rest.scatter(1, tok.masked_fill(~child, V), 0.0)[:, :V]
        none = (rest.sum(1) <= 0)[:, None]
        cum = torch.where(none, whole, rest).cumsum(1)
        final = (cum <= (s.u_last.double() * cum[:, -1])[:, None]).sum(1)
    tokens = torch.where(node < num[:, None], tokens,
                         torch.where(node == num[:, None], final[:, None], -1))
    return num.int(), path.masked_fill(path == n, -1).int(), tokens


def _plain_commit(s):
    n, cu = s.max_q, s.cu_q.long()
    base = (s.ctx_lens.long() - (cu[1:] - cu[:-1]))[:, None]
    node = torch.arange(n, device=s.key.device)
    # rows that stay: the root's, onto itself
    moves = (node > 0) & (node <= s.kept[:, None])
    dst = _slots(s.block_table, base + torch.where(moves, node, 0)).view(-1)
    src = _slots(s.block_table, base + torch.where(moves, s.path.long(), 0)).view(-1)
    s.key[:, dst] = s.key[:, src]
    s.value[:, dst] = s.value[:, src]
    return {"key": s.key, "value": s.value}


def work(case):
    nodes, second = _lengths(case)
    T, es = sum(nodes), 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "attend":
        Hq, KVH, D = case["heads"], case["kv_heads"], case["dim"]
        pairs = sum(n * (c - n) + n * (n + 1) / 2 for n, c in zip(nodes, second))
        return {"bytes": 2 * sum(second) * KVH * D * es + 2 * T * Hq * D * es +
                T * -(-max(nodes) // 32) * 4 + sum(second) / BS * 4, "flops": 4.0 * Hq * D * pairs}
    if case["kind"] == "commit":
        moved = sum(m for i, m in enumerate(second) if i % 4 != 3)
        row = case["kv_heads"] * case["dim"] * es
        return {"bytes": 2 * 2 * max(1, moved) * case["layers"] * row, "flops": 0}
    ints = T * 16 + len(nodes) * (4 + case["n_hi"] * 12)
    if case["mode"] == "match":
        return {"bytes": ints, "flops": 0}
    # one row of the target, and of the draft where there is one, for each sequence
    rows = 2 if case["mode"] == "sample" else 1
    return {"bytes": ints + len(nodes) * rows * case["vocab"] * es,
            "flops": 3.0 * len(nodes) * case["vocab"]}


# ------------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "verify": _exact_verify, "commit": _exact_commit}[
        case["kind"]](s)


def _exact_attend(s):
    f, at = torch.float64, 0
    out = torch.empty(s.q.shape, dtype=f, device="cuda")
    for b, (n, c) in enumerate(zip(s.nodes, s.ctx)):
        pos = torch.arange(c, device="cuda")
        slots = s.block_table[b].long()[pos // BS] * BS + pos % BS
        seen = torch.ones((n, c), dtype=torch.bool, device="cuda")
        for a in range(n):
            seen[:, c - n + a] = s.mask[at:at + n, a // 32] >> a % 32 & 1 != 0
        for h in range(s.key.shape[1]):
            k, v = s.key[slots, h].to(f), s.value[slots, h].to(f)
            for j in range(h * s.G, (h + 1) * s.G):
                x = s.q[at:at + n, j].to(f) @ k.t().contiguous() / math.sqrt(s.q.shape[2])
                out[at:at + n, j] = x.masked_fill(~seen, -math.inf).softmax(-1) @ v
        at += n
    return out


def _exact_verify(s):
    nums, paths, rows = [], [], []
    tokens, parents, u = s.tokens.tolist(), s.parents.tolist(), s.u.double().tolist()
    for b, n in enumerate(s.nodes):
        at = sum(s.nodes[:b])
        kids = {}
        for i in range(1, n):
            kids.setdefault(parents[at + i], []).append(i)
        path, out, tried = [0], [], []
        while True:
            here, tried = path[-1], []
            go = None
            total = 0.0
            for i in kids.get(here, []):
                x = tokens[at + i]
                if x in tried:
                    continue
                tried.append(x)
                if s.choice is not None:
                    ok = int(s.choice[at + here]) == x
                elif s.draft is not None:
                    ok = u[at + here] * float(s.draft[at - b + here, x]) < \
                        float(s.target[at + here, x])
                else:
                    total += float(s.target[at + here, x])
                    ok = u[at + here] < total
                if ok:
                    go = i
                    break
            if go is None:
                break
            path.append(go)
            out.append(tokens[at + go])
        here = path[-1]
        if s.choice is not None:
            out.append(int(s.choice[at + here]))
        else:
            p = s.target[at + here].double().cpu()
            rest = p.clone()
            if s.draft is not None:
                if here + 1 < n:
                    rest = (p - s.draft[at - b + here].double().cpu()).clamp(min=0)
            else:
                rest[tried] = 0
            if not rest.sum() > 0:
                rest = p
            cum = rest.cumsum(0)
            out.append(int(torch.searchsorted(cum, cum[-1] * s.u_last[b].double().cpu(),
                                              right=True)))
        nums.append(len(path) - 1)
        paths.append(path + [-1] * (s.max_q - len(path)))
        rows.append(out + [-1] * (s.max_q - len(out)))
    return (torch.tensor(nums, dtype=torch.int32), torch.tensor(paths, dtype=torch.int32),
            torch.tensor(rows))


def _exact_commit(s):
    key, value = s.key.double(), s.value.double()
    old_k, old_v = key.clone(), value.clone()
    for b, (n, c, m) in enumerate(zip(s.nodes, s.ctx_lens.tolist(), s.kept.tolist())):
        for j in range(1, m + 1):
            src, dst = (c - n + a for a in (int(s.path[b, j]), j))
            src, dst = (int(s.block_table[b, x // BS]) * BS + x % BS for x in (src, dst))
            key[:, dst] = old_k[:, src]
            value[:, dst] = old_v[:, src]
    return {"key": key, "value": value}
