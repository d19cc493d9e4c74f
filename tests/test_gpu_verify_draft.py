"""verify_draft and match_draft against the rules written out for one sequence at a time, with exact
sums (fractions) where the numbers allow it and float64 ones elsewhere."""

import random
from fractions import Fraction

import numpy as np
import pytest
import torch

from tests._tree import random_parents
from tests._util import gen

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _draw(r, whole, u):
    """The least v with r_0 + .. + r_v > u S; from `whole` where r is zero; -1 where that is too."""
    for row in (r, whole):
        row = np.where(row > 0, row, 0.0)
        cum = np.cumsum(row)
        if cum[-1] > 0:
            if not np.isfinite(cum[-1]):
                return -1
            at = int(np.searchsorted(cum, u * cum[-1], side="right"))
            return at if at < len(row) else int(np.nonzero(row)[0][-1])
    return -1


def _one(tokens, parents, p, q, u, u_last, width):
    """(num, path, tokens) of one sequence; p, q: float64 rows; u: float64."""
    n, V = len(tokens), p.shape[1]
    if not n:
        return 0, [-1] * width, [-1] * width
    path, out = [0], []
    while True:
        here = path[-1]
        kids = [i for i in range(here + 1, n) if parents[i] == here]
        go, held, total = None, [], Fraction(0)
        for i in kids:
            x = int(tokens[i])
            if not 0 <= x < V or x in held:
                continue
            held.append(x)
            if q is not None:
                ok = Fraction(u[here]) * Fraction(q[here, x]) < Fraction(p[here, x])
            else:
                total += Fraction(p[here, x]) if p[here, x] > 0 else 0
                ok = p[here, x] > 0 and Fraction(u[here]) < total
            if ok:
                go = i
                break
        if go is None:
            break
        path.append(go)
        out.append(int(tokens[go]))
    here = path[-1]
    rest = p[here].copy()
    if q is not None:
        if here + 1 < n:
            with np.errstate(invalid="ignore"):
                rest = rest - q[here]
    else:
        rest[[x for x in held]] = 0.0
    out.append(_draw(rest, p[here], u_last))
    return (len(path) - 1, path + [-1] * (width - len(path)), out + [-1] * (width - len(out)))


class Draft:
    def __init__(self, q_lens, V, dtype, seed, chain, kind="tree", peak=3.0):
        rng = random.Random(seed)
        g = gen(seed)
        self.q_lens, self.T, self.width, self.V = q_lens, sum(q_lens), max(q_lens + [1]), V
        self.chain = chain
        self.parents = [random_parents(n, rng, "chain" if chain else kind) for n in q_lens]
        logits = torch.randn((self.T, V), generator=g) * peak
        self.p = logits.softmax(-1).to(dtype)
        self.q = None
        self.tokens = torch.randint(0, V, (self.T,), generator=g)
        at = 0
        if chain:
            rows = [at + i for at, n in zip(np.cumsum([0] + q_lens), q_lens) for i in range(n - 1)]
            self.q = (logits + 0.5 * torch.randn((self.T, V), generator=g)).softmax(-1)[rows].to(dtype)
        else:
            for n, par in zip(q_lens, self.parents):      # children: likely tokens of their parent
                for i in range(1, n):
                    if par[i] >= 0 and rng.random() < 0.9:
                        top = logits[at + par[i]].topk(min(V, 4)).indices
                        self.tokens[at + i] = top[rng.randrange(len(top))]
                at += n
        if chain:
            first = 0
            for n in q_lens:
                for i in range(1, n):
                    self.tokens[at + i] = torch.multinomial(self.q[first + i - 1].float(), 1,
                                                            generator=g)[0]
                at += n
                first += max(0, n - 1)
        self.u = torch.rand(self.T, generator=g)
        self.u_last = torch.rand(len(q_lens), generator=g)
        self.cu = torch.tensor(np.concatenate([[0], np.cumsum(q_lens)]), dtype=torch.int32)

    def call(self, **kw):
        from dispec_amd.engine.hip_verify import verify_draft
        par = torch.tensor([x for t in self.parents for x in t], dtype=torch.int32)
        args = dict(parents=None if self.chain else par.to(DEV),
                    draft_probs=self.q.to(DEV) if self.chain else None, max_q_len=self.width)
        args.update(kw)
        return verify_draft(self.tokens.to(DEV), self.p.to(DEV), self.u.to(DEV),
                            self.u_last.to(DEV), self.cu.to(DEV), **args)

    def reference(self):
        rows, at, first = [], 0, 0
        p, u, ul = self.p.double().numpy(), self.u.double().numpy(), self.u_last.double().numpy()
        q = None if self.q is None else self.q.double().numpy()
        for b, n in enumerate(self.q_lens):
            rows.append(_one(self.tokens[at:at + n], self.parents[b], p[at:at + n],
                             None if q is None else q[first:first + max(0, n - 1)],
                             u[at:at + n], ul[b], self.width))
            at += n
            first += max(0, n - 1)
        return rows

    def check(self, got=None):
        got = self.call() if got is None else got
        num, path, tok = (t.cpu().tolist() for t in got)
        for b, (n, ps, ts) in enumerate(self.reference()):
            assert num[b] == n and path[b] == ps and tok[b] == ts, (b, num[b], n, path[b], ps, tok[b], ts)
        assert got[0].dtype == got[1].dtype == torch.int32 and got[2].dtype == torch.int64


LENGTHS = [[1], [6], [1, 9, 0, 4, 2], [0, 0, 3], [64, 65, 3], [130, 1, 64]]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1, 7, 1000, 4096, 8193, 50257])
@pytest.mark.parametrize("q_lens", LENGTHS)
@pytest.mark.parametrize("chain", [True, False])
def test_verdicts(hip, dtype, V, q_lens, chain):
    if V > 8193 and sum(q_lens) > 100:
        q_lens = q_lens[1:]
    for seed in range(3):
        Draft(q_lens, V, dtype, seed + V, chain).check()


@pytest.mark.parametrize("kind", ["chain", "star"])
@pytest.mark.parametrize("peak", [0.5, 3.0])
def test_proposed_chains_and_many_children(hip, kind, peak):
    d = Draft([70, 3, 200], 40, torch.float32, 5, False, kind=kind, peak=peak)
    d.check()
    if kind == "chain":
        d.check(d.call(parents=None))


def test_wide_vocabulary(hip):
    """More slices than the threads that add them up."""
    V = 4096 * 300 + 17
    for chain in (True, False):
        Draft([3, 2], V, torch.float32, 9, chain, peak=0.1).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("chain", [True, False])
@pytest.mark.parametrize("V", [33, 4099])
def test_rows_at_any_stride(hip, dtype, chain, V):
    d = Draft([4, 7], V, dtype, 3, chain)
    want = d.call()
    wide = torch.full((d.T, V + 5), float("nan"), dtype=dtype, device=DEV)[:, 3:3 + V]
    wide.copy_(d.p)
    from dispec_amd.engine.hip_verify import verify_draft
    par = torch.tensor([x for t in d.parents for x in t], dtype=torch.int32, device=DEV)
    got = verify_draft(d.tokens.to(DEV).int(), wide, d.u.to(DEV), d.u_last.to(DEV), d.cu.to(DEV),
                       parents=None if chain else par,
                       draft_probs=d.q.to(DEV) if chain else None)   # max_q_len from cu_q
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    d.check(got)


def test_borders(hip):
    """u on a border: sums of powers of two are exact in any order, so the rule's strictness shows.
    p = 1/4 each: u = 1/2 passes two tokens, draws the third; u = 0 keeps what has any weight."""
    p = torch.full((8, 4), 0.25)
    p[4:] = torch.tensor([0.0, 0.5, 0.0, 0.5])
    d = Draft([1] * 8, 4, torch.float32, 0, False)
    d.p, d.u_last = p, torch.tensor([0.0, 0.25, 0.5, 0.75, 0.0, 0.5, 0.25, 1 - 2.0 ** -24])
    d.check()
    assert d.call().tokens[:, 0].tolist() == [0, 1, 2, 3, 1, 3, 1, 3]
    # a child of p 1/2 is kept below 1/2, not at it
    d = Draft([2, 2, 3], 4, torch.float32, 0, False)
    d.parents = [[-1, 0], [-1, 0], [-1, 0, 0]]
    d.p = torch.tensor([0.5, 0.25, 0.25, 0.0]).repeat(7, 1)
    d.tokens = torch.tensor([0, 0, 0, 0, 0, 1, 0])
    d.u = torch.tensor([0.5 - 2.0 ** -25, 0, 0.5, 0, 0.5, 0, 0])
    d.check()
    assert d.call().num_accepted.tolist() == [1, 0, 1]
    # a chain: kept where u q < p, not where they are equal
    d = Draft([2, 2, 2], 4, torch.float32, 0, True)
    d.p = torch.tensor([0.25, 0.75, 0.0, 0.0]).repeat(6, 1)
    d.q = torch.tensor([0.5, 0.5, 0.0, 0.0]).repeat(3, 1)
    d.tokens = torch.zeros(6, dtype=torch.long)
    d.u = torch.tensor([0.5, 0, 0.5 - 2.0 ** -25, 0, 0.0, 0])
    d.check()
    assert d.call().num_accepted.tolist() == [0, 1, 1]
    assert d.call().tokens[0].tolist() == [1, -1]


def test_nothing_left_over(hip):
    """p <= q throughout (rows that do not add up to the same), or children that hold all of p: the
    token comes from p."""
    d = Draft([2], 5, torch.float32, 0, True)
    d.p = torch.tensor([[0.25, 0.5, 0.125, 0.0, 0.0], [0.2] * 5])
    d.q = torch.tensor([[0.5, 0.5, 0.25, 0.0, 0.0]])
    d.tokens = torch.tensor([0, 0])
    d.u = torch.tensor([0.75, 0.0])
    for u in (0.0, 0.3, 0.9):
        d.u_last = torch.tensor([u])
        d.check()
    d = Draft([3], 4, torch.float32, 0, False)
    d.parents = [[-1, 0, 0]]
    d.p = torch.tensor([0.5, 0.25, 0.0, 0.0]).repeat(3, 1)
    d.tokens = torch.tensor([9, 0, 1])
    d.u = torch.tensor([0.75, 0.0, 0.0])
    d.u_last = torch.tensor([0.7])
    d.check()
    assert d.call().tokens.tolist() == [[1, -1, -1]]


@pytest.mark.parametrize("V", [20, 5000])
@pytest.mark.parametrize("chain", [True, False])
def test_odd_values(hip, V, chain):
    """NaN and negative entries are never drawn; a row of zeros, or with an infinity, gives no token
    and is counted; tokens outside the vocabulary are never kept, and counted once each."""
    d = Draft([1, 1, 3, 1], V, torch.float32, 1, chain)
    d.p[0, ::2] = float("nan")
    d.p[1] = 0.0
    d.p[2, 5], d.p[2, 6] = -1.0, float("nan")
    d.p[5, 7] = float("inf")
    d.tokens[3], d.tokens[4] = V, -1
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = d.call(err=err)
    d.check(got)
    assert int(err) == 4 and got.tokens[1, 0] == got.tokens[3, 0] == -1
    assert got.num_accepted.tolist() == [0, 0, 0, 0] and 0 <= int(got.tokens[2, 0]) < V
    d.u_last[:] = 1.0                                      # outside [0, 1): the last that has weight
    got = d.call()
    assert all(t < V for t in got.tokens[:, 0].tolist())


def test_bad_parents_and_short_rows(hip):
    """A node whose parent is not an earlier one is never reached; nodes past max_q_len or past the
    rows do not count."""
    d = Draft([5], 6, torch.float32, 2, False)
    d.parents = [[-1, 4, 2, -7, 0]]
    d.p = torch.full((5, 6), 1 / 8.0)
    d.p[:, 3] = 3 / 8.0
    d.tokens = torch.tensor([0, 3, 3, 3, 3])
    d.u[:] = 0.1
    d.check()
    assert d.call().path.tolist() == [[0, 4, -1, -1, -1]]
    got = d.call(max_q_len=3)
    assert got.num_accepted.tolist() == [0] and got.path.tolist() == [[0, -1, -1]]
    d.cu = torch.tensor([0, 900], dtype=torch.int32)       # more rows than there are
    assert d.call(max_q_len=5).path.tolist() == [[0, 4, -1, -1, -1]]


@pytest.mark.parametrize("chain", [True, False])
def test_tokens_follow_the_target(hip, chain):
    """Whatever the draft proposes, the first token after the root is distributed as p: its shares
    over 2^18 draws lie within 6 standard deviations, sqrt(p (1 - p) / N)."""
    from dispec_amd.engine.hip_verify import verify_draft
    N, V, B = 1 << 18, 6, 1 << 14
    g = torch.Generator(device=DEV).manual_seed(3)
    p = torch.tensor([0.05, 0.3, 0.1, 0.15, 0.2, 0.2], device=DEV)
    q = torch.tensor([0.3, 0.1, 0.2, 0.1, 0.05, 0.25], device=DEV)
    seen = torch.zeros(V, device=DEV, dtype=torch.float64)
    n = 2 if chain else 4
    cu = torch.arange(B + 1, dtype=torch.int32, device=DEV) * n
    par = torch.tensor([-1, 0, 0, 0] * B, dtype=torch.int32, device=DEV)
    for _ in range(N // B):
        draft = torch.multinomial(q, B * n, replacement=True, generator=g)
        if not chain:
            draft = torch.tensor([0, 1, 4, 1], device=DEV).repeat(B)   # (one of them twice)
        got = verify_draft(draft, p.expand(B * n, V).contiguous(),
                           torch.rand(B * n, generator=g, device=DEV),
                           torch.rand(B, generator=g, device=DEV), cu,
                           parents=None if chain else par,
                           draft_probs=q.expand(B, V).contiguous() if chain else None, max_q_len=n)
        seen += torch.bincount(got.tokens[:, 0], minlength=V)
    share, pd = seen / N, p.double()
    assert float(((share - pd).abs() / (pd * (1 - pd) / N).sqrt()).max()) < 6


@pytest.mark.parametrize("kind", ["tree", "chain", "star"])
@pytest.mark.parametrize("q_lens", LENGTHS + [[1024]])
def test_match(hip, q_lens, kind):
    from dispec_amd.engine.hip_verify import match_draft
    rng = random.Random(len(q_lens))
    par = [random_parents(n, rng, kind) for n in q_lens]
    flat = [x for t in par for x in t]
    V = 3
    tok = [rng.randrange(V) for _ in flat]
    want = [rng.randrange(V) for _ in flat]
    cu = np.concatenate([[0], np.cumsum(q_lens)])
    width = max(q_lens)
    got = match_draft(torch.tensor(tok, device=DEV), torch.tensor(want, dtype=torch.int32, device=DEV),
                      torch.tensor(cu, dtype=torch.int32, device=DEV),
                      parents=None if kind == "chain" else
                      torch.tensor(flat, dtype=torch.int32, device=DEV), max_q_len=width)
    for b, n in enumerate(q_lens):
        at = int(cu[b])
        path = [0] if n else []
        while n:
            nxt = [i for i in range(path[-1] + 1, n)
                   if par[b][i] == path[-1] and tok[at + i] == want[at + path[-1]]]
            if not nxt:
                break
            path.append(nxt[0])
        assert int(got.num_accepted[b]) == max(0, len(path) - 1)
        assert got.path[b].tolist() == path + [-1] * (width - len(path))
        assert got.tokens[b].tolist() == [want[at + i] for i in path] + [-1] * (width - len(path))


def test_streams_graphs_and_repeats(hip):
    """The same verdict on another stream, twice, and replayed from a graph with other inputs."""
    a = Draft([6, 1, 20], 9000, torch.float32, 4, False)
    b = Draft([6, 1, 20], 9000, torch.float32, 5, False)
    want = [x.call() for x in (a, b)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = a.call()
    side.synchronize()
    for x, y in zip(got, want[0]):
        assert torch.equal(x, y)
    from dispec_amd.engine.hip_verify import match_draft, verify_draft
    par = [torch.tensor([x for t in d.parents for x in t], dtype=torch.int32, device=DEV)
           for d in (a, b)]
    st = [t.to(DEV) for t in (a.tokens, a.p, a.u, a.u_last, a.cu)] + [par[0].clone()]
    verify_draft(*st[:5], parents=st[5], max_q_len=20)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = verify_draft(*st[:5], parents=st[5], max_q_len=20)
        m = match_draft(st[0], st[0], st[4], parents=st[5], max_q_len=20)
    for i in (1, 0, 1, 0):
        d = (a, b)[i]
        for t, x in zip(st, (d.tokens, d.p, d.u, d.u_last, d.cu, par[i])):
            t.copy_(x)
        eager = verify_draft(*st[:5], parents=st[5], max_q_len=20)
        graph.replay()
        torch.cuda.synchronize()
        for x, y, z in zip(out, want[i], eager):
            assert torch.equal(x, y) and torch.equal(x, z)
        assert torch.equal(m.path, match_draft(st[0], st[0], st[4], parents=st[5], max_q_len=20).path)
