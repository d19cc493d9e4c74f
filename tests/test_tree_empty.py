"""Batches of drafted trees without a node, on the host: nothing is launched, and what a caller reads
is what the formulas give."""

import pytest
import torch

from dispec_amd import _lib
from dispec_amd.engine import hip_attn, hip_verify
from dispec_amd.kv.paged_cache import commit_path

I32, I64 = torch.int32, torch.int64


@pytest.fixture()
def no_launch(monkeypatch):
    monkeypatch.setattr(_lib, "require_gpu", lambda *t: None)

    def launched(*a):
        raise AssertionError("a batch without nodes reached the library")

    class Calls:
        def __getattr__(self, name):
            return launched

    monkeypatch.setattr(_lib, "calls", lambda: Calls())


@pytest.mark.parametrize("T,B,bound", [(T, B, bound) for T in (0, 4) for B in (0, 3)
                                       for bound in (None, 0, 5) if not (T and B and bound)])
def test_verdicts(no_launch, T, B, bound):
    """All sequences empty; T rows behind them (a padded batch)."""
    cu, tok = torch.zeros(B + 1, dtype=I32), torch.zeros(T, dtype=I64)
    p, u, last = torch.full((T, 7), 1 / 7), torch.zeros(T), torch.zeros(B)
    for got in (hip_verify.verify_draft(tok, p, u, last, cu, max_q_len=bound),
                hip_verify.verify_draft(tok, p, u, last, cu, max_q_len=bound, draft_probs=p),
                hip_verify.match_draft(tok, tok, cu, max_q_len=bound)):
        width = bound or 0
        assert torch.equal(got.num_accepted, torch.zeros(B, dtype=I32))
        assert torch.equal(got.path, torch.full((B, width), -1, dtype=I32))
        assert torch.equal(got.tokens, torch.full((B, width), -1, dtype=I64))


@pytest.mark.parametrize("B,width", [(0, 4), (0, 0), (3, 0), (3, 1)])
def test_commits(no_launch, B, width):
    """No sequence, or verdicts without a kept node."""
    pool = torch.zeros(2, 64, 2, 8)
    commit_path(pool, pool.clone(), torch.zeros((B, 4), dtype=I32), torch.zeros(B + 1, dtype=I32),
                torch.zeros(B, dtype=I32), torch.zeros((B, width), dtype=I32),
                torch.zeros(B, dtype=I32))


@pytest.mark.parametrize("B", [0, 3])
def test_masks(no_launch, B):
    cu = torch.zeros(B + 1, dtype=I32)
    for kw in (dict(num_tokens=0), dict(num_tokens=0, max_q_len=40)):
        mask = hip_attn.tree_mask(None, cu, **kw)
        assert mask.shape == (0, 2 if kw.get("max_q_len") else 1) and mask.dtype == I32
    assert hip_attn.tree_mask(torch.zeros(0, dtype=I32), cu).shape == (0, 1)


@pytest.mark.parametrize("T,B", [(0, 0), (0, 3), (4, 0), (4, 3)])
def test_attention(no_launch, T, B):
    """Rows behind the last sequence stay as they are."""
    q, kv = torch.zeros(T, 4, 64), torch.zeros(64, 2, 64)
    out = torch.full_like(q, 3.0)
    hip_attn.paged_tree_attention(q, kv, kv, torch.zeros((B, 4), dtype=I32),
                                  torch.zeros(B + 1, dtype=I32), torch.zeros(B, dtype=I32),
                                  torch.zeros((T, 1), dtype=I32), 2, out=out)
    assert bool((out == 3).all())
