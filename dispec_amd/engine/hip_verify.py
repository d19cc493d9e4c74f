"""The verdict on drafted tokens, on the device.

The reference samples with `rejection_sample(draft_tokens, draft_probs, target_probs)`
(dispec/spec/rejection.py:25-54): one chain, its loop on the host.  `verify_draft` decides a batch
of chains (with the draft's probabilities) or trees (proposed tokens) from given random numbers,
`match_draft` one whose target tokens are known; both return device tensors that
`PagedKVCache.commit_path` takes as they are, so nothing waits for the host between the forward
and the commit.
"""

from __future__ import annotations

import functools
from typing import NamedTuple

import torch

from dispec_amd import _lib

MAX_TREE_NODES = 1024   # of one sequence, its root included
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_INTS = (torch.int64, torch.int32)


class DraftVerdict(NamedTuple):
    """What the target keeps of each sequence's draft."""

    num_accepted: torch.Tensor   # (B,) int32: kept nodes besides the root
    path: torch.Tensor           # (B, max_q_len) int32: the kept nodes, the root (0) first; then -1
    tokens: torch.Tensor         # (B, max_q_len) int64: the kept tokens, the token after them; -1


@functools.lru_cache(maxsize=256)
def _ws_bytes(B, V) -> int:
    return _lib.lib().dsp_verify_workspace_bytes(B, V)


def _as(t, dtype):
    return t if t.dtype == dtype and t.is_contiguous() else t.to(dtype).contiguous()


def _ints(t, name, n):
    if t.shape != (n,) or t.dtype not in _INTS:
        raise ValueError(f"{name} must be ({n},) int32 or int64; got {tuple(t.shape)} {t.dtype}")
    return _as(t, torch.int64)


def _layout(draft_tokens, cu_q, parents, max_q_len):
    """(tokens int64, cu_q int32, parents int32 or None, T, B, max_q_len) of a draft."""
    T, B = draft_tokens.numel(), cu_q.numel() - 1
    if draft_tokens.dim() != 1:
        raise ValueError(f"draft_tokens has shape {tuple(draft_tokens.shape)}: expected (T,)")
    if cu_q.dim() != 1 or B < 0:
        raise ValueError(f"cu_q has shape {tuple(cu_q.shape)}: expected (B + 1,)")
    if parents is not None and parents.shape != (T,):
        raise ValueError(f"parents has shape {tuple(parents.shape)} for {T} nodes")
    cu_q = _as(cu_q, torch.int32)
    if max_q_len is None:
        max_q_len = int((cu_q[1:] - cu_q[:-1]).max().item()) if B else 0
    return (_ints(draft_tokens, "draft_tokens", T), cu_q,
            None if parents is None else _as(parents, torch.int32), T, B, int(max_q_len))


def _outputs(B, width, like):
    empty = like.new_empty   # (of the allocations a call makes the cheapest form)
    return DraftVerdict(empty(B, dtype=torch.int32), empty((B, width), dtype=torch.int32),
                        empty((B, width), dtype=torch.int64))


def verify_draft(draft_tokens, target_probs, uniforms, final_uniforms, cu_q, parents=None,
                 draft_probs=None, max_q_len=None, err=None):
    """Which path of each sequence's draft the target keeps, and the token after it.

    The T rows are those of the target's forward: node 0 of a sequence is the last token that was
    kept, the others are drafted tokens, each after its parent; row i of target_probs is the
    target's distribution p_i of the token after node i.

    With `draft_probs` the drafts are chains whose tokens were drawn from them (rejection
    sampling): the token x after node i is kept where u_i q_i(x) < p_i(x); where one is not, the
    next token is drawn from max(p_i - q_i, 0).  Without, they are trees of proposed tokens: of
    node i's children, in order, the first is kept with u_i < the sum of the p_i of the children so
    far; where none is, the next token is drawn from p_i without their tokens.  Both leave the
    target's distribution as it is.  Sums and comparisons are in 64 bits; the same inputs give the
    same tokens.

    draft_tokens:   (T,) int32 / int64 (a root's is not read)
    target_probs:   (T, V) bf16, fp16 or fp32, rows at any stride
    uniforms:       (T,) fp32 in [0, 1), final_uniforms: (B,) fp32 in [0, 1)
    cu_q:           (B+1,) int32 node offsets
    parents:        (T,) int32 parent of each node within its sequence (None: chains)
    draft_probs:    (T - B, V) like target_probs: q_0 .. q_{n-2} of each chain, packed (an empty
                    sequence has no row); with rows behind the last sequence, or empty ones,
                    T - B to T rows, of which those behind the last chain's are not read
    max_q_len:      bound of the nodes of a sequence, at most 1024 (computed from cu_q if omitted,
                    which costs a device->host copy)
    err:            optional int32 device counter of drafted tokens outside the vocabulary and of
                    rows without a positive, finite sum (whose token is -1)
    returns:        DraftVerdict
    """
    _lib.one_gpu(target_probs, draft_tokens, uniforms, final_uniforms, cu_q, parents, draft_probs,
                 err)
    if parents is not None and draft_probs is not None:
        raise ValueError("draft_probs are a chain's: parents and draft_probs exclude each other")
    tokens, cu_q, parents, T, B, max_q_len = _layout(draft_tokens, cu_q, parents, max_q_len)
    dtype, shape = target_probs.dtype, target_probs.shape
    if dtype not in _DTYPES or len(shape) != 2:
        raise ValueError(f"target_probs must be (T, V) bf16, fp16 or fp32; got {tuple(shape)} {dtype}")
    rows, V = shape
    if rows != T:
        raise ValueError(f"target_probs has {rows} rows for {T} nodes")
    stride, last = target_probs.stride()
    if last != 1 and V > 1:
        target_probs, stride = target_probs.contiguous(), V
    draft_stride = draft_rows = 0
    if draft_probs is not None:
        shape = draft_probs.shape
        if len(shape) != 2 or shape[1] != V or draft_probs.dtype != dtype:
            raise ValueError(f"draft_probs must be (rows, {V}) of {dtype}; got {tuple(shape)} "
                             f"{draft_probs.dtype}")
        draft_rows = shape[0]
        if not max(0, T - B) <= draft_rows <= T:
            raise ValueError(f"draft_probs has {draft_rows} rows for {T} nodes of {B} chains: one "
                             "for each drafted token")
        draft_stride, last = draft_probs.stride()
        if last != 1 and V > 1:
            draft_probs, draft_stride = draft_probs.contiguous(), V
    for t, name, n in ((uniforms, "uniforms", T), (final_uniforms, "final_uniforms", B)):
        if t.shape != (n,) or t.dtype != torch.float32:
            raise ValueError(f"{name} must be ({n},) float32; got {tuple(t.shape)} {t.dtype}")
    uniforms, final_uniforms = uniforms.contiguous(), final_uniforms.contiguous()
    got = _outputs(B, max_q_len, target_probs)
    if not (T and B and max_q_len):   # no node at all (T: rows behind the last sequence)
        return DraftVerdict(got[0].zero_(), got[1].fill_(-1), got[2].fill_(-1))
    need = _ws_bytes(B, V)
    ws = target_probs.new_empty(need, dtype=torch.uint8)
    with _lib.on_device(target_probs):
        _lib.check(_lib.calls().dsp_verify_draft(
            tokens.data_ptr(), _lib.ptr(parents), target_probs.data_ptr(), stride, T,
            _lib.ptr(draft_probs), draft_stride, draft_rows, uniforms.data_ptr(),
            final_uniforms.data_ptr(), cu_q.data_ptr(), B, max_q_len, V, _lib.dtype_code(dtype),
            ws.data_ptr(), need, got[0].data_ptr(), got[1].data_ptr(), got[2].data_ptr(),
            _lib.ptr(err), _lib.stream_of(target_probs)), "dsp_verify_draft")
    return got


def match_draft(draft_tokens, target_tokens, cu_q, parents=None, max_q_len=None):
    """`verify_draft` where the target's token after each node is known (greedy decoding, or
    sampled already): a drafted token is kept where it is the target's after its parent, the first
    of several; the token after the path is the target's.

    draft_tokens, target_tokens: (T,) int32 / int64; cu_q, parents, max_q_len: as there
    """
    _lib.one_gpu(draft_tokens, target_tokens, cu_q, parents)
    tokens, cu_q, parents, T, B, max_q_len = _layout(draft_tokens, cu_q, parents, max_q_len)
    target_tokens = _ints(target_tokens, "target_tokens", T)
    got = _outputs(B, max_q_len, tokens)
    if not (T and B and max_q_len):   # no node at all (T: rows behind the last sequence)
        return DraftVerdict(got[0].zero_(), got[1].fill_(-1), got[2].fill_(-1))
    with _lib.on_device(tokens):
        _lib.check(_lib.calls().dsp_match_draft(
            tokens.data_ptr(), target_tokens.data_ptr(), _lib.ptr(parents), cu_q.data_ptr(), T, B,
            max_q_len, got[0].data_ptr(), got[1].data_ptr(), got[2].data_ptr(),
            _lib.stream_of(tokens)), "dsp_match_draft")
    return got
