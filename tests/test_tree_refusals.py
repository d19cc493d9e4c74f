"""Calls that the tree operators refuse, on the host."""

import pytest
import torch

from dispec_amd import _lib
from dispec_amd.engine import hip_attn, hip_verify
from dispec_amd.kv.paged_cache import commit_path


@pytest.fixture()
def on_cpu(monkeypatch):
    """The argument checks run before any launch: let them see CPU tensors."""
    monkeypatch.setattr(_lib, "require_gpu", lambda *t: None)

    def launched(*a):
        raise AssertionError("a refused call reached the library")

    class Calls:
        def __getattr__(self, name):
            return launched

    monkeypatch.setattr(_lib, "calls", lambda: Calls())


def _attn(**kw):
    T, Hq, KVH, D = 5, 4, 2, 64
    a = dict(q=torch.zeros(T, Hq, D, dtype=torch.bfloat16),
             k=torch.zeros(64, KVH, D, dtype=torch.bfloat16),
             v=torch.zeros(64, KVH, D, dtype=torch.bfloat16),
             bt=torch.zeros((2, 4), dtype=torch.int32), cu=torch.tensor([0, 2, 5], dtype=torch.int32),
             lens=torch.tensor([2, 5], dtype=torch.int32),
             mask=torch.zeros((T, 1), dtype=torch.int32), G=2, kw={})
    a.update(kw)
    return hip_attn.paged_tree_attention(a["q"], a["k"], a["v"], a["bt"], a["cu"], a["lens"],
                                         a["mask"], a["G"], **{"max_q_len": 3, **a["kw"]})


@pytest.mark.parametrize("kw,match", [
    (dict(q=torch.zeros(5, 4, dtype=torch.bfloat16)), "expected q"),
    (dict(G=3), "kv_groups"),
    (dict(k=torch.zeros(64, 2, 64)), "dtypes"),
    (dict(v=torch.zeros(64, 2, 64, dtype=torch.bfloat16).transpose(0, 1).contiguous()
          .transpose(0, 1)), "strides"),
    (dict(cu=torch.zeros(4, dtype=torch.int32)), "cu_q"),
    (dict(bt=torch.zeros((3, 4), dtype=torch.int32)), "block_table"),
    (dict(mask=torch.zeros((4, 1), dtype=torch.int32)), "tree_mask"),
    (dict(mask=torch.zeros((5, 1), dtype=torch.int64)), "tree_mask"),
    (dict(kw={"max_q_len": 33}), "tree_mask"),
    (dict(kw={"max_ctx": 65}), "max_ctx"),
    (dict(kw={"out": torch.zeros(5, 4, 64)}), "out must"),
])
def test_tree_attention(on_cpu, kw, match):
    with pytest.raises(ValueError, match=match):
        _attn(**kw)


def test_tree_mask(on_cpu):
    cu = torch.tensor([0, 2], dtype=torch.int32)
    for args, kw, match in (((None, cu, 2), {}, "num_tokens"),
                            ((torch.zeros((2, 1), dtype=torch.int32), cu, 2), {}, "parents"),
                            ((torch.zeros(2, dtype=torch.int32), cu, 2), {"num_tokens": 3}, "parents"),
                            ((None, torch.zeros(0, dtype=torch.int32), 2), {"num_tokens": 2}, "cu_q")):
        with pytest.raises(ValueError, match=match):
            hip_attn.tree_mask(*args, **kw)


def _verify(**kw):
    T, B, V = 6, 2, 10
    a = dict(tok=torch.zeros(T, dtype=torch.int64), p=torch.zeros(T, V), u=torch.zeros(T),
             ul=torch.zeros(B), cu=torch.tensor([0, 3, 6], dtype=torch.int32), kw={})
    a.update(kw)
    return hip_verify.verify_draft(a["tok"], a["p"], a["u"], a["ul"], a["cu"],
                                   **{"max_q_len": 3, **a["kw"]})


@pytest.mark.parametrize("kw,match", [
    (dict(tok=torch.zeros(6)), "draft_tokens"),
    (dict(tok=torch.zeros((6, 1), dtype=torch.int64)), "draft_tokens"),
    (dict(p=torch.zeros(5, 10)), "rows"),
    (dict(p=torch.zeros(6, 10, dtype=torch.float64)), "target_probs"),
    (dict(u=torch.zeros(5)), "uniforms"),
    (dict(u=torch.zeros(6, dtype=torch.float64)), "uniforms"),
    (dict(ul=torch.zeros(3)), "final_uniforms"),
    (dict(cu=torch.zeros((2, 2), dtype=torch.int32)), "cu_q"),
    (dict(kw={"parents": torch.zeros(5, dtype=torch.int32)}), "parents"),
    (dict(kw={"parents": torch.zeros(6, dtype=torch.int32), "draft_probs": torch.zeros(4, 10)}),
     "exclude"),
    (dict(kw={"draft_probs": torch.zeros(3, 10)}), "draft_probs"),
    (dict(kw={"draft_probs": torch.zeros(7, 10)}), "draft_probs"),
    (dict(kw={"draft_probs": torch.zeros(4, 9)}), "draft_probs"),
    (dict(kw={"draft_probs": torch.zeros(4, 10, dtype=torch.bfloat16)}), "draft_probs"),
])
def test_verify_draft(on_cpu, kw, match):
    with pytest.raises(ValueError, match=match):
        _verify(**kw)


def test_match_draft(on_cpu):
    cu = torch.tensor([0, 4], dtype=torch.int32)
    tok = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="target_tokens"):
        hip_verify.match_draft(tok, tok[:3], cu, max_q_len=4)
    with pytest.raises(ValueError, match="parents"):
        hip_verify.match_draft(tok, tok, cu, parents=torch.zeros(3, dtype=torch.int32), max_q_len=4)


def _commit(**kw):
    i32 = dict(dtype=torch.int32)
    a = dict(key=torch.zeros(2, 64, 2, 8), value=torch.zeros(2, 64, 2, 8),
             bt=torch.zeros((3, 4), **i32), cu=torch.zeros(4, **i32), lens=torch.zeros(3, **i32),
             path=torch.zeros((3, 5), **i32), num=torch.zeros(3, **i32))
    a.update(kw)
    commit_path(a["key"], a["value"], a["bt"], a["cu"], a["lens"], a["path"], a["num"])


@pytest.mark.parametrize("kw,match", [
    (dict(key=torch.zeros(64, 2, 8)), "pools"),
    (dict(value=torch.zeros(2, 64, 2, 8, dtype=torch.bfloat16)), "pools"),
    (dict(key=torch.zeros(2, 64, 8, 2).transpose(2, 3), value=torch.zeros(2, 64, 8, 2)
          .transpose(2, 3)), "contiguous rows"),
    (dict(cu=torch.zeros(3, dtype=torch.int32)), "sequences"),
    (dict(path=torch.zeros((2, 5), dtype=torch.int32)), "sequences"),
    (dict(num=torch.zeros(2, dtype=torch.int32)), "sequences"),
    (dict(path=torch.zeros((3, 5), dtype=torch.int64)), "int32"),
    (dict(lens=torch.zeros(3, dtype=torch.int64)), "int32"),
])
def test_commit_path(on_cpu, kw, match):
    with pytest.raises(ValueError, match=match):
        _commit(**kw)


def test_cpu_tensors_are_refused():
    z = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU only"):
        hip_attn.tree_mask(z, torch.zeros(2, dtype=torch.int32), 1)
    with pytest.raises(RuntimeError, match="GPU only"):
        _commit()
    with pytest.raises(RuntimeError, match="GPU only"):
        _verify()
    with pytest.raises(RuntimeError, match="GPU only"):
        _attn()


P = 0x1000   # any address: the calls below return before touching memory


def test_library_statuses():
    lib = _lib.lib()

    def tree(B=1, Hq=4, KVH=2, D=64, words=1, max_q=3, max_ctx=64, bs=16, dtype=_lib.DSP_BF16,
             q=P, ws=None, wsb=0, bt_stride=4):
        return lib.dsp_paged_tree_attention(q, 256, 64, P, P, 64, 128, 64, P, bt_stride, bs, P, P,
                                            P, words, B, Hq, KVH, D, 0.1, max_q, max_ctx, ws, wsb,
                                            P, 256, 64, dtype, None, None)

    assert tree(B=0) == tree(max_q=0) == _lib.DSP_OK
    for kw in (dict(B=-1), dict(Hq=3), dict(words=0), dict(max_q=33), dict(bs=12), dict(q=None),
               dict(bt_stride=3)):
        assert tree(**kw) == _lib.DSP_EINVAL, kw
    for kw in (dict(D=48), dict(D=512), dict(dtype=7)):
        assert tree(**kw) == _lib.DSP_EUNSUPPORTED, kw
    assert tree(q=P + 1) == _lib.DSP_EALIGN
    big = dict(B=2, max_q=64, words=2, max_ctx=1 << 16, bt_stride=1 << 12)
    assert lib.dsp_paged_tree_workspace_bytes(2, 4, 2, 64, 64, 1 << 16) > 0
    assert tree(**big) == _lib.DSP_EWORKSPACE
    assert lib.dsp_paged_tree_workspace_bytes(1, 3, 2, 64, 4, 64) == 0

    def verify(tok=P, parents=None, draft=None, B=1, max_q=4, V=100, dtype=_lib.DSP_F32, ws=P,
               wsb=1 << 20, target=P):
        return lib.dsp_verify_draft(tok, parents, target, 100, 4, draft, 100, 3, P, P, P, B, max_q,
                                    V, dtype, ws, wsb, P, P, P, None, None)

    assert verify(B=0) == verify(max_q=0) == _lib.DSP_OK
    for kw in (dict(tok=None), dict(parents=P, draft=P), dict(B=-1), dict(V=0), dict(B=65536)):
        assert verify(**kw) == _lib.DSP_EINVAL, kw
    for kw in (dict(dtype=9), dict(max_q=1025), dict(V=1 << 31)):
        assert verify(**kw) == _lib.DSP_EUNSUPPORTED, kw
    for kw in (dict(ws=None), dict(wsb=8)):
        assert verify(**kw) == _lib.DSP_EWORKSPACE, kw
    for kw in (dict(target=P + 2), dict(ws=P + 4)):
        assert verify(**kw) == _lib.DSP_EALIGN, kw
    assert lib.dsp_verify_workspace_bytes(0, 10) == 0 < lib.dsp_verify_workspace_bytes(1, 10)

    assert lib.dsp_match_draft(P, P, None, P, 4, 0, 4, P, P, P, None) == _lib.DSP_OK
    assert lib.dsp_match_draft(P, None, None, P, 4, 1, 4, P, P, P, None) == _lib.DSP_EINVAL
    assert lib.dsp_match_draft(P, P, None, P, 4, 1, 1025, P, P, P, None) == _lib.DSP_EUNSUPPORTED
    assert lib.dsp_tree_mask(P, P, 4, 1, 33, 1, P, None) == _lib.DSP_EINVAL
    assert lib.dsp_tree_mask(P, P, 4, 0, 32, 1, P, None) == _lib.DSP_OK

    def commit(k=P, layers=2, B=1, cols=4, bs=16):
        return lib.dsp_kv_commit_path(k, P, layers, 1 << 16, 256, 64, 256, bs, P, 4, 4, P, P, P, 4,
                                      cols, P, B, None, None)

    assert commit(B=0) == commit(layers=0) == commit(cols=1) == _lib.DSP_OK
    for kw in (dict(k=None), dict(layers=-1), dict(bs=3), dict(B=-1)):
        assert commit(**kw) == _lib.DSP_EINVAL, kw
    for kw in (dict(B=65536), dict(cols=1025)):
        assert commit(**kw) == _lib.DSP_EUNSUPPORTED, kw


def test_the_runner_s_batches_of_trees():
    """What SeqMeta.parents may hold, before anything reaches the GPU."""
    import types

    from dispec_amd.engine.model_runner import ModelRunner, SeqMeta
    from tests.toy_lm import toy_lm
    runner = ModelRunner(toy_lm("qwen3"), attn_backend="native")
    cache = types.SimpleNamespace(block_size=16, key=torch.zeros(1))
    meta = lambda n, parents: SeqMeta(list(range(100)), n, 600 + n, parents)  # noqa: E731
    assert not meta(4, None).is_tree() and not meta(4, [-1, 0, 1, 2]).is_tree()
    assert meta(4, [-1, 0, 0, 2]).is_tree()
    for bad in ([-1, 0, 0], [0, 0, 0, 0], [-1, 1, 0, 0], [-1, 0, -1, 0], [-1, 0, 4, 0], []):
        with pytest.raises(ValueError, match="parents"):
            runner._batch([meta(4, bad)], cache)
    with pytest.raises(ValueError, match="1024 a sequence"):
        runner._batch([meta(4, [-1, 0, 0, 2]), SeqMeta(list(range(100)), 1025, 1025)], cache)
    got = runner._batch([meta(4, [-1, 0, 0, 2]), meta(1, None), meta(3, None)], cache)
    assert got.tree_mask is None and not got.shared_prefix and not got.balanced  # (native: on host)
    assert got.cu_q.tolist() == [0, 4, 5, 8] and got.max_q_len == 4


def test_native_attention_of_a_tree():
    """attn_backend="native": a node's output is that of its path run as a chain."""
    import types

    from dispec_amd.engine.model_runner import ModelRunner, SeqMeta
    from tests.toy_lm import toy_lm
    runner = ModelRunner(toy_lm("qwen3"), attn_backend="native")
    g = torch.Generator().manual_seed(1)
    parents, base = [-1, 0, 0, 1, 1, 2], 9
    n = len(parents)
    k, v = (torch.randn(base + n, 2, 64, generator=g) for _ in range(2))
    q = torch.randn(n, 4, 64, generator=g)
    rows = types.SimpleNamespace(context_slots=lambda ids, c: c, gather=lambda i, c: (k[:c], v[:c]))
    got = runner._torch_attention(q, rows, 0, (SeqMeta([0], n, base + n, parents),))
    for i in range(n):
        path = [i]
        while parents[path[0]] >= 0:
            path.insert(0, parents[path[0]])
        keys = list(range(base)) + [base + j for j in path]
        one = types.SimpleNamespace(context_slots=lambda ids, c: c,
                                    gather=lambda i, c: (k[keys], v[keys]))
        want = runner._torch_attention(q[path], one, 0, (SeqMeta([0], len(path), len(keys)),))
        torch.testing.assert_close(got[i], want[-1], rtol=1e-5, atol=1e-5)
