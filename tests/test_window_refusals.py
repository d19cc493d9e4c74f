"""Calls that the windowed attention and the quantised cache refuse, on the host."""

import pytest
import torch

from dispec_amd import _lib
from dispec_amd.engine import hip_attn
from dispec_amd.kv import quant_cache


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
    monkeypatch.setattr(hip_attn, "_window_ws_bytes", lambda *a: 0)


T, HQ, KVH, D, S = 5, 4, 2, 64, 64
BF16 = torch.bfloat16
U8 = torch.uint8


def _window(**kw):
    a = dict(q=torch.zeros(T, HQ, D, dtype=BF16), k=torch.zeros(S, KVH, D, dtype=BF16),
             v=torch.zeros(S, KVH, D, dtype=BF16), bt=torch.zeros((2, 4), dtype=torch.int32),
             cu=torch.tensor([0, 2, 5], dtype=torch.int32),
             lens=torch.tensor([2, 5], dtype=torch.int32), G=2, kw={})
    a.update(kw)
    return hip_attn.paged_window_attention(a["q"], a["k"], a["v"], a["bt"], a["cu"], a["lens"], a["G"],
                                           **{"window": 8, "max_q_len": 3, **a["kw"]})


@pytest.mark.parametrize("kw,match", [
    (dict(q=torch.zeros(5, 4, dtype=BF16)), "expected q"),
    (dict(G=3), "kv_groups"),
    (dict(k=torch.zeros(64, 2, 64)), "dtypes"),
    (dict(q=torch.zeros(T, HQ, 32, dtype=BF16)), "width"),
    (dict(v=torch.zeros(64, 2, 64, dtype=BF16).transpose(0, 1).contiguous().transpose(0, 1)),
     "strides"),
    (dict(cu=torch.zeros(4, dtype=torch.int32)), "cu_q"),
    (dict(cu=None), "without cu_q"),
    (dict(bt=torch.zeros((3, 4), dtype=torch.int32)), "block_table"),
    (dict(kw={"window": -1}), "window"),
    (dict(kw={"window": 0, "sinks": 4}), "window"),
    (dict(kw={"sinks": -4}), "window"),
    (dict(kw={"max_ctx": 65}), "max_ctx"),
    (dict(kw={"out": torch.zeros(5, 4, 64)}), "out must"),
])
def test_window_attention(on_cpu, kw, match):
    with pytest.raises(ValueError, match=match):
        _window(**kw)


def _quant(**kw):
    a = dict(q=torch.zeros(T, HQ, D, dtype=BF16), k=torch.zeros(S, KVH, D, dtype=U8),
             ks=torch.zeros(S, KVH, 2, dtype=U8), v=torch.zeros(S, KVH, D, dtype=U8),
             vs=torch.zeros(S, KVH, 2, dtype=U8), kw={})
    a.update(kw)
    return hip_attn.paged_quant_attention(
        a["q"], a["k"], a["ks"], a["v"], a["vs"], torch.zeros((2, 4), dtype=torch.int32),
        torch.tensor([0, 2, 5], dtype=torch.int32), torch.tensor([2, 5], dtype=torch.int32), 2,
        **{"max_q_len": 3, **a["kw"]})


@pytest.mark.parametrize("kw,match", [
    (dict(q=torch.zeros(T, HQ, D, dtype=torch.float64)), "uint8"),
    (dict(k=torch.zeros(S, KVH, D, dtype=BF16)), "uint8"),
    (dict(vs=torch.zeros(S, KVH, 2)), "uint8"),
    (dict(ks=torch.zeros(S, KVH, 4, dtype=U8)), "scales"),
    (dict(q=torch.zeros(T, HQ, 32, dtype=BF16), k=torch.zeros(S, KVH, 32, dtype=U8)), "scales"),
    (dict(ks=torch.zeros(KVH, S, 2, dtype=U8).transpose(0, 1)), "strides"),
    (dict(k=torch.zeros(S, KVH, 48, dtype=U8), v=torch.zeros(S, KVH, 48, dtype=U8)), "width"),
    (dict(kw={"scale": 0.0}), "scale"),
    (dict(kw={"scale": -1.0}), "scale"),
    (dict(kw={"scale": float("nan")}), "scale"),
])
def test_quant_attention(on_cpu, kw, match):
    with pytest.raises(ValueError, match=match):
        _quant(**kw)


def _rows(append=True, **kw):
    a = dict(k=torch.zeros(8, KVH, D, dtype=U8), ks=torch.zeros(8, KVH, 2, dtype=U8),
             v=torch.zeros(8, KVH, D, dtype=U8), vs=torch.zeros(8, KVH, 2, dtype=U8),
             slots=torch.arange(3), x=torch.zeros(3, KVH, D), y=torch.zeros(3, KVH, D),
             dtype=torch.float32)
    a.update(kw)
    pools = (a["k"], a["ks"], a["v"], a["vs"], a["slots"])
    if append:
        return quant_cache.quant_append(*pools, a["x"], a["y"])
    return quant_cache.quant_gather(*pools, a["dtype"])


@pytest.mark.parametrize("append", [True, False])
@pytest.mark.parametrize("kw,match", [
    (dict(k=torch.zeros(8, KVH, D)), "uint8"),
    (dict(v=torch.zeros(9, KVH, D, dtype=U8)), "codes"),
    (dict(ks=torch.zeros(8, KVH, 3, dtype=U8), vs=torch.zeros(8, KVH, 3, dtype=U8)), "scales"),
    (dict(k=torch.zeros(KVH, 8, D, dtype=U8).transpose(0, 1),
          v=torch.zeros(KVH, 8, D, dtype=U8).transpose(0, 1)), "strides"),
    (dict(slots=torch.arange(3, dtype=torch.int32)), "slots"),
    (dict(k=torch.zeros(16, D, dtype=U8), v=torch.zeros(16, D, dtype=U8)), "codes"),
])
def test_rows(on_cpu, append, kw, match):
    with pytest.raises(ValueError, match=match):
        _rows(append, **kw)


def test_rows_of_other_types(on_cpu):
    with pytest.raises(ValueError, match="shapes"):
        _rows(x=torch.zeros(2, KVH, D))
    with pytest.raises(ValueError, match="dtypes"):
        _rows(x=torch.zeros(3, KVH, D, dtype=BF16))
    with pytest.raises(ValueError, match="dtypes"):
        _rows(x=torch.zeros(3, KVH, D, dtype=torch.float64), y=torch.zeros(3, KVH, D, dtype=torch.float64))
    with pytest.raises(ValueError, match="values in"):
        _rows(False, dtype=torch.float64)


def test_cache_formats(on_cpu):
    for kw in (dict(format="int8"), dict(head_dim=96), dict(dtype=torch.float64)):
        with pytest.raises(ValueError):
            quant_cache.QuantPagedKVCache(**{**dict(num_layers=1, num_blocks=2, block_size=16,
                                                    num_kv_heads=1, head_dim=64, device="cpu"), **kw})


# ---- the C entry points, which return before any launch
PTR = 0x10000   # (never followed)


def _c_window(**kw):
    a = dict(q=PTR, qt=256, qh=64, k=PTR, v=PTR, slots=64, slot=256, head=128, ks=None, vs=None, ss=0,
             sh=0, fmt=_lib.DSP_KV_PLAIN, bt=PTR, bts=4, bs=16, cu=PTR, lens=PTR, B=2, Hq=4, KVH=2, D=64,
             scale=0.125, window=8, sinks=2, max_q=3, max_ctx=64, ws=None, ws_bytes=0, out=PTR, ot=256,
             oh=64, dtype=_lib.DSP_BF16, err=None, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.lib().dsp_paged_window_attention(*a.values())


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), _lib.DSP_EINVAL), (dict(lens=None), _lib.DSP_EINVAL),
    (dict(B=-1), _lib.DSP_EINVAL), (dict(Hq=5), _lib.DSP_EINVAL), (dict(window=-1), _lib.DSP_EINVAL),
    (dict(window=0), _lib.DSP_EINVAL), (dict(bs=24), _lib.DSP_EINVAL), (dict(max_ctx=65), _lib.DSP_EINVAL),
    (dict(cu=None), _lib.DSP_EINVAL), (dict(dtype=7), _lib.DSP_EUNSUPPORTED),
    (dict(fmt=3), _lib.DSP_EUNSUPPORTED), (dict(D=48), _lib.DSP_EUNSUPPORTED),
    (dict(fmt=_lib.DSP_KV_FP8), _lib.DSP_EINVAL),
    (dict(fmt=_lib.DSP_KV_FP8, ks=PTR, vs=PTR, D=32), _lib.DSP_EUNSUPPORTED),
    (dict(fmt=_lib.DSP_KV_FP8, ks=PTR, vs=PTR, bs=8, bts=8), _lib.DSP_EUNSUPPORTED),
    (dict(fmt=_lib.DSP_KV_FP8, ks=PTR, vs=PTR, slots=63), _lib.DSP_EUNSUPPORTED),
    (dict(fmt=_lib.DSP_KV_FP8, ks=PTR, vs=PTR, k=PTR + 8), _lib.DSP_EUNSUPPORTED),
    (dict(fmt=_lib.DSP_KV_FP8, ks=PTR, vs=PTR, scale=0.0), _lib.DSP_EUNSUPPORTED),
    (dict(q=PTR + 1), _lib.DSP_EALIGN),
    (dict(max_ctx=1 << 20, bts=1 << 16, window=0, sinks=0), _lib.DSP_EWORKSPACE),
    (dict(B=0), _lib.DSP_OK), (dict(max_q=0), _lib.DSP_OK),
])
def test_c_window(kw, status):
    assert _c_window(**kw) == status


def _c_append(gather=False, **kw):
    a = dict(k=PTR, ks=PTR, v=PTR, vs=PTR, L=1, code_layer=0, code_slot=128, scale_layer=0, scale_slot=4,
             S=8)
    rows = (dict(slots=PTR, T=3, KVH=2, D=64, fmt=_lib.DSP_KV_FP8, ko=PTR, vo=PTR, dtype=_lib.DSP_BF16)
            if gather else
            dict(x=PTR, xl=0, xt=128, xh=64, y=PTR, yl=0, yt=128, yh=64, slots=PTR, T=3, KVH=2, D=64,
                 fmt=_lib.DSP_KV_FP8, dtype=_lib.DSP_BF16))
    a.update(rows, err=None, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    fn = _lib.lib().dsp_kv_gather_quant if gather else _lib.lib().dsp_kv_append_quant
    return fn(*a.values())


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("kw,status", [
    (dict(k=None), _lib.DSP_EINVAL), (dict(slots=None), _lib.DSP_EINVAL), (dict(T=-1), _lib.DSP_EINVAL),
    (dict(D=40), _lib.DSP_EUNSUPPORTED), (dict(fmt=0), _lib.DSP_EUNSUPPORTED),
    (dict(dtype=9), _lib.DSP_EUNSUPPORTED), (dict(code_slot=64), _lib.DSP_EINVAL),
    (dict(scale_slot=2), _lib.DSP_EINVAL), (dict(code_slot=132), _lib.DSP_EALIGN),
    (dict(k=PTR + 4), _lib.DSP_EALIGN), (dict(KVH=1 << 15), _lib.DSP_EUNSUPPORTED),
    (dict(T=0), _lib.DSP_OK), (dict(L=0), _lib.DSP_OK),
])
def test_c_rows(gather, kw, status):
    assert _c_append(gather, **kw) == status


def test_c_alignment_of_rows():
    assert _c_append(x=PTR + 1) == _lib.DSP_EALIGN
    assert _c_append(True, ko=PTR + 8) == _lib.DSP_EALIGN
