"""What dsp_paged_window_attention refuses of shapes and strides, on the host: it returns before any
launch."""

import pytest

from dispec_amd import _lib

PTR = 0x10000   # (never followed)
FORMATS = [_lib.DSP_KV_FP8, _lib.DSP_KV_FP4]


def call(fmt, max_q=3, dtype=_lib.DSP_BF16, **kw):
    """A call over a quantised cache of heads of 64 whose arguments are right but for `kw`."""
    a = dict(q=PTR, qt=256, qh=64, k=PTR, v=PTR, slots=64, slot=128, head=64, ks=PTR, vs=PTR, ss=4, sh=2,
             fmt=fmt, bt=PTR, bts=4, bs=16, cu=PTR, lens=PTR, B=2, Hq=4, KVH=2, D=64, scale=0.125, window=8,
             sinks=2, max_q=max_q, max_ctx=64, ws=None, ws_bytes=0, out=PTR, ot=256, oh=64, dtype=dtype,
             err=None, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.lib().dsp_paged_window_attention(*a.values())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("max_q", [1, 3, 200])
@pytest.mark.parametrize("D", [-64, -8, 0, 1, 8, 16, 31, 32, 33, 96, 512])
def test_head_dims_of_a_quantised_cache(fmt, max_q, D):
    """64, 128 and 256 only, below the 32 elements of a group too."""
    assert call(fmt, max_q, D=D) == _lib.DSP_EUNSUPPORTED
    _lib.lib().dsp_paged_window_workspace_bytes(2, 4, 2, D, max_q, 64, 8, 2, fmt, _lib.DSP_BF16)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [_lib.DSP_BF16, _lib.DSP_F16, _lib.DSP_F32])
@pytest.mark.parametrize("max_q", [1, 50, 200])
@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("stride", [-(1 << 40), -4, -1, 1 << 26, 1 << 30, 1 << 32, 1 << 40])
def test_slot_strides_of_scales(fmt, dtype, max_q, D, stride):
    """A block's rows of scales are addressed in 32 bits: strides are bounded as those of codes are,
    for every kernel (few rows, up to 128, more).  Without a workspace a call that is not refused for
    its strides is for that."""
    kw = dict(D=D, qt=4 * D, qh=D, slot=2 * D, head=D, sh=D // 32, ot=4 * D, oh=D, max_ctx=1 << 20,
              bts=1 << 16, window=0, sinks=0)
    assert call(fmt, max_q, dtype, ss=stride, **kw) == _lib.DSP_EUNSUPPORTED
    assert call(fmt, max_q, dtype, ss=(1 << 26) - 8, **kw) == _lib.DSP_EWORKSPACE
    assert call(fmt, max_q, dtype, ss=0, **kw) == _lib.DSP_EWORKSPACE
