"""A paged KV pool in 8 or 4 bits an element.

The reference's pool holds the model's type (dispec/kv/paged_cache.py:39-41).  Here a row's elements
are e4m3 ("fp8": a byte each) or e2m1 ("fp4": two to a byte, the first in the low half), and 32
neighbouring elements of a head share a scale, a power of two whose exponent plus 127 is one byte:
1.03 or 0.53 bytes an element instead of 2.  Rows are quantised as they are written (`quant_append`)
and read back as values of the model's type (`quant_gather`); attention reads the codes themselves
(`engine.hip_attn.paged_quant_attention`).

`QuantPagedKVCache` is a `PagedKVCache` over such pools: the same interface, k and v in the model's
type on the way in and out.
"""

from __future__ import annotations

import torch

from dispec_amd import _lib
from dispec_amd.kv.paged_cache import PagedKVCache, commit_path

FORMATS = ("fp8", "fp4")
GROUP = 32   # elements that share a scale
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def code_width(format: str, head_dim: int) -> int:
    """Bytes of a head's codes."""
    return head_dim if _lib.kv_format(format) == _lib.DSP_KV_FP8 else head_dim // 2


def _pools(k_cache, k_scale, v_cache, v_scale):
    """(format, layers, slots, KVH, D, and code and scale strides of a layer and a slot) of pools
    (S, KVH, width) of one layer or (L, S, KVH, width) of all."""
    shape, stride, scales, s_stride = (k_cache.shape, k_cache.stride(), k_scale.shape,
                                       k_scale.stride())
    if not k_cache.dtype == k_scale.dtype == v_cache.dtype == v_scale.dtype == torch.uint8:
        raise ValueError(f"codes and scales must be uint8, got {k_cache.dtype}, {k_scale.dtype}, "
                         f"{v_cache.dtype}, {v_scale.dtype}")
    n = len(shape)
    if n not in (3, 4) or len(scales) != n or v_cache.shape != shape or v_scale.shape != scales:
        raise ValueError(f"expected codes (S, KVH, width) or (L, S, KVH, width) and scales alike for K "
                         f"and V; got {tuple(shape)}, {tuple(v_cache.shape)}, {tuple(scales)}, "
                         f"{tuple(v_scale.shape)}")
    S, KVH, width = shape[-3:]
    groups = scales[-1]
    D = GROUP * groups
    if scales[-2] != KVH or scales[-3] != S or scales[0] != shape[0] or width != D and 2 * width != D:
        raise ValueError(f"scales {tuple(scales)} for codes {tuple(shape)}: one for {GROUP} elements of "
                         "a byte or half a byte")
    if (v_cache.stride() != stride or v_scale.stride() != s_stride or stride[-1] != 1
            or s_stride[-1] != 1 or (stride[-2] != width or s_stride[-2] != groups) and KVH > 1):
        raise ValueError("codes and scales need the same strides for K and V with contiguous rows")
    fmt = _lib.DSP_KV_FP8 if width == D else _lib.DSP_KV_FP4
    if n == 3:
        return fmt, 1, S, KVH, D, (0, stride[0], 0, s_stride[0])
    return fmt, shape[0], S, KVH, D, (stride[0], stride[1], s_stride[0], s_stride[1])


def quant_append(k_cache, k_scale, v_cache, v_scale, slots, k, v, err=None) -> None:
    """Quantise rows k and v into the slots of a quantised pool (dsp_kv_append_quant).

    k_cache, v_cache: uint8 codes (S, KVH, width) of a layer, or (L, S, KVH, width) of all: width
                      head_dim ("fp8") or head_dim / 2 ("fp4")
    k_scale, v_scale: uint8 scales (S, KVH, head_dim / 32), or with L before
    slots:            (T,) int64 slot ids, unique, of every layer
    k, v:             (T, KVH, head_dim), or (L, T, KVH, head_dim); bf16, fp16 or fp32, at any
                      strides with head_dim contiguous
    err:              optional int32 device counter of slots outside the pool (skipped)

    Of each group of 32 elements the scale is the least power of two from 2^-100 to 2^118 by which
    the largest fits the format; a code is the nearest number's (halves: the even code).  fp16 rows
    are first clamped to +-61440 ("fp8") or +-49152 ("fp4"), so that they read back finite.  A group
    with an infinity or NaN reads back as NaN.
    """
    fast, stream = _lib.torch_calls(), _lib.current_stream(k_cache)
    if fast is not None and stream is not None and fast.append(
            k_cache, k_scale, v_cache, v_scale, slots, k, v, err, stream):
        return
    fmt, L, S, KVH, D, strides = _pools(k_cache, k_scale, v_cache, v_scale)
    T, rows = slots.numel(), k.shape
    n = len(rows)
    if (n != k_cache.dim() or v.shape != rows or rows[-1] != D or rows[-2] != KVH or rows[-3] != T
            or n == 4 and rows[0] != L):
        raise ValueError(f"k, v have shapes {tuple(k.shape)}, {tuple(v.shape)}: expected "
                         f"{((L,) if k_cache.dim() == 4 else ()) + (T, KVH, D)}")
    dtype = k.dtype
    if v.dtype != dtype or dtype not in _DTYPES:
        raise ValueError(f"k/v dtypes {k.dtype}/{v.dtype}: bf16, fp16 or fp32, both the same")
    if slots.dtype != torch.int64:
        raise ValueError(f"slots must be int64, got {slots.dtype}")
    dev = _lib.same_gpu(k_cache, k_scale, v_cache, v_scale, slots, k, v, err)
    if not (T and L):
        return
    if not slots.is_contiguous():
        slots = slots.contiguous()
    ks, vs = k.stride(), v.stride()
    if ks[-1] != 1:
        k = k.contiguous()
        ks = k.stride()
    if vs[-1] != 1:
        v = v.contiguous()
        vs = v.stride()
    status = _lib.call_on(dev, _lib.calls().dsp_kv_append_quant, (
        k_cache.data_ptr(), k_scale.data_ptr(), v_cache.data_ptr(), v_scale.data_ptr(), L, *strides, S,
        k.data_ptr(), ks[0] if n == 4 else 0, ks[-3], ks[-2], v.data_ptr(), vs[0] if n == 4 else 0,
        vs[-3], vs[-2], slots.data_ptr(), T, KVH, D, fmt, _lib.dtype_code(dtype),
        None if err is None else err.data_ptr(), _lib.stream_of(k_cache)))
    if status:
        _lib.check(status, "dsp_kv_append_quant")


def quant_gather(k_cache, k_scale, v_cache, v_scale, slots, dtype=torch.bfloat16, err=None, out=None):
    """The values (k, v) that slots of a quantised pool hold (dsp_kv_gather_quant): each (T, KVH,
    head_dim), or (L, T, KVH, head_dim) of pools of all layers, rounded to `dtype` (which loses
    nothing in bf16 and fp32, and in fp16 where the rows were written from fp16).  Arguments as for
    `quant_append`; a slot outside the pool leaves its rows as they were (undefined without `out`).
    out: optional pair of contiguous tensors of that shape and type to write."""
    fast, stream = _lib.torch_calls(), _lib.current_stream(k_cache)
    if fast is not None and stream is not None and out is None:
        got = fast.gather(k_cache, k_scale, v_cache, v_scale, slots, dtype, err, stream)
        if got is not None:
            return got
    fmt, L, S, KVH, D, strides = _pools(k_cache, k_scale, v_cache, v_scale)
    if dtype not in _DTYPES:
        raise ValueError(f"values in bf16, fp16 or fp32, not {dtype}")
    if slots.dtype != torch.int64:
        raise ValueError(f"slots must be int64, got {slots.dtype}")
    T = slots.numel()
    rows = (T, KVH, D) if k_cache.dim() == 3 else (L, T, KVH, D)
    if out is None:
        k = k_cache.new_empty(rows, dtype=dtype)
        v = torch.empty_like(k)
    else:
        k, v = out
        for t in out:
            if t.shape != rows or t.dtype != dtype or not t.is_contiguous():
                raise ValueError(f"out must be two contiguous tensors {rows} of {dtype}; got "
                                 f"{tuple(t.shape)} {t.dtype}")
    dev = _lib.same_gpu(k_cache, k_scale, v_cache, v_scale, slots, k, v, err)
    if not (T and L):
        return k, v
    if not slots.is_contiguous():
        slots = slots.contiguous()
    status = _lib.call_on(dev, _lib.calls().dsp_kv_gather_quant, (
        k_cache.data_ptr(), k_scale.data_ptr(), v_cache.data_ptr(), v_scale.data_ptr(), L, *strides, S,
        slots.data_ptr(), T, KVH, D, fmt, k.data_ptr(), v.data_ptr(), _lib.dtype_code(dtype),
        None if err is None else err.data_ptr(), _lib.stream_of(k_cache)))
    if status:
        _lib.check(status, "dsp_kv_gather_quant")
    return k, v


class QuantPagedKVCache(PagedKVCache):
    """A `PagedKVCache` whose pools hold codes and scales: `key`, `value` (L, slots, KVH, width) and
    `key_scale`, `value_scale` (L, slots, KVH, head_dim / 32), uint8.  `dtype` is the model's type, of
    what is written and read back; blocks, forks and prefix sharing work as they do there."""

    def __init__(self, num_layers: int, num_blocks: int, block_size: int, num_kv_heads: int,
                 head_dim: int, dtype: torch.dtype = torch.bfloat16, device: str = "cuda",
                 format: str = "fp8"):
        width = code_width(format, head_dim)
        if dtype not in _DTYPES or head_dim not in (64, 128, 256):
            raise ValueError(f"dtype {dtype}, head_dim {head_dim}: a quantised cache takes bf16, fp16 or "
                             "fp32 and head_dim 64, 128 or 256")
        super().__init__(num_layers, num_blocks, block_size, num_kv_heads, width, torch.uint8, device)
        self.head_dim, self.dtype, self.format = head_dim, dtype, format
        shape = self.key.shape[:3] + (head_dim // GROUP,)
        self.key_scale = torch.zeros(shape, dtype=torch.uint8, device=self.key.device)
        self.value_scale = torch.zeros_like(self.key_scale)

    @classmethod
    def for_model(cls, config, num_blocks: int, block_size: int, dtype, device="cuda",
                  format: str = "fp8") -> "QuantPagedKVCache":
        head_dim = getattr(config, "head_dim", None) or (
            config.hidden_size // config.num_attention_heads)
        return cls(num_layers=config.num_hidden_layers, num_blocks=num_blocks,
                   block_size=block_size, num_kv_heads=config.num_key_value_heads,
                   head_dim=head_dim, dtype=dtype, device=device, format=format)

    def memory_bytes(self) -> int:
        return 2 * (self.key.numel() + self.key_scale.numel())

    @property
    def row_bytes(self) -> int:
        """Bytes of one slot's codes of one layer (all KV heads)."""
        return self.key.shape[2] * self.key.shape[3]

    @property
    def scale_row_bytes(self) -> int:
        return self.key_scale.shape[2] * self.key_scale.shape[3]

    def layer(self, layer_idx: int):
        """(k_cache, k_scale, v_cache, v_scale) of a layer, as `paged_quant_attention` takes them."""
        return (self.key[layer_idx], self.key_scale[layer_idx], self.value[layer_idx],
                self.value_scale[layer_idx])

    def _all(self):
        return self.key, self.key_scale, self.value, self.value_scale

    # -- per-step IO ------------------------------------------------------------------
    def write(self, layer_idx: int, slots, k, v) -> None:
        """Quantise token rows into a layer (slots (T,), k and v (T, KVH, head_dim))."""
        n = slots.numel()
        k, v = self._rows(k, "k", n), self._rows(v, "v", n)
        quant_append(*self.layer(layer_idx), self._as_slots(slots.reshape(-1), self.key.device), k, v,
                     err=self._err)
        self._after()

    def gather(self, layer_idx: int, slots):
        """(k, v) values of the given flat slots, each (len(slots), KVH, head_dim)."""
        kv = quant_gather(*self.layer(layer_idx), self._as_slots(slots.reshape(-1), self.key.device),
                          self.dtype, err=self._err)
        self._after()
        return kv

    # -- whole-sequence export / import -------------------------------------------------
    def _slots_of(self, tables: list[list[int]], lengths: list[int]) -> torch.Tensor:
        """Slots of the sequences' first tokens, one after the other."""
        bs = self.block_size
        blocks = torch.cat([torch.tensor(ids[:-(-n // bs)], dtype=torch.int64)
                            for ids, n in zip(tables, lengths)] or [torch.zeros(0, dtype=torch.int64)])
        slots = (blocks[:, None] * bs + torch.arange(bs)).reshape(-1)
        keep = torch.cat([torch.arange(-(-n // bs) * bs) < n for n in lengths]
                         or [torch.zeros(0, dtype=torch.bool)])
        return slots[keep].to(self.key.device)

    def export_batch(self, seqs):
        """As `PagedKVCache.export_batch`, in values of the model's type: flat K and V buffers and the
        token offsets; sequence b is buffer[L*cu[b] : L*cu[b+1]] viewed as (L, T_b, H, D)."""
        cu = [0]
        for ids, n in seqs:
            self._check_blocks(ids, n)
            cu.append(cu[-1] + n)
        shape = (self.num_layers * cu[-1], self.num_kv_heads, self.head_dim)
        if len(seqs) == 1:
            k, v = self._read(*seqs[0])
            return k.view(shape), v.view(shape), cu
        parts = [self._read(ids, n) for ids, n in seqs]
        flat = [torch.cat([p[i].flatten(0, 1) for p in parts]) if parts
                else torch.empty(shape, dtype=self.dtype, device=self.key.device) for i in (0, 1)]
        return flat[0], flat[1], cu

    def _read(self, block_ids, n, out=None):
        kv = quant_gather(*self._all(), self._slots_of([block_ids], [n]), self.dtype, err=self._err,
                          out=out)
        self._after()
        return kv

    def export_into(self, block_ids, seq_len, k, v) -> None:
        self._check_blocks(block_ids, seq_len)
        self._read(block_ids, seq_len, (k, v))

    def import_batch(self, tables, k, v, cu) -> None:
        """Quantise flat buffers laid out as export_batch's into the given block tables."""
        for ids, a, b in zip(tables, cu[:-1], cu[1:]):
            self._check_blocks(ids, b - a)
        L = self.num_layers
        for ids, a, b in zip(tables, cu[:-1], cu[1:]):
            rows = (L, b - a, self.num_kv_heads, self.head_dim)
            quant_append(*self._all(), self._slots_of([ids], [b - a]), k[L * a:L * b].reshape(rows),
                         v[L * a:L * b].reshape(rows), err=self._err)
        self._after()

    def _device_slots(self, block_table, cu_seqlens, max_seqlen):
        raise NotImplementedError("a quantised cache has no device-table gather and scatter: "
                                  "use export_batch and import_batch")

    def gather_into(self, block_table, cu_seqlens, max_seqlen, k_buf, v_buf) -> None:
        self._device_slots(block_table, cu_seqlens, max_seqlen)

    def scatter_from(self, block_table, cu_seqlens, max_seqlen, k_buf, v_buf) -> None:
        self._device_slots(block_table, cu_seqlens, max_seqlen)

    # -- block moves: codes, then scales, as bytes -------------------------------------
    def _scales(self) -> "_ScalePool":
        return _ScalePool(self)

    def copy_blocks_device(self, src, src_ids, dst_ids) -> None:
        self._same_format(src)
        super().copy_blocks_device(src, src_ids, dst_ids)
        PagedKVCache.copy_blocks_device(self._scales(), src._scales(), src_ids, dst_ids)

    def copy_block_fanout_device(self, src, src_block, dst_ids) -> None:
        self._same_format(src)
        super().copy_block_fanout_device(src, src_block, dst_ids)
        PagedKVCache.copy_block_fanout_device(self._scales(), src._scales(), src_block, dst_ids)

    def copy_blocks_from(self, src, src_ids, dst_ids) -> None:
        """dst[l, block d] = src[l, block s] for every layer, K and V, codes and scales."""
        self._same_format(src)
        if len(src_ids) != len(dst_ids):
            raise ValueError("src_ids and dst_ids differ in length")
        if (src.num_layers, src.block_bytes) != (self.num_layers, self.block_bytes):
            raise ValueError("block copy between pools of different geometry")
        if not src_ids:
            return
        if src is self and set(src_ids) & set(dst_ids):
            raise ValueError("a block is both copied from and written in one copy_blocks call")
        ids = torch.tensor([list(src_ids), list(dst_ids)], dtype=torch.int32).to(self.key.device)
        if len(src_ids) > 1 and len(set(src_ids)) == 1 and 0 <= src_ids[0] < src.num_blocks:
            self.copy_block_fanout_device(src, src_ids[0], ids[1])
        else:
            self.copy_blocks_device(src, ids[0], ids[1])
        self._after()

    def commit_path(self, block_table, cu_q, ctx_lens, path, num_accepted) -> None:
        for k, v in ((self.key, self.value), (self.key_scale, self.value_scale)):
            commit_path(k, v, block_table, cu_q, ctx_lens, path, num_accepted,
                        block_size=self.block_size, err=self._err)
        self._after()


class _ScalePool(PagedKVCache):
    """The scales of a quantised cache as a pool whose blocks can be copied."""

    def __init__(self, cache: QuantPagedKVCache):
        self.num_layers, self.num_blocks = cache.num_layers, cache.num_blocks
        self.block_size, self.num_kv_heads = cache.block_size, cache.num_kv_heads
        self.key, self.value = cache.key_scale, cache.value_scale
        self.head_dim, self._err = self.key.shape[3], cache._err
