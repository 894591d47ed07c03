"""The quantised KV cache and the attention that reads it: Python host layer over tgaf_kv_* / tgaf_attention*.

What a decoder runs between its qkv linear and its o linear.  The cache is paged, and its rows are grouped-affine codes in
the layout of the weights; the reference's counterparts are its f16 KV store and decode attention kernels
(core/src/compute/cuda/kernels/ops/norm_rope_ops.cu:164, kernels/ops/attention_ops.cu:20-215).

All calls address tokens in one way: of the `lens[b]` cached tokens of sequence b the last `cu[b + 1] - cu[b]` are the
call's own, in rows cu[b] .. cu[b + 1] of its packed tensors; token t of a sequence lies in row t % page_tokens of page
table[b, t // page_tokens].  table, lens and cu are int32 tensors on the device, so a call captured into a CUDA graph
follows them from replay to replay.  Calls only enqueue on the context's stream.
"""
from __future__ import annotations

import ctypes as C
import math

from . import _capi
from .gaf import DTYPE_BF16, DTYPE_F32, Context, GafError, _STATUS_INVALID_ARGUMENT


def _refuse(message: str):
    raise GafError(_STATUS_INVALID_ARGUMENT, message)


def _check_device(ctx: Context, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and (t.device.type != "cuda" or t.device.index != ctx.device):
            _refuse(f"{name} must be on cuda:{ctx.device}, got {t.device}")


def _dtype_tag(name: str, dtype) -> int:
    import torch
    tag = {torch.float32: DTYPE_F32, torch.bfloat16: DTYPE_BF16}.get(dtype)
    if tag is None:
        _refuse(f"{name} must be bf16 or f32, got {dtype}")
    return tag


def _check_rows(name: str, t, heads: int, head_dim: int) -> None:
    if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != head_dim:
        _refuse(f"{name} must be [tokens, {heads}, {head_dim}], got {tuple(t.shape)}")
    if t.stride(2) != 1:
        _refuse(f"{name} must be contiguous along its last axis")


def _check_written(name: str, t) -> None:
    """A tensor that is written must not name one place twice."""
    reach = 1
    for stride, size in sorted(zip(t.stride(), t.shape)):
        if size > 1:
            if stride < reach:
                _refuse(f"{name} must not overlap itself")
            reach = stride * size


class KvCache:
    """A paged cache of grouped-affine K / V rows in device memory (tgaf_kv_cache).

    packed: int32 [pages, 2, kv_heads, page_tokens, head_dim * bits / 32], K at index 0 of the second axis, V at 1;
    scales, biases: 2-byte tensors [pages, 2, kv_heads, page_tokens, head_dim / group] of bf16 values."""

    def __init__(self, ctx: Context, handle, packed, scales, biases, group: int, bits: int):
        self.ctx, self._h = ctx, handle
        self.packed, self.scales, self.biases = packed, scales, biases
        self.pages, _, self.kv_heads, self.page_tokens, _ = packed.shape
        self.head_dim, self.group, self.bits = packed.shape[4] * 32 // bits, group, bits

    @classmethod
    def wrap_device(cls, ctx: Context, packed, scales, biases, group: int, bits: int):
        """Wrap torch device tensors without copying; they are kept alive by the cache."""
        import torch
        if bits not in (4, 8) or group not in (32, 64, 128):
            _refuse(f"bits must be 4 or 8 and group 32, 64 or 128, got {bits} and {group}")
        if packed.dim() != 5 or packed.shape[1] != 2 or packed.dtype != torch.int32:
            _refuse(f"packed must be int32 [pages, 2, kv_heads, page_tokens, words], got {packed.dtype} {tuple(packed.shape)}")
        head_dim = packed.shape[4] * 32 // bits
        want = (*packed.shape[:4], head_dim // group)
        for name, t in (("scales", scales), ("biases", biases)):
            if tuple(t.shape) != want or t.dtype not in (torch.bfloat16, torch.int16):
                _refuse(f"{name} must be bf16 (or int16 bit patterns) {want}, got {t.dtype} {tuple(t.shape)}")
        if not (packed.is_contiguous() and scales.is_contiguous() and biases.is_contiguous()):
            _refuse("cache buffers must be contiguous")
        _check_device(ctx, packed=packed, scales=scales, biases=biases)
        h = C.c_void_p()
        ctx._check(ctx._lib.tgaf_kv_cache_wrap_device(
            ctx._h, C.c_void_p(packed.data_ptr()), C.c_void_p(scales.data_ptr()), C.c_void_p(biases.data_ptr()), packed.shape[0],
            packed.shape[2], packed.shape[3], head_dim, group, bits, C.byref(h)))
        return cls(ctx, h, packed, scales, biases, group, bits)

    @classmethod
    def allocate(cls, ctx: Context, pages: int, kv_heads: int, head_dim: int, page_tokens: int = 64, bits: int = 8, group: int = 64):
        """A cache of `pages` empty pages: head_dim * bits / 8 + 4 * head_dim / group bytes per token, head and K or V."""
        import torch
        if bits not in (4, 8) or group not in (32, 64, 128) or head_dim % group:
            _refuse(f"bits must be 4 or 8, group 32, 64 or 128 and head_dim a multiple of it, got {bits}, {group}, {head_dim}")
        dev = f"cuda:{ctx.device}"
        packed = torch.zeros((pages, 2, kv_heads, page_tokens, head_dim * bits // 32), dtype=torch.int32, device=dev)
        scales = torch.zeros((pages, 2, kv_heads, page_tokens, head_dim // group), dtype=torch.bfloat16, device=dev)
        return cls.wrap_device(ctx, packed, scales, torch.zeros_like(scales), group, bits)

    def free(self) -> None:
        if getattr(self, "_h", None):
            self.ctx._lib.tgaf_kv_cache_free(self.ctx._h, self._h)
            self._h = None

    def __del__(self):
        try:
            if getattr(self.ctx, "_h", None):
                self.free()
        except Exception:
            pass


def _seqs(ctx: Context, table, lens, cu, total: int) -> _capi.KvSeqs:
    import torch
    if table.dtype != torch.int32 or table.dim() != 2 or (table.shape[1] > 1 and table.stride(1) != 1):
        _refuse(f"table must be int32 [batch, pages] with contiguous rows, got {table.dtype} {tuple(table.shape)}")
    batch = table.shape[0]
    if lens.dtype != torch.int32 or tuple(lens.shape) != (batch,) or not lens.is_contiguous():
        _refuse(f"lens must be contiguous int32 [{batch}], got {lens.dtype} {tuple(lens.shape)}")
    if cu is not None and (cu.dtype != torch.int32 or tuple(cu.shape) != (batch + 1,) or not cu.is_contiguous()):
        _refuse(f"cu must be contiguous int32 [{batch + 1}], got {cu.dtype} {tuple(cu.shape)}")
    if cu is None and (total % batch if batch else total):
        _refuse(f"{total} rows are no equal share of {batch} sequences: give cu")
    _check_device(ctx, table=table, lens=lens, cu=cu)
    stride = table.stride(0) if batch > 1 else max(table.stride(0), table.shape[1])
    if stride < table.shape[1]:
        _refuse("table rows must not overlap")
    return _capi.KvSeqs(table.data_ptr(), stride, table.shape[1], batch, lens.data_ptr(), cu.data_ptr() if cu is not None else None, total)


def _row_args(t):
    return C.c_void_p(t.data_ptr()), t.stride(0), t.stride(1)


def kv_append(ctx: Context, cache: KvCache, k, v, table, lens, cu=None) -> None:
    """Quantises the call's own rows k, v [tokens, kv_heads, head_dim] (bf16 or f32, any token and head strides) into the
    sequences' pages (tgaf_kv_append).  lens counts them already; without cu every sequence has tokens / batch of them."""
    tag = _dtype_tag("k", k.dtype)
    for name, t in (("k", k), ("v", v)):
        _check_rows(name, t, cache.kv_heads, cache.head_dim)
    if v.dtype != k.dtype or v.shape[0] != k.shape[0]:
        _refuse(f"k and v must have one dtype and length, got {k.dtype} {k.shape[0]} and {v.dtype} {v.shape[0]}")
    _check_device(ctx, k=k, v=v)
    s = _seqs(ctx, table, lens, cu, k.shape[0])
    ctx._check(ctx._lib.tgaf_kv_append(ctx._h, cache._h, C.byref(s), tag, *_row_args(k), *_row_args(v)))


def kv_read(ctx: Context, cache: KvCache, table, lens, cu=None, total: int | None = None, dtype=None, out=None):
    """The rows that kv_append with the same table, lens and cu wrote, read back: (k, v), each [total, kv_heads, head_dim],
    bf16 (default) or f32 (tgaf_kv_read).  total: rows of the call, needed unless `out` = (k, v) is given; whole sequences
    are cu = cumulated lens.  Rows that lie in no sequence are left as they were (undefined in new tensors)."""
    import torch
    if out is None:
        if total is None:
            _refuse("total (or out) is needed")
        dtype = torch.bfloat16 if dtype is None else dtype
        _dtype_tag("dtype", dtype)
        shape, dev = (total, cache.kv_heads, cache.head_dim), f"cuda:{ctx.device}"
        out = (torch.empty(shape, dtype=dtype, device=dev), torch.empty(shape, dtype=dtype, device=dev))
    k, v = out
    tag = _dtype_tag("out", k.dtype)
    for name, t in (("out k", k), ("out v", v)):
        _check_rows(name, t, cache.kv_heads, cache.head_dim)
        _check_written(name, t)
    if v.dtype != k.dtype or v.shape[0] != k.shape[0] or (total is not None and total != k.shape[0]):
        _refuse("out k and v must have one dtype and `total` rows")
    _check_device(ctx, k=k, v=v)
    s = _seqs(ctx, table, lens, cu, k.shape[0])
    ctx._check(ctx._lib.tgaf_kv_read(ctx._h, cache._h, C.byref(s), tag, *_row_args(k), *_row_args(v)))
    return k, v


def _attend(ctx: Context, cache: KvCache, q, prefix_table, prefix_len: int, table, lens, cu, max_new, scale, out):
    import torch
    tag = _dtype_tag("q", q.dtype)
    if q.dim() != 3 or q.shape[1] == 0 or q.shape[1] % cache.kv_heads:
        _refuse(f"q must be [tokens, heads, {cache.head_dim}] with heads a multiple of {cache.kv_heads}, got {tuple(q.shape)}")
    _check_rows("q", q, q.shape[1], cache.head_dim)
    _check_device(ctx, q=q)
    s = _seqs(ctx, table, lens, cu, q.shape[0])
    if max_new is None:
        if cu is not None:
            _refuse("max_new is needed with cu")
        max_new = q.shape[0] // max(1, table.shape[0])
    scale = 1.0 / math.sqrt(cache.head_dim) if scale is None else float(scale)
    if out is None:
        out = torch.empty((q.shape[0], q.shape[1], cache.head_dim), dtype=q.dtype, device=q.device)
    else:
        _check_rows("out", out, q.shape[1], cache.head_dim)
        _check_written("out", out)
        if out.dtype != q.dtype or out.shape[0] != q.shape[0]:
            _refuse(f"out must be {q.dtype} with {q.shape[0]} rows")
        _check_device(ctx, out=out)
    if q.shape[0] == 0:
        return out
    tail = (tag, *_row_args(q), q.shape[1], int(max_new), scale, *_row_args(out))
    if prefix_table is None:
        ctx._check(ctx._lib.tgaf_attention(ctx._h, cache._h, C.byref(s), *tail))
    else:
        ctx._check(ctx._lib.tgaf_attention_shared_prefix(ctx._h, cache._h, C.c_void_p(prefix_table.data_ptr()), prefix_len, C.byref(s), *tail))
    return out


def attention(ctx: Context, cache: KvCache, q, table, lens, cu=None, max_new=None, scale=None, out=None):
    """Causal attention of the call's own tokens over their sequences' cached tokens (tgaf_attention).

    q: [tokens, heads, head_dim], bf16 or f32, any token and head strides; heads / kv_heads query heads share a cached head.
    The tokens' own K / V rows are appended first (`lens` counts them).  max_new: an upper bound of the own tokens of any
    sequence (the launch is sized by it), needed with cu.  scale: default 1 / sqrt(head_dim).  Rows that see no key are 0."""
    return _attend(ctx, cache, q, None, 0, table, lens, cu, max_new, scale, out)


def attention_shared_prefix(ctx: Context, cache: KvCache, q, prefix_table, prefix_len: int, table, lens, cu=None, max_new=None,
                            scale=None, out=None):
    """`attention` for sequences that all continue one shared prefix of `prefix_len` tokens in the pages `prefix_table`
    (int32 [pages], on the device); table and lens do not count the prefix.  Its pages are read once for the whole batch
    (tgaf_attention_shared_prefix)."""
    import torch
    prefix_len = int(prefix_len)
    if prefix_table.dtype != torch.int32 or prefix_table.dim() != 1 or not prefix_table.is_contiguous():
        _refuse(f"prefix_table must be contiguous int32 [pages], got {prefix_table.dtype} {tuple(prefix_table.shape)}")
    if prefix_len < 0 or prefix_len > prefix_table.shape[0] * cache.page_tokens:
        _refuse(f"prefix_len {prefix_len} does not fit {prefix_table.shape[0]} pages of {cache.page_tokens} tokens")
    _check_device(ctx, prefix_table=prefix_table)
    return _attend(ctx, cache, q, prefix_table, prefix_len, table, lens, cu, max_new, scale, out)
