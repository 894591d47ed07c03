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

from . import _capi
from .gaf import DTYPE_BF16, DTYPE_F32, Context, GafError, _STATUS_INVALID_ARGUMENT


_BF16 = _F32 = _I32 = None   # torch's dtypes, once torch is loaded


def _torch():
    global _BF16, _F32, _I32
    import torch
    _BF16, _F32, _I32 = torch.bfloat16, torch.float32, torch.int32


def _refuse(message: str):
    raise GafError(_STATUS_INVALID_ARGUMENT, message)


# The checks below run in front of every launch of a decoder step, so they ask each tensor once for what they need
# (get_device() is the device's index, -1 on the CPU).

def _tag(name: str, dtype) -> int:
    if _BF16 is None:
        _torch()
    if dtype is _BF16:
        return DTYPE_BF16
    if dtype is not _F32:
        _refuse(f"{name} must be bf16 or f32, got {dtype}")
    return DTYPE_F32


def _count(name: str, value, least: int = 0, most: int = 2 ** 32 - 1) -> int:
    """An integer that the C entry takes as it is: ctypes would drop the bits above 32, and a sign."""
    if type(value) is int and least <= value <= most:
        return value
    if isinstance(value, bool) or not hasattr(value, "__index__") or not least <= value.__index__() <= most:
        _refuse(f"{name} must be an integer from {least} to {most}, got {value!r}")
    return value.__index__()


def _other_device(ctx: Context, cache: KvCache):
    _refuse(f"the cache is on cuda:{cache.ctx.device}, the context on cuda:{ctx.device}")


def _rows(ctx: Context, name: str, t, heads: int, head_dim: int, written: bool = False):
    """Rows of `t` and its pointer, token stride and head stride, if it is [rows, heads, head_dim] on the context's device."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 3 or shape[1] != heads or shape[2] != head_dim:
        _refuse(f"{name} must be [tokens, {heads}, {head_dim}], got {tuple(shape)}")
    if stride[2] != 1:
        _refuse(f"{name} must be contiguous along its last axis")
    if t.get_device() != ctx.device:
        _refuse(f"{name} must be on cuda:{ctx.device}, got {t.device}")
    if written:        # a tensor that is written must not name one place twice
        reach = 1
        for step, size in sorted(zip(stride, shape)):
            if size > 1:
                if step < reach:
                    _refuse(f"{name} must not overlap itself")
                reach = step * size
    if shape[0] > 2 ** 32 - 1:
        _refuse(f"{name} has too many rows: {shape[0]}")
    return shape[0], (t.data_ptr(), stride[0], stride[1])


class KvCache:
    """A paged cache of grouped-affine K / V rows in device memory (tgaf_kv_cache).  Any context of its device may use it.

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
        for name, t in (("packed", packed), ("scales", scales), ("biases", biases)):
            if t.get_device() != ctx.device:
                _refuse(f"{name} must be on cuda:{ctx.device}, got {t.device}")
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
    device = ctx.device
    shape = table.shape
    if table.dtype is not _I32 or len(shape) != 2:
        _refuse(f"table must be int32 [batch, pages], got {table.dtype} {tuple(shape)}")
    batch, width = shape
    stride, inner = table.stride()
    if (inner != 1 and width > 1) or (stride < width and batch > 1):
        _refuse("table must have contiguous rows that do not overlap")
    if lens.dtype is not _I32 or lens.shape != (batch,) or not lens.is_contiguous():
        _refuse(f"lens must be contiguous int32 [{batch}], got {lens.dtype} {tuple(lens.shape)}")
    if table.get_device() != device or lens.get_device() != device:
        _refuse(f"table and lens must be on cuda:{device}, got {table.device} and {lens.device}")
    at = None
    if cu is not None:
        if cu.dtype is not _I32 or cu.shape != (batch + 1,) or not cu.is_contiguous():
            _refuse(f"cu must be contiguous int32 [{batch + 1}], got {cu.dtype} {tuple(cu.shape)}")
        if cu.get_device() != device:
            _refuse(f"cu must be on cuda:{device}, got {cu.device}")
        at = cu.data_ptr()
    elif total % batch if batch else total:
        _refuse(f"{total} rows are no equal share of {batch} sequences: give cu")
    return _capi.KvSeqs(table.data_ptr(), stride if batch > 1 else max(stride, width), width, batch, lens.data_ptr(), at, total)


def kv_append(ctx: Context, cache: KvCache, k, v, table, lens, cu=None) -> None:
    """Quantises the call's own rows k, v [tokens, kv_heads, head_dim] (bf16 or f32, any token and head strides) into the
    sequences' pages (tgaf_kv_append).  lens counts them already; without cu every sequence has tokens / batch of them."""
    if cache.ctx.device != ctx.device:
        _other_device(ctx, cache)
    tag = _tag("k", k.dtype)
    total, k_args = _rows(ctx, "k", k, cache.kv_heads, cache.head_dim)
    v_rows, v_args = _rows(ctx, "v", v, cache.kv_heads, cache.head_dim)
    if v.dtype is not k.dtype or v_rows != total:
        _refuse(f"k and v must have one dtype and length, got {k.dtype} {total} and {v.dtype} {v_rows}")
    seqs = _seqs(ctx, table, lens, cu, total)
    st = ctx._lib.tgaf_kv_append(ctx._h, cache._h, seqs, tag, *k_args, *v_args)
    if st:
        ctx._check(st)


def kv_read(ctx: Context, cache: KvCache, table, lens, cu=None, total: int | None = None, dtype=None, out=None):
    """The rows that kv_append with the same table, lens and cu wrote, read back: (k, v), each [total, kv_heads, head_dim],
    bf16 (default) or f32 (tgaf_kv_read).  total: rows of the call, needed unless `out` = (k, v) is given; whole sequences
    are cu = cumulated lens.  Rows that lie in no sequence are left as they were (undefined in new tensors)."""
    if _BF16 is None:
        _torch()
    if cache.ctx.device != ctx.device:
        _other_device(ctx, cache)
    if out is None:
        if total is None:
            _refuse("total (or out) is needed")
        tag, rows = DTYPE_BF16 if dtype is None else _tag("dtype", dtype), _count("total", total)
        seqs = _seqs(ctx, table, lens, cu, rows)
        k, v = cache.scales.new_empty((2, rows, cache.kv_heads, cache.head_dim), dtype=dtype or _BF16).unbind(0)
        at, step = k.data_ptr(), cache.kv_heads * cache.head_dim
        k_args, v_args = (at, step, cache.head_dim), (v.data_ptr(), step, cache.head_dim)
    else:
        k, v = out
        tag = _tag("out", k.dtype)
        rows, k_args = _rows(ctx, "out k", k, cache.kv_heads, cache.head_dim, True)
        v_rows, v_args = _rows(ctx, "out v", v, cache.kv_heads, cache.head_dim, True)
        if v.dtype is not k.dtype or v_rows != rows or (total is not None and total != rows):
            _refuse("out k and v must have one dtype and `total` rows")
        if k_args[0] == v_args[0] and rows:
            _refuse("out k and v must not be one tensor")
        seqs = _seqs(ctx, table, lens, cu, rows)
    st = ctx._lib.tgaf_kv_read(ctx._h, cache._h, seqs, tag, *k_args, *v_args)
    if st:
        ctx._check(st)
    return k, v


def _attend(ctx: Context, cache: KvCache, q, prefix_at, prefix_len: int, table, lens, cu, max_new, scale, out):
    if cache.ctx.device != ctx.device:
        _other_device(ctx, cache)
    tag = _tag("q", q.dtype)
    heads, head_dim = q.shape[1] if q.dim() == 3 else 0, cache.head_dim
    if heads == 0 or heads % cache.kv_heads:
        _refuse(f"q must be [tokens, heads, {head_dim}] with heads a multiple of {cache.kv_heads}, got {tuple(q.shape)}")
    total, q_args = _rows(ctx, "q", q, heads, head_dim)
    seqs = _seqs(ctx, table, lens, cu, total)
    if max_new is None:
        if cu is not None:
            _refuse("max_new is needed with cu")
        max_new = total // max(1, seqs.batch)
    else:
        max_new = _count("max_new", max_new, 1 if total else 0)
    if out is None:
        out = q.new_empty((total, heads, head_dim))
        out_args = (out.data_ptr(), heads * head_dim, head_dim)
    else:
        out_rows, out_args = _rows(ctx, "out", out, heads, head_dim, True)
        if out.dtype is not q.dtype or out_rows != total:
            _refuse(f"out must be {q.dtype} with {total} rows")
    if total == 0:
        return out
    scale = head_dim ** -0.5 if scale is None else scale
    if prefix_at is None:
        st = ctx._lib.tgaf_attention(ctx._h, cache._h, seqs, tag, *q_args, heads, max_new, scale, *out_args)
    else:
        st = ctx._lib.tgaf_attention_shared_prefix(ctx._h, cache._h, prefix_at, prefix_len, seqs, tag, *q_args, heads, max_new, scale, *out_args)
    if st:
        ctx._check(st)
    return out


def attention(ctx: Context, cache: KvCache, q, table, lens, cu=None, max_new=None, scale=None, out=None):
    """Causal attention of the call's own tokens over their sequences' cached tokens (tgaf_attention).

    q: [tokens, heads, head_dim], bf16 or f32, any token and head strides; heads / kv_heads query heads share a cached head.
    The tokens' own K / V rows are appended first (`lens` counts them).  max_new: an upper bound of the own tokens of any
    sequence, needed with cu: the launch is sized by it, and it decides which kernel takes the call, so a close one is best.
    scale: default 1 / sqrt(head_dim).  Rows that see no key are 0.  `out` must not overlap q."""
    return _attend(ctx, cache, q, None, 0, table, lens, cu, max_new, scale, out)


def attention_shared_prefix(ctx: Context, cache: KvCache, q, prefix_table, prefix_len: int, table, lens, cu=None, max_new=None,
                            scale=None, out=None):
    """`attention` for sequences that all continue one shared prefix of `prefix_len` tokens in the pages `prefix_table`
    (int32 [pages], on the device); table and lens do not count the prefix (tgaf_attention_shared_prefix).  Its pages are read
    once for 256 rows of a cached head (at most 32 in small calls, 16 in f32) instead of once per sequence; head sizes other
    than 64 and 128 read them for every row.  Calls of more than some 16 k rows (tokens x heads of 128): see `attention_reserve`."""
    _tag("q", q.dtype)
    if prefix_table.dtype is not _I32 or prefix_table.dim() != 1 or not prefix_table.is_contiguous():
        _refuse(f"prefix_table must be contiguous int32 [pages], got {prefix_table.dtype} {tuple(prefix_table.shape)}")
    prefix_len = _count("prefix_len", prefix_len)
    if prefix_len > prefix_table.shape[0] * cache.page_tokens:
        _refuse(f"prefix_len {prefix_len} does not fit {prefix_table.shape[0]} pages of {cache.page_tokens} tokens")
    if prefix_table.get_device() != ctx.device:
        _refuse(f"prefix_table must be on cuda:{ctx.device}, got {prefix_table.device}")
    return _attend(ctx, cache, q, prefix_table.data_ptr(), prefix_len, table, lens, cu, max_new, scale, out)


def attention_reserve(ctx: Context, cache: KvCache, rows: int) -> None:
    """Makes the context's workspace large enough for `attention_shared_prefix` calls of up to `rows` = tokens x heads rows
    (tgaf_attention_reserve): in front of a capture of such calls, or so that the first of them need not wait for it."""
    if cache.ctx.device != ctx.device:
        _other_device(ctx, cache)
    rows = _count("rows", rows, 0, 2 ** 31 - 1)
    ctx._check(ctx._lib.tgaf_attention_reserve(ctx._h, cache._h, rows))
