"""Plain 64-bit forms of the quantised KV cache's operators, on any device, for the tests."""
from __future__ import annotations

import math

import torch


def quantise_f32(x, bits, group):
    """Codes, scales and biases of the quantiser's definition, evaluated in f32 on the CPU."""
    most = float(2 ** bits - 1)
    g = x.float().cpu().unflatten(-1, (-1, group))
    lo, hi = g.amin(-1), g.amax(-1)
    b = lo.to(torch.bfloat16)
    s = ((hi * 0.5 - lo * 0.5) * (torch.ones(()) / torch.tensor(most * 0.5))).to(torch.bfloat16)
    s = torch.where(s.float() < torch.finfo(torch.float32).tiny, torch.zeros_like(s), s)
    half = (s.float() * 0.5).unsqueeze(-1)
    q = ((g * 0.5 - b.float().unsqueeze(-1) * 0.5) / torch.where(half > 0, half, 1.0)).round().clamp(0.0, most)
    q = torch.where(half > 0, q, 0.0)
    return q.flatten(-2).to(torch.uint8), s, b


def pack(q, bits):
    if bits == 4:
        q = q[..., 0::2] | (q[..., 1::2] << 4)
    return q.contiguous().view(torch.int32)


def codes(packed, bits):
    shift = torch.arange(0, 32, bits, device=packed.device)
    return ((packed.long().unsqueeze(-1) >> shift) & (2 ** bits - 1)).flatten(-2)


def values(cache, table, n, which):
    """The first n tokens of one block table in 64 bits: (value, value without its bias) [kv_heads, n, head_dim]."""
    page = cache.page_tokens
    pages = table[:-(-n // page)].long()
    q = codes(cache.packed[pages, which], cache.bits).double()
    s, b = (t.view(torch.bfloat16)[pages, which].double().repeat_interleave(cache.group, -1) for t in (cache.scales, cache.biases))
    flat = lambda x: x.transpose(0, 1).reshape(cache.kv_heads, -1, cache.head_dim)[:, :n]  # noqa: E731
    return flat(q * s + b), flat(q * s)


def attention(cache, q, table, lens, cu, prefix_table=None, prefix_len=0, scale=None):
    """(out, weighted absolute values) in 64 bits: the second is what roundings of the weights are relative to."""
    out, mass = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    scale = 1.0 / math.sqrt(cache.head_dim) if scale is None else scale
    for b in range(len(lens)):
        n, m = max(0, lens[b]), cu[b + 1] - cu[b]
        if m == 0:
            continue
        parts = [(table[b], n)] if n else []
        if prefix_len:
            parts.insert(0, (prefix_table, prefix_len))
        if not parts:
            continue
        k = torch.cat([values(cache, t, c, 0)[0] for t, c in parts], 1)
        v, vs = (torch.cat(x, 1) for x in zip(*[values(cache, t, c, 1) for t, c in parts]))
        j = torch.arange(prefix_len + n, device=q.device)
        last = prefix_len + lens[b] - m + torch.arange(m, device=q.device)
        seen = j <= last[:, None]
        if prefix_len:
            seen |= j < prefix_len
        x = q[cu[b]:cu[b + 1]].double().unflatten(1, (cache.kv_heads, -1)).permute(1, 2, 0, 3)
        w = torch.einsum("hgmd,hnd->hgmn", x, k) * scale
        w = w.masked_fill(~seen, -math.inf)
        w = torch.where(seen.any(-1, keepdim=True), torch.softmax(w, -1), 0.0)
        out[cu[b]:cu[b + 1]] = torch.einsum("hgmn,hnd->mhgd", w, v).flatten(1, 2)
        mass[cu[b]:cu[b + 1]] = torch.einsum("hgmn,hnd->mhgd", w, vs.abs() + v.abs()).flatten(1, 2)
    return out, mass
