"""What the roundings of the attention kernels may put their results off by, per row and value, in 64 bits.

Notation: key j of a sequence, group g of value d, code c centred by h = 2^(bits - 1), scale s, z = b + h s the group's centre, so that a
stored value is s (c - h) + z; y scores, w weights of the softmax, o results.  Types round by half a step: f32 2^-24, f16 2^-11
(subnormals: 2^-25 absolute), bf16 2^-8 of the value.  Accumulators of the tensor cores may cut instead of round: 2^-23.

A score that is off by e_j multiplies its weight by exp(e_j).  Since sum_j w_j (v_j - o) = 0, o moves by
sum_j w_j (exp(e_j) - 1) (v_j - o) / sum_j w_j exp(e_j), which is at most sum_j w_j (exp(|e_j|) - 1) |v_j - o| / sum_j w_j exp(-|e_j|).
(|v_j - o| is taken for |v_j| + |o| where its table would be large.)

f32 scores (all kernels): q, the codes and the products are exact or in two f16 terms (2^-22); what is left are the sums of D terms and
the factor and the reference applied to them: (D + 16) 2^-24 of the absolute terms, and 2^-22 of 1 + |y| with exp2's own.
tcgen05 kernel: key elements are f16 of fma(c - h, s, f16(z)).  The centres' roundings add up along a group, 2^-11 |z sum_g q|; those
of the elements to 2^-11 sum |q k| at most: a key whose elements are of one size has one rounding error in all of them, so that
they cannot be taken for independent.
Its values are rounded alike, 2^-11 (|v| + |z|), its weights by 2^-11; elements below 2^-39 of the largest of 32 keys are lost.
Register path: w s is one f16 (2^-11), or two (2^-22), times the exact centred code; w z is f32.
Weights below the normal f16 numbers are 2^-25 off, where the largest one of the row (w T, T: largest element of 32 keys), or of
the row and group (w s), is 2^top at least.
Sums of n keys: n / 16 accumulations by the tensor cores, 16 further ones.
"""
import math

import torch

import kv_reference as ref


def _parts(cache, parts, which):
    """(s (c - h), z, s) by value of the tokens of all parts [(block table, tokens)], each [kv_heads, n, head_dim]."""
    out = []
    for table, n in parts:
        value, code = ref.values(cache, table, n, which)
        s = cache.scales.view(torch.bfloat16)[table[:-(-n // cache.page_tokens)].long(), which].double().repeat_interleave(cache.group, -1)
        s = s.transpose(0, 1).reshape(cache.kv_heads, -1, cache.head_dim)[:, :n]
        z = value - code + s * 2 ** (cache.bits - 1)
        out.append((value - z, z, s))
    return [torch.cat(t, 1) for t in zip(*out)]


def _sequence(cache, x, parts, seen, scale, f32, wide, top):
    """(o, bound) of one sequence: x [kv_heads, heads, rows, D] 64 bits, parts [(table, n)], seen [rows, n]."""
    D, group = cache.head_dim, cache.group
    (kc, kz, _), (vc, vz, vs) = _parts(cache, parts, 0), _parts(cache, parts, 1)
    k, v = kc + kz, vc + vz
    n = k.shape[1]
    y = torch.einsum("hgmd,hnd->hgmn", x, k) * scale
    w = torch.softmax(y.masked_fill(~seen, -math.inf), -1)
    w = torch.where(seen.any(-1, keepdim=True), w, 0.0)
    mass = lambda t: torch.einsum("hgmn,hnd->hgmd", w, t.abs())  # noqa: E731
    o = torch.einsum("hgmn,hnd->hgmd", w, v)

    off = (D + 16) * 2.0 ** -24 * abs(scale) * torch.einsum("hgmd,hnd->hgmn", x.abs(), kc.abs() + kz.abs()) + 2.0 ** -22 * (1 + y.abs())
    if wide:
        sums = x.unflatten(-1, (-1, group)).sum(-1).abs()
        centres = kz.abs().unflatten(-1, (-1, group))[..., 0]
        off = off + abs(scale) * 2.0 ** -11 * (torch.einsum("hgmd,hnd->hgmn", sums, centres) + torch.einsum("hgmd,hnd->hgmn", x.abs(), k.abs()))
    least = (w * torch.exp(-off)).sum(-1, keepdim=True).clamp(min=1e-300)
    off = w * torch.expm1(off.clamp(max=30.0))
    if w.numel() * D <= 2 ** 27:
        away = torch.stack([(v[:, None] - o[..., i, None, :]).abs() for i in range(x.shape[2])], 2)      # [h, g, m, n, d]
        bound = torch.einsum("hgmn,hgmnd->hgmd", off, away)
    else:
        bound = torch.einsum("hgmn,hnd->hgmd", off, v.abs()) + off.sum(-1, keepdim=True) * o.abs()
    bound = bound / least

    bound = bound + (n / 16 + 16) * 2.0 ** -23 * (mass(vc) + mass(vz) + o.abs())
    if wide:
        bound = bound + 2.0 ** -11 * (2 * mass(v) + mass(vz))
        size, at = [], 0
        for _, m in parts:
            t = torch.nn.functional.pad((vc.abs() + vz.abs())[:, at:at + m], (0, 0, 0, -m % 32))
            size.append(t.unflatten(1, (-1, 32)).amax((2, 3)).repeat_interleave(32, 1)[:, :m])
            at += m
        size = w * torch.cat(size, 1)[:, None, None]
        bound = bound + (2.0 ** -39 * size.sum(-1) + n * 2.0 ** (-25 - top) * size.amax(-1)).unsqueeze(-1)
    else:
        bound = bound + (2.0 ** -22 if f32 else 2.0 ** -11) * mass(vc)
        largest = torch.stack([(w * vs[:, None, None, :, i].abs()).amax(-1) for i in range(0, D, group)], -1)
        bound = bound + n * 2.0 ** (-25 - top) * 2.0 ** (cache.bits - 1) * largest.repeat_interleave(group, -1)
    return o, bound


def takes_wide(q, cache, rows, sequences, prefix=False):
    """Whether the tcgen05 kernel takes a call of that many rows per cached head and sequence (narrow_rows in gaf_kv.cu)."""
    few = sequences * cache.kv_heads < torch.cuda.get_device_properties(0).multi_processor_count
    most = (24 if not few else 16 if prefix else 8) if cache.head_dim == 128 else 16 if few else 32
    return q.dtype == torch.bfloat16 and cache.head_dim in (64, 128) and rows > most


def attention(cache, q, table, lens, cu, wide, prefix_table=None, prefix_len=0, scale=None, top=0):
    """(o, bound), each [tokens, heads, D] in 64 bits; rows that lie in no sequence are zero with a bound of zero.
    wide: the tcgen05 kernel takes the call (bf16 and many rows).  top: see above."""
    scale = 1.0 / math.sqrt(cache.head_dim) if scale is None else scale
    o, bound = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    for b, n in enumerate(lens):
        m, mine = cu[b + 1] - cu[b], slice(cu[b], cu[b + 1])
        parts = ([(prefix_table, prefix_len)] if prefix_len else []) + ([(table[b], n)] if n > 0 else [])
        if m == 0 or not parts:
            continue
        seen = torch.arange(max(0, n), device=q.device) <= n - m + torch.arange(m, device=q.device)[:, None]
        seen = torch.cat((seen.new_ones(m, prefix_len), seen), 1)
        x = q[mine].double().unflatten(1, (cache.kv_heads, -1)).permute(1, 2, 0, 3)
        y, t = _sequence(cache, x, parts, seen, scale, q.dtype == torch.float32, wide, top)
        o[mine], bound[mine] = (u.permute(2, 0, 1, 3).flatten(1, 2) for u in (y, t))
    if q.dtype == torch.bfloat16:
        bound = bound * (1 + 2.0 ** -8) + 2.0 ** -8 * o.abs()
    return o, bound
