"""The attention kernels against bounds that follow from their roundings, row by row and value by value (kv_bounds)."""
import math

import pytest
import torch

import kv_bounds
from test_kv_cache import claim, cumulate, ctx, dev, filled_cache, make_tables  # noqa: F401

gpu = pytest.mark.gpu


def worst(out, want, bound):
    """Largest error in units of its bound; NaN counts as infinite."""
    return ((out.double() - want).abs() / (bound + 1e-300)).nan_to_num(nan=math.inf).max().item()


def check(ctx, cache, q, table, lens, cu, wide, **kw):  # noqa: F811
    """Within the bound everywhere; and the bound is worth something: results of zero would miss it somewhere in every head."""
    import talu_b200 as gaf
    prefix = [kw.get("prefix_table"), kw.get("prefix_len", 0)]
    call = dict(cu=dev(cu), max_new=max(b - a for a, b in zip(cu, cu[1:])), scale=kw.get("scale"))
    if prefix[1]:
        out = gaf.attention_shared_prefix(ctx, cache, q, *prefix, table, dev(lens), **call)
    else:
        out = gaf.attention(ctx, cache, q, table, dev(lens), **call)
    ctx.synchronize()
    want, bound = kv_bounds.attention(cache, q, table, lens, cu, wide, **kw)
    out = out[:cu[-1]]
    assert bool((bound < 0.1 * want.abs()).any(-1).any(0).all())
    most = worst(out, want, bound)
    assert most <= 1.0
    return out, want, bound


@gpu
@pytest.mark.parametrize("dim, bits, group", [(64, 8, 64), (64, 4, 32), (128, 8, 32), (128, 4, 128), (128, 8, 64)])
@pytest.mark.parametrize("rise", [6.5, 12.0, -6.5])
def test_scores_that_rise_from_chunk_to_chunk(ctx, dim, bits, group, rise):  # noqa: F811
    """Scores rise by more than 8 (base 2: 6.5 natural ones are 9.4) from every 32 keys to the next, so that each chunk of a
    unit rescales what the chunks before it have left; falling, and in steps that leave the earlier chunks a share."""
    import talu_b200 as gaf
    n, new, kv_heads, per_kv, page = 330, 70, 2, 4, 32
    table, pages, _ = make_tables([n], page, 1)
    cache = gaf.KvCache.allocate(ctx, pages, kv_heads, dim, page, bits, group)
    gen = torch.Generator(device="cuda").manual_seed(4)
    # one direction for q; a key's part along it sets its score
    unit = torch.where(torch.rand(dim, generator=gen, device="cuda") < 0.5, -1.0, 1.0)
    step = rise * (torch.arange(n, device="cuda") // 32)
    step = step + rise * 0.35 * (torch.arange(n, device="cuda") % 32 == 5)      # one key of each chunk well above the others
    k = 0.02 * torch.randn(n, kv_heads, dim, generator=gen, device="cuda") + (step / math.sqrt(dim))[:, None, None] * unit
    v = torch.randn(n, kv_heads, dim, generator=gen, device="cuda")
    v = v * torch.exp2(-9.4 * ((n - 1 - torch.arange(n, device="cuda")) // 32 < 1))[:, None, None] if rise > 0 else v
    gaf.kv_append(ctx, cache, k.bfloat16(), v.bfloat16(), table, dev([n]))
    q = (unit * (1 + 0.02 * torch.randn(new, kv_heads * per_kv, dim, generator=gen, device="cuda"))).bfloat16()
    check(ctx, cache, q, table, [n], [0, new], True)
