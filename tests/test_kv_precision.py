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
    """Within the bound everywhere; and the bound is worth something: results of zero, or of twice the size, would miss it in every
    head."""
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
    assert bool((bound < 0.5 * want.abs()).any(-1).any(0).all())
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


def scaled_groups(cache, table, lens, seed, by_key):
    """A claimed cache whose value groups differ in size: by 2^-10, 2^-16 and 2^-20 of the first inside every row, or by a power of
    two between 2^0 and 2^-20 drawn for every key and group."""
    claim(cache, table, lens, seed)
    shape = cache.scales[:, 1].shape
    if by_key:
        gen = torch.Generator(device="cuda").manual_seed(seed)
        e = -torch.randint(0, 21, shape, generator=gen, device="cuda").float()
    else:
        e = torch.tensor([0.0, -16.0, -20.0, -10.0], device="cuda")[:shape[-1]].expand(shape)
    for t in (cache.scales, cache.biases):
        t[:, 1] *= torch.exp2(e).bfloat16()


@gpu
@pytest.mark.parametrize("dtype, new", [(torch.bfloat16, 1), (torch.bfloat16, 5), (torch.bfloat16, 40), (torch.float32, 1), (torch.float32, 5), (torch.float32, 40)])
@pytest.mark.parametrize("dim, bits, group", [(64, 8, 32), (64, 4, 32), (128, 8, 32), (128, 4, 64), (128, 8, 64), (96, 8, 32)])
@pytest.mark.parametrize("by_key", [False, True])
def test_groups_of_different_size(ctx, dtype, new, dim, bits, group, by_key):  # noqa: F811
    """Every group of a value row to its own precision, however large its neighbours are."""
    lens, kv_heads, per_kv = [701, 90, 40], 2, 4 if new == 1 else 3
    table, pages, _ = make_tables(lens, 32, 1)
    cache = filled_cache(ctx, pages, kv_heads, dim, 32, bits, group)
    scaled_groups(cache, table, lens, 3, by_key)
    cu = [0, new, 2 * new, 3 * new]
    q = torch.randn(cu[-1], kv_heads * per_kv, dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(dtype)
    wide = kv_bounds.takes_wide(q, cache, new * per_kv, len(lens))
    out, want, bound = check(ctx, cache, q, table, lens, cu, wide, top=6 if wide else 4)
    # the whole of each group: roundings of single weights are independent
    err, size = ((x.unflatten(-1, (-1, group)) ** 2).sum((0, 1, 3)).sqrt() for x in (out.double() - want, want))
    assert bool((err <= (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -18) * size).all())


@gpu
@pytest.mark.parametrize("dim, bits, new, dtype", [(128, 8, 40, torch.bfloat16), (64, 4, 40, torch.bfloat16), (128, 8, 1, torch.bfloat16), (128, 4, 1, torch.float32)])
@pytest.mark.parametrize("below", [18.4, 22.2, 25.3])
def test_a_long_tail_behind_one_key(ctx, dtype, dim, bits, new, below):  # noqa: F811
    """One key takes nearly all the weight and has values of zero; what counts are 40000 others, each 2^-18 to 2^-25 of it.  As many
    sequences (of the same pages) as it takes to keep each in one piece: the parts of a cut one have references of their own."""
    import talu_b200 as gaf
    n, batch, kv_heads, per_kv, page = 40000, 40, 8, 2, 64
    table, pages, _ = make_tables([n], page, 1)
    cache = gaf.KvCache.allocate(ctx, pages, kv_heads, dim, page, bits, 64)
    gen = torch.Generator(device="cuda").manual_seed(4)
    unit = torch.where(torch.rand(dim, generator=gen, device="cuda") < 0.5, -1.0, 1.0)
    k = torch.zeros(n, kv_heads, dim, device="cuda")
    k[3] = unit * below * math.log(2.0) / math.sqrt(dim)
    v = 1 + 0.1 * torch.randn(n, kv_heads, dim, generator=gen, device="cuda")
    v[3] = 0
    gaf.kv_append(ctx, cache, k.bfloat16(), v.bfloat16(), table, dev([n]))
    flips = torch.rand(new, kv_heads * per_kv, dim, generator=gen, device="cuda") < 0.015
    q = torch.where(flips, -unit, unit).to(dtype)
    wide = kv_bounds.takes_wide(q, cache, new * per_kv, batch)
    _, want, bound = check(ctx, cache, q, table, [n], [0, new], wide, top=6 if wide else 4)
    out = gaf.attention(ctx, cache, q.repeat(batch, 1, 1), table.expand(batch, -1).contiguous(), dev([n] * batch))
    ctx.synchronize()
    assert max(worst(x, want, bound) for x in out.split(new)) <= 1.0


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("dim, group", [(128, 64), (64, 32), (96, 32)])
@pytest.mark.parametrize("k_size, v_size, q_size, scale", [(1e-12, 1e-9, 1.0, 1e11), (1e30, 1e30, 1e-30, 0.1), (1.0, 1e20, 0.0, 1.0), (1.0, 1.0, 30.0, 1.0),
                                                         (1.0, 1.0, 1.0, -0.3), (1.0, 1.0, 1.0, 0.0), (30.0, 1e-6, 3e4, 1e-4)])
def test_sizes_and_scales(ctx, dtype, new, dim, group, k_size, v_size, q_size, scale):  # noqa: F811
    """Values of any size that f32 sums hold, scores in the hundreds, scale of either sign or zero, q of zeros: by rows, each to
    the bound of its own scores, so that scores in the hundreds are checked as well as others."""
    lens, kv_heads = [150, 700], 2
    table, pages, _ = make_tables(lens, 32, 7)
    cache = filled_cache(ctx, pages, kv_heads, dim, 32, 8, group)
    claim(cache, table, lens)
    for t in (cache.scales, cache.biases):
        t[:, 0] *= k_size
        t[:, 1] *= v_size
    gen = torch.Generator(device="cuda").manual_seed(3)
    q = (torch.randn(2 * new, 4 * kv_heads, dim, device="cuda", generator=gen) * q_size).to(dtype)
    wide = kv_bounds.takes_wide(q, cache, 4 * new, 2)
    check(ctx, cache, q, table, lens, cumulate([new, new]), wide, scale=scale, top=6 if wide else 4)


@gpu
@pytest.mark.parametrize("dtype, new", [(torch.bfloat16, 1), (torch.bfloat16, 40), (torch.float32, 5)])
@pytest.mark.parametrize("v_size", [2.0 ** -45, 2.0 ** -60, 2.0 ** -74])
def test_small_values(ctx, dtype, new, v_size):  # noqa: F811
    """Values far below one, in a whole cache and in every other page beside ordinary ones: sums of weights and weighted values
    stay in range."""
    lens, kv_heads, dim = [150, 700], 2, 128
    table, pages, _ = make_tables(lens, 32, 7)
    cache = filled_cache(ctx, pages, kv_heads, dim, 32, 8, 64)
    claim(cache, table, lens)
    for t in (cache.scales, cache.biases):
        t[:, 1] *= v_size
    q = torch.randn(2 * new, 4 * kv_heads, dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).to(dtype)
    wide = kv_bounds.takes_wide(q, cache, 4 * new, 2)
    check(ctx, cache, q, table, lens, cumulate([new, new]), wide, top=6 if wide else 4)
    for t in (cache.scales, cache.biases):
        t[table[1, ::2].long(), 1] *= 1 / v_size
    check(ctx, cache, q, table, lens, cumulate([new, new]), wide, top=6 if wide else 4)


@gpu
@pytest.mark.parametrize("dtype, new", [(torch.bfloat16, 1), (torch.bfloat16, 30), (torch.float32, 2)])
@pytest.mark.parametrize("dim, bits, group", [(64, 8, 32), (128, 4, 64), (128, 8, 128), (96, 8, 32)])
@pytest.mark.parametrize("prefix", [1, 333])
def test_shared_prefix_to_the_bound(ctx, dtype, new, dim, bits, group, prefix):  # noqa: F811
    """Prefix and own pass together, groups of different size in both, rows that see the prefix alone."""
    lens, news, kv_heads, per_kv = [300, 0, 31, 64], [new, 2, min(31, new), new], 2, 3
    table, pages, _ = make_tables(lens + [prefix], 32, 1)
    cache = filled_cache(ctx, pages, kv_heads, dim, 32, bits, group)
    scaled_groups(cache, table, lens + [prefix], 3, True)
    cu = cumulate(news)
    q = torch.randn(cu[-1], kv_heads * per_kv, dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(dtype)
    most = max(news) * per_kv
    wide = [kv_bounds.takes_wide(q, cache, most, len(lens)), kv_bounds.takes_wide(q, cache, cu[-1] * per_kv, 1, True)]
    head = table[-1, :-(-prefix // 32)].contiguous()
    kw = dict(prefix_table=head, prefix_len=prefix)
    if all(wide) or not any(wide):
        check(ctx, cache, q, table[:-1], lens, cu, wide[0], top=6 if wide[0] else 4, **kw)
    else:                                   # one pass on either kernel: off by the sum of both bounds at most
        import talu_b200 as gaf
        out = gaf.attention_shared_prefix(ctx, cache, q, head, prefix, table[:-1], dev(lens), cu=dev(cu), max_new=max(news))
        ctx.synchronize()
        (want, a), (_, b) = (kv_bounds.attention(cache, q, table[:-1], lens, cu, w, top=4, **kw) for w in (True, False))
        assert worst(out, want, a + b) <= 1.0
