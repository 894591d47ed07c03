"""The quantised KV cache (tgaf_kv_*) and its attention (tgaf_attention*) against plain 64-bit forms."""
import ctypes as C
import math
import random

import pytest
import torch

import kv_reference as ref

gpu = pytest.mark.gpu


# ---- refusals: everything that the host can see -----------------------------------------------------------------------

class _FakeLib:
    def __getattr__(self, name):
        raise AssertionError(f"{name} was called: the arguments should have been refused before")


class _FakeCtx:
    """Stands for a context whose device tensors are on the CPU: the checks run, no call may come through."""
    _lib, _h = _FakeLib(), 1

    def __init__(self, device=-1):         # -1: what a tensor on the CPU gives as its device's index
        self.device = device


@pytest.fixture
def fake():
    from talu_b200 import kv
    packed = torch.zeros(4, 2, 2, 16, 16, dtype=torch.int32)
    scales = torch.zeros(4, 2, 2, 16, 1, dtype=torch.bfloat16)
    return kv.KvCache(_FakeCtx(), None, packed, scales, scales, 64, 8)


def _args(tokens=3, heads=2, dim=64, batch=3):
    return (torch.zeros(tokens, heads, dim, dtype=torch.bfloat16), torch.zeros(batch, 2, dtype=torch.int32),
            torch.zeros(batch, dtype=torch.int32))


@pytest.mark.parametrize("change", [
    dict(x=torch.zeros(3, 2, 64, dtype=torch.float16)),
    dict(x=torch.zeros(3, 3, 64, dtype=torch.bfloat16)),
    dict(x=torch.zeros(3, 2, 32, dtype=torch.bfloat16)),
    dict(x=torch.zeros(3, 128, dtype=torch.bfloat16)),
    dict(x=torch.zeros(3, 2, 128, dtype=torch.bfloat16)[:, :, ::2]),
    dict(x=torch.zeros(4, 2, 64, dtype=torch.bfloat16)),                        # 4 rows, 3 sequences, no cu
    dict(table=torch.zeros(3, 2, dtype=torch.int64)),
    dict(table=torch.zeros(3, dtype=torch.int32)),
    dict(table=torch.zeros(2, 3, dtype=torch.int32).t()),
    dict(lens=torch.zeros(2, dtype=torch.int32)),
    dict(lens=torch.zeros(3, dtype=torch.int64)),
    dict(lens=torch.zeros(6, dtype=torch.int32)[::2]),
    dict(cu=torch.zeros(3, dtype=torch.int32)),
    dict(cu=torch.zeros(4, dtype=torch.int64)),
])
def test_bad_rows_and_tables_are_refused(fake, change):
    from talu_b200 import GafError, attention, kv_append, kv_read
    x, table, lens = _args()
    x, table, lens, cu = change.get("x", x), change.get("table", table), change.get("lens", lens), change.get("cu")
    with pytest.raises(GafError) as e:
        kv_append(fake.ctx, fake, x, x, table, lens, cu=cu)
    assert e.value.invalid_argument
    if not (x.dim() == 3 and x.shape[1] == 3):
        with pytest.raises(GafError):
            attention(fake.ctx, fake, x, table, lens, cu=cu, max_new=3 if cu is not None else None)
    with pytest.raises(GafError):
        kv_read(fake.ctx, fake, table, lens, cu=cu, out=(x, x))


def test_bad_outputs_and_bounds_are_refused(fake):
    from talu_b200 import GafError, attention, attention_shared_prefix, kv_append, kv_read
    x, table, lens = _args()
    cu = torch.zeros(4, dtype=torch.int32)
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    bad = [
        lambda: kv_append(fake.ctx, fake, x, x.float(), table, lens),
        lambda: kv_append(fake.ctx, fake, x, x[:2], table, lens),
        lambda: kv_read(fake.ctx, fake, table, lens),
        lambda: kv_read(fake.ctx, fake, table, lens, total=3, dtype=torch.float16),
        lambda: kv_read(fake.ctx, fake, table, lens, total=4, out=(x, x.clone())),
        lambda: kv_read(fake.ctx, fake, table, lens, out=(x[:1].expand(3, 2, 64), x)),
        lambda: attention(fake.ctx, fake, torch.zeros(3, 3, 64, dtype=torch.bfloat16), table, lens),   # 3 heads on 2
        lambda: attention(fake.ctx, fake, q, table, lens, cu=cu),                                      # max_new is missing
        lambda: attention(fake.ctx, fake, q, table, lens, out=q.float()),
        lambda: attention(fake.ctx, fake, q, table, lens, out=q[:, :1].expand(3, 4, 64)),
        lambda: attention_shared_prefix(fake.ctx, fake, q, torch.zeros(2, dtype=torch.int32), 33, table, lens),
        lambda: attention_shared_prefix(fake.ctx, fake, q, torch.zeros(2, dtype=torch.int32), -1, table, lens),
        lambda: attention_shared_prefix(fake.ctx, fake, q, torch.zeros(2, dtype=torch.int64), 8, table, lens),
    ]
    for call in bad:
        with pytest.raises(GafError) as e:
            call()
        assert e.value.invalid_argument


@pytest.mark.parametrize("bits, group, words, groups", [(5, 64, 16, 1), (8, 16, 16, 4), (8, 64, 16, 2), (4, 64, 16, 1)])
def test_bad_caches_are_refused(bits, group, words, groups):
    from talu_b200 import GafError, KvCache
    with pytest.raises(GafError):
        KvCache.wrap_device(_FakeCtx(), torch.zeros(4, 2, 2, 16, words, dtype=torch.int32),
                            torch.zeros(4, 2, 2, 16, groups, dtype=torch.bfloat16),
                            torch.zeros(4, 2, 2, 16, groups, dtype=torch.bfloat16), group, bits)


def test_tensors_off_the_device_are_refused():
    from talu_b200 import GafError, KvCache, kv
    packed = torch.zeros(4, 2, 2, 16, 16, dtype=torch.int32)
    scales = torch.zeros(4, 2, 2, 16, 1, dtype=torch.bfloat16)
    with pytest.raises(GafError):
        KvCache.wrap_device(_FakeCtx(0), packed, scales, scales, 64, 8)
    cache = kv.KvCache(_FakeCtx(0), None, packed, scales, scales, 64, 8)
    x, table, lens = _args()
    with pytest.raises(GafError) as e:
        kv.kv_append(cache.ctx, cache, x, x, table, lens)
    assert "cuda:0" in e.value.message


def test_null_arguments_at_the_c_entries():
    from talu_b200 import _capi
    lib = _capi.load()
    h = C.c_void_p()
    assert lib.tgaf_kv_cache_wrap_device(None, 16, 16, 16, 1, 1, 16, 64, 64, 8, C.byref(h)) == 1
    assert lib.tgaf_kv_cache_wrap_device(None, 16, 16, 16, 1, 1, 16, 64, 64, 8, None) == 1
    assert lib.tgaf_kv_append(None, None, None, 1, None, 0, 0, None, 0, 0) == 1
    assert lib.tgaf_kv_read(None, None, None, 1, None, 0, 0, None, 0, 0) == 1
    assert lib.tgaf_attention(None, None, None, 1, None, 0, 0, 1, 1, 1.0, None, 0, 0) == 1
    assert lib.tgaf_attention_shared_prefix(None, None, None, 0, None, 1, None, 0, 0, 1, 1, 1.0, None, 0, 0) == 1
    assert lib.tgaf_kv_cache_free(None, None) == 0


# ---- on the GPU --------------------------------------------------------------------------------------------------------

@pytest.fixture(scope="module")
def ctx():
    import talu_b200 as gaf
    c = gaf.Context(0)
    yield c
    c.close()


def make_tables(lens, page, seed, spare=3):
    """Block tables over pages in random order, -1 behind each sequence's last page; the number of pages."""
    need = [-(-max(0, n) // page) for n in lens]
    order = list(range(sum(need) + spare))
    random.Random(seed).shuffle(order)
    table = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    return table.cuda(), sum(need) + spare, order


def filled_cache(ctx, pages, kv_heads, dim, page, bits, group, seed=0, garbage=True):
    """A cache of random quantised rows.  garbage: rows are NaN scales and biases until a sequence claims them."""
    import talu_b200 as gaf
    gen = torch.Generator(device="cuda").manual_seed(seed)
    cache = gaf.KvCache.allocate(ctx, pages, kv_heads, dim, page, bits, group)
    cache.packed.copy_(torch.randint(-2 ** 31, 2 ** 31, cache.packed.shape, generator=gen, device="cuda", dtype=torch.int64).int())
    if garbage:
        cache.scales.fill_(float("nan"))
        cache.biases.fill_(float("nan"))
    return cache


def claim(cache, table, lens, seed=1):
    """Gives every row that a sequence holds an ordinary scale and bias (the codes are random already)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shape = cache.scales.shape
    step = torch.rand(shape, generator=gen, device="cuda") * (6.0 / (2 ** cache.bits - 1)) + 0.2 / (2 ** cache.bits - 1)
    bias = -step * (2 ** cache.bits - 1) * (0.3 + 0.4 * torch.rand(shape, generator=gen, device="cuda"))
    for row, n in zip(table.tolist(), lens):
        for i in range(0, max(0, n), cache.page_tokens):
            p, m = row[i // cache.page_tokens], min(cache.page_tokens, n - i)
            cache.scales[p, :, :, :m] = step[p, :, :, :m].bfloat16()
            cache.biases[p, :, :, :m] = bias[p, :, :, :m].bfloat16()


def dev(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def cumulate(news):
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    return cu


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bits, group, dim, kv_heads, page", [(8, 64, 128, 8, 64), (4, 32, 64, 2, 16), (8, 32, 96, 3, 32),
                                                              (4, 128, 128, 1, 128), (4, 64, 64, 5, 256), (8, 128, 256, 2, 16)])
def test_append_then_read(ctx, dtype, bits, group, dim, kv_heads, page):
    """Codes, scales and biases are the definition's, bit for bit; other rows of the cache keep theirs; the values read back
    are q s + b rounded once, and off by half a step at most wherever the rounded scale reaches."""
    import talu_b200 as gaf
    lens, news = [1, 70, 0, 33, 300, 16], [1, 70, 0, 2, 41, 16]
    table, pages, _ = make_tables(lens, page, 3)
    cache = filled_cache(ctx, pages, kv_heads, dim, page, bits, group)
    cu = cumulate(news)
    tail = 2                                                   # rows behind the last sequence
    gen = torch.Generator(device="cuda").manual_seed(5)
    qkv = torch.randn(cu[-1] + tail, 3 * kv_heads, dim, generator=gen, device="cuda") * torch.exp(torch.randn(dim, generator=gen, device="cuda"))
    qkv[0, :, :group] = 0.75                                   # one value for a whole group
    qkv[1, :, :group] = 0.0
    qkv = qkv.to(dtype)
    k, v = qkv[:, kv_heads:2 * kv_heads], qkv[:, 2 * kv_heads:]
    before = [t.clone() for t in (cache.packed, cache.scales, cache.biases)]
    gaf.kv_append(ctx, cache, k, v, table, dev(lens), cu=dev(cu))
    out = [torch.full((cu[-1] + tail, kv_heads, dim), 7.0, dtype=torch.float32, device="cuda") for _ in range(2)]
    gaf.kv_read(ctx, cache, table, dev(lens), cu=dev(cu), out=out)
    low = gaf.kv_read(ctx, cache, table, dev(lens), cu=dev(cu), total=cu[-1] + tail)
    ctx.synchronize()
    want = [t.clone() for t in before]
    x = torch.stack((k, v), 1)
    q, s, b = ref.quantise_f32(x, bits, group)
    tab = table.cpu()
    for seq, (n, m) in enumerate(zip(lens, news)):
        for i in range(m):
            pos, t = n - m + i, cu[seq] + i
            p = int(tab[seq, pos // page])
            want[0][p, :, :, pos % page] = ref.pack(q[t], bits).cuda()
            want[1][p, :, :, pos % page] = s[t].cuda()
            want[2][p, :, :, pos % page] = b[t].cuda()
    for got, w in zip((cache.packed, cache.scales, cache.biases), want):
        assert torch.equal(got.view(torch.int16 if got.dtype == torch.bfloat16 else got.dtype), w.view(torch.int16 if w.dtype == torch.bfloat16 else w.dtype))
    wide = lambda z: z.repeat_interleave(group, -1)  # noqa: E731
    value = (q.double() * wide(s.double()) + wide(b.double())).float()      # exact in 64 bits, rounded once
    for i in range(2):
        assert torch.equal(out[i][:cu[-1]].cpu(), value[:cu[-1], i])
        assert (out[i][cu[-1]:] == 7.0).all()
        assert torch.equal(low[i][:cu[-1]].cpu(), value[:cu[-1], i].bfloat16())
    # half a step, or, at the top, what the rounded scale (2^-8 of itself a step, 2^bits - 1 steps) leaves; f32 minima are
    # rounded to bf16, which is 2^-8 of them
    most = 2 ** bits - 1
    bound = wide(s.double()) * (0.5 + most * 2.0 ** -8) * (1 + 2.0 ** -20) + (0 if dtype == torch.bfloat16 else 2.0 ** -8) * wide(b.double()).abs()
    err = (value.double() - x.double().cpu()).abs()[:cu[-1]]
    assert (err <= bound[:cu[-1]]).all()


@gpu
@pytest.mark.parametrize("bits", [4, 8])
def test_append_of_extreme_values(ctx, bits):
    """Largest and smallest finite values are stored; a group with an infinity or a NaN reads back as NaN, its neighbours not."""
    import talu_b200 as gaf
    dim, group = 128, 32
    cache = gaf.KvCache.allocate(ctx, 2, 1, dim, 16, bits, group)
    x = torch.randn(6, 1, dim, device="cuda")
    big = torch.finfo(torch.bfloat16).max
    x[0, 0, :group] = torch.linspace(-1, 1, group) * big
    x[1, 0, :group] = torch.linspace(-1, 1, group) * torch.finfo(torch.float32).tiny   # a step below the smallest normal
    x[2, 0, 5] = math.inf
    x[3, 0, 40] = -math.inf
    x[4, 0, 70] = math.nan
    for x in (x, x.bfloat16()):
        gaf.kv_append(ctx, cache, x, x, dev([[0]]), dev([6]))
        k, v = gaf.kv_read(ctx, cache, dev([[0]]), dev([6]), total=6, dtype=torch.float32)
        ctx.synchronize()
        assert torch.equal(k.isnan(), v.isnan())
        bad = torch.zeros(6, dim // group, dtype=torch.bool, device="cuda")
        bad[2, 0] = bad[3, 1] = bad[4, 2] = True
        assert torch.equal(k.isnan()[:, 0], bad.repeat_interleave(group, -1))
        step = 2 * big / (2 ** bits - 1)
        assert (k[0, 0, :group].double() - x[0, 0, :group].double()).abs().max() <= step * (0.5 + (2 ** bits - 1) * 2.0 ** -8)
        assert k[1, 0, :group].abs().max() <= torch.finfo(torch.float32).tiny


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_of_any_stride_and_alignment(ctx, dtype):
    import talu_b200 as gaf
    cache = gaf.KvCache.allocate(ctx, 4, 3, 64, 16, 8, 32)
    raw = torch.randn(3, 21, 67, device="cuda").to(dtype)          # [heads, tokens, odd pitch]
    k = raw[:, :20, 3:67].transpose(0, 1)
    v = raw[:, 1:, 1:65].transpose(0, 1)
    table, lens = dev([[2, 0]]), dev([20])
    gaf.kv_append(ctx, cache, k, v, table, lens)
    a = gaf.kv_read(ctx, cache, table, lens, total=20, dtype=dtype)
    wide = torch.zeros(3, 20, 65, device="cuda", dtype=dtype)
    b = (wide[:, :, 1:].transpose(0, 1), torch.zeros(20, 3, 64, device="cuda", dtype=dtype))
    gaf.kv_read(ctx, cache, table, lens, out=b)
    dense = gaf.KvCache.allocate(ctx, 4, 3, 64, 16, 8, 32)
    gaf.kv_append(ctx, dense, k.contiguous(), v.contiguous(), table, lens)
    ctx.synchronize()
    assert torch.equal(cache.packed, dense.packed) and torch.equal(cache.scales, dense.scales) and torch.equal(cache.biases, dense.biases)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and (wide[:, :, 0] == 0).all()


@gpu
def test_bad_tables_are_reported_and_skipped(ctx):
    """A table entry outside the cache or a length beyond the table: an error at the next synchronize, nothing written or seen."""
    import talu_b200 as gaf
    cache = gaf.KvCache.allocate(ctx, 3, 2, 64, 16, 8, 64)
    x = torch.randn(2, 2, 64, device="cuda").bfloat16()
    for table, lens in (([[0, 3], [1, 1]], [17, 3]), ([[0, -1], [1, 1]], [17, 3]), ([[0, 2], [1, 1]], [40, 3])):
        cache.scales.zero_()
        gaf.kv_append(ctx, cache, x, x, dev(table), dev(lens))
        with pytest.raises(gaf.GafError) as e:
            ctx.synchronize()
        assert e.value.status == 7 and "page" in e.value.message
        assert set(cache.scales.float().nonzero()[:, 0].tolist()) == {1}
        out = [torch.full((2, 2, 64), 7.0, device="cuda") for _ in range(2)]
        gaf.kv_read(ctx, cache, dev(table), dev(lens), out=out)
        with pytest.raises(gaf.GafError):
            ctx.synchronize()
        assert (out[0][0] == 7.0).all() and (out[0][1] != 7.0).all()
        y = gaf.attention(ctx, cache, torch.randn(2, 4, 64, device="cuda").bfloat16(), dev(table), dev(lens))
        with pytest.raises(gaf.GafError):
            ctx.synchronize()
        assert y.isfinite().all()
        ctx.synchronize()


def check_attention(ctx, cache, q, table, lens, cu, max_new, prefix_table=None, prefix_len=0, scale=None, cu_given=True):
    """Against 64 bits.  Each bf16 weight and each bf16 value w may be half a step, 2^-8 of itself, off (of the values'
    part without bias, or of the value), and the result is rounded once more; a score that is off by e changes all weights by
    a factor of e^(2e) at most.  f32 sums of n terms add n 2^-24 of their absolute terms."""
    import talu_b200 as gaf
    kw = {"cu": dev(cu) if cu_given else None, "max_new": max_new if cu_given else None, "scale": scale}
    out = torch.full((q.shape[0], q.shape[1] * cache.head_dim), 7.0, dtype=q.dtype, device="cuda").unflatten(1, (q.shape[1], -1))
    if prefix_table is None:
        gaf.attention(ctx, cache, q, table, dev(lens), out=out, **kw)
    else:
        gaf.attention_shared_prefix(ctx, cache, q, prefix_table, prefix_len, table, dev(lens), out=out, **kw)
    ctx.synchronize()
    want, mass = ref.attention(cache, q, table, lens, cu, prefix_table, prefix_len, scale)
    assert (out[cu[-1]:] == 7.0).all()
    out, want, mass = out[:cu[-1]].double(), want[:cu[-1]], mass[:cu[-1]]
    # bf16: 2^-8 of the weights, 2^-8 of the result and, where keys or values pass through bf16, twice 2^-8 again;
    # f32: 2^-16 of the weights (two bf16 halves) and sums
    tol = (2.0 ** -8 * (3 * mass + want.abs()) if q.dtype == torch.bfloat16 else 2.0 ** -15 * mass) + 1e-7
    worst = ((out - want).abs() / tol).max().item() if out.numel() else 0.0
    assert worst <= 1.0, worst
    if out.numel() and want.norm() > 0:
        # errors of single weights are independent: in the norm they cancel
        rel = ((out - want).norm() / want.norm()).item()
        assert rel <= (2.0 ** -8 if q.dtype == torch.bfloat16 else 2.0 ** -16), rel
    return out


SHAPES = [  # kv_heads, per_kv, dim, bits, group, page
    (8, 4, 128, 8, 64, 64), (2, 8, 128, 4, 64, 64), (2, 4, 64, 8, 32, 16), (1, 1, 128, 8, 128, 128), (3, 5, 64, 4, 32, 32),
    (2, 7, 128, 4, 32, 16), (1, 16, 128, 8, 32, 256), (2, 3, 64, 4, 64, 64), (2, 2, 96, 8, 32, 16), (1, 3, 256, 4, 128, 32),
    (4, 1, 128, 4, 128, 64), (1, 71, 64, 8, 64, 64), (2, 4, 32, 4, 32, 16)]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention_one_token(ctx, shape, dtype):
    """One new token each: lengths of zero and one, ends inside pages and at their borders, NaN in all rows behind the ends."""
    kv_heads, per_kv, dim, bits, group, page = shape
    lens = [1, 0, 15, 16, 17, 63, 64, 65, 129, 700]
    table, pages, _ = make_tables(lens, page, 1)
    cache = filled_cache(ctx, pages, kv_heads, dim, page, bits, group)
    claim(cache, table, lens)
    q = torch.randn(len(lens), kv_heads * per_kv, dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(dtype)
    out = check_attention(ctx, cache, q, table, lens, list(range(len(lens) + 1)), 1, cu_given=False)
    assert (out[1] == 0).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention_ragged(ctx, shape, dtype):
    """New tokens from none to whole prompts, more new tokens than cached ones, rows behind the last sequence, strided q."""
    kv_heads, per_kv, dim, bits, group, page = shape
    lens, news = [40, 7, 200, 3, 0, 131, 65], [3, 7, 0, 5, 2, 77, 1]
    table, pages, _ = make_tables(lens, page, 1)
    cache = filled_cache(ctx, pages, kv_heads, dim, page, bits, group)
    claim(cache, table, lens)
    cu = cumulate(news)
    heads = kv_heads * per_kv
    q = torch.randn(cu[-1] + 3, heads + 1, dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(dtype)[:, 1:]
    check_attention(ctx, cache, q, table, lens, cu, max(news))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("prefix", [1, 70, 1000])
def test_attention_shared_prefix(ctx, shape, dtype, prefix):
    kv_heads, per_kv, dim, bits, group, page = shape
    lens, news = [40, 1, 0, 3, 131, 65, 2], [3, 1, 0, 5, 2, 1, 2]
    table, pages, _ = make_tables(lens + [prefix], page, 1)
    cache = filled_cache(ctx, pages, kv_heads, dim, page, bits, group)
    claim(cache, table, lens + [prefix])
    cu = cumulate(news)
    prefix_table = table[-1, :-(-prefix // page)].contiguous()
    q = torch.randn(cu[-1] + 1, kv_heads * per_kv, dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(dtype)
    check_attention(ctx, cache, q, table[:-1], lens, cu, max(news), prefix_table, prefix)


@gpu
@pytest.mark.parametrize("shape", [(8, 4, 128, 8, 64, 64), (4, 8, 64, 4, 32, 16), (2, 2, 128, 4, 128, 128)])
def test_attention_of_prompts_over_long_caches(ctx, shape):
    """Hundreds of new tokens over a thousand cached ones: row tiles that start inside a token's heads, units and tiles at
    every kind of border, sequences that leave half of a row tile empty."""
    kv_heads, per_kv, dim, bits, group, page = shape
    lens, news = [1500, 64, 333, 1100], [300, 64, 1, 129]
    table, pages, _ = make_tables(lens, page, 7)
    cache = filled_cache(ctx, pages, kv_heads, dim, page, bits, group)
    claim(cache, table, lens)
    cu = cumulate(news)
    q = torch.randn(cu[-1], kv_heads * per_kv, dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).bfloat16()
    check_attention(ctx, cache, q, table, lens, cu, max(news))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("k_size, v_size, q_size, scale", [(1e-12, 1e-9, 1.0, 1e11), (1e30, 1e30, 1e-30, 0.1), (1.0, 1e20, 0.0, 1.0), (1.0, 1.0, 30.0, 1.0),
                                                         (1.0, 1.0, 1.0, -0.3), (1.0, 1.0, 1.0, 0.0), (30.0, 1e-6, 3e4, 1e-4)])
def test_attention_of_large_and_small_values(ctx, dtype, new, k_size, v_size, q_size, scale):
    """Values of any size that f32 sums hold, scores in the hundreds, scale of either sign or zero, q of zeros."""
    lens, news = [150, 700], [new, new]
    table, pages, _ = make_tables(lens, 32, 7)
    cache = filled_cache(ctx, pages, 2, 128, 32, 8, 64)
    claim(cache, table, lens)
    for t in (cache.scales, cache.biases):
        t[:, 0] *= k_size
        t[:, 1] *= v_size
    q = (torch.randn(2 * new, 8, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) * q_size).to(dtype)
    out = torch.empty_like(q)
    import talu_b200 as gaf
    gaf.attention(ctx, cache, q, table, dev(lens), cu=dev(cumulate(news)), max_new=new, scale=scale, out=out)
    ctx.synchronize()
    want, mass = ref.attention(cache, q, table, lens, cumulate(news), scale=scale)
    # a score y is a sum of 128 products: off by 128 2^-24 of their absolute sum in f32, and by 2^-12 sqrt(128) of a product's
    # size where keys are rounded to f16; it changes its weight, and with it the result, by that share
    k = torch.cat([ref.values(cache, table[b], lens[b], 0)[0].abs() for b in range(2)], 1)
    size = abs(scale) * q.double().abs().amax() * k.amax()
    share = size.item() * (2.0 ** -12 * 12 if dtype == torch.bfloat16 else 2.0 ** -17)
    tol = mass * (2.0 ** -8 * 3 + 2 * share if dtype == torch.bfloat16 else 2.0 ** -15 + 2 * share) + 2.0 ** -8 * want.abs() * (dtype == torch.bfloat16)
    assert ((out.double() - want).abs() <= tol + 1e-30).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("per_kv, new", [(1, 5), (4, 5), (4, 60)])
def test_values_that_are_not_finite(ctx, dtype, per_kv, new):
    """A NaN group of a key makes every row that sees the key NaN, one of a value only its group's part; rows that do not see
    it, behind a causal border or in another sequence, are untouched."""
    import talu_b200 as gaf
    lens, news, group = [90, 200], [new, new], 32
    table, pages, _ = make_tables(lens, 16, 7)
    cache = filled_cache(ctx, pages, 2, 128, 16, 8, group)
    claim(cache, table, lens)
    q = torch.randn(2 * new, 2 * per_kv, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).to(dtype)
    run = lambda: gaf.attention(ctx, cache, q, table, dev(lens), cu=dev([0, new, 2 * new]), max_new=new)  # noqa: E731
    clean = run()
    at = lens[1] - 3                                            # seen by the last three tokens of the second sequence
    page, row = int(table[1, at // 16]), at % 16
    saved = cache.scales[page, 1, 1, row, 2].clone()
    cache.scales[page, 1, 1, row, 2] = float("nan")             # V, head 1, values 64..95
    bad_v = run()
    cache.scales[page, 1, 1, row, 2] = saved
    cache.biases[page, 0, 0, row, 0] = float("nan")             # K, head 0
    bad_k = run()
    ctx.synchronize()
    hit = torch.zeros_like(clean, dtype=torch.bool)
    hit[2 * new - 3:, per_kv:, 64:96] = True
    assert torch.equal(bad_v.isnan(), hit) and torch.equal(bad_v[~hit], clean[~hit])
    hit = torch.zeros_like(clean, dtype=torch.bool)
    hit[2 * new - 3:, :per_kv] = True
    assert torch.equal(bad_k.isnan(), hit) and torch.equal(bad_k[~hit], clean[~hit])


@gpu
@pytest.mark.parametrize("new, per_kv", [(1, 4), (5, 4), (90, 4)])
def test_captured_calls_follow_their_tables(ctx, new, per_kv):
    """Append and attention captured once; lengths, tables and rows change between replays.  Equal inputs give equal bits."""
    import talu_b200 as gaf
    own = gaf.Context(0, own_stream=True)
    stream = torch.cuda.Stream()
    own.set_stream(stream.cuda_stream)
    batch, kv_heads, dim, page = 3, 2, 128, 32
    cache = gaf.KvCache.allocate(own, 200, kv_heads, dim, page, 8, 64)
    gen = torch.Generator(device="cuda").manual_seed(5)
    table = torch.arange(150, device="cuda").view(3, 50).int()
    lens, cu = dev([new] * 3), dev([new * i for i in range(4)])
    qkv = torch.randn(batch * new, (per_kv + 2) * kv_heads, dim, device="cuda", generator=gen).bfloat16()
    q, k, v = qkv.split([per_kv * kv_heads, kv_heads, kv_heads], 1)
    out = torch.zeros(batch * new, per_kv * kv_heads, dim, device="cuda", dtype=torch.bfloat16)

    def step():
        gaf.kv_append(own, cache, k, v, table, lens, cu=cu)
        gaf.attention(own, cache, q, table, lens, cu=cu, max_new=new, out=out)

    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        step()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
    for turn in range(5):
        qkv.copy_(torch.randn(qkv.shape, device="cuda", generator=gen))
        lens.copy_(dev([new * (turn + 1)] * 3))
        if turn == 3:                                           # the pages move
            old = table.clone()
            table.copy_(199 - table)
            for t in (cache.packed, cache.scales, cache.biases):
                t[table.long().flatten()] = t[old.long().flatten()].clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        first = out.clone()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(first, out)
        n = [new * (turn + 1)] * 3
        want, mass = ref.attention(cache, q, table, n, [new * i for i in range(4)])
        assert ((out.double() - want).abs() <= 2.0 ** -8 * (3 * mass + want.abs()) + 1e-7).all()
    own.synchronize()
    del graph
    cache.free()
    own.close()


@gpu
def test_two_contexts_at_once():
    """Each context has its own workspace: calls of two contexts on two streams may overlap."""
    import talu_b200 as gaf
    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [gaf.Context(0, stream=s.cuda_stream) for s in streams]
    jobs = []
    for i, c in enumerate(ctxs):
        lens = [3000 + 100 * i, 40, 900]
        table, pages, _ = make_tables(lens, 64, i)
        cache = filled_cache(c, pages, 2, 128, 64, 8, 64, seed=i)
        claim(cache, table, lens, seed=i)
        q = torch.randn(3, 8, 128, device="cuda").bfloat16()
        jobs.append((c, cache, q, table, dev(lens), lens))
    torch.cuda.synchronize()
    outs = [[gaf.attention(c, cache, q, table, lens) for _ in range(20)] for c, cache, q, table, lens, _ in jobs]
    torch.cuda.synchronize()
    for (c, cache, q, table, _, lens), many in zip(jobs, outs):
        want, mass = ref.attention(cache, q, table, lens, [0, 1, 2, 3])
        for out in many:
            assert torch.equal(out, many[0])
        assert ((many[0].double() - want).abs() <= 2.0 ** -8 * (3 * mass + want.abs()) + 1e-7).all()
        c.synchronize()
        cache.free()
        c.close()


@gpu
def test_prefix_is_the_head_of_every_sequence(ctx):
    """A prefix that ends with a page gives what tables that begin with its pages give, up to the roundings of the weights."""
    import talu_b200 as gaf
    lens, page, prefix = [70, 3, 129, 64], 32, 320
    table, pages, _ = make_tables(lens + [prefix], page, 1)
    cache = filled_cache(ctx, pages, 2, 128, page, 8, 64)
    claim(cache, table, lens + [prefix])
    head = table[-1, :prefix // page].contiguous()
    q = torch.randn(4, 16, 128, device="cuda").bfloat16()
    a = gaf.attention_shared_prefix(ctx, cache, q, head, prefix, table[:-1], dev(lens))
    whole = torch.cat((head.expand(4, -1), table[:-1, :5]), 1).contiguous()
    b = gaf.attention(ctx, cache, q, whole, dev([n + prefix for n in lens]))
    none = gaf.attention_shared_prefix(ctx, cache, q, head, 0, table[:-1], dev(lens))
    plain = gaf.attention(ctx, cache, q, table[:-1], dev(lens))
    ctx.synchronize()
    assert (a.float() - b.float()).norm() <= 2.0 ** -8 * b.float().norm()
    assert torch.equal(none, plain)


@gpu
@pytest.mark.parametrize("new", [2, 50])
def test_more_new_tokens_than_announced(ctx, new):
    """A sequence with more than max_new own tokens: reported, its rows from max_new on left as they were."""
    import talu_b200 as gaf
    lens = [100, 80]
    table, pages, _ = make_tables(lens, 16, 1)
    cache = filled_cache(ctx, pages, 2, 64, 16, 8, 64)
    claim(cache, table, lens)
    q = torch.randn(2 * new, 8, 64, device="cuda").bfloat16()
    out = torch.full_like(q, 7.0)
    gaf.attention(ctx, cache, q, table, dev(lens), cu=dev([0, new - 1, 2 * new]), max_new=new - 1, out=out)
    with pytest.raises(gaf.GafError) as e:
        ctx.synchronize()
    assert e.value.status == 7 and "max_new" in e.value.message
    assert (out[2 * new - 2:] == 7.0).all() and (out[:2 * new - 2] != 7.0).any(-1).all()
    assert gaf.attention(ctx, cache, q[:0], table, dev(lens), cu=dev([0, 0, 0]), max_new=1).shape == (0, 8, 64)
    gaf.kv_append(ctx, cache, q[:0, :2], q[:0, :2], table, dev(lens), cu=dev([0, 0, 0]))
    ctx.synchronize()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new, offset", [(1, 0), (1, 1), (30, 0), (30, 1)])
def test_attention_with_any_strides(ctx, dtype, new, offset):
    """Queries and results with odd pitches, heads in front of tokens, and bases that are not 16-byte aligned."""
    import talu_b200 as gaf
    lens = [100, 80]
    table, pages, _ = make_tables(lens, 16, 1)
    wide = torch.full((2, pages + 5), -1, dtype=torch.int32, device="cuda")      # a table with a pitch of its own
    wide[:, :table.shape[1]] = table
    cache = filled_cache(ctx, pages, 2, 128, 16, 8, 64)
    claim(cache, table, lens)
    raw = torch.randn(8, 2 * new, 128 + 2 * offset + 1, device="cuda").to(dtype)
    q = raw[:, :, offset:offset + 128].transpose(0, 1)
    buf = torch.full((8, 2 * new, 131 + offset), 7.0, device="cuda", dtype=dtype)
    out = buf[:, :, offset:offset + 128].transpose(0, 1)
    gaf.attention(ctx, cache, q, wide[:, :table.shape[1]], dev(lens), out=out)
    dense = gaf.attention(ctx, cache, q.contiguous(), table, dev(lens))
    ctx.synchronize()
    assert torch.equal(out, dense)
    assert (buf[:, :, :offset] == 7.0).all() and (buf[:, :, offset + 128:] == 7.0).all()


@gpu
@pytest.mark.parametrize("new", [1, 64])
def test_pages_beyond_four_gigabytes(ctx, new):
    """Offsets of codes and of scales that do not fit 32 bits."""
    import talu_b200 as gaf
    kv_heads, dim, page = 8, 128, 64
    pages = (2 ** 32 // (2 * kv_heads * page * dim) + 1) * 2 + 8            # codes: over 8 GB; the last pages are used
    free, _ = torch.cuda.mem_get_info()
    if free < 12 * 2 ** 30:
        pytest.skip("not enough device memory")
    cache = gaf.KvCache.allocate(ctx, pages, kv_heads, dim, page, 8, 32)
    lens = [200, 130]
    table = dev([[pages - 1, 5, pages - 3, pages - 8], [pages - 2, pages // 2 + 1, pages - 4, 0]])
    q = torch.randn(2 * new, 32, dim, device="cuda").bfloat16()
    for b, n in enumerate(lens):
        kv = torch.randn(2, n, kv_heads, dim, device="cuda").bfloat16()
        gaf.kv_append(ctx, cache, kv[0], kv[1], table[b:b + 1], dev([n]))
        got = gaf.kv_read(ctx, cache, table[b:b + 1], dev([n]), total=n)
        step = (kv.float().amax(-1) - kv.float().amin(-1)).amax() / 255
        assert (got[0].float() - kv[0].float()).abs().amax() <= 1.1 * step + 2.0 ** -8 * 6
        assert (got[1].float() - kv[1].float()).abs().amax() <= 1.1 * step + 2.0 ** -8 * 6
    check_attention(ctx, cache, q, table, lens, [0, new, 2 * new], new)
    cache.free()


@gpu
def test_decoder_layer_from_linears_and_cache(ctx, oracle):
    """qkv linear, append, attention and o linear as a decoder runs them: a prompt of two sequences, then single tokens, against
    the same layer in 64 bits on the dequantised weights and the cache's values."""
    import talu_b200 as gaf
    from helpers import make_weights
    heads, kv_heads, dim, hidden = 8, 2, 64, 512
    parts = {}
    for i, (name, n, k) in enumerate((("qkv", (heads + 2 * kv_heads) * dim, hidden), ("o", hidden, heads * dim))):
        packed, scales, biases = make_weights(oracle, n, k, 64, 4, seed=i)
        parts[name] = gaf.Weight.from_host(ctx, packed, scales, biases, 64, 4)
    cache = gaf.KvCache.allocate(ctx, 12, kv_heads, dim, 32, 8, 64)
    table = dev([[3, 7, 1, 0], [2, 9, 11, 4]])
    lens, gen = [0, 0], torch.Generator(device="cuda").manual_seed(1)
    for news in ([70, 33], [1, 1], [1, 1]):
        lens = [a + b for a, b in zip(lens, news)]
        cu = cumulate(news)
        x = torch.randn(cu[-1], hidden, device="cuda", generator=gen).bfloat16()
        qkv = gaf.linear(ctx, parts["qkv"], x).unflatten(1, (-1, dim))
        q, k, v = qkv.split([heads, kv_heads, kv_heads], 1)
        gaf.kv_append(ctx, cache, k, v, table, dev(lens), cu=dev(cu))
        a = gaf.attention(ctx, cache, q, table, dev(lens), cu=dev(cu), max_new=max(news))
        y = gaf.linear(ctx, parts["o"], a.flatten(1))
        ctx.synchronize()
        want, mass = ref.attention(cache, q, table, lens, cu)
        assert ((a.double() - want).abs() <= 2.0 ** -8 * (3 * mass + want.abs()) + 1e-7).all()
        w = gaf.dequant_f32(ctx, parts["o"]).double()
        exact = a.double().flatten(1) @ w.T
        assert (y.double() - exact).norm() <= 1e-2 * exact.norm()
        k_back, _ = gaf.kv_read(ctx, cache, table, dev(lens), cu=dev(cu), total=cu[-1])
        ctx.synchronize()
        assert (k_back.float() - k.float()).norm() <= 2.0 ** -6 * k.float().norm()   # half a 1/255 step of a range of some six sigma
    for w in parts.values():
        w.free()


@gpu
@pytest.mark.parametrize("dtype, new", [(torch.bfloat16, 1), (torch.bfloat16, 70), (torch.float32, 70)])
def test_a_bad_page_hides_its_keys_only(ctx, dtype, new):
    """A table entry outside the cache in the middle of a sequence, or of a shared prefix: its 32 keys are not seen, all others are."""
    import talu_b200 as gaf
    n, page, hole = 300, 32, slice(64, 96)
    table, pages, _ = make_tables([n], page, 1)
    cache = filled_cache(ctx, pages, 2, 128, page, 8, 64)
    claim(cache, table, [n])
    q = torch.randn(new, 8, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).to(dtype)
    bad = table.clone()
    bad[0, 2] = pages
    a = gaf.attention(ctx, cache, q, bad, dev([n]))
    with pytest.raises(gaf.GafError) as e:
        ctx.synchronize()
    assert e.value.status == 7
    b = gaf.attention_shared_prefix(ctx, cache, q, bad[0], 224, table[:, 7:], dev([n - 224]))
    with pytest.raises(gaf.GafError):
        ctx.synchronize()
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[hole] = False
    k, v = ref.values(cache, table[0], n, 0)[0][:, keep], ref.values(cache, table[0], n, 1)
    v, vs = v[0][:, keep], v[1][:, keep]
    seen = (torch.arange(n, device="cuda") <= n - new + torch.arange(new, device="cuda")[:, None])[:, keep]
    x = q.double().unflatten(1, (2, -1)).permute(1, 2, 0, 3)
    w = torch.softmax((torch.einsum("hgmd,hnd->hgmn", x, k) / math.sqrt(128)).masked_fill(~seen, -math.inf), -1)
    want = torch.einsum("hgmn,hnd->mhgd", w, v).flatten(1, 2)
    mass = torch.einsum("hgmn,hnd->mhgd", w, vs.abs() + v.abs()).flatten(1, 2)
    tol = (2.0 ** -8 * (3 * mass + want.abs()) if dtype == torch.bfloat16 else 2.0 ** -15 * mass) + 1e-7
    for out in (a, b):
        assert ((out.double() - want).abs() <= tol).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new", [1, 5, 40])
def test_a_generous_bound_and_a_row_that_is_not_finite(ctx, dtype, new):
    """max_new far above what any sequence has; a NaN or an infinity in q spoils its own row and no other."""
    import talu_b200 as gaf
    lens = [100, 260, 31]
    table, pages, _ = make_tables(lens, 16, 1)
    cache = filled_cache(ctx, pages, 2, 128, 16, 4, 64)
    claim(cache, table, lens)
    cu = [0, new, 2 * new, 2 * new + min(new, 31)]
    q = torch.randn(cu[-1], 8, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).to(dtype)
    clean = check_attention(ctx, cache, q, table, lens, cu, 1000)
    q[new, 3, 17] = float("nan")
    q[0, 0, 5] = float("inf")
    out = gaf.attention(ctx, cache, q, table, dev(lens), cu=dev(cu), max_new=1000)
    ctx.synchronize()
    hit = torch.zeros(clean.shape, dtype=torch.bool, device="cuda")
    hit[new, 3] = hit[0, 0] = True
    assert out[new, 3].isnan().all() and not out[0, 0].isfinite().any()
    assert torch.equal(out.double()[~hit], clean[~hit])


@gpu
def test_a_prefix_call_that_outgrows_its_workspace_in_a_capture_is_refused():
    import talu_b200 as gaf
    own = gaf.Context(0, own_stream=True)
    stream = torch.cuda.Stream()
    own.set_stream(stream.cuda_stream)
    cache = gaf.KvCache.allocate(own, 8, 8, 128, 16, 8, 64)
    table, lens = dev([[0]] * 3), dev([1] * 3)
    small, large = (torch.zeros(n, 64, 128, dtype=torch.bfloat16, device="cuda") for n in (3, 1200))
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        call = lambda q: gaf.attention_shared_prefix(own, cache, q, dev_prefix, 40, table, lens, cu=cu, max_new=400)  # noqa: E731
        dev_prefix, cu = dev([1, 2, 3]), dev([0, 1, 2, 3])
        call(small)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call(small)
            with pytest.raises(gaf.GafError) as e:
                call(large)
        assert e.value.status == 5
        graph.replay()
        call(large)
    own.synchronize()
    del graph
    cache.free()
    own.close()
