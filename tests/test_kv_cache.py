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
