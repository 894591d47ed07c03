"""The quantised KV cache and its attention: contexts, workspaces, and calls at the edge of what is documented."""
import pytest
import torch

import kv_reference as ref
from test_kv_cache import _FakeCtx, _args, claim, ctx, cumulate, dev, fake, filled_cache, make_tables  # noqa: F401

gpu = pytest.mark.gpu


def close(out, cache, q, table, lens, cu, **kw):
    want, mass = ref.attention(cache, q, table, lens, cu, **kw)
    return bool(((out.double() - want).abs() <= 2.0 ** -8 * (mass + want.abs()) + 1e-7).all())


def test_a_cache_of_another_device_is_refused(fake):  # noqa: F811
    from talu_b200 import GafError, attention, attention_shared_prefix, kv_append, kv_read
    x, table, lens = _args()
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    here = _FakeCtx()
    fake.ctx = _FakeCtx(0)                    # the tensors are on the context's device, the cache is not
    for call in (lambda: kv_append(here, fake, x, x, table, lens), lambda: kv_read(here, fake, table, lens, total=3),
                 lambda: attention(here, fake, q, table, lens),
                 lambda: attention_shared_prefix(here, fake, q, table[0], 8, table, lens)):
        with pytest.raises(GafError) as e:
            call()
        assert e.value.invalid_argument and "cuda:0" in e.value.message


@gpu
@pytest.mark.parametrize("new", [1, 40])
def test_a_context_without_a_cache_of_its_own(new):
    """A cache that another context has wrapped: the first call makes the workspace, and cannot be captured."""
    import talu_b200 as gaf
    owner, other = gaf.Context(0), gaf.Context(0, own_stream=True)
    stream = torch.cuda.Stream()
    other.set_stream(stream.cuda_stream)
    lens = [2000, 130]
    table, pages, _ = make_tables(lens, 32, 1)
    cache = filled_cache(owner, pages, 2, 128, 32, 8, 64)
    claim(cache, table, lens)
    cu = [0, new, 2 * new]
    q = torch.randn(2 * new, 8, 128, device="cuda").bfloat16()
    out = torch.zeros_like(q)
    args = (other, cache, q, table, dev(lens))
    kw = dict(cu=dev(cu), max_new=new, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            gaf.kv_append(other, cache, q[:, :2], q[:, 2:4], table, args[4], cu=kw["cu"])      # needs no workspace
            with pytest.raises(gaf.GafError) as e:
                gaf.attention(*args, **kw)
            assert e.value.status == 5
        del graph
        gaf.attention(*args, **kw)
        other.synchronize()
        assert close(out, cache, q, table, lens, cu)
        out.zero_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            gaf.attention(*args, **kw)
        graph.replay()
    other.synchronize()
    assert close(out, cache, q, table, lens, cu)
    del graph
    cache.free()
    other.close()
    owner.close()


def _prefix_calls(own, heads=64, most=600):
    """A cache and a function that makes a shared-prefix call of n tokens, all tensors of the largest call in hand."""
    import talu_b200 as gaf
    cache = filled_cache(own, 6, 8, 128, 16, 8, 64)
    prefix, table, lens = dev([1, 2, 3]), dev([[0]]), dev([16])
    claim(cache, dev([[1, 2, 3], [0, 0, 0]]), [40, 16])
    q = torch.randn(most, heads, 128, device="cuda").bfloat16()
    out, cu = torch.zeros_like(q), [dev([0, n]) for n in range(most + 1)]
    torch.cuda.synchronize()
    return cache, lambda n: gaf.attention_shared_prefix(own, cache, q[:n], prefix, 40, table, lens, cu=cu[n], max_new=n, out=out[:n]), q, out


@gpu
def test_the_prefix_workspace_of_growing_calls():
    """Calls that grow step by step hold twice what the largest of them needs at most, whatever was needed before."""
    import talu_b200 as gaf
    own = gaf.Context(0)
    cache, call, q, out = _prefix_calls(own)
    call(1)
    own.synchronize()
    free = torch.cuda.mem_get_info()[0]
    for n in range(20, 601, 20):
        call(n)
    own.synchronize()
    assert free - torch.cuda.mem_get_info()[0] <= 2 * 600 * 64 * 129 * 4 + 2 ** 22
    want, mass = ref.attention(cache, q, dev([[0]]), [16], [0, 600], dev([1, 2, 3]), 40)
    assert ((out.double() - want).abs() <= 2.0 ** -8 * (mass + want.abs()) + 1e-7).all()
    cache.free()
    own.close()


def test_bad_reservations_are_refused(fake):  # noqa: F811
    from talu_b200 import GafError, attention_reserve
    for rows in (-1, 2 ** 31, 2 ** 64 + 5):
        with pytest.raises(GafError) as e:
            attention_reserve(fake.ctx, fake, rows)
        assert e.value.invalid_argument
    from talu_b200 import _capi
    assert _capi.load().tgaf_attention_reserve(None, None, 5) == 1


@gpu
def test_a_reserved_workspace_and_captured_calls():
    """Reserved calls neither allocate nor are refused in a capture; a graph keeps its block when later calls outgrow it."""
    import talu_b200 as gaf
    own = gaf.Context(0, own_stream=True)
    stream = torch.cuda.Stream()
    own.set_stream(stream.cuda_stream)
    cache, call, q, out = _prefix_calls(own)
    gaf.attention_reserve(own, cache, 300 * 64)
    want, mass = ref.attention(cache, q, dev([[0]]), [16], [0, 600], dev([1, 2, 3]), 40)
    good = lambda n: bool(((out[:n].double() - w[:n]).abs() <= 2.0 ** -8 * (m[:n] + w[:n].abs()) + 1e-7).all())  # noqa: E731
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call(300)
        w, m = ref.attention(cache, q, dev([[0]]), [16], [0, 300], dev([1, 2, 3]), 40)
        free = torch.cuda.mem_get_info()[0]
        call(600)
        gaf.attention_reserve(own, cache, 600 * 64)
        own.synchronize()
        assert torch.cuda.mem_get_info()[0] < free                 # the graph's block is kept beside the new one
        gaf.attention_reserve(own, cache, 2500 * 64)               # ... the one of the call in between is not
        gaf.attention_reserve(own, cache, 5000 * 64)
        own.synchronize()
        assert free - torch.cuda.mem_get_info()[0] <= 2 * 2500 * 64 * 129 * 4 + 2 ** 22
        out.zero_()
        graph.replay()
        own.synchronize()
        assert good(300)
        call(600)
        own.synchronize()
        w, m = want, mass
        assert good(600)
    del graph
    cache.free()
    own.close()


@gpu
@pytest.mark.parametrize("dtype, new, dim", [(torch.bfloat16, 1, 128), (torch.bfloat16, 40, 64), (torch.float32, 5, 128), (torch.bfloat16, 2, 96), (torch.bfloat16, 40, 128)])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("prefix", [0, 40])
def test_a_query_row_that_is_not_finite(ctx, dtype, new, dim, value, prefix):  # noqa: F811
    """Keys whose values are all negative where the row has its infinity: every score is -inf (or inf), and the row is NaN as a
    softmax of such scores is.  Rows that see no key stay zero, all others as they were."""
    import talu_b200 as gaf
    lens, page = [300, 0, 90], 32
    table, pages, _ = make_tables(lens + [prefix], page, 1)
    cache = gaf.KvCache.allocate(ctx, pages, 2, dim, page, 8, 32)
    gen = torch.Generator(device="cuda").manual_seed(4)
    for row, n in zip(table, lens + [prefix]):
        if n:
            kv = torch.randn(2, n, 2, dim, device="cuda", generator=gen)
            kv[0] = -1 - kv[0].abs()
            gaf.kv_append(ctx, cache, kv[0], kv[1], row[None].contiguous(), dev([n]))
    cu = [0, new, 2 * new, 3 * new]
    q = torch.randn(3 * new, 6, dim, device="cuda", generator=gen).to(dtype)
    head = table[-1, :2].contiguous()

    def run():
        args = (ctx, cache, q) + ((head, prefix) if prefix else ()) + (table[:3], dev(lens))
        return (gaf.attention_shared_prefix if prefix else gaf.attention)(*args, cu=dev(cu), max_new=new)
    clean = run()
    hit = torch.zeros(clean.shape, dtype=torch.bool, device="cuda")
    for t, h in ((0, 1), (new, 4), (3 * new - 1, 0)):
        q[t, h, 7] = value
        hit[t, h] = prefix > 0 or t != new
    out = run()
    ctx.synchronize()
    assert clean.isfinite().all() and torch.equal(out.isnan(), hit) and torch.equal(out[~hit], clean[~hit])


@gpu
@pytest.mark.parametrize("dtype, new, dim", [(torch.bfloat16, 3, 128), (torch.bfloat16, 40, 64), (torch.float32, 3, 64), (torch.bfloat16, 3, 96)])
def test_own_rows_beyond_those_of_the_call(ctx, dtype, new, dim):  # noqa: F811
    """cu ends two rows behind the tensors: every call works on the rows that there are, as if there were two more, and reports it."""
    import talu_b200 as gaf
    lens, page = [100, 80], 32
    table, pages, _ = make_tables(lens, page, 1)
    caches = [filled_cache(ctx, pages, 2, dim, page, 8, 32, garbage=False) for _ in range(2)]
    for c in caches:
        claim(c, table, lens)
    x = torch.randn(2 * new, 8, dim, device="cuda").to(dtype)
    cu, short, results = dev([0, new, 2 * new]), 2 * new - 2, []
    for c, n in zip(caches, (2 * new, short)):
        def call(f, c=c, n=n):
            y = f(c, n)
            if n == short:
                with pytest.raises(gaf.GafError) as e:
                    ctx.synchronize()
                assert e.value.status == 7 and "rows" in e.value.message
            ctx.synchronize()
            return y
        call(lambda c, n: gaf.kv_append(ctx, c, x[:n, :2], x[:n, 2:4], table, dev(lens), cu=cu))
        k, v = call(lambda c, n: gaf.kv_read(ctx, c, table, dev(lens), cu=cu, total=n, dtype=dtype))
        a = call(lambda c, n: gaf.attention(ctx, c, x[:n], table, dev(lens), cu=cu, max_new=new))
        p = call(lambda c, n: gaf.attention_shared_prefix(ctx, c, x[:n], table[0, :2].contiguous(), 50, table, dev(lens), cu=cu, max_new=new))
        results.append((k, v, a, p))
        if n == 2 * new:                       # the two rows that the other cache does not get
            for t, s in zip((caches[1].packed, caches[1].scales, caches[1].biases), (c.packed, c.scales, c.biases)):
                last = table[1, 2].long()
                t[last, :, :, 14:16] = s[last, :, :, 14:16]
    whole, part = results
    for w, y in zip(whole[:2], part[:2]):
        assert torch.equal(w[:short], y)
    bound = 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -18
    for w, y in zip(whole[2:], part[2:]):      # the row tiles differ, and with them the order of the sums
        assert (w[:short].double() - y.double()).abs().max() <= bound * w.abs().max()


def test_counts_that_do_not_fit_are_refused(fake):  # noqa: F811
    """Negative numbers, numbers above 32 bits and numbers that are none: what C would read from them is something else."""
    from talu_b200 import GafError, attention, attention_shared_prefix, kv_append, kv_read
    x, table, lens = _args()
    q, cu = torch.zeros(3, 4, 64, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int32)
    head = torch.zeros(2, dtype=torch.int32)
    many = torch.zeros(1, 2, 64, dtype=torch.bfloat16).expand(2 ** 32 + 3, 2, 64)
    calls = [lambda: kv_append(fake.ctx, fake, many, many, table, lens, cu=cu),
             lambda: attention(fake.ctx, fake, torch.zeros(1, 4, 64, dtype=torch.bfloat16).expand(2 ** 32 + 3, 4, 64), table, lens, cu=cu, max_new=3)]
    for bad in (-1, 2 ** 32 + 1, 1.0, True, "3"):
        calls += [lambda bad=bad: kv_read(fake.ctx, fake, table, lens, cu=cu, total=bad),
                  lambda bad=bad: attention(fake.ctx, fake, q, table, lens, cu=cu, max_new=bad),
                  lambda bad=bad: attention_shared_prefix(fake.ctx, fake, q, head, 8, table, lens, cu=cu, max_new=bad),
                  lambda bad=bad: attention_shared_prefix(fake.ctx, fake, q, head, bad, table, lens)]
    calls.append(lambda: attention(fake.ctx, fake, q, table, lens, cu=cu, max_new=0))
    for call in calls:
        with pytest.raises(GafError) as e:
            call()
        assert e.value.invalid_argument


@gpu
def test_tables_wider_than_positions_are_refused(ctx):  # noqa: F811
    """Wider than what 32 bits with a sign count (rows of a table may overlap where their stride says so, so no memory is needed)."""
    import ctypes as C
    import talu_b200 as gaf
    from talu_b200 import _capi
    cache = gaf.KvCache.allocate(ctx, 1, 1, 64, 256, 8, 64)
    t, n, q = dev([[0]]), dev([1]), torch.zeros(1, 1, 64, device="cuda", dtype=torch.bfloat16)
    width = 2 ** 31 // 256
    seqs = _capi.KvSeqs(t.data_ptr(), width, width, 1, n.data_ptr(), None, 1)
    p = C.c_void_p(q.data_ptr())
    assert ctx._lib.tgaf_kv_append(ctx._h, cache._h, seqs, gaf.gaf.DTYPE_BF16, p, 64, 64, p, 64, 64) == 1
    assert ctx._lib.tgaf_attention(ctx._h, cache._h, seqs, gaf.gaf.DTYPE_BF16, p, 64, 64, 1, 1, C.c_float(1.0), p, 64, 64) == 1
    assert ctx._lib.tgaf_attention_shared_prefix(ctx._h, cache._h, C.c_void_p(t.data_ptr()), 2 ** 31 - 100, _capi.KvSeqs(t.data_ptr(), 1, 1, 1, n.data_ptr(), None, 1),
                                                 gaf.gaf.DTYPE_BF16, p, 64, 64, 1, 1, C.c_float(1.0), p, 64, 64) == 1
    cache.free()


@gpu
def test_calls_right_behind_a_reported_error():
    """The reset of a context's counters after an error is over before the next launch, on a non-blocking stream too."""
    import talu_b200 as gaf
    own = gaf.Context(0, own_stream=True)
    lens = [3000, 500]
    table, pages, _ = make_tables(lens, 32, 1)
    cache = filled_cache(own, pages, 2, 128, 32, 8, 64)
    claim(cache, table, lens)
    bad, n, q = table.clone(), dev(lens), torch.randn(2, 8, 128, device="cuda").bfloat16()
    bad[0, 3] = pages
    outs = [torch.zeros_like(q) for _ in range(50)]
    torch.cuda.synchronize()
    for out in outs:
        gaf.attention(own, cache, q, bad, n, out=out)
        with pytest.raises(gaf.GafError):
            own.synchronize()
        gaf.attention(own, cache, q, table, n, out=out)
    own.synchronize()
    assert close(outs[0], cache, q, table, lens, [0, 1, 2])
    assert all(torch.equal(out, outs[0]) for out in outs)
    cache.free()
    own.close()


def test_one_tensor_for_keys_and_values_is_refused(fake):  # noqa: F811
    """Read back into one place, keys and values would overwrite each other in no order."""
    from talu_b200 import GafError, kv_read
    x, table, lens = _args()
    with pytest.raises(GafError) as e:
        kv_read(fake.ctx, fake, table, lens, out=(x, x))
    assert e.value.invalid_argument and "one tensor" in e.value.message
