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
