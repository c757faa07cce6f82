"""The scratch of chunk attention when memory is short: a call that needs it says so, one that can do without it does, from then
on in the same way, and can be captured."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import test_gpu_paged as floats  # noqa: E402
from test_gpu_paged import PAGE, Case, order  # noqa: E402
from test_gpu_paged_q4 import Q4Case, attend, check_attention  # noqa: E402


@pytest.fixture()
def own():
    import gsvcu
    c = gsvcu.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("ty", ["f16", "bf16"])
def test_without_memory_for_unpacked_pages_the_4_bits_are_read(own, ty):
    """Long chunks whose pages would be unpacked first: right without the memory for it, the same bits every time, in a captured
    graph too, and also after there is memory again; smaller calls are unpacked then."""
    import gsvcu
    c = Q4Case(ty, [400] * 12, [1500] * 12, 16, 4, 64)   # (336 CTAs: no splits, so the unpacked pages are all the scratch)
    other = gsvcu.Context(0)
    x, unpacked, _ = attend(other, c)
    kernels = [0, 0]
    for i, ctx in enumerate((own, other)):
        if ctx is own:
            own.set_memory_fault(True)
        before = ctx.kernel_launches()
        _, first, _ = attend(ctx, c, q=x)
        kernels[i] = ctx.kernel_launches() - before
        if ctx is own:
            a = first
    assert kernels == [1, 2]
    assert torch.equal(attend(own, c, q=x)[1], a)
    cache, chunks = c.objects()
    out = torch.empty_like(x)
    stream = torch.cuda.ExternalStream(own.stream_handle())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        own.op_chunk_attention(cache, chunks, c.layer, x, out)
    own.set_memory_fault(False)
    for _ in range(2):
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        own.sync()
        assert torch.equal(out, a)
    check_attention(c, x, out, None, 0.125)
    assert torch.equal(attend(own, c, q=x)[1], a)
    small = Q4Case(ty, [400] * 8, [900] * 8, 16, 4, 64, seed=1)
    before = own.kernel_launches()
    y, b, _ = attend(own, small)
    assert own.kernel_launches() - before == 2
    assert torch.equal(attend(other, small, q=y)[1], b)
    del graph
    other.close()


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("q", [1, 60])
def test_split_results_without_memory_are_refused(own, q4, q):
    import gsvcu
    c = (Q4Case if q4 else Case)("f16", [q], [9000 + q], 8, 2, 64)
    x = c.rand(q, 8, 64)
    out = torch.full_like(x, 7.0)
    cache, chunks = c.objects()
    own.set_memory_fault(True)
    for _ in range(2):
        with pytest.raises(gsvcu.GsvcuError) as e:
            order(own).op_chunk_attention(cache, chunks, c.layer, x, out)
        assert e.value.code == -3 and "memory" in str(e.value)
    own.sync()
    assert (out == 7.0).all()
    own.set_memory_fault(False)
    (attend if q4 else floats.attend)(own, c, q=x)


@pytest.mark.parametrize("captured", [False, True])
def test_outgrown_unpacked_pages_are_freed_unless_a_graph_may_use_them(own, captured):
    """Calls that need 105, 236 and 524 MB for unpacked pages (the table's length bounds it) hold what the last one needs, and
    before that only what a graph was captured with, whose replays stay right."""
    c = Q4Case("bf16", [400], [1500], 32, 8, 128, max_pages=400)
    table = c.table.clone()
    x, first, _ = attend(own, c)
    cache, chunks = c.objects()
    out = torch.empty_like(x)
    stream = torch.cuda.ExternalStream(own.stream_handle())
    torch.cuda.synchronize()
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            own.op_chunk_attention(cache, chunks, c.layer, x, out)
    free, reserved = torch.cuda.mem_get_info()[0], torch.cuda.memory_reserved()
    for pages in (900, 2000):
        c.table = torch.full((1, pages), 2 ** 30, dtype=torch.int32, device="cuda")
        c.table[:, :400] = table
        attend(own, c, q=x)
        attend(own, c, q=x)
    grown = free - torch.cuda.mem_get_info()[0] - (torch.cuda.memory_reserved() - reserved)
    block = 400 * 8 * 4 * PAGE * 128   # bytes of the first
    want = block * 5 - (0 if captured else block)
    assert abs(grown - want) < block // 2, (grown, want)   # (splits: up to 40 MB)
    if captured:
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        own.sync()
        assert torch.equal(out, first)
        del graph


@pytest.mark.parametrize("ty,dim,heads,kv_heads", [("bf16", 128, 32, 8), ("f16", 64, 16, 4)])
@pytest.mark.parametrize("window", [0, 1000])
def test_a_long_chunk_beside_many_single_tokens(own, ty, dim, heads, kv_heads, window):
    """The slots' pages are not unpacked for the chunk's sake; without slots, or with idle ones, its own are."""
    for q_len, kernels in (([512] + [1] * 32, 1), ([512] + [0] * 11, 2)):
        c = Q4Case(ty, q_len, [1900] + [700 + 31 * s for s in range(1, len(q_len))], heads, kv_heads, dim)
        before = own.kernel_launches()
        attend(own, c, window=window)
        assert own.kernel_launches() - before == kernels   # (enough CTAs: the keys are not split)


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("max_kv", [64, 1 << 20])
def test_batches_too_large_for_one_launch_are_refused(own, q4, max_kv):
    """2^16 sequences times 2^15 row tiles: refused from the sizes, on the host."""
    import ctypes as C

    import gsvcu
    c = (Q4Case if q4 else Case)("f16", [1], [5], 1, 1, 32)
    cache, _ = c.objects()
    x, out = c.rand(1, 1, 32), torch.full((1, 1, 32), 7.0, dtype=torch.float16, device="cuda")
    batch = gsvcu.ChunkBatchDesc(c.row_start.data_ptr(), c.kv.data_ptr(), c.table.data_ptr(), 1 << 16, max_kv // PAGE, 1 << 20,
                                 1 << 20, max_kv)
    args = gsvcu.ChunkAttentionArgs(cache.addr, C.addressof(batch), x.data_ptr(), out.data_ptr(), None, None, 32, 32, c.layer, 1, 0, 0.0)
    before = own.kernel_launches()
    assert order(own).lib.gsvcu_op_chunk_attention(own.h, C.byref(args)) == -1
    assert own.kernel_launches() == before
    own.sync()
    assert (out == 7.0).all()
