"""The paged-cache operators where rows, warps or batches differ from one another: against the same 64-bit definition
and with the same derived tolerances as the other tests of these operators."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_paged import PAGE, Case, attend, check_append, check_attention, ctx  # noqa: E402,F401


def set_keys(c, s, dim, values):
    """Component `dim` of every key of sequence s (all kv heads) gets values [kv_len]."""
    for j in range(-(-c.kv_len[s] // PAGE)):
        part = values[j * PAGE:(j + 1) * PAGE]
        c.pool[int(c.table[s, j]), c.layer, 0, :, :len(part), dim] = part.to(c.dtype)


@pytest.mark.parametrize("ty,dim", [("bf16", 128), ("f16", 128), ("f16", 64), ("bf16", 32)])
@pytest.mark.parametrize("rows", [128, 101])
def test_warps_of_a_row_tile_at_their_own_pace(ctx, ty, dim, rows):  # noqa: F811
    """One tile of up to 128 rows over 12 key tiles in one pass: scores that climb by 14 (log2) per key tile, so that the
    running maximum is raised in every tile, but only for the rows of one warp of 32, of two, of every second one, or of
    all, beside rows whose maximum stays. 80 units keep the keys in one split."""
    n_seq, kv = 10, 1500
    c = Case(ty, [rows] * n_seq, [kv] * n_seq, 8, 8, dim)
    q = c.rand(c.rows, c.heads, dim)
    q[:, :, 0] = 0.0
    per_tile = torch.arange(kv, device="cuda") // 128
    warp = torch.arange(rows, device="cuda") // 32
    climbs = [warp == 0, warp == 1, warp == 2, warp == 3, (warp == 0) | (warp == 3), warp % 2 == 0, warp >= 0, warp < 0,
              (torch.arange(rows, device="cuda") % 5) == 0, warp == 2]
    for s in range(n_seq):
        step = per_tile if s != 9 else per_tile // 2   # the last: raised in every second tile
        set_keys(c, s, 0, step.float())
        q[s * rows:(s + 1) * rows, :, 0] = (climbs[s].float() * 10.0 * dim ** 0.5)[:, None].to(c.dtype)
    x, a, la = attend(ctx, c, q=q)
    for _ in range(5):
        _, b, lb = attend(ctx, c, q=x)
        assert torch.equal(a, b) and torch.equal(la, lb)


def decode_case(ty="f16", n=2, kv=3000, heads=4, kv_heads=2, dim=64, q=1, seed=0):
    return Case(ty, [q] * n, [kv] * n, heads, kv_heads, dim, seed=seed)


@pytest.mark.parametrize("q", [1, 5, 60])
def test_captured_graphs_keep_their_scratch(tmp_path, q):
    """A split call (joined by its last CTA, by a kernel of its own, on tcgen05) captured in a graph, then a larger call
    that outgrows the scratch, then a model file that does not load: replays still give the result, on new contents."""
    import gsvcu
    own = gsvcu.Context(0)
    small, large = decode_case(q=q), decode_case(n=6, kv=20000, heads=16, kv_heads=4, dim=128, q=q)
    x = small.rand(small.rows, small.heads, small.dim)
    out = torch.empty_like(x)
    cache, chunks = small.objects()
    attend(own, small, q=x)
    stream = torch.cuda.ExternalStream(own.stream_handle())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        own.op_chunk_attention(cache, chunks, small.layer, x, out)
    attend(own, large)
    bad = tmp_path / "none.gguf"
    bad.write_bytes(b"GGUF")
    with pytest.raises(gsvcu.GsvcuError):
        own.load(str(bad))
    keep = [torch.full((1 << 20,), float("nan"), device="cuda") for _ in range(64)]   # (freed memory would be reused)
    for _ in range(3):
        x.normal_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        own.sync()
        check_attention(small, x, out, None, small.dim ** -0.5)
        attend(own, large)
    del graph, keep
    own.close()


@pytest.mark.parametrize("mode", ["relaxed", "thread_local", "global"])
def test_scratch_does_not_grow_in_a_capture(mode):
    """A first split call inside a capture is refused and leaves nothing behind: the capture ends as usual, the same call
    outside it is right, and then it can be captured."""
    import gsvcu
    own = gsvcu.Context(0)
    c = decode_case()
    x = c.rand(c.rows, c.heads, c.dim)
    out = torch.empty_like(x)
    cache, chunks = c.objects()
    torch.cuda.synchronize()
    stream = torch.cuda.ExternalStream(own.stream_handle())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode=mode):
        out.zero_()
        with pytest.raises(gsvcu.GsvcuError) as e:
            own.op_chunk_attention(cache, chunks, c.layer, x, out)
    assert e.value.code == -6 and "once before" in str(e.value)
    attend(own, c, q=x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode=mode):
        own.op_chunk_attention(cache, chunks, c.layer, x, out)
    for _ in range(2):
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        own.sync()
        check_attention(c, x, out, None, c.dim ** -0.5)
    del graph
    own.close()


@pytest.mark.parametrize("ty", ["f16", "f32"])
@pytest.mark.parametrize("group", [1, 3, 5, 7])
@pytest.mark.parametrize("bounds", [(0, -723922764), (7, -1292124672), (8, -1199745), (0, -1599320890), (3, -2 ** 31),
                                    (-5, 3), (-2 ** 31, 2 ** 31 - 1), (8, 2 ** 31 - 1), (2 ** 31 - 1, -2 ** 31), (9, 9)])
def test_row_bounds_far_outside_the_batch(ctx, ty, group, bounds):  # noqa: F811
    """row_start with values whose differences and products pass 32 bits: the call reports them and writes nothing outside
    its rows and pages."""
    import gsvcu
    c = Case(ty, [8], [70], 2 * group, 2, 64)
    c.row_start.copy_(torch.tensor(bounds, dtype=torch.int32))
    x, kv = c.rand(8, 2 * group, 64), c.rand(8, 2, 64)
    guard = torch.full((72, 2 * group, 64), 7.0, dtype=c.dtype, device="cuda")
    out = guard[32:40]
    cache, chunks = c.objects()
    for lens in (70, 0, -2 ** 31, 2 ** 31 - 1):
        c.kv.fill_(lens)
        torch.cuda.synchronize()
        ctx.op_chunk_attention(cache, chunks, 1, x, out)
        with pytest.raises(gsvcu.GsvcuError) as e:
            ctx.sync()
        assert e.value.code == -1 and "row_start" in str(e.value)
        before = c.pool.clone()
        torch.cuda.synchronize()
        ctx.op_kv_append(cache, chunks, 1, x, kv, kv, out)
        with pytest.raises(gsvcu.GsvcuError) as e:
            ctx.sync()
        assert e.value.code == -1
        assert (guard[:32] == 7.0).all() and (guard[40:] == 7.0).all()
        assert torch.equal(torch.nan_to_num(before[:, 0]), torch.nan_to_num(c.pool[:, 0]))   # (the other layer)
    ctx.sync()


@pytest.mark.parametrize("ty", ["f16", "f32"])
@pytest.mark.parametrize("q", [2, 70])
def test_both_operators_report_the_same_bounds(ctx, ty, q):  # noqa: F811
    """Lengths inside the table but outside the given sizes, and rows that no sequence owns, are reported after either
    operator; a bound on the chunks that is wider than the batch is none of these."""
    import gsvcu
    c = Case(ty, [q, q], [q + 100, q + 30], 4, 2, 64, max_pages=8)
    x, kv = c.rand(2 * q, 4, 64), c.rand(2 * q, 2, 64)
    out = torch.empty_like(x)

    def reported(chunks):
        cache = gsvcu.PagedKV(c.pool)
        found = []
        for call in (lambda: ctx.op_kv_append(cache, chunks, 1, x, kv, kv, out),
                     lambda: ctx.op_chunk_attention(cache, chunks, 1, x, out)):
            torch.cuda.synchronize()
            call()
            try:
                ctx.sync()
                found.append(None)
            except gsvcu.GsvcuError as e:
                assert e.code == -1
                found.append("kv_len" in str(e))
        return found

    def batch(max_chunk=q, max_kv=q + 100):
        return gsvcu.ChunkBatch(c.row_start, c.kv, c.table, 2 * q, max_chunk, max_kv)

    assert reported(batch()) == [None, None]
    assert reported(batch(max_chunk=2 * q + 999)) == [None, None]
    assert reported(batch(max_kv=q + 99)) == [True, True]
    assert reported(batch(max_chunk=q - 1)) == [True, True]
    for bounds in ((0, q, 2 * q - 1), (1, q, 2 * q)):
        c.row_start.copy_(torch.tensor(bounds, dtype=torch.int32))
        assert reported(batch()) == [True, True], bounds
    c.row_start.copy_(torch.tensor([0, q, 2 * q], dtype=torch.int32))
    c.kv[1] = -1
    assert reported(batch()) == [True, True]
    c.kv[1] = q + 30
    attend(ctx, c, max_chunk=100000)


@pytest.mark.parametrize("ty,dim,q", [("bf16", 128, 1), ("bf16", 64, 60), ("bf16", 128, 200), ("bf16", 32, 300), ("f32", 64, 1),
                                      ("f32", 64, 40)])
@pytest.mark.parametrize("at", [5, 6, 7, 63, 70, 134, 391])
@pytest.mark.parametrize("kv", [400, 5000])
def test_scores_that_overflow_make_their_rows_nan(ctx, ty, dim, q, at, kv):  # noqa: F811
    """Finite queries and keys whose product is infinite: as exp(inf - inf) the row and its log-sum-exp are NaN, whichever
    key it is; a product of minus infinity has weight 0 (F32: NaN, its two parts overflow apart); other rows are not
    touched."""
    c = Case(ty, [q], [kv + q], 2, 1, dim)
    x = c.rand(q, 2, dim)
    x[:, :, :3] = 0.0
    zero = torch.zeros(kv + q, device="cuda")
    for d in range(3):
        set_keys(c, 0, d, zero)
    _, base, base_lse = attend(ctx, c, q=x)
    big = zero.clone()
    big[at] = 1e30
    set_keys(c, 0, 0, big)
    set_keys(c, 0, 1, -big)
    rows = torch.arange(q, device="cuda") % 40 == 0
    cache, chunks = c.objects()
    out, lse = torch.empty_like(x), torch.empty(q, 2, device="cuda")
    for d in (0, 1):
        y = x.clone()
        y[rows, 0, d] = 1e30
        torch.cuda.synchronize()
        ctx.op_chunk_attention(cache, chunks, c.layer, y, out, lse=lse)
        ctx.sync()
        if d == 0 or ty == "f32":
            assert out[rows, 0].isnan().all() and lse[rows, 0].isnan().all(), d
        else:
            assert torch.isfinite(out).all() and torch.isfinite(lse).all()
            # one key of weight about exp(|q| |k| / sqrt(dim)) / kv less
            assert ((lse[rows, 0] - base_lse[rows, 0]).abs() < 0.2).all()
        rest = torch.ones_like(lse, dtype=torch.bool)
        rest[rows, 0] = False
        assert torch.allclose(out[rest].float(), base[rest].float(), rtol=2.0 ** -6, atol=2.0 ** -6), d
        assert torch.allclose(lse[rest], base_lse[rest], rtol=1e-5, atol=1e-4), d


@pytest.mark.parametrize("ty,dim,q", [("f16", 32, 1), ("bf16", 128, 5), ("f32", 64, 40), ("f16", 64, 60), ("bf16", 128, 300)])
@pytest.mark.parametrize("kv", [70, 5000])
def test_a_query_of_nan_makes_its_row_nan(ctx, ty, dim, q, kv):  # noqa: F811
    c = Case(ty, [q], [kv + q], 2, 1, dim)
    x, base, base_lse = attend(ctx, c)
    y = x.clone()
    y[q // 2, 1, 3] = float("nan")
    cache, chunks = c.objects()
    out, lse = torch.empty_like(x), torch.empty(q, 2, device="cuda")
    torch.cuda.synchronize()
    ctx.op_chunk_attention(cache, chunks, c.layer, y, out, lse=lse)
    ctx.sync()
    assert out[q // 2, 1].isnan().all() and lse[q // 2, 1].isnan()
    rest = torch.ones_like(lse, dtype=torch.bool)
    rest[q // 2, 1] = False
    assert torch.allclose(out[rest].float(), base[rest].float(), rtol=2.0 ** -6, atol=2.0 ** -6)
    assert torch.allclose(lse[rest], base_lse[rest], rtol=1e-5, atol=1e-4)


def test_scales_past_the_range_are_refused(ctx):  # noqa: F811
    import gsvcu
    c = Case("f16", [1], [5], 1, 1, 32)
    x = c.rand(1, 1, 32)
    cache, chunks = c.objects()
    for scale in (3e38, -3e38, float("inf"), float("nan")):
        with pytest.raises(gsvcu.GsvcuError) as e:
            ctx.op_chunk_attention(cache, chunks, 1, x, x.clone(), scale=scale)
        assert e.value.code == -1 and "scale" in str(e.value)


@pytest.mark.parametrize("ty", ["f16", "bf16"])
@pytest.mark.parametrize("at", [4, 5, 6, 7, 77, 78, 79])
def test_one_key_that_outweighs_the_rest(ctx, ty, at):  # noqa: F811
    """One key holds all but a ten-thousandth of the weight, at any place among the columns: its exponential alone decides
    the sum, so that the log-sum-exp shows the exponential's error."""
    c = Case(ty, [200], [500], 2, 2, 32)
    q = torch.zeros(200, 2, 32, dtype=c.dtype, device="cuda")
    q[:, :, 0] = 5.0
    for d in range(32):
        set_keys(c, 0, d, torch.zeros(500, device="cuda"))
    key = torch.zeros(500, device="cuda")
    key[at] = 17.0
    set_keys(c, 0, 0, key)
    attend(ctx, c, q=q)


@pytest.mark.parametrize("ty,q", [("f16", 1), ("f16", 4), ("f16", 24), ("f16", 40), ("f16", 150), ("bf16", 1), ("bf16", 40)])
@pytest.mark.parametrize("below,spread", [(25.1, 0.0), (24.0, 0.3), (22.0, 0.0)])
def test_a_sink_beside_a_long_light_tail(ctx, ty, q, below, spread):  # noqa: F811
    """One key of value 0 holds nearly all the weight, 16383 others 2^-22 to 2^-25 of its weight each: the output is the
    tail's. F16 holds weights down to 2^-24 with few bits and none below 2^-25."""
    n_seq, kv = 10, 16384
    c = Case(ty, [q] * n_seq, [kv] * n_seq, 8, 8, 64)
    x = torch.zeros(c.rows, 8, 64, dtype=c.dtype, device="cuda")
    x[:, :, 0] = 8.0
    c.pool[:, :, 1] = c.pool[:, :, 1].abs() + 0.5
    for s in range(n_seq):
        key = torch.randn(kv, generator=c.gen, device="cuda") * spread
        key[0] = below * 0.6931
        set_keys(c, s, 0, key)
        c.pool[int(c.table[s, 0]), c.layer, 1, :, 0] = 0.0
    attend(ctx, c, q=x)


def test_append_refuses_half_given_arguments(ctx):  # noqa: F811
    """A table of angles with broadcast dimensions (its rows would be taken for other positions' angles), one table without
    the other, queries without their output."""
    c = Case("f16", [2], [70], 4, 2, 64)
    cache, chunks = c.objects()
    q, kv = c.rand(2, 4, 64), c.rand(2, 2, 64)
    out, angle = torch.empty_like(q), torch.zeros(80, 32, device="cuda")
    for bad in (dict(cos=angle[:, None], sin=angle[:, None]), dict(cos=angle[:, :, None], sin=angle[:, :, None]), dict(cos=angle),
                dict(sin=angle), dict(cos=angle[0], sin=angle[0]), dict(q_out=None), dict(q=None)):
        args = dict(q=q, k=kv, v=kv, q_out=out)
        args.update(bad)
        with pytest.raises(ValueError):
            ctx.op_kv_append(cache, chunks, 1, **args)
    ctx.op_kv_append(cache, chunks, 1, q, kv, kv, out, cos=angle, sin=angle)
    ctx.sync()


@pytest.mark.parametrize("rows", [1500, 3000, 6000])
@pytest.mark.parametrize("ty,row_ty,dim,rot,pairs", [("bf16", "bf16", 128, 128, False), ("f16", "f32", 32, 32, True),
                                                     ("f32", "f32", 64, 32, False), ("f16", "f16", 32, 16, False)])
def test_append_of_many_rows(ctx, ty, row_ty, dim, rot, pairs, rows):  # noqa: F811
    """Prompt chunks of so many rows that a row takes 128, 64 or 32 threads, beside short ones."""
    check_append(ctx, ty, row_ty, 6, 2, dim, rot, pairs, q_len=(rows - 141, 1, 0, 140), kv_len=(rows - 141, 77, 5, 200))


@pytest.mark.parametrize("dim", [64, 128])
def test_f32_row_tiles_of_24_are_joined(ctx, dim):  # noqa: F811
    """F32 chunks whose plan takes 24-row tiles and splits the keys."""
    attend(ctx, Case("f32", [240, 240, 131, 240, 5], [4000, 3999, 4000, 700, 3000], 5, 5, dim))


@pytest.mark.parametrize("ty,dim", [("f16", 64), ("bf16", 128)])
@pytest.mark.parametrize("q,kv", [(60, 60), (60, 900), (300, 300), (300, 2000), (90, 9000)])
def test_page_waits_that_run_out_are_reported(ctx, ty, dim, q, kv):  # noqa: F811
    """Every pair of page copies from the second on expects 16 bytes more than it gets (the copies themselves complete) and
    its wait has a short limit: the call ends with products under way, the next sync reports it once, and the same call
    without the fault is right."""
    import gsvcu
    c = Case(ty, [q, 0, q], [kv, 5, kv], 4, 2, dim)
    x = c.rand(c.rows, c.heads, dim)
    out = torch.empty_like(x)
    cache, chunks = c.objects()
    torch.cuda.synchronize()
    ctx.set_wait_fault(True)
    try:
        ctx.op_chunk_attention(cache, chunks, c.layer, x, out)
        with pytest.raises(gsvcu.GsvcuError) as e:
            ctx.sync()
        assert e.value.code == -2 and "gave up" in str(e.value)
    finally:
        ctx.set_wait_fault(False)
    ctx.sync()
    attend(ctx, c, q=x)


def test_addresses_off_their_elements_are_refused(ctx):  # noqa: F811
    """Through the C structs: every array at an address that is not a multiple of its element is refused before a launch."""
    import ctypes
    import gsvcu
    c = Case("f16", [2], [70], 4, 2, 64)
    q, kv = c.rand(2, 4, 64), c.rand(2, 2, 64)
    f32, ints = torch.zeros(80 * 32, device="cuda"), torch.zeros(8, dtype=torch.int32, device="cuda")
    cache, chunks = c.objects()
    before, launches = c.pool.clone(), ctx.kernel_launches()
    append = dict(q=q.data_ptr(), k=kv.data_ptr(), v=kv.data_ptr(), q_out=q.data_ptr(), cos=f32.data_ptr(), sin=f32.data_ptr(),
                  pos=ints.data_ptr(), q_stride=256, k_stride=128, v_stride=128, q_out_stride=256, layer=1, row_dtype=0,
                  n_q_head=4, n_pos=80, rot_dim=64)
    attention = dict(q=q.data_ptr(), out=q.data_ptr(), lse=f32.data_ptr(), prefix=ints.data_ptr(), q_stride=256, out_stride=256,
                     layer=1, n_q_head=4, scale=1.0)
    torch.cuda.synchronize()

    def call(fn, struct, args, batch=chunks.desc):
        a = struct(kv=ctypes.addressof(cache.desc), batch=ctypes.addressof(batch), **args)
        return getattr(ctx.lib, fn)(ctx.h, ctypes.byref(a))

    for fn, struct, args, names in (("gsvcu_op_kv_append", gsvcu.KvAppendArgs, append, ("q", "k", "v", "q_out", "cos", "sin", "pos")),
                                    ("gsvcu_op_chunk_attention", gsvcu.ChunkAttentionArgs, attention, ("q", "out", "lse", "prefix"))):
        for name in names:
            for off in (1, 2, 3) if name in ("cos", "sin", "pos", "lse", "prefix") else (1,):
                assert call(fn, struct, dict(args, **{name: args[name] + off})) == -1, (fn, name, off)
        for name in ("row_start", "kv_len", "block_table"):
            batch = gsvcu.ChunkBatchDesc.from_buffer_copy(chunks.desc)
            setattr(batch, name, getattr(batch, name) + 2)
            assert call(fn, struct, args, batch) == -1, (fn, name)
    ctx.sync()
    assert ctx.kernel_launches() == launches
    assert torch.equal(torch.nan_to_num(before), torch.nan_to_num(c.pool))
