"""The paged-cache operators on a cache held in 4 bits, the head norms of the append and the read-back, against their
formulas in 64 bits, through the Python binding of the C ABI.

Tolerances, set per element before the first run. u: unit roundoff of the rows' type, s: a group's scale.
  attention  as for the float caches (test_gpu_paged.py): the codes' products are exact in F16, so a score's error is that
             of an f32 sum; few rows multiply unrounded weights, many rows F16 weights (2^-11, less than the u they get
             there for BF16 rows).
             The weights are F16 for BF16 rows too, kept 2^14 (few rows, two parts) or 2^11 (many rows) up, and F16 ends at
             steps of 2^-24: a weight is off by up to 2^-25 / 2^14 = 2^-39 (2^-25 / 2^11 = 2^-36) of its row's largest
             however light it is. The sum of the weights is at least the largest, so an output is off by up to n max|v|
             2^-39 (2^-36) more: where the heavy keys' values are 0 and the others' weights below that, all of it.
  norm       in units of 2^-24: the sum's rounding and eps 1 each, halved by the root, the root and the division 1 each, two
             products: 5; a rotation adds a product and a sum of two such terms: 7, rounded up to 10 (times |a| + |b|).
  store      half a step s / 2 of the nearest code, a whole one and 4 % (the scale's rounding, 8 times 2^-8) where the code
             was cut off at 15; on top the norm's and rotation's error; groups below 2^-22 may vanish.
  read       exact; BF16 rows one rounding u.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import q4_format  # noqa: E402
from test_gpu_paged import PAGE, ROUND, TYPES, Case, attention_oracle, ctx, order, rotate_oracle  # noqa: E402,F401


class Q4Case(Case):
    """Ragged sequences in a shuffled 4-bit cache whose unused tokens have NaN scales and whose unused table entries name
    pages far outside the pool."""

    def __init__(self, ty, *args, **kw):
        super().__init__(ty, *args, **kw)
        self.pool = q4_format.encode(self.pool.float())

    def objects(self, max_kv=0, max_chunk=None):
        import gsvcu
        longest = max(self.q_len, default=0) if max_chunk is None else max_chunk
        return (gsvcu.PagedKV(self.pool, rows=self.dtype),
                gsvcu.ChunkBatch(self.row_start, self.kv, self.table, self.rows, longest, max_kv))

    def keys(self, s, h, which):
        n = self.kv_len[s]
        p = self.table[s, :-(-n // PAGE)].long()
        return q4_format.decode(self.pool[p, self.layer, which, h])[0].reshape(-1, self.dim)[:n]

    def set_values(self, values):
        """The whole layer's keys and values [page][2][kv head][64][dim] are quantised anew."""
        self.pool[:, self.layer] = q4_format.encode(values.float())


def check_attention(c, q, out, lse, scale, window=0, prefix=None):
    ro, rl, amp, mag = attention_oracle(c, q, scale, window, prefix)
    n, u = max(c.kv_len, default=0), ROUND[c.ty]
    weight = (c.dim + 8) * 2.0 ** -24 * mag + 2.0 ** -20 + (n / 64 + 64) * 2.0 ** -24
    light = 2.0 ** (-36 if max(c.q_len, default=0) * (c.heads // c.kv_heads) > 32 else -39)
    largest = torch.zeros(c.rows, dtype=torch.float64, device="cuda")
    for s, m in enumerate(c.q_len):
        if m and c.kv_len[s]:
            largest[int(c.starts[s]):int(c.starts[s]) + m] = max(float(c.keys(s, h, 1).abs().max()) for h in range(c.kv_heads))
    tol = u * ro.abs() + (2 * weight[..., None] + u) * amp + (2.0 ** -25 if c.ty == "f16" else 0.0) + \
        n * light * largest[:, None, None]
    err = (out.double() - ro).abs()
    assert torch.isfinite(out).all()
    assert (err <= tol).all(), float((err / tol.clamp_min(1e-300)).max())
    if lse is not None:
        empty = torch.isinf(rl)
        assert torch.equal(torch.isneginf(lse), empty)
        e, t = (lse.double() - rl).abs()[~empty], (weight + 2.0 ** -22 * rl.abs())[~empty]
        assert (e <= t).all(), float((e / t).max()) if e.numel() else 0


def attend(ctx, c, q=None, window=0, prefix=None, scale=None, max_kv=0, lse=True):  # noqa: F811
    q = c.rand(c.rows, c.heads, c.dim) if q is None else q
    out = torch.full((c.rows, c.heads, c.dim), float("nan"), dtype=c.dtype, device="cuda")
    ls = torch.full((c.rows, c.heads), float("nan"), device="cuda") if lse else None
    pf = None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device="cuda")
    cache, chunks = c.objects(max_kv)
    order(ctx).op_chunk_attention(cache, chunks, c.layer, q, out, scale=scale, prefix=pf, window=window, lse=ls)
    ctx.sync()
    check_attention(c, q, out, ls, c.dim ** -0.5 if scale is None else scale, window, prefix)
    return q, out, ls


def test_format_round_trip():
    """The tests' own encoder and decoder belong together."""
    x = torch.randn(3, 2, PAGE, 128, device="cuda")
    v, s, _ = q4_format.decode(q4_format.encode(x))
    assert ((v - x.double()).abs() <= 1.04 * s.abs()).all()


# ------------------------------------------------------------------ attention

@pytest.mark.parametrize("ty", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(16, 16), (8, 2), (7, 1), (32, 2), (24, 1)])
def test_single_tokens(ctx, ty, dim, heads, kv_heads):  # noqa: F811
    """One new token per sequence: one key, page ends inside and at a tile, ragged lengths."""
    attend(ctx, Q4Case(ty, [1] * 9, [1, 2, 15, 63, 64, 65, 127, 200, 517], heads, kv_heads, dim))


@pytest.mark.parametrize("ty", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (6, 2), (8, 1), (5, 1)])
def test_ragged_chunks(ctx, ty, dim, heads, kv_heads):  # noqa: F811
    """Chunks of 0, 1, a few and many rows, with and without cached keys before them."""
    attend(ctx, Q4Case(ty, [5, 0, 1, 17, 33, 130, 64, 300], [5, 40, 1, 17, 95, 131, 700, 301], heads, kv_heads, dim))


@pytest.mark.parametrize("ty,dim,heads,kv_heads,q", [("f16", 64, 16, 4, 2), ("bf16", 128, 8, 2, 4), ("f16", 32, 16, 16, 7),
                                                     ("bf16", 64, 12, 1, 2), ("f16", 128, 3, 1, 8)])
def test_drafts(ctx, ty, dim, heads, kv_heads, q):  # noqa: F811
    """A few rows per sequence: 8, 16, 24 and 32 packed rows."""
    attend(ctx, Q4Case(ty, [q, 1, q, q - 1], [q, 200, 900, 63 + q], heads, kv_heads, dim))


@pytest.mark.parametrize("ty,dim,heads,kv_heads", [("f16", 64, 16, 4), ("bf16", 128, 8, 2), ("f16", 32, 16, 16), ("bf16", 64, 12, 1)])
@pytest.mark.parametrize("window,prefix", [(1, None), (16, None), (100, None), (64, [0, 3, 200, 64, 90]),
                                           (0, [1, 3, 333, 64, 90]), (37, [0, 0, 5000, 129, 500]), (4096, None)])
@pytest.mark.parametrize("q_len", [(70, 1, 200, 129, 3), (1, 1, 2, 1, 1)])
def test_windows_and_prefixes(ctx, ty, dim, heads, kv_heads, window, prefix, q_len):  # noqa: F811
    attend(ctx, Q4Case(ty, list(q_len), [400, 333, 200, 640, 90], heads, kv_heads, dim), window=window, prefix=prefix)


@pytest.mark.parametrize("ty,dim", [("f16", 32), ("bf16", 128), ("f16", 64)])
@pytest.mark.parametrize("q", [3, 150])
def test_rows_that_see_nothing(ctx, ty, dim, q):  # noqa: F811
    """No keys at all, or a chunk longer than its keys: those rows give 0 and -infinity."""
    _, out, lse = attend(ctx, Q4Case(ty, [q, q, 1], [0, 2, 0], 4, 2, dim))
    assert (out[:q] == 0).all() and torch.isneginf(lse[:q]).all()
    assert (out[q:2 * q - 2] == 0).all() and torch.isneginf(lse[q:2 * q - 2]).all()
    assert torch.isfinite(lse[2 * q - 2:2 * q]).all()


@pytest.mark.parametrize("ty,dim,heads,kv_heads,q", [("bf16", 128, 32, 8, 1), ("f16", 32, 16, 16, 1), ("f16", 64, 4, 1, 5),
                                                     ("bf16", 128, 8, 2, 40), ("f16", 64, 4, 4, 150), ("f16", 32, 4, 4, 150)])
def test_long_caches_are_split(ctx, ty, dim, heads, kv_heads, q):  # noqa: F811
    """Few rows over long caches (work split over the keys and joined); the same result twice, bit for bit, also with a
    looser bound on the length."""
    c = Q4Case(ty, [q, q, q], [9000, 4097, q], heads, kv_heads, dim, max_pages=200)
    x, a, la = attend(ctx, c, max_kv=9000)
    _, b, lb = attend(ctx, c, q=x, max_kv=9000)
    assert torch.equal(a, b) and torch.equal(la, lb)
    attend(ctx, c, q=x, max_kv=0, lse=False)


@pytest.mark.parametrize("ty,dim,heads,kv_heads,q", [("f16", 32, 16, 16, 1), ("bf16", 128, 8, 2, 1), ("f16", 64, 16, 4, 1), ("bf16", 128, 8, 2, 5),
                                                     ("f16", 64, 9, 1, 3), ("bf16", 32, 8, 4, 12), ("f16", 128, 2, 2, 20)])
@pytest.mark.parametrize("n_seq", [1, 7, 60, 300])
@pytest.mark.parametrize("window", [0, 200])
def test_pages_dealt_out_over_ragged_batches(ctx, ty, dim, heads, kv_heads, q, n_seq, window):  # noqa: F811
    """Lengths from a few keys to thousands, sequences without rows and without keys among them: units that one CTA has to
    itself, that two or many share, and CTAs with many units. The same result twice, bit for bit, and after a smaller batch."""
    lens = [(37 * i * i + 11) % 700 + (5000 if i % 50 == 3 else 0) + (9000 if n_seq == 1 else 0) for i in range(n_seq)]
    rows = [0 if i % 9 == 4 else q if i % 4 else 1 for i in range(n_seq)]
    c = Q4Case(ty, rows, [max(n, r) if i % 11 else n for i, (n, r) in enumerate(zip(lens, rows))], heads, kv_heads, dim)
    x, a, la = attend(ctx, c, window=window, prefix=[i % 90 for i in range(n_seq)] if window else None)
    attend(ctx, Q4Case(ty, [1, 1], [900, 2000], heads, kv_heads, dim))
    _, b, lb = attend(ctx, c, q=x, window=window, prefix=[i % 90 for i in range(n_seq)] if window else None, max_kv=max(c.kv_len) + 500)
    assert torch.equal(a, b) and torch.equal(la, lb)


@pytest.mark.parametrize("ty,dim,heads,kv_heads,q,kv", [("f16", 64, 40, 1, 1, 500), ("bf16", 128, 40, 1, 1, 9000), ("f16", 32, 66, 2, 1, 3000)])
def test_wide_groups(ctx, ty, dim, heads, kv_heads, q, kv):  # noqa: F811
    """More than 32 query heads of a kv head: single tokens on the kernel for many rows."""
    attend(ctx, Q4Case(ty, [q, q], [kv, 70], heads, kv_heads, dim))


def test_a_zero_scale_over_a_long_cache(ctx):  # noqa: F811
    """Many rows on the kernel for few, several row tiles of a sequence, pages dealt out."""
    attend(ctx, Q4Case("f16", [70, 3, 140], [6000, 90, 3000], 4, 2, 64), scale=0.0)
    attend(ctx, Q4Case("bf16", [50, 1], [5000, 4000], 8, 2, 128), scale=0.0, window=900)


@pytest.mark.parametrize("scale", [0.0, 1.7, -0.3])
@pytest.mark.parametrize("ty,q", [("f16", 1), ("bf16", 140), ("f16", 140)])
def test_scales(ctx, scale, ty, q):  # noqa: F811
    attend(ctx, Q4Case(ty, [q, 9], [257, 80], 8, 2, 64), scale=scale)


@pytest.mark.parametrize("ty,dim,q", [("f16", 64, 4), ("bf16", 128, 200), ("bf16", 32, 5), ("f16", 32, 300)])
def test_growing_scores(ctx, ty, dim, q):  # noqa: F811
    """Keys whose scores grow along the cache by far more than the range of the weights."""
    c = Q4Case(ty, [q], [900], 4, 2, dim)
    x = c.rand(c.rows, c.heads, c.dim).abs() + 0.5
    v = torch.randn(c.pool.shape[0], 2, 2, PAGE, dim, generator=c.gen, device="cuda")
    ramp = torch.linspace(-4.0, 4.0, 15 * PAGE, device="cuda").view(15, PAGE)
    v[c.table[0, :15].long(), 0] = ramp[:, None, :, None].expand(15, 2, PAGE, dim)
    c.set_values(v)
    attend(ctx, c, q=x.to(c.dtype))


@pytest.mark.parametrize("ty,q", [("f16", 1), ("f16", 4), ("f16", 24), ("f16", 40), ("f16", 150), ("bf16", 1), ("bf16", 40)])
@pytest.mark.parametrize("below,spread", [(25.1, 0.0), (24.0, 0.3), (22.0, 0.0)])
def test_a_sink_beside_a_long_light_tail(ctx, ty, q, below, spread):  # noqa: F811
    """One key of value 0 holds nearly all the weight, 16383 others 2^-22 to 2^-25 of its weight each: the output is the
    tail's."""
    n_seq, kv, dim = 10, 16384, 64
    c = Q4Case(ty, [q] * n_seq, [kv] * n_seq, 8, 8, dim)
    x = torch.zeros(c.rows, 8, dim, dtype=c.dtype, device="cuda")
    x[:, :, 0] = 8.0
    v = torch.randn(c.pool.shape[0], 2, 8, PAGE, dim, generator=c.gen, device="cuda")
    v[:, 0] *= 0.02
    v[:, 1] = v[:, 1].abs() + 0.5
    for s in range(n_seq):
        key = torch.randn(kv, generator=c.gen, device="cuda") * spread
        key[0] = below * 0.6931
        p = c.table[s, :kv // PAGE].long()
        v[p, 0, :, :, 0] = key.view(-1, 1, PAGE)
        v[p[0], 1, :, 0] = 0.0
    c.set_values(v)
    attend(ctx, c, q=x)


@pytest.mark.parametrize("ty", ["f16", "bf16"])
@pytest.mark.parametrize("q", [1, 9, 90])
def test_strided_and_unaligned_rows(ctx, ty, q):  # noqa: F811
    """Queries and outputs as slices of wider rows, at offsets and strides that 16-byte accesses do not fit; what lies
    between the rows stays."""
    c = Q4Case(ty, [q, q], [130, q], 4, 2, 64)
    for width, off in ((4 * 64 + 5, 1), (4 * 64 + 64, 32)):
        qs = c.rand(c.rows, width)
        os_ = torch.full((c.rows, width), 7.0, dtype=c.dtype, device="cuda")
        q3, o3 = qs[:, off:off + 256].unflatten(1, (4, 64)), os_[:, off:off + 256].unflatten(1, (4, 64))
        cache, chunks = c.objects()
        order(ctx).op_chunk_attention(cache, chunks, c.layer, q3, o3)
        ctx.sync()
        check_attention(c, q3, o3, None, 0.125)
        assert (os_[:, :off] == 7.0).all() and (os_[:, off + 256:] == 7.0).all()


@pytest.mark.parametrize("q", [1, 140])
def test_offsets_past_32_bits(ctx, q):  # noqa: F811
    """Pages whose byte offset passes 2^32: appended, read back and attended."""
    import gsvcu
    dim, heads = 128, 2
    n_page = 2 ** 32 // (2 * heads * 36 * dim) + 40
    pool = torch.empty(n_page, 1, 2, heads, PAGE, 72, dtype=torch.uint8, device="cuda")
    c = Q4Case("f16", [q], [150], heads, heads, dim, layers=1, layer=0)
    far = torch.tensor([[n_page - 1, n_page - 7, n_page - 30]], dtype=torch.int32, device="cuda")
    pool[far[0].long()] = c.pool[c.table[0].long()]
    pool[:3] = 255
    x, kv = c.rand(c.rows, heads, dim), c.rand(c.rows, 2, heads, dim)
    out, qo, k, v = (torch.empty_like(x) for _ in range(4))
    c.pool, c.table = pool, far
    cache, chunks = c.objects()
    order(ctx).op_kv_append(cache, chunks, 0, x, kv[:, 0], kv[:, 1], qo)
    ctx.op_kv_read(cache, chunks, 0, k, v)
    ctx.op_chunk_attention(cache, chunks, 0, qo, out)
    ctx.sync()
    code, scale = q4_format.quantise(kv)
    want = (code.double() - 8) * scale.double().repeat_interleave(32, -1)
    assert torch.equal(qo, x) and torch.equal(k.double(), want[:, 0]) and torch.equal(v.double(), want[:, 1])
    check_attention(c, x, out, None, dim ** -0.5)
    del pool, c


@pytest.mark.parametrize("ty,q,dim", [("f16", 1, 32), ("f16", 1, 64), ("bf16", 3, 128), ("bf16", 200, 64), ("f16", 40, 128)])
def test_masked_values_may_be_anything(ctx, ty, q, dim):  # noqa: F811
    """Tokens past kv_len, in the same pages: bits of the result do not depend on them."""
    c = Q4Case(ty, [q], [q + 70], 4, 4, dim)
    x, a, _ = attend(ctx, c)
    values, _, _ = q4_format.decode(c.pool)
    for fill in (float("inf"), 3.0, 0.0):
        c.pool = q4_format.encode(torch.where(values.isnan(), fill, values).float())
        _, b, _ = attend(ctx, c, q=x)
        assert torch.equal(a, b)


@pytest.mark.parametrize("ty,dim,q", [("f16", 32, 1), ("bf16", 128, 5), ("f16", 64, 150), ("bf16", 128, 300)])
@pytest.mark.parametrize("prefix", [None, 70])
def test_pages_behind_the_window_may_be_gone(ctx, ty, dim, q, prefix):  # noqa: F811
    """Pages that no row sees any more: stale table entries, NaN scales. Neither is touched nor reported."""
    c = Q4Case(ty, [q, 1], [2000, 900], 8, 2, dim)
    window = 130
    full = c.table.clone()
    whole = c.pool.clone()
    for s, (n, total) in enumerate(zip(c.q_len, c.kv_len)):
        for j in range(-(-total // PAGE)):
            if (j + 1) * PAGE <= total - n - window + 1 and not (prefix and j * PAGE < prefix):
                c.pool[int(c.table[s, j])] = 255
                c.table[s, j] = -7
    x = c.rand(c.rows, c.heads, c.dim)
    out = torch.empty_like(x)
    pf = None if prefix is None else torch.tensor([prefix] * 2, dtype=torch.int32, device="cuda")
    cache, chunks = c.objects()
    order(ctx).op_chunk_attention(cache, chunks, c.layer, x, out, prefix=pf, window=window)
    ctx.sync()
    c.table.copy_(full)
    c.pool = whole
    check_attention(c, x, out, None, dim ** -0.5, window, None if prefix is None else [prefix] * 2)


@pytest.mark.parametrize("ty,dim,q", [("f16", 32, 1), ("bf16", 128, 5), ("f16", 64, 60), ("bf16", 128, 300), ("bf16", 64, 800), ("f16", 32, 800)])
@pytest.mark.parametrize("kv", [70, 5000])
@pytest.mark.parametrize("bad", [float("nan"), 1e30])
def test_a_query_of_nan_or_past_the_range_makes_its_row_nan(ctx, ty, dim, q, kv, bad):  # noqa: F811
    """1e30: infinite in F16 rows, and past the F16 range that BF16 queries are read in."""
    c = Q4Case(ty, [q], [kv + q], 2, 1, dim)
    x, base, base_lse = attend(ctx, c)
    y = x.clone()
    y[q // 2, 1, 3] = bad
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


@pytest.mark.parametrize("ty,dim,q", [("f16", 64, 2), ("bf16", 128, 60), ("f16", 32, 1)])
def test_large_and_tiny_groups(ctx, ty, dim, q):  # noqa: F811
    """Groups at the top of the scales' range beside groups of subnormal scales and of zeros."""
    c = Q4Case(ty, [q], [300], 4, 2, dim)
    v = torch.randn(c.pool.shape[0], 2, 2, PAGE, dim, generator=c.gen, device="cuda")
    size = torch.tensor([6000.0, 2.0 ** -20, 0.0, 1.0], device="cuda")
    v[:, 1] *= size[torch.arange(PAGE, device="cuda") % 4][:, None]
    v[:, 0] *= torch.tensor([1.0, 2.0 ** -17], device="cuda")[torch.arange(PAGE, device="cuda") // 3 % 2][:, None]
    c.set_values(v)
    x, out, _ = attend(ctx, c)
    assert float(out.abs().max()) > 100.0


@pytest.mark.parametrize("ty,dim,heads,kv_heads,q", [("bf16", 128, 16, 2, 260), ("f16", 64, 8, 1, 300), ("bf16", 32, 16, 1, 130),
                                                     ("f16", 128, 2, 2, 1700), ("bf16", 64, 9, 1, 500)])
@pytest.mark.parametrize("window,prefix", [(0, None), (0, [3, 700, 64]), (300, None), (1600, [0, 70, 900])])
def test_chunks_whose_pages_are_unpacked_first(ctx, ty, dim, heads, kv_heads, q, window, prefix):  # noqa: F811
    """At least 1536 packed rows in a chunk, beside short ones and single tokens; windows that leave fewer rows to a key."""
    c = Q4Case(ty, [q, 1, q // 3], [q + 1111, 900, q // 3], heads, kv_heads, dim)
    attend(ctx, c, window=window, prefix=prefix)


@pytest.mark.parametrize("ty,dim,heads,kv_heads,q_len,kv_len,window", [
    ("bf16", 128, 32, 8, [1300], [9000], 0), ("f16", 64, 16, 4, [900, 700, 5, 1200], [7000, 6500, 9000, 8000], 0),
    ("bf16", 32, 16, 16, [1500], [9000], 0), ("f16", 128, 8, 8, [3000, 1900], [9500, 1900], 0), ("f16", 64, 16, 4, [1500, 1100], [9000, 9000], 3000)])
def test_chunks_of_more_than_one_wave(ctx, ty, dim, heads, kv_heads, q_len, kv_len, window):  # noqa: F811
    """More CTAs than the GPU takes at once, over many keys. Twice the same."""
    c = Q4Case(ty, q_len, kv_len, heads, kv_heads, dim)
    x, a, la = attend(ctx, c, window=window)
    _, b, lb = attend(ctx, c, q=x, window=window)
    assert torch.equal(a, b) and torch.equal(la, lb)


def test_pages_are_unpacked_again_for_every_call(ctx):  # noqa: F811
    """Two caches, two layers and two lengths through the same scratch, captured in a graph too: nothing is kept from one
    call for the next; a call past the scratch's limit reads the 4 bits themselves."""
    import gsvcu
    own = gsvcu.Context(0)
    a = Q4Case("bf16", [400], [1500], 8, 2, 64, seed=1)
    b = Q4Case("f16", [410, 3], [700, 90], 8, 2, 64, seed=2, layer=0)
    x, first, _ = attend(own, a)
    attend(own, b)
    _, again, _ = attend(own, a, q=x)
    assert torch.equal(first, again)
    cache, chunks = a.objects()
    out = torch.empty_like(x)
    stream = torch.cuda.ExternalStream(own.stream_handle())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        own.op_chunk_attention(cache, chunks, a.layer, x, out)
    attend(own, Q4Case("bf16", [400, 400, 400], [9000, 8000, 7000], 16, 2, 64))   # outgrows the scratch
    a.set_values(torch.randn(a.pool.shape[0], 2, 2, PAGE, 64, device="cuda"))
    for _ in range(2):
        x.normal_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        own.sync()
        check_attention(a, x, out, None, 0.125)
    wide = Q4Case("bf16", [400], [1500], 8, 2, 64, seed=1, max_pages=90000)   # (the table's length bounds the scratch)
    attend(own, wide, q=x)
    del graph
    own.close()


@pytest.mark.parametrize("ty,dim", [("bf16", 128), ("f16", 64), ("bf16", 32)])
@pytest.mark.parametrize("rows", [128, 101])
def test_warps_of_a_row_tile_at_their_own_pace(ctx, ty, dim, rows):  # noqa: F811
    """One tile of up to 128 rows over 12 key tiles in one pass: scores that climb from key tile to key tile for the rows of
    one warp, of two, of every fifth row or of all, beside rows whose maximum stays."""
    n_seq, kv = 10, 1500
    c = Q4Case(ty, [rows] * n_seq, [kv] * n_seq, 8, 8, dim)
    q = c.rand(c.rows, c.heads, dim)
    q[:, :, 0] = 0.0
    v = torch.randn(c.pool.shape[0], 2, 8, PAGE, dim, generator=c.gen, device="cuda")
    warp = torch.arange(rows, device="cuda") // 32
    climbs = [warp == 0, warp == 1, warp == 2, warp == 3, (warp == 0) | (warp == 3), warp % 2 == 0, warp >= 0, warp < 0,
              (torch.arange(rows, device="cuda") % 5) == 0, warp == 2]
    for s in range(n_seq):
        step = torch.arange(24 * PAGE, device="cuda") // 128 // (1 if s != 9 else 2)
        p = c.table[s, :24].long()
        v[p, 0, :, :, 0] = step.float().view(24, 1, PAGE).expand(24, 8, PAGE)
        q[s * rows:(s + 1) * rows, :, 0] = (climbs[s].float() * 10.0 * dim ** 0.5)[:, None].to(c.dtype)
    c.set_values(v)
    x, a, la = attend(ctx, c, q=q)
    for _ in range(3):
        _, b, lb = attend(ctx, c, q=x)
        assert torch.equal(a, b) and torch.equal(la, lb)


@pytest.mark.parametrize("ty,dim", [("f16", 64), ("bf16", 128), ("f16", 32)])
@pytest.mark.parametrize("q,kv", [(1, 700), (1, 9000), (3, 5000), (60, 60), (60, 900), (300, 300), (300, 2000), (90, 9000)])
def test_page_waits_that_run_out_are_reported(ctx, ty, dim, q, kv):  # noqa: F811
    """Every copy from the second on is expected to bring 16 bytes more than it does (the copies themselves complete) and its
    wait has a short limit: the call ends, the next sync reports it once, and the same call without the fault is right."""
    import gsvcu
    c = Q4Case(ty, [q, 0, q], [kv, 5, kv], 4, 2, dim)
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


# ------------------------------------------------------------------ append: norms and 4 bits

def norm_oracle(x, weight, eps):
    if weight is None:
        return x.double()
    x = x.double()
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()


def check_append(ctx, ty, row_ty, heads, kv_heads, dim, rot, pairs=False, own_pos=False, q_len=(3, 0, 1, 70, 130),  # noqa: F811
                 kv_len=(3, 5, 64, 200, 129), off=0, in_place=False, no_q=False, norms=(True, True), eps=1e-6, q4=False, size=1.0):
    """Rows through op_kv_append against the norm, the rotation and the quantiser in 64 bits; then read back."""
    c = (Q4Case if q4 else Case)(ty, list(q_len), list(kv_len), heads, kv_heads, dim, layers=3)
    rd = TYPES[row_ty]
    rows = (torch.randn(c.rows, (heads + 2 * kv_heads) * dim + off, generator=c.gen, device="cuda") * size).to(rd)
    x = rows[:, off:].unflatten(1, (heads + 2 * kv_heads, dim))
    q, k, v = x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
    q0 = q.clone()
    place = torch.cat([torch.arange(t - n, t) for n, t in zip(q_len, kv_len)]).cuda()
    seq = torch.repeat_interleave(torch.arange(len(q_len)), torch.tensor(q_len)).cuda()
    at = place.clamp_min(0)
    cos = sin = pos = ct = st = None
    if rot:
        ang = torch.arange(max(kv_len) + 1, dtype=torch.float64, device="cuda")[:, None] * \
            10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64, device="cuda") * 2 / rot)
        cos, sin = ang.cos().float(), ang.sin().float()
        if own_pos:
            at = torch.randint(0, max(kv_len), (c.rows,), generator=c.gen, device="cuda")
            pos = at.to(torch.int32)
        ct, st = cos[at], sin[at]
    wq, wk = (1.0 + 0.3 * torch.randn(dim, generator=c.gen, device="cuda") if on else None for on in norms)
    before = c.pool.clone()
    qo = q if in_place else torch.full((c.rows, heads, dim), float("nan"), dtype=c.dtype, device="cuda")
    cache, chunks = c.objects()
    order(ctx).op_kv_append(cache, chunks, 1, None if no_q else q, k, v, None if no_q else qo, cos=cos, sin=sin, pos=pos,
                            pairs=pairs, q_norm=wq, k_norm=wk, eps=eps)
    back = [torch.full((c.rows, kv_heads, dim), 7.0, dtype=t, device="cuda") for t in (c.dtype, c.dtype, torch.float32, torch.float32)]
    ctx.op_kv_read(cache, chunks, 1, back[0], back[1])
    ctx.op_kv_read(cache, chunks, 1, back[2], back[3])
    ctx.sync()
    want_q, mag_q = rotate_oracle(norm_oracle(q0, wq, eps), ct, st, pairs)
    want_k, mag_k = rotate_oracle(norm_oracle(k, wk, eps), ct, st, pairs)
    u = ROUND[ty]
    tiny = 2.0 ** -25 if ty == "f16" else 0.0
    if not no_q:
        assert ((qo.double() - want_q).abs() <= u * want_q.abs() + 10 * 2.0 ** -24 * mag_q + tiny).all()
    ok = place >= 0
    page, slot = c.table[seq[ok], place[ok] // PAGE].long(), place[ok] % PAGE
    if q4:
        values, scales, codes = q4_format.decode(c.pool)
        gk, gv = values[page, 1, 0, :, slot], values[page, 1, 1, :, slot]
        s, code = scales[page, 1, 0, :, slot], codes[page, 1, 0, :, slot]
        step = torch.where(code == 15, 1.04, 0.5 + 2.0 ** -18) * s.abs()
        assert ((gk - want_k[ok]).abs() <= step + 10 * 2.0 ** -24 * mag_k[ok] + 2.0 ** -22).all()
        big = want_k[ok].abs().unflatten(-1, (-1, 32)).amax(-1).repeat_interleave(32, -1)
        mk = mag_k[ok].unflatten(-1, (-1, 32)).amax(-1).repeat_interleave(32, -1)
        assert ((8 * s.abs() - big).abs() <= 2.0 ** -8 * big + 10 * 2.0 ** -24 * mk + 2.0 ** -21).all()
        want_code, want_scale = q4_format.quantise(v[ok])
        assert torch.equal(codes[page, 1, 1, :, slot], want_code.long())
        assert torch.equal(scales[page, 1, 1, :, slot], want_scale.double().repeat_interleave(32, -1))
        blank, now = (q4_format.decode(p) for p in (before, c.pool))
        for a, b in zip(blank, now):
            b[page, 1, :, :, slot] = a[page, 1, :, :, slot]
            assert torch.equal(torch.nan_to_num(a, 9.0), torch.nan_to_num(b, 9.0))
    else:
        gk, gv = c.pool[page, 1, 0, :, slot].double(), c.pool[page, 1, 1, :, slot].double()
        assert ((gk - want_k[ok]).abs() <= u * want_k[ok].abs() + 10 * 2.0 ** -24 * mag_k[ok] + tiny).all()
        assert torch.equal(gv, v[ok].to(c.dtype).double())
        before[page, 1, :, :, slot] = c.pool[page, 1, :, :, slot]
        assert ((before == c.pool) | (before.isnan() & c.pool.isnan())).all()
    for got, ref in zip(back, (gk, gv, gk, gv)):
        assert torch.equal(got[ok], ref.to(got.dtype))
        assert (got[~ok] == 7.0).all()


@pytest.mark.parametrize("ty,row_ty,q4", [("f16", "f32", False), ("f16", "f16", False), ("bf16", "bf16", False), ("f32", "f32", False),
                                          ("f16", "f32", True), ("f16", "f16", True), ("bf16", "f32", True), ("bf16", "bf16", True)])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("rot_share,pairs,own_pos", [(0, False, False), (1, False, False), (1, True, True), (2, False, True),
                                                     (2, True, False)])
def test_append_with_norms(ctx, ty, row_ty, q4, dim, rot_share, pairs, own_pos):  # noqa: F811
    check_append(ctx, ty, row_ty, 8, 2, dim, dim // rot_share if rot_share else 0, pairs, own_pos, q4=q4)


@pytest.mark.parametrize("norms", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("ty,q4", [("f16", True), ("bf16", True), ("bf16", False)])
@pytest.mark.parametrize("dim,rot", [(32, 32), (64, 0), (128, 96)])
def test_append_with_some_norms(ctx, norms, ty, q4, dim, rot):  # noqa: F811
    check_append(ctx, ty, ty, 6, 3, dim, rot, norms=norms, q4=q4)


@pytest.mark.parametrize("rot", [2, 6, 24, 40, 62])
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("q4", [False, True])
def test_append_odd_rotation_widths(ctx, rot, pairs, q4):  # noqa: F811
    check_append(ctx, "f16", "f32", 4, 2, 64, rot, pairs, q4=q4)


@pytest.mark.parametrize("off", [1, 3, 8])
@pytest.mark.parametrize("q4", [False, True])
def test_append_unaligned_rows(ctx, off, q4):  # noqa: F811
    check_append(ctx, "f16", "f16", 4, 2, 64, 64, off=off, q4=q4)
    check_append(ctx, "f16", "f32", 5, 1, 128, 128, off=off, q4=q4, pairs=True)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (16, 16), (48, 1), (7, 7), (40, 8)])
@pytest.mark.parametrize("dim", [32, 128])
@pytest.mark.parametrize("q4", [False, True])
def test_append_head_counts(ctx, heads, kv_heads, dim, q4):  # noqa: F811
    check_append(ctx, "bf16", "bf16", heads, kv_heads, dim, dim, q4=q4)


@pytest.mark.parametrize("rows", [1500, 6000])
@pytest.mark.parametrize("q4", [False, True])
def test_append_of_many_rows(ctx, rows, q4):  # noqa: F811
    """Row counts that take a warp, two or more for a row."""
    check_append(ctx, "bf16", "bf16", 8, 2, 128, 128, q_len=(rows, 1, 17), kv_len=(rows + 5, 90, 17), q4=q4)
    check_append(ctx, "f16", "f32", 4, 4, 32, 32, q_len=(rows, 3), kv_len=(rows, 90), q4=q4, pairs=True)


def test_append_in_place_without_queries_and_past_its_keys(ctx):  # noqa: F811
    for q4 in (False, True):
        check_append(ctx, "f16", "f16", 8, 2, 64, 64, in_place=True, q4=q4)
        check_append(ctx, "bf16", "f32", 4, 4, 32, 32, pairs=True, no_q=True, q4=q4)
        check_append(ctx, "f16", "f32", 4, 2, 64, 0, q_len=(9, 4), kv_len=(2, 4), q4=q4)
        check_append(ctx, "f16", "f32", 2, 1, 32, 32, q_len=[i % 3 for i in range(1200)],
                     kv_len=[1 + (i * 7) % 150 + i % 3 for i in range(1200)], q4=q4)


@pytest.mark.parametrize("size,eps", [(1e-4, 1e-6), (1e-12, 1e-5), (300.0, 0.0), (1e15, 1e-6), (2.0 ** -70, 2.0 ** -130)])
@pytest.mark.parametrize("q4", [False, True])
def test_norms_of_small_and_large_rows(ctx, size, eps, q4):  # noqa: F811
    """Sums of squares far from 1 (1e15: past 2^100; 2^-70: below F32's normal range): summed in 64 bits, rounded once."""
    check_append(ctx, "bf16", "f32", 4, 2, 64, 0, eps=eps, size=min(size, 1e15), q4=q4 and size < 1e4)


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("row_ty,ty", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "f16")])
def test_norms_of_heads_that_are_not_finite(ctx, row_ty, ty, off):  # noqa: F811
    """A NaN makes its head NaN; an infinity, or squares that overflow, the rest of its head 0 (an infinity itself NaN); other
    heads, and values, are as without them. 16-byte accesses and single elements."""
    import gsvcu
    n, heads, dim = 9, 3, 64
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    rows = torch.randn(n, 2 * heads * dim + off, generator=g, device="cuda")
    x = rows[:, off:].unflatten(1, (2 * heads, dim))
    x[1, 0, 5], x[2, 1, 63], x[3, 2, 0] = float("nan"), float("inf"), float("-inf")
    x[4, 0, 7], x[4, 0, 40] = float("inf"), float("nan")
    if row_ty != "f16":
        x[5, 1] = 1e30
    x[6, heads:] = float("nan")   # values
    rows = rows.to(TYPES[row_ty])
    x = rows[:, off:].unflatten(1, (2 * heads, dim))
    k, v = x[:, :heads], x[:, heads:]
    w = torch.rand(dim, generator=g, device="cuda") + 0.5
    i32 = dict(dtype=torch.int32, device="cuda")
    pool = torch.zeros(1, 1, 2, heads, PAGE, dim, dtype=TYPES[ty], device="cuda")
    chunks = gsvcu.ChunkBatch(torch.tensor([0, n], **i32), torch.tensor([n], **i32), torch.zeros(1, 1, **i32), n, n)
    out = torch.empty(n, heads, dim, dtype=TYPES[ty], device="cuda")
    order(ctx).op_kv_append(gsvcu.PagedKV(pool), chunks, 0, k, k, v, out, q_norm=w, k_norm=w)
    ctx.sync()
    f = k.float()
    want = f * (1.0 / (f.square().sum(-1, keepdim=True) / dim + 1e-6).sqrt()) * w
    for got in (out, pool[0, 0, 0, :, :n].transpose(0, 1)):
        got = got.float()
        assert torch.equal(got.isnan(), want.isnan())
        fine = ~want.isnan()
        assert ((got - want)[fine].abs() <= ROUND[ty] * want[fine].abs() + 2.0 ** -20).all()
    assert torch.equal(torch.nan_to_num(pool[0, 0, 1, :, :n].transpose(0, 1).float(), 9.0), torch.nan_to_num(v.to(TYPES[ty]).float(), 9.0))


def test_quantiser_borders(ctx):  # noqa: F811
    """Groups of zeros, of one magnitude in both signs, of subnormals, past the largest scale, with NaN or infinities,
    values exactly between two codes: codes and scales as the definition gives them, in F32, F16 and BF16 rows."""
    import gsvcu
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    n, dim = 64, 128
    x = torch.randn(n, 1, dim, generator=g, device="cuda")
    x[0] = 0.0
    x[1, 0, :32] = -0.0
    x[2, 0, 5], x[2, 0, 9] = 9.0, -9.0
    x[3, 0, 5], x[3, 0, 9] = -9.0, 9.0
    x[4] *= 2.0 ** -22
    x[5] *= 2.0 ** -26
    x[6] *= 1e4
    x[7] *= 6e4
    x[8, 0, 70] = float("nan")
    x[9, 0, 70] = float("inf")
    x[10, 0, 3] = float("-inf")
    x[11] = torch.arange(-64, 64, device="cuda").float()[None] / 8     # scales of 1: x / s ends in .5 and .0
    x[12:40] = (x[12:40] * 4).round() / 4
    x[40:] *= torch.logspace(-6, 4, n - 40, device="cuda")[:, None, None]
    for row_ty, ty in (("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")):
        rows = x.to(TYPES[row_ty])
        pool = torch.zeros(2, 1, 2, 1, PAGE, 72, dtype=torch.uint8, device="cuda")
        i32 = dict(dtype=torch.int32, device="cuda")
        cache = gsvcu.PagedKV(pool, rows=TYPES[ty])
        chunks = gsvcu.ChunkBatch(torch.tensor([0, n], **i32), torch.tensor([n], **i32), torch.tensor([[1]], **i32), n, n)
        order(ctx).op_kv_append(cache, chunks, 0, None, rows, rows, None)
        ctx.sync()
        want = q4_format.encode(rows[:, 0].float())
        values, scales, codes = q4_format.decode(pool[1, 0, :, 0])
        ref, ref_scales, ref_codes = q4_format.decode(want)
        fine = torch.isfinite(rows[:, 0].float()).unflatten(-1, (-1, 32)).all(-1).repeat_interleave(32, -1)
        assert int((~fine).sum()) >= 3 * 32
        for which in (0, 1):
            assert torch.equal(codes[which][fine], ref_codes[fine]) and torch.equal(scales[which][fine], ref_scales[fine])
            assert scales[which][~fine].isnan().all()
        assert (values[0][fine].abs() <= 21760).all() and not pool[0].any()


def test_every_code_and_scale_is_read_exactly(ctx):  # noqa: F811
    """All 16 codes under all finite F16 scales of 8 significant bits, subnormal ones among them, read back in F32 and F16;
    a weight of one token alone gives the value itself."""
    import gsvcu
    bits = torch.arange(0, 0x7c00, device="cuda")
    scale = bits.to(torch.int16).view(torch.float16)
    keep = (scale.float() == scale.float().bfloat16().float()) & (scale.float() <= 2720)
    scale = torch.cat((scale[keep], -scale[keep]))
    n = -(-scale.numel() // PAGE) * PAGE
    scale = torch.nn.functional.pad(scale, (0, n - scale.numel()), value=1.0)
    code = (torch.arange(32, device="cuda") + torch.arange(n, device="cuda")[:, None]) % 16
    byte, shift = (t.cuda() for t in q4_format.places(32))
    rows = torch.zeros(n, 16, dtype=torch.uint8, device="cuda")
    for e in range(32):
        rows[:, byte[e]] |= (code[:, e] << shift[e]).to(torch.uint8)
    pages = n // PAGE
    block = torch.cat((rows.view(pages, -1), scale.view(torch.uint8).view(pages, -1)), 1)
    pool = block.view(pages, 1, 1, 1, PAGE, 18).repeat(1, 1, 2, 1, 1, 1).contiguous()
    i32 = dict(dtype=torch.int32, device="cuda")
    cache = gsvcu.PagedKV(pool, rows=torch.float16)
    chunks = gsvcu.ChunkBatch(torch.tensor([0, n], **i32), torch.tensor([n], **i32), torch.arange(pages, **i32)[None], n, n)
    want = (code - 8).double() * scale.double()[:, None]
    for ty in (torch.float32, torch.float16):
        k, v = (torch.empty(n, 1, 32, dtype=ty, device="cuda") for _ in range(2))
        order(ctx).op_kv_read(cache, chunks, 0, k, v)
        ctx.sync()
        assert torch.equal(k[:, 0].double(), want) and torch.equal(v[:, 0].double(), want)
    each = gsvcu.ChunkBatch(torch.arange(n + 1, **i32), torch.arange(n, **i32) + 1, torch.arange(pages, **i32).repeat(n, 1), n, 1)
    q, out = torch.zeros(n, 1, 32, dtype=torch.float16, device="cuda"), torch.empty(n, 1, 32, dtype=torch.float16, device="cuda")
    order(ctx).op_chunk_attention(cache, each, 0, q, out, window=1)
    ctx.sync()
    assert torch.equal(out[:, 0].double(), want)


# ------------------------------------------------------------------ read back

@pytest.mark.parametrize("ty,q4", [("f16", False), ("bf16", False), ("f32", False), ("f16", True), ("bf16", True)])
@pytest.mark.parametrize("dim,kv_heads", [(32, 1), (64, 3), (128, 8)])
def test_read_back(ctx, ty, q4, dim, kv_heads):  # noqa: F811
    """Whole sequences and last tokens, in F32 and the cache's row type, into strided and unaligned rows; rows before the
    cache's start stay as they are."""
    kv_len = [1, 0, 64, 200, 65, 3]
    q_len = [1, 0, 64, 77, 65, 5]
    c = (Q4Case if q4 else Case)(ty, q_len, kv_len, kv_heads, kv_heads, dim)
    cache, chunks = c.objects()
    width = kv_heads * dim
    for dtype in {torch.float32, c.dtype}:
        for off, extra in ((0, 0), (1, 5), (8, 16)):
            k, v = (torch.full((c.rows, off + width + extra), 7.0, dtype=dtype, device="cuda") for _ in range(2))
            kr, vr = (t[:, off:off + width].unflatten(1, (kv_heads, dim)) for t in (k, v))
            order(ctx).op_kv_read(cache, chunks, c.layer, kr, vr)
            ctx.sync()
            for s, (n, total) in enumerate(zip(q_len, kv_len)):
                at, have = int(c.starts[s]), min(n, total)
                for which, rows in ((0, kr), (1, vr)):
                    assert (rows[at:at + n - have] == 7.0).all()
                    for h in range(kv_heads):
                        want = c.keys(s, h, which)[total - have:]
                        assert torch.equal(rows[at + n - have:at + n, h], want.to(dtype))
            for t in (k, v):
                assert (t[:, :off] == 7.0).all() and (t[:, off + width:] == 7.0).all()


def test_a_cache_moves_from_one_type_to_another(ctx):  # noqa: F811
    """Sequences read from a 4-bit cache, appended to an F16 one and back: the same codes, for the scales are kept."""
    import gsvcu
    c = Q4Case("f16", [200, 64, 1], [200, 64, 1], 4, 4, 64)
    cache, chunks = c.objects()
    k, v, k2, v2 = (torch.empty(c.rows, 4, 64, dtype=torch.float16, device="cuda") for _ in range(4))
    wide = torch.zeros(c.pool.shape[0], 1, 2, 4, PAGE, 64, dtype=torch.float16, device="cuda")
    again = torch.full_like(c.pool, 255)
    order(ctx).op_kv_read(cache, chunks, 1, k, v)
    ctx.op_kv_append(gsvcu.PagedKV(wide), chunks, 0, None, k, v, None)
    ctx.op_kv_read(gsvcu.PagedKV(wide), chunks, 0, k2, v2)
    ctx.op_kv_append(gsvcu.PagedKV(again, rows=torch.float16), chunks, 1, None, k2, v2, None)
    ctx.sync()
    assert torch.equal(k, k2) and torch.equal(v, v2)
    for s in range(3):
        for h in range(4):
            for which in (0, 1):
                old, new = c.keys(s, h, which), None
                p = c.table[s, :-(-c.kv_len[s] // PAGE)].long()
                new = q4_format.decode(again[p, 1, which, h])[0].reshape(-1, 64)[:c.kv_len[s]]
                _, scale, _ = q4_format.decode(c.pool[p, 1, which, h])
                assert ((old - new).abs() <= 1.04 * scale.reshape(-1, 64)[:c.kv_len[s]].abs()).all()
                full = (q4_format.decode(c.pool[p, 1, which, h])[2].reshape(-1, 2, 32)[:c.kv_len[s]] == 0).any(-1)
                assert torch.equal(old.view(-1, 2, 32)[full], new.view(-1, 2, 32)[full])   # code 0: the scale again


# ------------------------------------------------------------------ together, streams, graphs, refusals

@pytest.mark.parametrize("ty", ["f16", "bf16"])
def test_chunks_of_any_size_give_the_whole_prompt(ctx, ty):  # noqa: F811
    """A prompt normalised, rotated, quantised and attended in chunks (one token, many, odd ones): the same cache bit for
    bit, and what one chunk gives within the rounding."""
    import gsvcu
    heads, kv_heads, dim, total = 8, 2, 64, 331
    c = Q4Case(ty, [total], [total], heads, kv_heads, dim)
    ang = torch.arange(total, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(32, device="cuda") / 32.0)
    turn = dict(cos=ang.cos().float(), sin=ang.sin().float(), q_norm=torch.rand(dim, device="cuda") + 0.5,
                k_norm=torch.rand(dim, device="cuda") + 0.5)
    q, k, v = c.rand(total, heads, dim), c.rand(total, kv_heads, dim), c.rand(total, kv_heads, dim)
    cache, chunks = c.objects()
    qr, whole = torch.empty_like(q), torch.empty_like(q)
    order(ctx).op_kv_append(cache, chunks, 1, q, k, v, qr, **turn)
    ctx.op_chunk_attention(cache, chunks, 1, qr, whole)
    ctx.sync()
    check_attention(c, qr, whole, None, dim ** -0.5)
    pool = c.pool.clone()
    used = c.table[0, :6].long()
    c.pool[used, 1] = 255
    out = torch.empty_like(q)
    at = 0
    for n in (1, 1, 60, 5, 130, 1, 64, 69):
        part = gsvcu.ChunkBatch(torch.tensor([0, n], dtype=torch.int32, device="cuda"),
                                torch.tensor([at + n], dtype=torch.int32, device="cuda"), c.table, n, n)
        sl = slice(at, at + n)
        qp = torch.empty_like(q[sl])
        order(ctx).op_kv_append(cache, part, 1, q[sl], k[sl], v[sl], qp, **turn)
        ctx.op_chunk_attention(cache, part, 1, qp, out[sl])
        ctx.sync()
        assert torch.equal(qp, qr[sl])
        at += n
    assert at == total
    for a, b in zip(q4_format.decode(pool[used, 1]), q4_format.decode(c.pool[used, 1])):
        a, b = (t.permute(1, 2, 0, 3, 4).reshape(2, 2, -1, dim)[:, :, :total] for t in (a, b))
        assert torch.equal(a, b)
    check_attention(c, qr, out, None, dim ** -0.5)


@pytest.mark.parametrize("q", [1, 70])
def test_work_queued_on_the_contexts_stream(ctx, q):  # noqa: F811
    """Ordered with torch's work on the context's stream, captured in a CUDA graph and replayed on new contents."""
    c = Q4Case("f16", [q] * 4, [q + 300, q + 41, q + 64, q], 8, 2, 64, max_pages=8)
    cache, chunks = c.objects()
    n = c.rows
    x, k, v = c.rand(n, 8, 64), c.rand(n, 2, 64), c.rand(n, 2, 64)
    qo, out, kb, vb = torch.empty_like(x), torch.empty_like(x), torch.empty_like(k), torch.empty_like(v)
    w = torch.rand(64, device="cuda") + 0.5

    def step():
        ctx.op_kv_append(cache, chunks, 1, x, k, v, qo, q_norm=w, k_norm=w)
        ctx.op_chunk_attention(cache, chunks, 1, qo, out)
        ctx.op_kv_read(cache, chunks, 1, kb, vb)

    torch.cuda.synchronize()
    st = torch.cuda.ExternalStream(ctx.stream_handle())
    with torch.cuda.stream(st):
        x *= 2.0
        step()
        y = out + 0.0
    torch.cuda.synchronize()
    check_attention(c, qo, y, None, 0.125)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        step()
    for _ in range(2):
        x.normal_()
        k.normal_()
        v.normal_()
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            graph.replay()
        torch.cuda.synchronize()
        check_attention(c, qo, out, None, 0.125)
        code, scale = q4_format.quantise(v)
        assert torch.equal(vb.double(), (code.double() - 8) * scale.double().repeat_interleave(32, -1))
    ctx.sync()


def test_refusals(ctx):  # noqa: F811
    import ctypes
    import gsvcu
    c = Q4Case("f16", [2], [70], 4, 2, 64)
    cache, chunks = c.objects()
    q, kv = c.rand(2, 4, 64), c.rand(2, 2, 64)
    out, w = torch.empty_like(q), torch.ones(64, device="cuda")
    lib = ctx.lib
    assert lib.gsvcu_op_kv_read(ctx.h, None) == -1 and lib.gsvcu_op_kv_append_norm(ctx.h, None, None) == -1
    assert lib.gsvcu_op_kv_read(ctx.h, ctypes.byref(gsvcu.KvReadArgs())) == -1
    launches = ctx.kernel_launches()
    for bad in (dict(q_norm=w[:63].contiguous()), dict(k_norm=w.half()), dict(q_norm=w.cpu()), dict(k_norm=torch.ones(128, device="cuda")[::2])):
        with pytest.raises(ValueError):
            ctx.op_kv_append(cache, chunks, 1, q, kv, kv, out, **bad)
    for eps in (-1e-6, float("nan"), float("inf")):
        with pytest.raises(gsvcu.GsvcuError) as e:
            ctx.op_kv_append(cache, chunks, 1, q, kv, kv, out, q_norm=w, eps=eps)
        assert e.value.code == -1 and "eps" in str(e.value)
    with pytest.raises(gsvcu.GsvcuError):   # BF16 rows beside an F16 cache of 4 bits
        ctx.op_kv_append(cache, chunks, 1, q.bfloat16(), kv.bfloat16(), kv.bfloat16(), out)
    with pytest.raises(ValueError):         # q_out of another type than the cache's rows
        ctx.op_kv_append(cache, chunks, 1, q.float(), kv.float(), kv.float(), out.float())
    with pytest.raises(ValueError):
        ctx.op_chunk_attention(cache, chunks, 1, q.float(), out)
    for k, v in ((kv, kv.float()), (kv[:1], kv[:1]), (kv.cpu(), kv), (q, q)):
        with pytest.raises(ValueError):
            ctx.op_kv_read(cache, chunks, 1, k, v)
    with pytest.raises(gsvcu.GsvcuError):
        ctx.op_kv_read(cache, chunks, 1, kv.bfloat16(), kv.bfloat16())
    with pytest.raises(gsvcu.GsvcuError) as e:
        ctx.op_kv_read(cache, chunks, 2, kv, kv.clone())
    assert "layer" in str(e.value)
    odd = torch.zeros(3, 1, 2, 1, PAGE, 27, dtype=torch.uint8, device="cuda")   # heads of 48
    one = torch.empty(2, 1, 48, dtype=torch.float16, device="cuda")
    with pytest.raises(gsvcu.GsvcuError) as e:
        ctx.op_chunk_attention(gsvcu.PagedKV(odd, rows=torch.float16), chunks, 0, one, one.clone())
    assert "head_dim" in str(e.value)

    def call(fn, struct, args, *more, kv_dtype=None):
        desc = gsvcu.PagedKVDesc.from_buffer_copy(cache.desc)
        if kv_dtype is not None:
            desc.kv_dtype = kv_dtype
        a = struct(kv=ctypes.addressof(desc), batch=ctypes.addressof(chunks.desc), **args)
        return getattr(lib, fn)(ctx.h, ctypes.byref(a), *more)

    read = dict(k=kv.data_ptr(), v=kv.data_ptr(), k_stride=128, v_stride=128, layer=1, row_dtype=0)
    append = dict(q=q.data_ptr(), k=kv.data_ptr(), v=kv.data_ptr(), q_out=out.data_ptr(), q_stride=256, k_stride=128, v_stride=128,
                  q_out_stride=256, layer=1, row_dtype=0, n_q_head=4)
    for bad in (dict(k=0), dict(v=0), dict(k=read["k"] + 1), dict(v=read["v"] + 1), dict(k_stride=127), dict(v_stride=0), dict(row_dtype=2),
                dict(row_dtype=3), dict(layer=-1)):
        assert call("gsvcu_op_kv_read", gsvcu.KvReadArgs, dict(read, **bad)) == -1, bad
    for dtype in (-1, 5, 100):
        assert call("gsvcu_op_kv_read", gsvcu.KvReadArgs, read, kv_dtype=dtype) == -1
        assert call("gsvcu_op_kv_append", gsvcu.KvAppendArgs, append, kv_dtype=dtype) == -1
    for norm in (gsvcu.HeadNorm(w.data_ptr() + 2, 0, 0.0), gsvcu.HeadNorm(0, w.data_ptr() + 1, 0.0), gsvcu.HeadNorm(0, 0, -1.0)):
        assert call("gsvcu_op_kv_append_norm", gsvcu.KvAppendArgs, append, ctypes.byref(norm)) == -1
    assert call("gsvcu_op_kv_append", gsvcu.KvAppendArgs, dict(append, row_dtype=3)) == -1
    ctx.sync()
    assert ctx.kernel_launches() == launches


@pytest.mark.parametrize("q", [2, 150])
def test_bad_device_arrays_are_reported(ctx, q):  # noqa: F811
    """A page outside the pool, lengths beyond the table or the given bounds, a position outside the table of angles: memory
    outside the arrays stays untouched, the other sequences are right, and the next sync reports it once."""
    import gsvcu

    def expect(words):
        with pytest.raises(gsvcu.GsvcuError) as e:
            ctx.sync()
        assert e.value.code == -1 and words in str(e.value)
        ctx.sync()

    c = Q4Case("f16", [q, q], [q + 100, q + 30], 4, 2, 64)
    x, kv = c.rand(2 * q, 4, 64), c.rand(2 * q, 2, 64)
    out, qo, back = torch.empty_like(x), torch.empty_like(x), torch.empty_like(kv)
    w = torch.ones(64, device="cuda")
    cache, chunks = c.objects()
    good = c.table.clone()
    for page in (-1, c.pool.shape[0], 2 ** 31 - 1):
        c.table[1, (q + 29) // PAGE] = page
        before = c.pool.clone()
        order(ctx).op_kv_append(cache, chunks, 1, x, kv, kv, qo, q_norm=w)
        expect("page")
        seen = torch.zeros(c.pool.shape[0], dtype=torch.bool, device="cuda")
        seen[good[0, :(q + 99) // PAGE + 1].long()] = True
        seen[good[1, :(q + 29) // PAGE].long()] = True
        assert torch.equal(before[~seen], c.pool[~seen])
        order(ctx).op_kv_read(cache, chunks, 1, back, back.clone())
        expect("page")
        assert torch.equal(back[:q, 0].double(), c.keys(0, 0, 0)[100:])
        order(ctx).op_chunk_attention(cache, chunks, 1, x, out)
        expect("page")
        check = Q4Case.__new__(Q4Case)
        check.__dict__.update(c.__dict__, q_len=[q, 0], kv_len=[q + 100, 0], rows=q, heads=4)
        check_attention(check, x[:q], out[:q], None, 0.125)
    c.table.copy_(good)
    c.table[1] = good[0]
    c.kv[1] = 64 * c.table.shape[1] + 5
    for op in (lambda: ctx.op_chunk_attention(cache, chunks, 1, x, out), lambda: ctx.op_kv_append(cache, chunks, 1, x, kv, kv, qo),
               lambda: ctx.op_kv_read(cache, chunks, 1, back, back.clone())):
        order(ctx)
        op()
        expect("kv_len")
    c.kv[1] = q + 30
    c.table.copy_(good)
    ang = torch.ones(q + 50, 32, device="cuda")
    order(ctx).op_kv_append(cache, chunks, 1, x, kv, kv, qo, cos=ang, sin=ang, k_norm=w)
    expect("position")


@pytest.mark.parametrize("group", [1, 5, 7])
@pytest.mark.parametrize("max_kv", [0, 9000])
@pytest.mark.parametrize("bounds", [(0, -723922764), (7, -1292124672), (8, -1199745), (0, -1599320890), (3, -2 ** 31),
                                    (-5, 3), (-2 ** 31, 2 ** 31 - 1), (8, 2 ** 31 - 1), (2 ** 31 - 1, -2 ** 31), (9, 9)])
def test_row_bounds_far_outside_the_batch(ctx, group, max_kv, bounds):  # noqa: F811
    """row_start with values whose differences and products pass 32 bits, lengths far off: all three operators report them and
    write nothing outside their rows and pages. With the wider bound on the lengths the pages are dealt out."""
    import gsvcu
    c = Q4Case("f16", [8], [70], 2 * group, 2, 64, max_pages=200 if max_kv else None)
    c.table.fill_(1)
    c.row_start.copy_(torch.tensor(bounds, dtype=torch.int32))
    x, kv = c.rand(8, 2 * group, 64), c.rand(8, 2, 64)
    guard, back = torch.full((72, 2 * group, 64), 7.0, dtype=c.dtype, device="cuda"), torch.full((72, 2, 64), 7.0, dtype=c.dtype, device="cuda")
    w = torch.ones(64, device="cuda")
    cache, chunks = c.objects(max_kv)
    for lens in (70, 0, -2 ** 31, 2 ** 31 - 1):
        c.kv.fill_(lens)
        before = c.pool.clone()
        for call in (lambda: ctx.op_chunk_attention(cache, chunks, 1, x, guard[32:40]),
                     lambda: ctx.op_kv_append(cache, chunks, 1, x, kv, kv, guard[32:40], q_norm=w, k_norm=w),
                     lambda: ctx.op_kv_read(cache, chunks, 1, back[32:40], back[32:40].clone())):
            order(ctx)
            call()
            with pytest.raises(gsvcu.GsvcuError) as e:
                ctx.sync()
            assert e.value.code == -1
        for g in (guard, back):
            assert (g[:32] == 7.0).all() and (g[40:] == 7.0).all()
        assert torch.equal(before[:, 0], c.pool[:, 0])   # (the other layer)
    ctx.sync()


@pytest.mark.parametrize("q", [2, 70])
@pytest.mark.parametrize("kv", [100, 5000])
def test_the_operators_report_the_same_bounds(ctx, q, kv):  # noqa: F811
    """Lengths inside the table but outside the given sizes, and rows that no sequence owns, are reported after every operator; a
    bound on the chunks that is wider than the batch is none of these."""
    import gsvcu
    c = Q4Case("f16", [q, q], [q + kv, q + 30], 4, 2, 64, max_pages=90)
    x, rows = c.rand(2 * q, 4, 64), c.rand(2 * q, 2, 64)
    out = torch.empty_like(x)
    cache, _ = c.objects()

    def reported(max_chunk=q, max_kv=q + kv):
        chunks = gsvcu.ChunkBatch(c.row_start, c.kv, c.table, 2 * q, max_chunk, max_kv)
        found = []
        for call in (lambda: ctx.op_kv_append(cache, chunks, 1, x, rows, rows, out), lambda: ctx.op_chunk_attention(cache, chunks, 1, x, out),
                     lambda: ctx.op_kv_read(cache, chunks, 1, rows.clone(), rows.clone())):
            order(ctx)
            call()
            try:
                ctx.sync()
                found.append(None)
            except gsvcu.GsvcuError as e:
                assert e.code == -1
                found.append("kv_len" in str(e))
        return found

    assert reported() == [None] * 3
    assert reported(max_chunk=2 * q + 999) == [None] * 3
    assert reported(max_kv=q + kv - 1) == [True] * 3
    assert reported(max_chunk=q - 1) == [True] * 3
    for bounds in ((0, q, 2 * q - 1), (1, q, 2 * q)):
        c.row_start.copy_(torch.tensor(bounds, dtype=torch.int32))
        assert reported() == [True] * 3, bounds
    c.row_start.copy_(torch.tensor([0, q, 2 * q], dtype=torch.int32))
    c.kv[1] = -1
    assert reported() == [True] * 3


def test_nothing_to_do(ctx):  # noqa: F811
    """No rows: nothing is touched, nothing is launched."""
    c = Q4Case("f16", [0, 0], [5, 70], 4, 2, 64)
    out, w = torch.zeros(0, 4, 64, dtype=torch.float16, device="cuda"), torch.ones(64, device="cuda")
    cache, chunks = c.objects()
    before = ctx.kernel_launches()
    ctx.op_chunk_attention(cache, chunks, 0, out, out.clone())
    ctx.op_kv_append(cache, chunks, 0, out, out[:, :2], out[:, :2], out.clone(), q_norm=w, k_norm=w)
    ctx.op_kv_read(cache, chunks, 0, out[:, :2], out[:, :2].clone())
    ctx.sync()
    assert ctx.kernel_launches() == before


def test_example_with_a_4_bit_cache():
    """examples/chunked_decoder.py over 4 bits. Chunks and whole prompts round their products to BF16 in another order, so a
    key or value may differ by 2^-8 of itself and, where that crosses a border between codes, by a step s. With elements of up
    to 8 steps, 3 on average, 2 * 3 * 2^-8 = 2.3 % of the codes cross: 0.15 s over all, and s is at most a quarter of the
    elements' size: 4 % per layer, under 10 % for both layers' residuals."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "chunked_decoder.py")
    spec = importlib.util.spec_from_file_location("chunked_decoder", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    assert mod.main(lengths=(130, 9, 65), pieces=(50, 1, 64), bits=4) < 0.1
