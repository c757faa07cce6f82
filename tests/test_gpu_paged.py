"""The paged-cache operators (Context.op_kv_append, Context.op_chunk_attention) against their formulas in 64
bits, through the Python binding of the C ABI.

Tolerances follow from the arithmetic and are set per element. With u the unit roundoff of the cache's type:
  append     one rounding of an f32 sum of two products: u |y| + 4 * 2^-24 (|a| + |b|), plus half a subnormal
             step of F16.
  attention  the output's rounding u |o|, plus the relative error of the weights times A = sum w |v| / sum w.
             A weight's error: the score's (f32 sum of D products, at most (D + 8) 2^-24 sum_d |q_d k_d| scale,
             doubled for F32's two-part products), its scaling and the exponential (2^-20 covers scores up to
             16 and both), twice for numerator and denominator; the sums of n keys (n / 64 + 64) 2^-24. Where the
             weights themselves are rounded to 16 bits (many rows), u A on top.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

PAGE = 64
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
ROUND = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}


@pytest.fixture(scope="module")
def ctx():
    import gsvcu
    c = gsvcu.Context(0)
    yield c
    c.close()


def order(ctx):
    """The context's stream waits for what torch has queued (the operators run on the context's stream)."""
    torch.cuda.synchronize()
    return ctx


class Case:
    """Ragged sequences in a shuffled paged cache whose unused parts hold NaN and whose unused table entries
    name pages far outside the pool."""

    def __init__(self, ty, q_len, kv_len, heads, kv_heads, dim, layers=2, layer=1, spare=2, seed=0, max_pages=None):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.ty, self.dtype, self.layer = ty, TYPES[ty], layer
        self.q_len, self.kv_len, self.heads, self.kv_heads, self.dim = q_len, kv_len, heads, kv_heads, dim
        pages = [-(-n // PAGE) for n in kv_len]
        n_pages = sum(pages) + spare
        width = max_pages or max(1, max(pages, default=1))
        perm = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((len(kv_len), width), 2 ** 30, dtype=torch.int32, device="cuda")
        self.pool = torch.full((n_pages, layers, 2, kv_heads, PAGE, dim), float("nan"), dtype=self.dtype, device="cuda")
        at = 0
        for s, n in enumerate(pages):
            self.table[s, :n] = perm[at:at + n]
            for j in range(n):
                here = min(PAGE, kv_len[s] - j * PAGE)
                self.pool[int(perm[at + j]), layer, :, :, :here] = torch.randn(
                    2, kv_heads, here, dim, generator=g, device="cuda").to(self.dtype)
            at += n
        starts = np.concatenate([[0], np.cumsum(q_len)]).astype(np.int32)
        self.rows = int(starts[-1])
        self.starts = starts
        self.row_start = torch.from_numpy(starts).cuda()
        self.kv = torch.tensor(kv_len, dtype=torch.int32, device="cuda")
        self.gen = g

    def rand(self, *shape, dtype=None):
        return torch.randn(*shape, generator=self.gen, device="cuda").to(dtype or self.dtype)

    def objects(self, max_kv=0, max_chunk=None):
        import gsvcu
        longest = max(self.q_len, default=0) if max_chunk is None else max_chunk
        return gsvcu.PagedKV(self.pool), gsvcu.ChunkBatch(self.row_start, self.kv, self.table, self.rows, longest, max_kv)

    def keys(self, s, h, which):
        n = self.kv_len[s]
        p = self.table[s, :-(-n // PAGE)].long()
        return self.pool[p, self.layer, which, h].reshape(-1, self.dim)[:n].double()


def attention_oracle(c, q, scale, window=0, prefix=None):
    """(out, lse, A, S): the definition in 64 bits; A = sum w |v| / sum w, S = the largest sum |q_d k_d| scale."""
    out = torch.zeros(c.rows, c.heads, c.dim, dtype=torch.float64, device="cuda")
    amp, lse = torch.zeros_like(out), torch.full((c.rows, c.heads), float("-inf"), dtype=torch.float64, device="cuda")
    mag = torch.zeros(c.rows, c.heads, dtype=torch.float64, device="cuda")
    g = c.heads // c.kv_heads
    for s, (n, total) in enumerate(zip(c.q_len, c.kv_len)):
        if n == 0 or total == 0:
            continue
        at = int(c.starts[s])
        pos = torch.arange(total - n, total, device="cuda")[:, None]
        key = torch.arange(total, device="cuda")[None]
        seen = key <= pos
        if window:
            seen = seen & (key > pos - window)
        if prefix is not None:
            seen = seen | (key < int(prefix[s]))
        for h in range(c.heads):
            k, v = c.keys(s, h // g, 0), c.keys(s, h // g, 1)
            x = q[at:at + n, h].double()
            sc = (x @ k.T * scale).masked_fill(~seen, float("-inf"))
            top = sc.amax(1, keepdim=True).clamp_min(-1e300)
            w = (sc - top).exp()
            tot = w.sum(1, keepdim=True)
            safe = torch.where(tot > 0, tot, 1.0)
            out[at:at + n, h] = w @ v / safe
            amp[at:at + n, h] = w @ v.abs() / safe
            lse[at:at + n, h] = (top + tot.log())[:, 0]
            mag[at:at + n, h] = (x.abs() @ k.abs().T * abs(scale)).amax(1)
    return out, lse, amp, mag


def check_attention(c, q, out, lse, scale, window=0, prefix=None, label=""):
    ro, rl, amp, mag = attention_oracle(c, q, scale, window, prefix)
    n = max(c.kv_len, default=0)
    u = ROUND[c.ty]
    weight = (2.0 if c.ty == "f32" else 1.0) * (c.dim + 8) * 2.0 ** -24 * mag + 2.0 ** -20 + (n / 64 + 64) * 2.0 ** -24
    tol = u * ro.abs() + (2 * weight[..., None] + (u if c.ty != "f32" else 0.0)) * amp + (2.0 ** -25 if c.ty == "f16" else 0.0)
    err = (out.double() - ro).abs()
    assert torch.isfinite(out).all(), label
    assert (err <= tol).all(), (label, float((err / tol.clamp_min(1e-300)).max()))
    if lse is not None:
        empty = torch.isinf(rl)
        assert torch.equal(torch.isneginf(lse), empty), label
        e = (lse.double() - rl).abs()[~empty]
        t = (weight + 2.0 ** -22 * rl.abs())[~empty]
        assert (e <= t).all(), (label, float((e / t).max()) if e.numel() else 0)


def attend(ctx, c, q=None, window=0, prefix=None, scale=None, max_kv=0, max_chunk=None, lse=True, label=""):
    q = c.rand(c.rows, c.heads, c.dim) if q is None else q
    out = torch.full((c.rows, c.heads, c.dim), float("nan"), dtype=c.dtype, device="cuda")
    ls = torch.full((c.rows, c.heads), float("nan"), device="cuda") if lse else None
    pf = None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device="cuda")
    cache, chunks = c.objects(max_kv, max_chunk)
    order(ctx).op_chunk_attention(cache, chunks, c.layer, q, out, scale=scale, prefix=pf, window=window, lse=ls)
    ctx.sync()
    check_attention(c, q, out, ls, c.dim ** -0.5 if scale is None else scale, window, prefix, label)
    return q, out, ls


# ------------------------------------------------------------------ attention

@pytest.mark.parametrize("ty", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(16, 16), (8, 2), (7, 1), (32, 2)])
def test_single_tokens(ctx, ty, dim, heads, kv_heads):
    """One new token per sequence: one key, page ends inside and at a tile, ragged lengths."""
    attend(ctx, Case(ty, [1] * 9, [1, 2, 15, 63, 64, 65, 127, 200, 517], heads, kv_heads, dim))


@pytest.mark.parametrize("ty", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (6, 2), (8, 1), (5, 1)])
def test_ragged_chunks(ctx, ty, dim, heads, kv_heads):
    """Chunks of 0, 1, a few and many rows, with and without cached keys before them."""
    attend(ctx, Case(ty, [5, 0, 1, 17, 33, 130, 64, 300], [5, 40, 1, 17, 95, 131, 700, 301], heads, kv_heads, dim))


@pytest.mark.parametrize("ty,dim,heads,kv_heads", [("f16", 64, 16, 4), ("bf16", 128, 8, 2), ("f32", 32, 4, 4),
                                                   ("f16", 32, 16, 16), ("bf16", 64, 12, 1)])
@pytest.mark.parametrize("window,prefix", [(1, None), (16, None), (100, None), (64, [0, 3, 200, 64, 90]),
                                           (0, [1, 3, 333, 64, 90]), (37, [0, 0, 5000, 129, 500]), (4096, None)])
def test_windows_and_prefixes(ctx, ty, dim, heads, kv_heads, window, prefix):
    """Sliding windows, prefixes that every row sees (longer than the sequence included), both together."""
    attend(ctx, Case(ty, [70, 1, 200, 129, 3], [400, 333, 200, 640, 90], heads, kv_heads, dim), window=window, prefix=prefix)


@pytest.mark.parametrize("ty,dim", [("f16", 32), ("bf16", 128), ("f32", 64)])
@pytest.mark.parametrize("q", [3, 150])
def test_rows_that_see_nothing(ctx, ty, dim, q):
    """No keys at all, or a chunk longer than its keys: those rows give 0 and -infinity."""
    c = Case(ty, [q, q, 1], [0, 2, 0], 4, 2, dim)
    _, out, lse = attend(ctx, c)
    assert (out[:q] == 0).all() and torch.isneginf(lse[:q]).all()
    assert (out[q:2 * q - 2] == 0).all() and torch.isneginf(lse[q:2 * q - 2]).all()
    assert torch.isfinite(lse[2 * q - 2:2 * q]).all()


@pytest.mark.parametrize("ty,dim,heads,kv_heads,q", [("bf16", 128, 32, 8, 1), ("f16", 32, 16, 16, 1), ("f32", 64, 4, 1, 2),
                                                     ("bf16", 128, 8, 2, 40), ("f16", 64, 4, 4, 150), ("f16", 32, 4, 4, 150)])
def test_long_caches_are_split(ctx, ty, dim, heads, kv_heads, q):
    """Few rows over long caches (work split over the keys and joined); the same result twice, bit for bit, also
    with a looser bound on the length."""
    c = Case(ty, [q, q, q], [9000, 4097, q], heads, kv_heads, dim, max_pages=200)
    x, a, la = attend(ctx, c, max_kv=9000)
    _, b, lb = attend(ctx, c, q=x, max_kv=9000)
    assert torch.equal(a, b) and torch.equal(la, lb)
    attend(ctx, c, q=x, max_kv=0, lse=False)


@pytest.mark.parametrize("scale", [0.0, 1.7, -0.3])
@pytest.mark.parametrize("q", [1, 140])
def test_scales(ctx, scale, q):
    attend(ctx, Case("f16", [q, 9], [257, 80], 8, 2, 64), scale=scale)


@pytest.mark.parametrize("ty,dim,q", [("f16", 64, 4), ("bf16", 128, 200), ("f32", 32, 5), ("f16", 32, 300)])
def test_growing_scores(ctx, ty, dim, q):
    """Keys whose scores grow along the cache by far more than the type's range of weights: every tile raises the
    running maximum, and the first keys' weights vanish."""
    c = Case(ty, [q], [900], 4, 2, dim)
    x = c.rand(c.rows, c.heads, c.dim).abs() + 0.5
    ramp = torch.linspace(-4.0, 4.0, 900, device="cuda")
    p = c.table[0, :-(-900 // PAGE)].long()
    k = c.pool[p, c.layer, 0].permute(1, 0, 2, 3).reshape(2, -1, dim)
    k[:, :900] = (torch.ones(2, 900, dim, device="cuda") * ramp[None, :, None]).to(c.dtype)
    c.pool[p, c.layer, 0] = k.reshape(2, -1, PAGE, dim).permute(1, 0, 2, 3)
    attend(ctx, c, q=x.to(c.dtype))


@pytest.mark.parametrize("ty", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("q", [1, 90])
def test_strided_and_unaligned_rows(ctx, ty, q):
    """Queries and outputs as slices of wider rows, at offsets and strides that 16-byte accesses do not fit; what
    lies between the rows stays."""
    c = Case(ty, [q, q], [130, q], 4, 2, 64)
    for width, off in ((4 * 64 + 5, 1), (4 * 64 + 64, 32)):
        qs = c.rand(c.rows, width)
        os_ = torch.full((c.rows, width), 7.0, dtype=c.dtype, device="cuda")
        q3 = qs[:, off:off + 256].unflatten(1, (4, 64))
        o3 = os_[:, off:off + 256].unflatten(1, (4, 64))
        cache, chunks = c.objects()
        order(ctx).op_chunk_attention(cache, chunks, c.layer, q3, o3)
        ctx.sync()
        check_attention(c, q3, o3, None, 0.125)
        assert (os_[:, :off] == 7.0).all() and (os_[:, off + 256:] == 7.0).all()


@pytest.mark.parametrize("ty,dim", [("f16", 128), ("f32", 32)])
@pytest.mark.parametrize("q", [1, 140])
def test_offsets_past_32_bits(ctx, ty, dim, q):
    """Pages whose element offset passes 2^32."""
    import gsvcu
    dtype, heads = TYPES[ty], 2
    n_page = (2 ** 32) // (2 * heads * PAGE * dim) + 40
    pool = torch.empty(n_page, 1, 2, heads, PAGE, dim, dtype=dtype, device="cuda")
    c = Case(ty, [q], [150], heads, heads, dim, layers=1, layer=0)
    far = torch.tensor([[n_page - 1, n_page - 7, n_page - 30]], dtype=torch.int32, device="cuda")
    pool[far[0].long()] = c.pool[c.table[0].long()]
    pool[:3] = float("nan")
    x = c.rand(c.rows, heads, dim)
    kv = c.rand(c.rows, 2, heads, dim)
    out, qo = torch.empty_like(x), torch.empty_like(x)
    c.pool, c.table = pool, far
    cache, chunks = c.objects()
    order(ctx).op_kv_append(cache, chunks, 0, x, kv[:, 0], kv[:, 1], qo)
    ctx.op_chunk_attention(cache, chunks, 0, qo, out)
    ctx.sync()
    got = torch.cat([c.keys(0, h, 0)[150 - q:, None] for h in range(heads)], 1)
    assert torch.equal(qo, x) and torch.equal(got, kv[:, 0].double())
    check_attention(c, x, out, None, dim ** -0.5)
    del pool, c


def test_masked_values_may_be_anything(ctx):
    """Keys and values past kv_len, in the same pages, may be infinite or NaN (also covered by every other case's
    NaN): bits of the result do not depend on them."""
    for ty, q in (("f16", 1), ("bf16", 200), ("f32", 40)):
        c = Case(ty, [q], [q + 70], 4, 4, 64)
        x, a, _ = attend(ctx, c)
        c.pool.masked_fill_(c.pool.isnan(), float("inf"))
        _, b, _ = attend(ctx, c, q=x)
        c.pool.masked_fill_(c.pool.isinf(), 0.0)
        _, d, _ = attend(ctx, c, q=x)
        assert torch.equal(a, b) and torch.equal(a, d)


@pytest.mark.parametrize("ty,dim,q", [("f16", 32, 1), ("bf16", 128, 5), ("f32", 64, 40), ("f16", 64, 150), ("bf16", 128, 300)])
@pytest.mark.parametrize("prefix", [None, 70])
def test_pages_behind_the_window_may_be_gone(ctx, ty, dim, q, prefix):
    """A server with a sliding window gives back pages that no row sees any more: their table entries are stale and
    what they hold is another sequence's, or NaN. Neither is touched nor reported."""
    c = Case(ty, [q, 1], [2000, 900], 8, 2, dim)
    window = 130
    for s, (n, total) in enumerate(zip(c.q_len, c.kv_len)):
        first = total - n - window + 1
        for j in range(-(-total // PAGE)):
            seen = (j + 1) * PAGE > first or (prefix and j * PAGE < prefix)
            if not seen:
                c.pool[int(c.table[s, j])] = float("nan")
    x = c.rand(c.rows, c.heads, c.dim)
    full = c.table.clone()
    for s, (n, total) in enumerate(zip(c.q_len, c.kv_len)):
        for j in range(-(-total // PAGE)):
            if (j + 1) * PAGE <= total - n - window + 1 and not (prefix and j * PAGE < prefix):
                c.table[s, j] = -7
    out = torch.empty_like(x)
    pf = None if prefix is None else torch.tensor([prefix] * 2, dtype=torch.int32, device="cuda")
    cache, chunks = c.objects()
    order(ctx).op_chunk_attention(cache, chunks, c.layer, x, out, prefix=pf, window=window)
    ctx.sync()
    c.table.copy_(full)
    c.pool.nan_to_num_(0.0)
    check_attention(c, x, out, None, dim ** -0.5, window, None if prefix is None else [prefix] * 2)


def test_nothing_to_do(ctx):
    """No rows, or no sequences: nothing is touched, nothing is launched."""
    import gsvcu
    c = Case("f16", [0, 0], [5, 70], 4, 2, 64)
    out = torch.zeros(0, 4, 64, dtype=torch.float16, device="cuda")
    cache, chunks = c.objects()
    before = ctx.kernel_launches()
    ctx.op_chunk_attention(cache, chunks, 0, out, out.clone())
    ctx.op_kv_append(cache, chunks, 0, out, out[:, :2], out[:, :2], out.clone())
    ctx.sync()
    assert ctx.kernel_launches() == before


# ------------------------------------------------------------------ append

def rotate_oracle(x, cos, sin, pairs):
    x = x.double().clone()
    if cos is None:
        return x, x.abs()
    half = cos.shape[1]
    c, s = cos.double()[:, None], sin.double()[:, None]
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if pairs else (i, i + half)
    xa, xb = x[..., a], x[..., b]
    mag = x.abs()
    mag[..., a] = mag[..., b] = xa.abs() + xb.abs()
    x[..., a], x[..., b] = xa * c - xb * s, xa * s + xb * c
    return x, mag


def check_append(ctx, ty, row_ty, heads, kv_heads, dim, rot, pairs=False, own_pos=False, q_len=(3, 0, 1, 70, 130),
                 kv_len=(3, 5, 64, 200, 129), off=0, in_place=False, no_q=False):
    c = Case(ty, list(q_len), list(kv_len), heads, kv_heads, dim, layers=3)
    rd = TYPES[row_ty]
    width = (heads + 2 * kv_heads) * dim + off
    rows = c.rand(c.rows, width, dtype=rd)
    x = rows[:, off:].unflatten(1, (heads + 2 * kv_heads, dim))
    q, k, v = x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
    q0 = q.clone()
    cos = sin = pos = None
    place = torch.cat([torch.arange(t - n, t) for n, t in zip(q_len, kv_len)]).cuda()
    seq = torch.repeat_interleave(torch.arange(len(q_len)), torch.tensor(q_len)).cuda()
    at = place.clamp_min(0)
    if rot:
        ang = torch.arange(max(kv_len) + 1, dtype=torch.float64, device="cuda")[:, None] * \
            10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64, device="cuda") * 2 / rot)
        cos, sin = ang.cos().float(), ang.sin().float()
        if own_pos:
            at = torch.randint(0, max(kv_len), (c.rows,), generator=c.gen, device="cuda")
            pos = at.to(torch.int32)
    before = c.pool.clone()
    qo = q if in_place else torch.full((c.rows, heads, dim), float("nan"), dtype=c.dtype, device="cuda")
    cache, chunks = c.objects()
    order(ctx).op_kv_append(cache, chunks, 1, None if no_q else q, k, v, None if no_q else qo, cos=cos, sin=sin, pos=pos,
                            pairs=pairs)
    ctx.sync()
    ct, st = (None, None) if cos is None else (cos[at], sin[at])
    want_q, mag_q = rotate_oracle(q0, ct, st, pairs)
    want_k, mag_k = rotate_oracle(k, ct, st, pairs)
    u = ROUND[ty]
    tiny = 2.0 ** -25 if ty == "f16" else 0.0
    if not no_q:
        assert ((qo.double() - want_q).abs() <= u * want_q.abs() + 4 * 2.0 ** -24 * mag_q + tiny).all()
    ok = place >= 0
    page = c.table[seq[ok], place[ok] // PAGE].long()
    gk, gv = c.pool[page, 1, 0, :, place[ok] % PAGE], c.pool[page, 1, 1, :, place[ok] % PAGE]
    assert ((gk.double() - want_k[ok]).abs() <= u * want_k[ok].abs() + 4 * 2.0 ** -24 * mag_k[ok] + tiny).all()
    assert torch.equal(gv, v[ok].to(c.dtype))
    # nothing else changed
    before[page, 1, 0, :, place[ok] % PAGE] = gk
    before[page, 1, 1, :, place[ok] % PAGE] = gv
    same = (before == c.pool) | (before.isnan() & c.pool.isnan())
    assert same.all()


@pytest.mark.parametrize("ty,row_ty", [("f16", "f32"), ("f16", "f16"), ("bf16", "f32"), ("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("rot_share,pairs,own_pos", [(0, False, False), (1, False, False), (1, True, True), (2, False, True),
                                                     (2, True, False)])
def test_append(ctx, ty, row_ty, dim, rot_share, pairs, own_pos):
    check_append(ctx, ty, row_ty, 8, 2, dim, dim // rot_share if rot_share else 0, pairs, own_pos)


@pytest.mark.parametrize("rot", [2, 6, 24, 40, 62])
@pytest.mark.parametrize("pairs", [False, True])
def test_append_odd_rotation_widths(ctx, rot, pairs):
    check_append(ctx, "f16", "f32", 4, 4, 64, rot, pairs)


@pytest.mark.parametrize("off", [1, 3, 8])
def test_append_unaligned_rows(ctx, off):
    check_append(ctx, "bf16", "bf16", 4, 2, 128, 128, off=off)
    check_append(ctx, "f16", "f32", 4, 2, 32, 32, pairs=True, off=off)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (16, 16), (48, 1), (7, 7), (40, 8)])
@pytest.mark.parametrize("dim", [32, 128])
def test_append_head_counts(ctx, heads, kv_heads, dim):
    check_append(ctx, "bf16", "f32", heads, kv_heads, dim, dim)


def test_append_in_place_and_without_queries(ctx):
    check_append(ctx, "f16", "f16", 8, 2, 64, 64, in_place=True)
    check_append(ctx, "f16", "f16", 8, 2, 64, 24, in_place=True)
    check_append(ctx, "f32", "f32", 4, 4, 32, 32, pairs=True, no_q=True)


def test_append_chunk_longer_than_its_keys(ctx):
    """Rows whose cache position would be negative are rotated but not stored."""
    check_append(ctx, "f16", "f32", 4, 2, 64, 0, q_len=(9, 4), kv_len=(2, 4))


def test_append_many_sequences(ctx):
    n = 1200
    check_append(ctx, "f16", "f32", 2, 1, 32, 32, q_len=[i % 3 for i in range(n)], kv_len=[1 + (i * 7) % 150 + i % 3 for i in range(n)])


# ------------------------------------------------------------------ together, streams, graphs, refusals

@pytest.mark.parametrize("ty", ["f16", "bf16", "f32"])
def test_chunks_of_any_size_give_the_whole_prompt(ctx, ty):
    """A prompt appended and attended in chunks (one token, many, odd ones) gives what one chunk gives."""
    import gsvcu
    heads, kv_heads, dim, total = 8, 2, 64, 331
    c = Case(ty, [total], [total], heads, kv_heads, dim)
    ang = torch.arange(total, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(32, device="cuda") / 32.0)
    cos, sin = ang.cos().float(), ang.sin().float()
    q, k, v = c.rand(total, heads, dim), c.rand(total, kv_heads, dim), c.rand(total, kv_heads, dim)
    cache, chunks = c.objects()
    qr, whole = torch.empty_like(q), torch.empty_like(q)
    order(ctx).op_kv_append(cache, chunks, 1, q, k, v, qr, cos=cos, sin=sin)
    ctx.op_chunk_attention(cache, chunks, 1, qr, whole)
    ctx.sync()
    check_attention(c, qr, whole, None, dim ** -0.5)
    pool = c.pool.clone()
    c.pool.fill_(float("nan"))
    out = torch.empty_like(q)
    at = 0
    for n in (1, 1, 60, 5, 130, 1, 64, 69):
        row_start = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        kv = torch.tensor([at + n], dtype=torch.int32, device="cuda")
        part = gsvcu.ChunkBatch(row_start, kv, c.table, n, n)
        sl = slice(at, at + n)
        qp = torch.empty_like(q[sl])
        order(ctx).op_kv_append(cache, part, 1, q[sl], k[sl], v[sl], qp, cos=cos, sin=sin)
        ctx.op_chunk_attention(cache, part, 1, qp, out[sl])
        ctx.sync()
        assert torch.equal(qp, qr[sl])
        at += n
    assert at == total
    assert torch.equal(torch.nan_to_num(pool[:, 1]), torch.nan_to_num(c.pool[:, 1]))
    check_attention(c, qr, out, None, dim ** -0.5)


def test_work_queued_on_the_contexts_stream(ctx):
    """A torch stream over the context's stream orders torch's work with the operators' without host waits, and
    the calls can be captured in a CUDA graph and replayed on new contents."""
    c = Case("f16", [1] * 4, [300, 41, 64, 1], 8, 2, 64, max_pages=8)
    cache, chunks = c.objects()
    q, k, v = c.rand(4, 8, 64), c.rand(4, 2, 64), c.rand(4, 2, 64)
    qo, out = torch.empty_like(q), torch.empty_like(q)
    torch.cuda.synchronize()
    st = torch.cuda.ExternalStream(ctx.stream_handle())
    with torch.cuda.stream(st):
        x = q * 2.0
        ctx.op_kv_append(cache, chunks, 1, x, k, v, qo)
        ctx.op_chunk_attention(cache, chunks, 1, qo, out)
        y = out + 0.0
    torch.cuda.synchronize()
    assert torch.equal(qo, q * 2.0)
    check_attention(c, qo, y, None, 0.125)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        ctx.op_kv_append(cache, chunks, 1, q, k, v, qo)
        ctx.op_chunk_attention(cache, chunks, 1, qo, out)
    for seed in range(2):
        q.normal_()
        k.normal_()
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            graph.replay()
        torch.cuda.synchronize()
        check_attention(c, q, out, None, 0.125)
    ctx.sync()


def test_refusals(ctx):
    import ctypes
    import gsvcu
    assert ctx.lib.gsvcu_op_kv_append(ctx.h, None) == -1 and ctx.lib.gsvcu_op_chunk_attention(ctx.h, None) == -1
    empty = gsvcu.KvAppendArgs(), gsvcu.ChunkAttentionArgs()   # null cache and batch
    assert ctx.lib.gsvcu_op_kv_append(ctx.h, ctypes.byref(empty[0])) == -1
    assert ctx.lib.gsvcu_op_chunk_attention(ctx.h, ctypes.byref(empty[1])) == -1
    c = Case("f16", [2], [70], 4, 2, 64)
    cache, chunks = c.objects()
    q, kv = c.rand(2, 4, 64), c.rand(2, 2, 64)
    out = torch.empty_like(q)
    with pytest.raises(gsvcu.GsvcuError) as e:
        ctx.op_chunk_attention(cache, chunks, 2, q, out)
    assert e.value.code == -1 and "layer" in str(e.value)
    with pytest.raises(gsvcu.GsvcuError) as e:
        ctx.op_chunk_attention(cache, chunks, 1, c.rand(2, 5, 64), c.rand(2, 5, 64))
    assert e.value.code == -1 and "multiple" in str(e.value)
    for bad in (dict(window=-1), dict(scale=float("nan"))):
        with pytest.raises(gsvcu.GsvcuError):
            ctx.op_chunk_attention(cache, chunks, 1, q, out, **bad)
    with pytest.raises(ValueError):
        ctx.op_chunk_attention(cache, chunks, 1, q.float(), out)
    with pytest.raises(ValueError):
        ctx.op_chunk_attention(cache, chunks, 1, q[:1], out)
    with pytest.raises(ValueError):
        ctx.op_chunk_attention(cache, chunks, 1, q.transpose(1, 2).contiguous().transpose(1, 2), out)
    with pytest.raises(ValueError):
        ctx.op_chunk_attention(cache, chunks, 1, q, out, prefix=torch.zeros(1, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        ctx.op_kv_append(cache, chunks, 1, q, kv, kv.float(), out)
    with pytest.raises(gsvcu.GsvcuError):   # bf16 rows into an f16 cache
        ctx.op_kv_append(cache, chunks, 1, q.bfloat16(), kv.bfloat16(), kv.bfloat16(), out)
    cos = torch.zeros(80, 40, device="cuda")
    with pytest.raises(gsvcu.GsvcuError):   # rotates more than a head holds
        ctx.op_kv_append(cache, chunks, 1, q, kv, kv, out, cos=cos, sin=cos)
    for bad in (dict(q=q.cpu()), dict(out=out.cpu()), dict(cache=gsvcu.PagedKV(c.pool.cpu()))):   # host memory
        with pytest.raises(ValueError):
            ctx.op_chunk_attention(bad.get("cache", cache), chunks, 1, bad.get("q", q), bad.get("out", out))
    with pytest.raises(ValueError):
        gsvcu.ChunkBatch(c.row_start, c.kv.cpu(), c.table, 2, 2)
    odd = torch.empty(3, 1, 2, 1, PAGE, 48, dtype=torch.float16, device="cuda")
    one = torch.empty(2, 1, 48, dtype=torch.float16, device="cuda")
    with pytest.raises(gsvcu.GsvcuError) as e:
        ctx.op_chunk_attention(gsvcu.PagedKV(odd), chunks, 0, one, one.clone())
    assert "head_dim" in str(e.value)
    ctx.sync()


@pytest.mark.parametrize("ty", ["f16", "f32"])
@pytest.mark.parametrize("q", [2, 150])
def test_bad_device_arrays_are_reported(ctx, ty, q):
    """A page outside the pool, lengths beyond the table or the given bounds, a position outside the table of
    angles: memory outside the arrays stays untouched, the other sequences are right, and the next sync reports
    it once."""
    import gsvcu

    def expect(words):
        with pytest.raises(gsvcu.GsvcuError) as e:
            ctx.sync()
        assert e.value.code == -1 and words in str(e.value)
        ctx.sync()

    c = Case(ty, [q, q], [q + 100, q + 30], 4, 2, 64)
    x, kv = c.rand(2 * q, 4, 64), c.rand(2 * q, 2, 64)
    out, qo = torch.empty_like(x), torch.empty_like(x)
    cache, chunks = c.objects()
    good = c.table.clone()
    for page in (-1, c.pool.shape[0], 2 ** 31 - 1):
        c.table[1, (q + 29) // PAGE] = page
        before = c.pool.clone()
        order(ctx).op_kv_append(cache, chunks, 1, x, kv, kv, qo)
        expect("page")
        seen = torch.zeros(c.pool.shape[0], dtype=torch.bool, device="cuda")
        seen[good[0, :(q + 99) // PAGE + 1].long()] = True
        seen[good[1, :(q + 29) // PAGE].long()] = True
        assert torch.equal(torch.nan_to_num(before[~seen]), torch.nan_to_num(c.pool[~seen]))
        order(ctx).op_chunk_attention(cache, chunks, 1, x, out)
        expect("page")
        check = Case.__new__(Case)
        check.__dict__.update(c.__dict__, q_len=[q, 0], kv_len=[q + 100, 0], rows=q, heads=4)
        check_attention(check, x[:q], out[:q], None, 0.125)
    c.table.copy_(good)
    c.table[1] = good[0]
    c.kv[1] = 64 * c.table.shape[1] + 5
    order(ctx).op_chunk_attention(cache, chunks, 1, x, out)
    expect("kv_len")
    order(ctx).op_kv_append(cache, chunks, 1, x, kv, kv, qo)
    expect("kv_len")
    c.kv[1] = q + 30
    c.table.copy_(good)
    _, short = c.objects(max_chunk=q - 1)
    order(ctx).op_chunk_attention(cache, short, 1, x, out)
    expect("kv_len")
    ang = torch.ones(q + 50, 32, device="cuda")
    order(ctx).op_kv_append(cache, chunks, 1, x, kv, kv, qo, cos=ang, sin=ang)
    expect("position")
    attend(ctx, Case(ty, [q], [q + 7], 4, 2, 64))


def test_example_of_streaming_requests():
    """examples/chunked_decoder.py: prompts in pieces beside single tokens against the same prompts whole. Two BF16
    layers: the paths round the same sums in another order, 2^-8 each time, over 2 layers' products and residuals."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "chunked_decoder.py")
    spec = importlib.util.spec_from_file_location("chunked_decoder", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    assert mod.main(lengths=(130, 9, 65), pieces=(50, 1, 64)) < 4 * 2.0 ** -8
