"""Chunk attention at the ends of its range, over float and 4-bit caches: scores far above the steps of F32 and queries far
below those of F16.

Tolerances, set before the first run. u: unit roundoff of the rows' type.
  large scores   two keys with the same score, all others so far below that their weight is 0: the output is the mean of the
                 two values, off by a rounding of each weight to the type's bits (u, of the values' magnitudes), one of the
                 output (u) and F32's sums and quotient (2^-20). The log-sum-exp S + log 2 has a rounding of the scale's
                 factor, the product, the reference, its sum with the logarithm and the factor log 2: 5 times 2^-24 of S,
                 rounded up to 2^-21, and 1 for the logarithm.
"""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_paged import PAGE, ROUND, Case, ctx, order  # noqa: E402,F401
from test_gpu_paged_q4 import Q4Case, attend  # noqa: E402


def case(ty, q4, *args, **kw):
    return (Q4Case if q4 else Case)(ty, *args, **kw)


def set_layer(c, v):
    """The layer's keys and values [page][2][kv head][64][dim]."""
    if isinstance(c, Q4Case):
        c.set_values(v)
    else:
        c.pool[:, c.layer] = v.to(c.dtype)


# ------------------------------------------------------------------ large scores

TYPES = [("f16", False), ("bf16", False), ("f32", False), ("f16", True), ("bf16", True)]


@pytest.mark.parametrize("ty,q4", TYPES)
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("q,kv", [(1, 700), (1, 9000), (7, 5000), (14, 70), (60, 900), (60, 9000), (800, 2000)])
@pytest.mark.parametrize("scale", [1.0, 37.0, 1e12])
def test_finite_scores_of_any_size(ctx, ty, q4, dim, q, kv, scale):  # noqa: F811
    """Scores of 2^24 to 2^70, in few rows, in chunks, split and with their pages unpacked first: two keys share the weight,
    in every row as its own query decides how large they are."""
    c = case(ty, q4, [q], [kv + q], 2, 1, dim)
    a, b = 5, kv - 9
    v = torch.zeros(c.pool.shape[0], 2, 1, PAGE, dim, device="cuda")
    v[:, 1].normal_(generator=c.gen)
    for key in (a, b):
        v[int(c.table[0, key // PAGE]), 0, 0, key % PAGE, 0] = -16384.0
    set_layer(c, v)
    x = torch.zeros(q, 2, dim, device="cuda")
    x[..., 0] = -1024.0 * 2.0 ** (5.0 * torch.rand(q, 2, generator=c.gen, device="cuda"))
    x = x.bfloat16().to(c.dtype)   # (8 bits: the products are exact in every type)
    out, lse = torch.empty_like(x), torch.empty(q, 2, device="cuda")
    cache, chunks = c.objects()
    order(ctx).op_chunk_attention(cache, chunks, c.layer, x, out, scale=scale, lse=lse)
    ctx.sync()
    values = c.keys(0, 0, 1)
    va, vb = values[a], values[b]
    u = ROUND[ty]
    tol = u * ((va + vb) / 2).abs() + (u + 2.0 ** -20) * (va.abs() + vb.abs()) / 2 + (2.0 ** -25 if ty == "f16" else 0.0)
    score = x[..., 0].double() * -16384.0 * scale
    assert torch.isfinite(out).all(), (~torch.isfinite(out[..., 0])).sum()
    err = (out.double() - (va + vb) / 2).abs()
    assert (err <= tol).all(), float((err / tol).max())
    assert ((lse.double() - score).abs() <= 2.0 ** -21 * score + 1.0).all()


# ------------------------------------------------------------------ small queries

@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads,q,kv", [(16, 4, 1, 900), (8, 1, 1, 9000), (8, 2, 4, 700), (8, 2, 40, 900), (8, 1, 130, 300), (8, 1, 260, 900)])
@pytest.mark.parametrize("size", [2.0 ** -20, 2.0 ** -40, 2.0 ** -126, 2.0 ** -132, 1.0])
def test_bf16_queries_of_any_size(ctx, dim, heads, kv_heads, q, kv, size):  # noqa: F811
    """BF16 queries below F16's range with a scale that makes up for them, over 4 bits: in few rows, in chunks and with the
    pages unpacked first. Rows of one tile differ by 2^10, one is 0, and one has an element that outweighs its others by
    2^12. The tolerances are the usual ones: nothing of a query is lost."""
    c = Q4Case("bf16", [q, 1, q], [kv + q, 90, kv + 3], heads, kv_heads, dim)
    x = torch.randn(c.rows, heads, dim, generator=c.gen, device="cuda")
    x *= 2.0 ** -(torch.arange(c.rows * heads, device="cuda") % 11).float().view(c.rows, heads, 1)
    x[c.rows // 2, heads // 2] = 0.0
    x[0, heads - 1, 1:] *= 2.0 ** -12
    x = (x.bfloat16().double() * size).bfloat16()
    cut = 126 if size < 2.0 ** -126 else 0   # (the scale is at most 1e38)
    attend(ctx, c, q=x, scale=(1.0 / size if not cut else 2.0 ** cut) * dim ** -0.5)


@pytest.mark.parametrize("q", [1, 9, 60, 800])
def test_bf16_queries_of_any_size_with_a_negative_scale_and_masks(ctx, q):  # noqa: F811
    c = Q4Case("bf16", [q, 3], [q + 900, 70], 2, 1, 64)
    x = (c.rand(c.rows, 2, 64).double() * 2.0 ** -50).bfloat16()
    attend(ctx, c, q=x, scale=-0.125 * 2.0 ** 50)
    attend(ctx, c, q=x, scale=0.125 * 2.0 ** 50, window=100, prefix=[70, 3])
    attend(ctx, c, q=x, scale=0.0)
    attend(ctx, c, q=x, scale=1e-38)   # (scores far below 1: every key weighs the same)


# ------------------------------------------------------------------ many units

@pytest.mark.parametrize("ty,dim,heads,kv_heads,q,n_seq", [("bf16", 128, 8, 8, 1, 230), ("bf16", 128, 32, 8, 8, 150), ("f16", 32, 16, 16, 1, 190)])
@pytest.mark.parametrize("longest", [4096, 4097])
def test_many_units_at_the_border_of_64_pages(ctx, ty, dim, heads, kv_heads, q, n_seq, longest):  # noqa: F811
    """A block for each unit, or the pages dealt out. Twice the same."""
    lens = [q + 37 * s % 600 for s in range(n_seq - 2)] + [longest, 4000]
    c = Q4Case(ty, [q] * n_seq, lens, heads, kv_heads, dim)
    x, a, la = attend(ctx, c, max_kv=longest)
    cache, chunks = c.objects(longest)
    b, lb = torch.empty_like(a), torch.empty_like(la)
    order(ctx).op_chunk_attention(cache, chunks, c.layer, x, b, lse=lb)
    ctx.sync()
    assert torch.equal(a, b) and torch.equal(la, lb)
