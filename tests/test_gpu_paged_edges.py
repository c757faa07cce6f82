"""The paged-cache operators where rows, warps or batches differ from one another: against the same 64-bit definition
and with the same derived tolerances as the other tests of these operators."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_paged import PAGE, Case, attend, ctx  # noqa: E402,F401


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
