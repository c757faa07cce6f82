"""How a call of chunk attention over the paged cache is cut up, from its sizes alone: no GPU."""
import json
import os
import subprocess

import pytest

import gsvcu

HERE = os.path.dirname(os.path.abspath(__file__))
EXE = os.path.join(HERE, "cpp", "bin", "paged_plan")
F16, F32, BF16, Q4_F16, Q4_BF16 = range(5)


def plan(kv_dtype=Q4_BF16, head_dim=128, kv_heads=8, heads=32, n_seq=1, n_rows=1, max_chunk=None, max_kv=8192, window=0,
         scale=0.125):
    assert os.path.exists(EXE), "build with `make -C tests/cpp`"
    chunk = n_rows if max_chunk is None else max_chunk
    args = [kv_dtype, head_dim, kv_heads, heads, n_seq, -(-max_kv // 64), n_rows, chunk, max_kv, window, scale]
    out = subprocess.run([EXE] + [str(a) for a in args], capture_output=True, text=True, check=True, timeout=60)
    return json.loads(out.stdout)


@pytest.mark.parametrize("sizes,unpacked", [
    (dict(n_rows=384), True), (dict(n_rows=383), False),                       # 1536 rows times query heads of a kv head
    (dict(n_seq=8, n_rows=8 * 128, max_chunk=384), True), (dict(n_seq=8, n_rows=8 * 128 - 1, max_chunk=384), False),
    (dict(n_seq=33, n_rows=512 + 32, max_chunk=512), False),                   # one chunk beside 32 decoding slots
    (dict(n_seq=33, n_rows=4096, max_chunk=4096), True),                       # the slots are idle
    (dict(n_seq=33, n_rows=4096 + 1, max_chunk=4096), True),                   # one of them decodes
    (dict(n_seq=33, n_rows=4096 + 1, max_chunk=2048), False), (dict(n_seq=32, n_rows=4096 + 1, max_chunk=2048), True),
    (dict(n_seq=2, n_rows=4096, max_chunk=2048), True),
    (dict(n_rows=2048, window=384), True), (dict(n_rows=2048, window=383), False),
    (dict(n_seq=9, n_rows=2048 + 8, max_chunk=2048, window=400), True),
    (dict(n_seq=17, n_rows=2048 + 16, max_chunk=2048, window=400), False),
    (dict(n_rows=2048, kv_dtype=BF16), False), (dict(n_rows=2048, scale=0.0), False),
    (dict(n_rows=2048, n_seq=1, max_kv=1 << 20), False),                       # more than 2 GB
])
def test_pages_are_unpacked_for_many_rows_of_every_sequence(sizes, unpacked):
    """The pages of every sequence in the call are: that pays where the longest chunk has 1536 rows times query heads of a kv
    head and the others not too few (512 on average), not for one chunk beside many single tokens."""
    c = plan(**sizes)
    assert (c["unpack_pages"] > 0) == unpacked, c


@pytest.mark.parametrize("kv_dtype", [F16, F32, BF16, Q4_F16, Q4_BF16])
@pytest.mark.parametrize("head_dim", [32, 128])
@pytest.mark.parametrize("sizes,least", [
    (dict(kv_heads=1, heads=1, n_seq=1 << 16, n_rows=1 << 20, scale=0.0, max_kv=64), 1 << 31),      # row tiles of 32 rows
    (dict(kv_heads=1, heads=1, n_seq=1 << 16, n_rows=1 << 20, scale=0.0, max_kv=1 << 20), 1 << 31),
    (dict(kv_heads=1 << 10, heads=1 << 10, n_seq=1 << 21, n_rows=1 << 20, max_chunk=1, max_kv=64), 1 << 31),
    (dict(kv_heads=1 << 10, heads=1 << 10, n_seq=(1 << 31) - 1, n_rows=1 << 20, max_chunk=1, max_kv=1 << 20), 1 << 40),
    (dict(kv_heads=1 << 10, heads=1 << 10, n_seq=1 << 20, n_rows=1 << 20, max_chunk=1, max_kv=64), 1 << 30),   # (fits)
    (dict(kv_heads=8, heads=8, n_seq=64, n_rows=64, max_chunk=1, max_kv=2048), 512),
])
def test_the_blocks_of_a_launch_are_counted_in_64_bits(kv_dtype, head_dim, sizes, least):
    """What a call compares with the largest grid: a CTA at least for every sequence, row tile and kv head, whichever kernel."""
    assert plan(kv_dtype, head_dim, **sizes)["ctas"] >= least


@pytest.mark.parametrize("head_dim", [32, 64, 128])
@pytest.mark.parametrize("group,chunk", [(1, 1), (4, 5), (4, 8)])
def test_short_units_have_a_block_of_their_own(head_dim, group, chunk):
    """4-bit caches, few rows: up to 64 pages when there are many units, up to 40 (heads of 128 when there are few: 16) else."""
    many, some, few = ((n, dict(kv_heads=8, heads=8 * group, n_seq=n, n_rows=n * chunk, max_chunk=chunk)) for n in (1000, 75, 4))
    for (n, sizes), pages in ((many, 64), (some, 40), (few, 16 if head_dim == 128 else 40)):
        c = plan(Q4_BF16, head_dim, max_kv=64 * pages, **sizes)
        assert not c["dealt"] and c["ctas"] == n * 8 * -(-group * chunk // 32)
        assert plan(Q4_BF16, head_dim, max_kv=64 * pages + 1, **sizes)["dealt"]


def test_the_switch_for_missing_memory_takes_a_context():
    assert gsvcu.load_library().gsvcu_set_memory_fault(None, 1) == -1
