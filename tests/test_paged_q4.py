"""The 4-bit paged cache without a GPU: what the descriptions and entry points refuse, and the tests' own format helper."""
import ctypes as C

import pytest

import gsvcu

torch = pytest.importorskip("torch")

import q4_format  # noqa: E402


def test_null_arguments_are_rejected():
    lib = gsvcu.load_library()
    assert lib.gsvcu_op_kv_read(None, C.byref(gsvcu.KvReadArgs())) == -1
    assert lib.gsvcu_op_kv_append_norm(None, C.byref(gsvcu.KvAppendArgs()), C.byref(gsvcu.HeadNorm())) == -1


def test_a_pool_of_bytes_describes_a_4_bit_cache():
    for dim in (32, 64, 128):
        pool = torch.zeros(3, 2, 2, 4, 64, 9 * dim // 16, dtype=torch.uint8)
        for rows, code in ((torch.float16, 3), (torch.bfloat16, 4)):
            kv = gsvcu.PagedKV(pool, rows=rows)
            d = kv.desc
            assert (d.pool, d.kv_dtype, d.n_page, d.n_layer, d.n_kv_head, d.head_dim) == (pool.data_ptr(), code, 3, 2, 4, dim)
            assert kv.dtype == rows and kv.head_dim == dim
    for rows in (None, torch.float32, torch.uint8, "float16"):
        with pytest.raises(ValueError):
            gsvcu.PagedKV(pool, rows=rows)
    for bad in (pool[..., :70].contiguous(), pool[:, :, :1], pool[..., :36], pool.to(torch.int8)):
        with pytest.raises(ValueError):
            gsvcu.PagedKV(bad, rows=torch.float16)
    half = torch.zeros(3, 2, 2, 4, 64, 32, dtype=torch.float16)
    assert gsvcu.PagedKV(half, rows=torch.float16).desc.kv_dtype == 0
    with pytest.raises(ValueError):
        gsvcu.PagedKV(half, rows=torch.bfloat16)


def test_the_format_helper():
    """Encoded values come back within the quantiser's step; scales have 8 significant bits, so that scale * (code - 8) and
    24 * scale are F16 numbers."""
    g = torch.Generator()
    g.manual_seed(0)
    for dim in (32, 64, 128):
        x = torch.randn(2, 64, dim, generator=g) * torch.logspace(-4, 3, 64)[:, None]
        v, s, code = q4_format.decode(q4_format.encode(x))
        assert int(code.min()) == 0 and int(code.max()) == 15
        tol = torch.where(code == 15, 1.04, 0.5 + 2.0 ** -18) * s.abs() + 2.0 ** -22
        assert ((v - x.double()).abs() <= tol).all()
        assert torch.equal(v.half().double(), v) and torch.equal((24 * s).half().double(), 24 * s)
