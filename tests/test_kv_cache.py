"""The paged cache's and the router's host side: sizes, refusals and the Python layer's checks (no GPU)."""

import ctypes
import os

import pytest

from conftest import load_package


@pytest.fixture(scope="module")
def pkg():
    m = load_package()
    if not os.path.exists(m.LIB_PATH):
        m.build()
    return m


def up(n):
    return -(-n // 256) * 256


@pytest.mark.parametrize("heads,dim,page,pages", [(8, 128, 16, 5), (1, 64, 48, 3), (3, 96, 4096, 1), (4, 256, 32, 70000)])
def test_cache_bytes(pkg, heads, dim, page, pages):
    L = pkg.lib()
    rows = heads * page * pages
    assert L.b200_kv_cache_nbytes(pkg.F16, heads, dim, page, pages) == 2 * up(rows * dim * 2)
    assert L.b200_kv_cache_nbytes(pkg.Q8_0, heads, dim, page, pages) == 2 * up(rows * dim) + 2 * up(rows * dim // 32 * 2)


@pytest.mark.parametrize("qtype,heads,dim,page,pages", [
    (0, 8, 128, 16, 5), (12, 8, 128, 16, 5), (1, 0, 128, 16, 5), (1, 8, 80, 16, 5), (1, 8, 0, 16, 5), (1, 8, 512, 16, 5), (1, 8, 128, 0, 5),
    (1, 8, 128, 8, 5), (1, 8, 128, 24, 5), (1, 8, 128, 8192, 5), (1, 8, 128, 16, 0), (8, 8, 128, 16, -1), (8, 65536, 256, 4096, 1 << 31),
    (8, 65535, 256, 4096, (1 << 31) - 1),
])
def test_caches_that_are_not_supported_have_no_bytes(pkg, qtype, heads, dim, page, pages):
    assert pkg.lib().b200_kv_cache_nbytes(qtype, heads, dim, page, pages) == 0


def test_null_arguments_are_refused(pkg):
    L = pkg.lib()
    c = pkg.KvCacheStruct()
    r = ctypes.byref(c)
    assert L.b200_kv_cache_alloc(None, pkg.F16, 8, 128, 16, 1, r) == pkg.ERR_INVALID
    assert L.b200_kv_cache_alloc(None, pkg.F16, 8, 128, 16, 1, None) == pkg.ERR_INVALID
    assert L.b200_kv_cache_view(None, pkg.F16, 8, 128, 16, 1, None, 0, r) == pkg.ERR_INVALID
    assert L.b200_kv_cache_free(None, r) == pkg.ERR_INVALID
    assert L.b200_kv_write(None, None, r, None, 0, None, 1, 1, None, 0, None, 0) == pkg.ERR_INVALID
    assert L.b200_kv_read(None, None, r, None, 0, None, None, 1, 1, 0, None, None) == pkg.ERR_INVALID
    assert L.b200_kv_attention(None, None, r, None, 0, None, 1, 1, 8, None, 0, 1.0, None, None, 0) == pkg.ERR_INVALID
    assert L.b200_kv_attention_workspace(None, None, 0, 0, 0, 0) == 0
    assert L.b200_moe_router(None, None, ctypes.byref(pkg.Router()), None, None, 1, None, None) == pkg.ERR_INVALID
    assert b"moe_router" in L.b200_last_error(None)


def bare(pkg):
    """A context whose checks of tensors can be called without a device."""
    ctx = pkg.Context.__new__(pkg.Context)
    ctx.device = 0
    return ctx


def test_the_python_layer_refuses_what_it_cannot_pass_on(pkg):
    import torch

    ctx = bare(pkg)
    cache = pkg.KvCache.__new__(pkg.KvCache)
    cache.ctx, cache.open, cache.n_kv_head, cache.head_dim, cache.data = ctx, True, 2, 64, None
    x = torch.zeros(1, 1, 2, 64)
    table, lens = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="cuda:0"):  # host tensors
        ctx.kv_write(cache, x, x, table, lens)
    with pytest.raises(ValueError, match="cuda:0"):
        ctx.kv_attention(cache, x, table, lens, 1.0)
    with pytest.raises(ValueError, match="n_seq, n_tok"):
        ctx.kv_attention(cache, x[0], table, lens, 1.0)
    with pytest.raises(ValueError, match="both k and v"):
        ctx.kv_read(cache, table, lens, k=x)
    with pytest.raises(ValueError, match="n_tok"):
        ctx.kv_read(cache, table, lens)
    with pytest.raises(ValueError, match="float32 or float16"):
        ctx.kv_read(cache, table, lens, k=x.double(), v=x.double())
    with pytest.raises(ValueError, match="unknown score"):
        ctx.moe_router(torch.zeros(1, 8), 2, score="relu")
    with pytest.raises(ValueError, match="T, n_expert"):
        ctx.moe_router(torch.zeros(8), 2)
    with pytest.raises(ValueError, match="cuda:0"):
        ctx.moe_router(torch.zeros(1, 8), 2)
