"""CPU tests of the paged cache's boundary: bad parameters are status codes or exceptions before a device is touched."""
import ctypes

import pytest
import torch


def _cache(cabi, **kw):
    c = cabi.FmhaPagedCache()
    c.k, c.v, c.block_table, c.k_scale, c.v_scale = 0x1000, 0x2000, 0x3000, 0x4001, 0x5003  # never dereferenced
    c.num_pages, c.page_size, c.max_pages, c.block_table_stride = 10, 32, 4, 4
    for s in (c.k_strides, c.v_strides):
        s.batch, s.row, s.head = 32 * 2 * 128, 2 * 128, 128
    for s in (c.k_scale_strides, c.v_scale_strides):
        s.batch, s.row, s.head = 32 * 2, 2, 1
    for k, v in kw.items():
        setattr(c, k, v)
    return c


BAD_CACHE = [
    (dict(k=None), 1), (dict(v=None), 1), (dict(block_table=None), 1), (dict(format=1, k_scale=None), 1),
    (dict(format=1, v_scale=None), 1), (dict(format=2), 11), (dict(num_pages=0), 3), (dict(page_size=0), 3),
    (dict(page_size=24), 3), (dict(page_size=-16), 3), (dict(max_pages=0), 3), (dict(k=0x1008), 5),
    (dict(max_pages=1 << 26), 10), (dict(block_table_stride=-1), 4),
]


def _calls(cabi, cache):
    """The three entry points with good parameters but for the cache."""
    lib = cabi.load_library()
    w = cabi.FmhaCacheWriteParams()
    w.cache, w.k, w.v, w.seqlens = cache, 0x6000, 0x7000, 0x8000
    r = cabi.FmhaCacheReadParams()
    r.cache, r.k, r.v, r.seqused_k = cache, 0x6000, 0x7000, 0x8000
    a = cabi.FmhaPagedFwdParams()
    a.cache, a.q, a.o, a.lse, a.seqused_k, a.scale = cache, 0x6000, 0x7000, 0x9000, 0x8000, 0.1
    for p in (w, r):
        p.batch, p.heads, p.seqlen, p.head_dim = 2, 2, 5, 128
        for s in (p.k_strides, p.v_strides):
            s.batch, s.row, s.head = 5 * 2 * 128, 2 * 128, 128
    a.batch, a.heads_q, a.heads_k, a.seqlen_q, a.head_dim = 2, 4, 2, 5, 128
    for s in (a.q_strides, a.o_strides):
        s.batch, s.row, s.head = 5 * 4 * 128, 4 * 128, 128
    return (w, lambda: lib.fmha_cache_write(ctypes.byref(w), None)), (r, lambda: lib.fmha_cache_read(ctypes.byref(r), None)), \
        (a, lambda: lib.fmha_paged_fwd(ctypes.byref(a), None, 0, None))


@pytest.mark.parametrize("change,status", BAD_CACHE)
def test_a_bad_cache_is_a_status(built_library, change, status):
    from flash_attn_v100 import cabi

    for _, call in _calls(cabi, _cache(cabi, **change)):
        assert call() == status


@pytest.mark.parametrize("pool", ["k_strides", "v_strides"])
@pytest.mark.parametrize("field", ["batch", "row", "head"])
def test_strides_of_pools(built_library, pool, field):
    """Rows are read 16 bytes at a time: 8 elements of 16 bits, 16 of 8."""
    from flash_attn_v100 import cabi

    for fmt, value in ((0, 132), (1, 136), (0, 0), (1, -128)):
        c = _cache(cabi, format=fmt)
        setattr(getattr(c, pool), field, value)
        for _, call in _calls(cabi, c):
            assert call() == 4, (fmt, value)


@pytest.mark.parametrize("change,status", [
    (dict(dtype=2), 11), (dict(head_dim=80), 2), (dict(head_dim=256), 2), (dict(batch=-1), 3), (dict(seqlen=-1), 3),
    (dict(heads=0), 3), (dict(k=None), 1), (dict(v=None), 1), (dict(k=0x6002), 5), (dict(batch=1 << 20, seqlen=1 << 20), 10)])
def test_write_and_read_reject(built_library, change, status):
    from flash_attn_v100 import cabi

    for p, call in _calls(cabi, _cache(cabi))[:2]:
        for k, v in change.items():
            setattr(p, k, v)
        assert call() == status


@pytest.mark.parametrize("change,status", [
    (dict(dtype=-1), 11), (dict(head_dim=32), 2), (dict(heads_q=5), 3), (dict(heads_q=0), 3), (dict(heads_k=0), 3),
    (dict(heads_q=258), 3), (dict(seqlen_q=-1), 3), (dict(scale=0.0), 3), (dict(scale=float("inf")), 3), (dict(q=None), 1),
    (dict(o=None), 1), (dict(lse=None), 1), (dict(seqused_k=None), 1), (dict(q=0x6004), 5), (dict(seqlen_q=0x7fffffff), 10)])
def test_attention_rejects(built_library, change, status):
    from flash_attn_v100 import cabi

    p, call = _calls(cabi, _cache(cabi))[2]
    for k, v in change.items():
        setattr(p, k, v)
    assert call() == status


def test_nothing_to_do_is_no_error(built_library):
    from flash_attn_v100 import cabi

    for p, call in _calls(cabi, _cache(cabi)):
        p.batch = 0
        assert call() == 0
    assert cabi.load_library().fmha_cache_write(None, None) == 1
    assert cabi.load_library().fmha_cache_read(None, None) == 1
    assert cabi.load_library().fmha_paged_fwd(None, None, 0, None) == 1


def test_cpu_tensors_are_refused(built_library):
    from flash_attn_v100 import flash_attn_paged_func, paged_cache_read, paged_cache_write

    cache = torch.zeros(2, 16, 1, 64, dtype=torch.float16)
    x, table, lens = torch.zeros(1, 1, 1, 64, dtype=torch.float16), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        flash_attn_paged_func(x, cache, cache, table, lens)
    with pytest.raises(RuntimeError):
        paged_cache_write(x, x, cache, cache, table, lens)
    with pytest.raises(RuntimeError):
        paged_cache_read(cache, cache, table, lens)


def test_derivatives_are_refused(built_library):
    """The cache has none: an output without a gradient would say that it is zero."""
    import torch.autograd.forward_ad as fw

    from flash_attn_v100 import flash_attn_paged_func, paged_cache_read, paged_cache_write

    def tensors():
        cache = torch.zeros(2, 16, 1, 64, dtype=torch.float16)
        return [torch.zeros(1, 1, 1, 64, dtype=torch.float16), cache, cache.clone(), torch.zeros(1, 2, dtype=torch.int32),
                torch.zeros(1, dtype=torch.int32)]

    calls = (lambda x, k, v, t, n: flash_attn_paged_func(x, k, v, t, n), lambda x, k, v, t, n: paged_cache_write(x, x, k, v, t, n),
             lambda x, k, v, t, n: paged_cache_read(k, v, t, n))
    for call in calls:
        for which in (0, 1, 2):
            if call is calls[2] and which == 0:
                continue
            a = tensors()
            a[which].requires_grad_()
            with pytest.raises(RuntimeError, match="no derivative"):
                call(*a)
            a = tensors()
            with fw.dual_level():
                a[which] = fw.make_dual(a[which], torch.ones_like(a[which]))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(*a)
        with pytest.raises(RuntimeError, match="functorch"):
            a = tensors()
            torch.vmap(lambda k: call(a[0], k, a[2], a[3], a[4]))(torch.stack([a[1], a[1]]))
