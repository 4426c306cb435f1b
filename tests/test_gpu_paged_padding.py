"""GPU tests of padding queries over long caches, whose items have many tiles to a block: what they hold changes nothing."""
import functools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
LENS = [20000, 9000, 30000, 16384]


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@functools.lru_cache(maxsize=1)
def long_cache(d, dtype, e4m3, heads=8, page=64):
    """Pools, table and scales of four long entries of N(0, 1)."""
    from flash_attn_v100 import paged_cache_write

    pages = -(-max(LENS) // page)
    table = torch.randperm(4 * pages, generator=torch.Generator().manual_seed(3)).to(torch.int32).reshape(4, pages).cuda()
    shape = (4 * pages, page, heads, d)
    g = torch.Generator(device="cuda").manual_seed(7)
    k, v = (torch.empty(shape, dtype=torch.uint8 if e4m3 else dtype, device="cuda") for _ in range(2))
    scales = {}
    if e4m3:
        k, v = k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn)
        scales = {n: torch.empty(shape[:3], dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for n in ("k_scale", "v_scale")}
    new = [torch.randn((4, max(LENS), heads, d), generator=g, device="cuda").to(dtype) for _ in range(2)]
    paged_cache_write(*new, k, v, table, _i32([0] * 4), **scales)
    return k, v, table, scales


@pytest.mark.parametrize("d,dtype,e4m3", [(128, BF16, True), (64, F16, True), (96, BF16, False), (64, F16, False)])
@pytest.mark.parametrize("n,new", [(1, [1, 0, 1, 1]), (4, [1, 3, 0, 4]), (8, [5, 8, 1, 2]), (12, [12, 1, 7, 0]), (16, [2, 15, 16, 9]),
                                   (40, [1, 40, 0, 33])])
@pytest.mark.parametrize("causal", [True, False])
def test_padding_queries_change_nothing(n, new, d, dtype, e4m3, causal):
    """Bit for bit: not even the references of the others' exponentials.  (Renewing them costs a tile of few rows more than the
    tile itself.)"""
    from flash_attn_v100 import flash_attn_paged_func

    k, v, table, scales = long_cache(d, dtype, e4m3)
    g = torch.Generator(device="cuda").manual_seed(n)
    q = torch.randn((4, n, 32, d), generator=g, device="cuda").to(dtype)
    noise = torch.randn((4, n, 32, d), generator=g, device="cuda")
    padding = (torch.arange(n, device="cuda")[None, :] >= _i32(new)[:, None])[:, :, None, None]
    call = lambda q: flash_attn_paged_func(q, k, v, table, _i32(LENS), _i32(new), causal=causal, return_lse=True, **scales)  # noqa: E731
    want = call(torch.where(padding, torch.zeros_like(q), q))
    for junk in (2.0 ** 3, 2.0 ** 15, math.inf, math.nan):
        dirty = (noise * junk).to(dtype) if math.isfinite(junk) else torch.full_like(q, junk)
        got = call(torch.where(padding, dirty, q))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), junk
