"""GPU tests of what the paged attention's values do to one another: scales of V that fp16 cannot take, group of keys by group
of keys, and what a NaN reaches."""
import math

import pytest
import torch

from tests.paged_helpers import Cache, check_attention
from tests.test_gpu_paged_use import Held

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _q(z, n, h, d, dtype, seed=1, size=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((z, n, h, d), generator=g) * size).to(dtype).cuda()


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("n", [4, 8, 12, 16])
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("where", ["first", "second", "one row", "all"])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_values_whose_scale_fp16_does_not_hold(n, d, where, dtype):
    """Items of 16, 32, 48 and 64 rows over an 8-bit cache: rows of V beyond what a scale in fp16 can be, in the first or the
    second 16 keys of 32, in a single key, or everywhere."""
    from flash_attn_v100 import flash_attn_paged_func, paged_cache_read, paged_cache_write

    length, lens = 700, [700, 333]
    low, high = (-40, 17) if dtype == BF16 else (-22, 6)
    c = Cache([0, 0], 2, d, 32, dtype, True, room=length)
    k, v = _q(2, length, 2, d, BF16, 5).float(), _q(2, length, 2, d, BF16, 6).float()
    t = torch.arange(length, device="cuda")
    odd = {"first": t % 32 < 16, "second": t % 32 >= 16, "one row": t == 277, "all": t >= 0}[where]
    size = torch.where(t % 3 == 0, 2.0 ** low, 2.0 ** high)
    v = torch.where(odd[None, :, None, None], v * size[None, :, None, None], v)
    v = v.clamp(-6e4, 6e4) if dtype == F16 else v
    paged_cache_write(k.to(dtype), v.to(dtype), *c.args(), _i32([0, 0]), **c.scales())
    held = Held(*paged_cache_read(*c.args(), _i32(lens), length, dtype=dtype, **c.scales()), lens, True)
    q = _q(2, n, 8, d, dtype, n)
    got = flash_attn_paged_func(q, *c.args(), _i32(lens), causal=True, return_lse=True, **c.scales())
    check_attention(got, q, held, d ** -0.5, True)


@pytest.mark.parametrize("n", [1, 6, 12, 16, 80])
@pytest.mark.parametrize("dtype,e4m3", [(BF16, False), (BF16, True), (F16, False), (F16, True)])
def test_a_nan_reaches_who_sees_it(n, dtype, e4m3):
    """A NaN in a key: rows that see it are NaN, all others what they are without it, tokens before it among them (to the
    rounding: with many rows, neighbours of a row that needs a new reference take the same way as it).  One in a
    value: its element, of its entry and the heads that read its head, where that sees it and maybe before (0 times it is
    NaN); nothing else."""
    from flash_attn_v100 import flash_attn_paged_func

    c = Cache([300, 200], 2, 128, 32, dtype, e4m3, seed=3)
    q = _q(2, n, 8, 128, dtype)
    call = lambda: flash_attn_paged_func(q, *c.args(), c.seqused_k, causal=True, return_lse=True, **c.scales())  # noqa: E731
    o0, l0 = call()
    assert torch.isfinite(o0).all() and torch.isfinite(l0).all()
    page, slot = c.where(0, [297])  # seen by the last 3 new tokens
    k, v = (x.view(torch.uint8) if e4m3 else x for x in (c.k_cache, c.v_cache))
    nan, first = 0x7F if e4m3 else math.nan, max(0, n - 3)
    was = k[page, slot, 1, 5].clone()
    k[page, slot, 1, 5] = nan
    o, lse = call()
    assert torch.isnan(o[0, first:, 4:]).all() and torch.isnan(lse[0, 4:, first:]).all()
    o[0, first:, 4:], lse[0, 4:, first:] = o0[0, first:, 4:], l0[0, 4:, first:]
    check_attention((o, lse), q, c, 128 ** -0.5, True)
    assert torch.equal(o[1], o0[1]) and torch.equal(o[0, :, :4], o0[0, :, :4])
    k[page, slot, 1, 5] = was
    v[page, slot, 0, 7] = nan
    o, lse = call()
    assert torch.equal(lse, l0) and torch.isnan(o[0, first:, :4, 7]).all()
    o[0, :, :4, 7] = o0[0, :, :4, 7]
    assert torch.equal(o, o0)


@pytest.mark.parametrize("dtype,e4m3", [(BF16, False), (BF16, True), (F16, True)])
def test_entries_that_share_pages(dtype, e4m3):
    """Three entries with the same first pages, one of which has a page twice, and a token that two of them write to one place."""
    from flash_attn_v100 import flash_attn_paged_func, paged_cache_read, paged_cache_write

    d, page = 128, 32
    one = Cache([200], 2, d, page, dtype, e4m3, room=page, seed=9)
    pages = one.host_table[0, :7].tolist()
    spare = next(p for p in range(one.k_cache.shape[0]) if p not in pages)
    table = _i32([pages, pages, pages[:4] + [pages[1], spare, spare]])  # (the third has 150 tokens: four pages and 22 of page 1)
    new = _q(1, 1, 2, d, dtype, 3)
    k = torch.cat([new, new, _q(1, 1, 2, d, dtype, 4)])
    paged_cache_write(k, -k, one.k_cache, one.v_cache, table, _i32([200, 200, 160]), None, one.k_scale, one.v_scale)
    lens = [201, 201, 150]
    kr, vr = paged_cache_read(one.k_cache, one.v_cache, table, _i32(lens), 201, dtype=dtype, **one.scales())
    assert torch.equal(kr[0], kr[1]) and torch.equal(vr[0, 200], -kr[0, 200])
    assert torch.equal(kr[2, 128:150], kr[0, page:page + 22])
    if not e4m3:
        assert torch.equal(kr[0, 200], new[0, 0])
    held = Held(kr, vr, lens, e4m3)
    for n in (1, 7, 40):
        q = _q(3, n, 8, d, dtype, n)
        got = flash_attn_paged_func(q, one.k_cache, one.v_cache, table, _i32(lens), causal=True, return_lse=True, **one.scales())
        check_attention(got, q, held, d ** -0.5, True)
        assert n != 1 or not torch.equal(got[0][0], got[0][2])
