"""GPU tests of the paged key/value cache: what is written, what is read back, and the attention over it, against
their definitions in 64 bits."""
import math

import pytest
import torch

from tests.paged_helpers import Cache, attend64, check_attention, encode64

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _q(z, n, h, d, dtype, seed=1, size=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((z, n, h, d), generator=g) * size).to(dtype).cuda()


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------------ writing
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("page,layout", [(16, "nhd"), (48, "hnd"), (128, "nhd")])
def test_written_rows_are_the_format_s(d, dtype, e4m3, page, layout):
    from flash_attn_v100 import paged_cache_write

    lens, new, n = [0, 5, 130, 16], [7, 1, 0, 3], 7
    c = Cache(lens, 3, d, page, dtype, e4m3, room=n, layout=layout)
    k, v = _q(4, n, 3, d, dtype, 3, 4.0), _q(4, n, 3, d, dtype, 4)
    k[0, 1, 0], v[0, 2, 1] = 0.0, 0.0
    k[0, 3, 2, ::5] = math.inf
    k[1, 0, 1, 3] = math.nan
    before = [t.clone().view(torch.uint8 if e4m3 else dtype) for t in (c.k_cache, c.v_cache)]
    paged_cache_write(k, v, *c.args(), c.seqused_k, _i32(new), **c.scales())
    for x, cache, scale, was in ((k, c.k_cache, c.k_scale, before[0]), (v, c.v_cache, c.v_scale, before[1])):
        untouched = torch.ones(cache.shape[:2], dtype=torch.bool, device="cuda")
        for z in range(4):
            where = c.where(z, range(lens[z], lens[z] + new[z]))
            untouched[where] = False
            rows = x[z, :new[z]]
            if e4m3:
                codes, e = encode64(rows)
                got = cache.view(torch.uint8)[where].view(torch.float8_e4m3fn).double()
                assert torch.equal(got.nan_to_num(777.0), codes.nan_to_num(777.0))
                assert torch.equal(scale.view(torch.uint8)[where].double() - 127, e)
            else:
                assert torch.equal(cache[where].nan_to_num(777.0), rows.nan_to_num(777.0))
        now = cache.view(torch.uint8 if e4m3 else dtype)
        assert torch.equal(now[untouched].nan_to_num(3.0), was[untouched].nan_to_num(3.0))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_rows_at_the_ends_of_the_types(dtype):
    """Largest and smallest values, rows whose largest value is 448 * 2^k and its neighbours, values half way
    between two codes."""
    from flash_attn_v100 import paged_cache_read, paged_cache_write

    d, rows = 64, []
    top = torch.finfo(dtype).max
    step = 1 + torch.finfo(dtype).eps
    for big in (top, 448.0, 448.0 * step, 448.0 / step, 3.5, 3.5 * step, torch.finfo(dtype).tiny, 0.0,
                torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps, 57344.0, 63488.0):
        x = torch.linspace(-1, 1, d) * big
        x[0] = big
        rows.append(x)
    rows.append(torch.arange(d) * 8.0)  # codes and the middles between them: 16-step from 128, 32-step from 256 on
    x = torch.stack(rows).to(dtype).reshape(1, len(rows), 1, d).cuda()
    c = Cache([0], 1, d, 16, dtype, True, room=len(rows))
    paged_cache_write(x, -x, *c.args(), _i32([0]), **c.scales())
    codes, e = encode64(x[0])
    value = codes * torch.exp2(e).unsqueeze(-1)
    k, v = paged_cache_read(*c.args(), _i32([len(rows)]), len(rows), dtype=dtype, **c.scales())
    assert torch.isfinite(k).all()
    assert torch.equal(k[0].double(), value) and torch.equal(v[0].double(), -value)
    # e4m3 has three bits behind the point: off by 2^-4 of the value, or by half of the row's least step
    least = torch.exp2(e).unsqueeze(-1) * 2.0 ** -10
    # (a value that would round beyond the type goes down: a whole step, 2^-3)
    bound = torch.maximum(x[0].double().abs() * 2.0 ** -4, least)
    bound = torch.where(x[0].double().abs() > 0.96875 * top, x[0].double().abs() * 2.0 ** -3, bound)
    assert ((k[0].double() - x[0].double()).abs() <= bound).all()


def test_tokens_without_a_place_are_dropped():
    from flash_attn_v100 import paged_cache_write

    c = Cache([30, 4, 8], 2, 64, 16, F16, False)
    table = c.table[:, :2].contiguous()
    table[1, 0], table[2, 0] = -1, c.k_cache.shape[0]
    k = _q(3, 9, 2, 64, F16)
    c.k_cache.zero_(), c.v_cache.zero_()
    paged_cache_write(k, k, c.k_cache, c.v_cache, table, _i32([30, 4, -3]))
    page, slot = c.where(0, [30, 31])
    want = torch.zeros_like(c.k_cache)
    want[page, slot] = k[0, :2]  # 32 tokens fit; entry 1's page is none; entry 2 starts before its first
    assert torch.equal(c.k_cache, want) and torch.equal(c.v_cache, want)


# ------------------------------------------------------------------------------------------ reading
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("page,layout", [(16, "nhd"), (80, "hnd"), (256, "nhd")])
def test_read_back(d, dtype, e4m3, page, layout):
    from flash_attn_v100 import paged_cache_read

    lens = [0, 1, 77, 300, 16]
    c = Cache(lens, 3, d, page, dtype, e4m3, layout=layout)
    for seqlen in (301, 75, None):
        got = paged_cache_read(*c.args(), c.seqused_k, seqlen, dtype=dtype if e4m3 else None, **c.scales())
        for t, rows in zip(got, (c.k, c.v)):
            width = c.table.shape[1] * page if seqlen is None else seqlen
            assert t.dtype == dtype and t.shape == (5, width, 3, d)
            for z, n in enumerate(lens):
                m = min(n, width)
                assert torch.equal(t[z, :m].double(), rows[z][:m])
                assert (t[z, m:] == 0).all()


def test_missing_pages_read_as_zeros_and_other_types_round():
    from flash_attn_v100 import flash_attn_paged_func, paged_cache_read

    c = Cache([64, 40], 2, 64, 16, BF16, True)
    table = c.table.clone()
    table[0, 1], table[1, 0] = -7, 1 << 20
    for dtype in (F16, BF16):
        k, v = paged_cache_read(c.k_cache, c.v_cache, table, _i32([64, 1000]), 64, dtype=dtype, **c.scales())
        for t, rows in ((k, c.k), (v, c.v)):
            assert (t[0, 16:32] == 0).all() and (t[1, :16] == 0).all()
            assert torch.equal(t[0, :16], rows[0][:16].to(dtype)) and torch.equal(t[1, 16:40], rows[1][16:].to(dtype))


# ------------------------------------------------------------------------------------------ attention
CASES = [
    # lens, n, new, heads of the cache, group, page
    ([200, 1, 128, 517], 1, None, 2, 1, 16),
    ([200, 0, 129, 1024, 640], 1, [1, 1, 0, 1, 1], 2, 4, 64),
    ([77, 1500], 1, None, 1, 8, 48),
    ([300, 40, 3], 5, [5, 2, 5], 3, 3, 32),     # (the last entry's first two tokens see nothing)
    ([700], 3, None, 2, 7, 128),
    ([2100, 64], 9, None, 1, 5, 256),
    ([900, 130, 128], 40, [40, 1, 33], 2, 2, 16),
    ([600, 257], 130, [130, 7], 2, 4, 112),
    ([1300], 300, None, 1, 6, 64),
    ([520, 1, 2000], 257, [257, 1, 1], 3, 1, 32),
    ([400], 20, None, 1, 128, 64),
]


@pytest.mark.parametrize("d,dtype,e4m3", [(128, BF16, False), (128, BF16, True), (128, F16, False), (128, F16, True),
                                          (64, F16, False), (64, BF16, True), (64, F16, True), (96, BF16, False),
                                          (96, F16, True), (96, BF16, True), (64, BF16, False), (96, F16, False)])
@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("causal", [True, False])
def test_attention_over_pages(d, dtype, e4m3, case, causal):
    from flash_attn_v100 import flash_attn_paged_func

    lens, n, new, hk, group, page = CASES[case]
    c = Cache(lens, hk, d, page, dtype, e4m3, seed=case, layout="hnd" if case % 3 == 1 else "nhd")
    q = _q(len(lens), n, hk * group, d, dtype, case, 2.0)
    got = flash_attn_paged_func(q, *c.args(), c.seqused_k, None if new is None else _i32(new), causal=causal,
                                return_lse=True, **c.scales())
    check_attention(got, q, c, d ** -0.5, causal, new)
    assert torch.equal(got[0], flash_attn_paged_func(q, *c.args(), c.seqused_k, None if new is None else _i32(new),
                                                     causal=causal, **c.scales()))
