"""GPU tests of the paged attention's numbers: weights that are small but many, scores and factors at the ends of fp32."""
import pytest
import torch

from tests.paged_helpers import UNIT, Cache, attend64, check_attention
from tests.test_gpu_paged_use import Held

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _q(z, n, h, d, dtype, seed=1, size=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((z, n, h, d), generator=g) * size).to(dtype).cuda()


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _attend(q, c, lens, new=None, causal=True, **kw):
    from flash_attn_v100 import flash_attn_paged_func

    return flash_attn_paged_func(q, *c.args(), lens, None if new is None else _i32(new), causal=causal, return_lse=True,
                                 **c.scales(), **kw)


@pytest.mark.parametrize("n", [1, 16, 17, 33, 49, 64])
@pytest.mark.parametrize("dtype,e4m3", [(BF16, True), (F16, True), (F16, False), (BF16, False)])
def test_small_shares_add_up(n, dtype, e4m3):
    """A first key that has all the weight but 2^-26 for each of 8191 others, and a value of zero: the output is what the
    others leave, 1.2e-4.  P of up to 64 rows is 2^5 times the exponential over the reference, so an fp16 P, whose least step
    is 2^-24, is off by 2^-30 of the first key's at most, an output by 2^-30 of the sum of |v| over the keys seen."""
    from flash_attn_v100 import paged_cache_read, paged_cache_write

    z, h, d, length = 10, 16, 64, 8192  # (more items than SMs: few of them are cut)
    c = Cache([0] * z, h, d, 64, dtype, e4m3, room=length)
    k, v = (torch.zeros((z, length, h, d), dtype=dtype, device="cuda") for _ in range(2))
    k[:, 0, :, 0] = 72.0
    v[:, 1:] = 1.0 + torch.arange(8, device="cuda", dtype=dtype).repeat(8) / 8
    paged_cache_write(k, v, *c.args(), _i32([0] * z), **c.scales())
    lens = [length] * z
    held = Held(*paged_cache_read(*c.args(), _i32(lens), length, dtype=dtype, **c.scales()), lens, e4m3)
    q = torch.zeros((z, n, h, d), dtype=dtype, device="cuda")
    q[..., 0] = 2.0
    o, lse = _attend(q, c, _i32(lens), causal=False)
    r_o, r_lse, a, b, size = attend64(q[:2], held, 0.125, False)
    e = 2.0 ** -23 * ((d + 4) * float(size.max()) + 8)
    u = UNIT[dtype]
    limit = u * (1 + u) * (a + r_o.abs()) + 4 * e * a + 2.0 ** -24
    if dtype == F16 or e4m3:
        limit = limit + 2.0 ** -30 * b
    assert ((o[:2].double() - r_o).abs() <= limit).all()
    assert ((lse[:2].double() - r_lse).abs() <= e + 2.0 ** -22 * r_lse.abs()).all()


@pytest.mark.parametrize("n", [1, 5, 8, 12, 16, 40])
@pytest.mark.parametrize("d,dtype,e4m3,up", [(128, BF16, False, 60), (64, BF16, False, 30), (96, BF16, True, 60), (128, BF16, True, 27),
                                             (64, F16, False, 27), (128, F16, True, 27), (128, BF16, False, 22), (64, BF16, True, 22)])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_whose_rounding_is_larger_than_an_exponent(n, d, dtype, e4m3, up, sign):
    """Finite scores of 2^up and more, over several tiles to a block: every row is its largest key's value, wherever the
    second largest score is further below than the rounding of both."""
    c = Cache([2500, 700, 5000], 8, d, 64, dtype, e4m3, seed=n)
    q, scale = _q(3, n, 32, d, dtype, n), sign * 2.0 ** up
    got = _attend(q, c, c.seqused_k, softmax_scale=scale)
    check_attention(got, q, c, scale, True)
    clear = 0
    for z in range(3):
        k, v = (x[z].repeat_interleave(4, 1).permute(1, 0, 2) for x in (c.k, c.v))
        s = scale * q[z].double().permute(1, 0, 2) @ k.transpose(1, 2)
        i, j = torch.arange(n, device="cuda")[:, None], torch.arange(c.lens[z], device="cuda")[None, :]
        s = torch.where(j <= c.lens[z] - n + i, s, -torch.inf)
        top, where = s.topk(2, -1)
        size = abs(scale) * q[z].double().permute(1, 0, 2).abs() @ k.abs().transpose(1, 2)
        # each score is off by e; one that is 40 below the largest has a weight of 2^-57
        e = 2.0 ** -23 * ((d + 4) * size.amax(-1) + 8)
        alone = top[..., 0] - top[..., 1] > 2 * e + 40
        want = torch.gather(v, 1, where[..., :1].expand(-1, -1, d))
        off = (got[0][z].double().permute(1, 0, 2) - want).abs()
        assert (off <= UNIT[dtype] * 1.01 * want.abs() + 2.0 ** -24)[alone].all()
        clear += int(alone.sum())
    assert clear > 3 * n * 32 // 2


@pytest.mark.parametrize("n", [1, 6, 9, 16, 40])
@pytest.mark.parametrize("up", [-122, -60, 60, 110])
def test_tiny_queries_of_huge_keys(n, up):
    """Queries of 2^up and keys of 2^-up (8 bits): ordinary scores, whose two factors are beyond, or below, normal numbers."""
    from flash_attn_v100 import paged_cache_read, paged_cache_write

    d, lens = 64, [300, 140]
    c = Cache([0, 0], 2, d, 32, BF16, True, room=300)
    k, v = (_q(2, 300, 2, d, BF16, i, 1.0) for i in (2, 3))
    k = torch.ldexp(k.double(), torch.tensor(-up, device="cuda")).to(BF16)
    paged_cache_write(k, v, *c.args(), _i32([0, 0]), **c.scales())
    held = Held(*paged_cache_read(*c.args(), _i32(lens), 300, dtype=BF16, **c.scales()), lens, True)
    q = torch.ldexp(_q(2, n, 8, d, BF16, 4).double(), torch.tensor(up, device="cuda")).to(BF16)
    check_attention(_attend(q, c, _i32(lens)), q, held, d ** -0.5, True)


@pytest.mark.parametrize("n", [1, 2, 5, 8, 11, 16, 40])
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("up", [12, 30, 60, 100])
def test_queries_of_very_unequal_size(n, d, e4m3, up):
    """Heads and tokens of one item: ordinary ones, zeros, 2^up and 2^-up times the ordinary (bf16), over several tiles to a
    block.  None of them is less exact for its neighbours."""
    c = Cache([2500, 700, 5000], 8, d, 32, BF16, e4m3, seed=n)
    q = _q(3, n, 32, d, BF16, n)
    size = torch.ones((3, n, 32, 1), device="cuda")
    size[:, :, 1::4] = 2.0 ** up
    size[1, :, 2::4] = 2.0 ** -up
    size[2, n // 2:, 3::4] = 0.0
    q = (q.float() * size).to(BF16)
    check_attention(_attend(q, c, c.seqused_k), q, c, d ** -0.5, True)
