"""GPU tests of the paged attention's rows as neighbours: what one row of queries holds (padding, a huge or a tiny query) is
nothing to the others, and small shares of a row's weight are not lost."""
import math

import pytest
import torch

from tests.paged_helpers import UNIT, Cache, attend64, check_attention

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


# new tokens and how many of them are real: items of 16, 32, 48, 64 and 256 rows with four query heads per cache head
RAGGED = [(4, [1, 3, 0, 4]), (8, [5, 8, 1, 2]), (12, [12, 1, 7, 0]), (16, [2, 15, 16, 9]), (40, [1, 40, 0, 33])]


def _padded(n, new, dtype, d, junk):
    """Queries with zeros, and with junk, in their padding."""
    clean = _q(len(new), n, 8, d, dtype, n)
    padding = torch.arange(n, device="cuda")[None, :, None, None] >= _i32(new)[:, None, None, None]
    noise = _q(len(new), n, 8, d, dtype, n + 1)
    other = torch.full_like(clean, junk) if not math.isfinite(junk) else (noise.sign() * junk).to(dtype)
    return torch.where(padding, torch.zeros_like(clean), clean), torch.where(padding, other, clean)


@pytest.mark.parametrize("n,new", RAGGED)
@pytest.mark.parametrize("d,dtype,e4m3", [(128, BF16, True), (64, BF16, True), (96, BF16, True), (128, F16, True), (128, BF16, False)])
@pytest.mark.parametrize("junk", [2.0 ** 15, 2.0 ** 60, math.inf, math.nan])
def test_padding_queries_may_hold_anything(n, new, d, dtype, e4m3, junk):
    c = Cache([900, 130, 300, 2000], 2, d, 64, dtype, e4m3, seed=n)
    q, dirty = _padded(n, new, dtype, d, junk)
    check_attention(_attend(dirty, c, c.seqused_k, new), q, c, d ** -0.5, True, new)
