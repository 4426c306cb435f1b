"""GPU test of calls in a row whose every tile comes from HBM: the copies land late and in any order, and every call's answer
is the first one's, bit for bit."""
import pytest
import torch

from tests.test_gpu_paged_padding import LENS, _i32, long_cache

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("d,dtype,e4m3", [(128, BF16, False), (96, BF16, False), (64, F16, False), (128, BF16, True)])
@pytest.mark.parametrize("n", [1, 8, 12, 16, 40])
def test_calls_in_a_row_are_alike(n, d, dtype, e4m3):
    from flash_attn_v100 import flash_attn_paged_func

    k, v, table, scales = long_cache(d, dtype, e4m3)
    g = torch.Generator(device="cuda").manual_seed(n)
    q, lens = torch.randn((4, n, 32, d), generator=g, device="cuda").to(dtype), _i32(LENS)
    call = lambda: flash_attn_paged_func(q, k, v, table, lens, causal=True, return_lse=True, **scales)  # noqa: E731
    o, lse = call()
    assert torch.isfinite(o).all() and torch.isfinite(lse).all()
    for _ in range(6):
        got = [call() for _ in range(25)]
        assert all(torch.equal(a, o) and torch.equal(b, lse) for a, b in got)
