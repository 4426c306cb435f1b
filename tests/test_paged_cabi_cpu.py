"""CPU tests of ``cabi.paged_cache`` and ``cabi.paged_fwd``: tensors that do not belong together are refused before their pointers
go anywhere (8-bit pools without scales would be read as 16-bit ones, beyond their ends)."""
import pytest
import torch

F16, E4M3, E8M0 = torch.float16, torch.float8_e4m3fn, torch.float8_e8m0fnu


def _bytes(shape, dtype):
    return torch.zeros(shape, dtype=torch.uint8).view(dtype)


def _pools(e4m3=False):
    shape = (4, 16, 2, 64)
    k, v = (_bytes(shape, E4M3) if e4m3 else torch.zeros(shape, dtype=F16) for _ in range(2))
    scale = _bytes(shape[:3], E8M0) if e4m3 else None
    return dict(k_cache=k, v_cache=v, block_table=torch.zeros((3, 2), dtype=torch.int32), k_scale=scale, v_scale=scale)


@pytest.mark.parametrize("e4m3,change,match", [
    (True, dict(k_scale=None, v_scale=None), "belong to"), (True, dict(k_scale=None), "belong to"), (True, dict(v_scale=None), "belong to"),
    (False, dict(k_scale=_bytes((4, 16, 2), E8M0), v_scale=_bytes((4, 16, 2), E8M0)), "belong to"),
    (True, dict(k_scale=_bytes((4, 16, 1), E8M0)), "k_scale and v_scale must"), (True, dict(v_scale=torch.zeros((4, 16, 2))), "k_scale and v_scale must"),
    (False, dict(v_cache=torch.zeros((3, 16, 2, 64), dtype=F16)), "k_cache and v_cache"), (False, dict(v_cache=torch.zeros((4, 16, 2, 64), dtype=torch.bfloat16)), "k_cache and v_cache"),
    (False, dict(k_cache=torch.zeros((4, 16, 2, 64)), v_cache=torch.zeros((4, 16, 2, 64))), "k_cache and v_cache"),
    (False, dict(k_cache=torch.zeros((4, 16, 64, 2), dtype=F16).transpose(2, 3)), "k_cache and v_cache"), (True, dict(v_cache=torch.zeros((4, 16, 2, 64), dtype=F16)), "k_cache and v_cache"),
    (False, dict(block_table=torch.zeros((3, 2), dtype=torch.int64)), "block_table"), (False, dict(block_table=torch.zeros(6, dtype=torch.int32)), "block_table"),
    (False, dict(block_table=torch.zeros((2, 3), dtype=torch.int32).t()), "block_table"), (False, {}, "CUDA device"), (True, {}, "CUDA device")])
def test_tensors_that_do_not_belong_together(e4m3, change, match):
    from flash_attn_v100 import cabi

    with pytest.raises(RuntimeError, match=match):
        cabi.paged_cache(**dict(_pools(e4m3), **change))


@pytest.mark.parametrize("shape,dtype,heads,ok", [((3, 1, 4, 64), F16, 2, True), ((2, 1, 4, 64), F16, 2, False), ((3, 1, 4, 128), F16, 2, False),
                                                  ((3, 1, 4, 64), F16, 4, False), ((3, 1, 4, 64), torch.bfloat16, 2, False)])
@pytest.mark.parametrize("e4m3", [False, True])
def test_a_cache_of_other_tensors(shape, dtype, heads, ok, e4m3):
    from flash_attn_v100 import cabi

    c, x = cabi.FmhaPagedCache(), torch.zeros(shape, dtype=dtype)
    cabi._require_fit(c, 7, 7, x)  # a struct that was filled by hand says nothing of its tensors
    c.tensors = tuple(_pools(e4m3).values())
    if ok or (e4m3 and dtype == torch.bfloat16):  # (8 bits are read as either type)
        return cabi._require_fit(c, shape[0], heads, x)
    with pytest.raises(RuntimeError, match="the cache must have"):
        cabi._require_fit(c, shape[0], heads, x)
