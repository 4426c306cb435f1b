"""GPU tests of the paged ops as PyTorch sees them: versions of what is written, schemas, traced calls."""
import pytest
import torch

from tests.paged_helpers import Cache

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _q(z, n, h, d, dtype, seed=1):
    return torch.randn((z, n, h, d), generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("e4m3", [False, True])
def test_every_write_counts_once(e4m3):
    """Whatever way it takes: what autograd saved of the caches before is seen to be overwritten."""
    from flash_attn_v100 import paged_cache_write

    c = Cache([20, 3], 2, 64, 16, BF16, e4m3, room=4)
    x = _q(2, 2, 2, 64, BF16)
    args = (x, x, *c.args(), c.seqused_k, None, c.k_scale, c.v_scale)
    written = [t for t in (c.k_cache, c.v_cache, c.k_scale, c.v_scale) if t is not None]

    def inference():
        with torch.inference_mode():
            torch.ops.flash_attn_v100.paged_write(*args)

    ways = [lambda: paged_cache_write(*args), lambda: torch.ops.flash_attn_v100.paged_write(*args), inference,
            lambda: torch.compile(paged_cache_write, backend="eager")(*args)]
    for i, way in enumerate(ways):
        before = [t._version for t in written]
        way()
        assert [t._version for t in written] == [n + 1 for n in before], i


def test_a_saved_cache_is_seen_to_be_overwritten():
    c = Cache([20], 2, 64, 16, BF16, False, room=4)
    x = _q(1, 2, 2, 64, BF16)
    w = torch.ones((), device="cuda", requires_grad=True)
    loss = (w * c.k_cache).sum()
    torch.ops.flash_attn_v100.paged_write(x, x, *c.args(), c.seqused_k)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("e4m3", [False, True])
def test_schemas_and_fake_tensors(e4m3):
    import flash_attn_v100  # noqa: F401

    c = Cache([40, 9], 2, 64, 16, BF16, e4m3, room=4)
    for t in (c.k_cache, c.v_cache):  # (junk NaN would not compare equal to itself)
        t.view(torch.uint8 if e4m3 else BF16).zero_()
    for t in (c.k_scale, c.v_scale):
        if t is not None:
            t.view(torch.uint8).fill_(127)
    x, q = _q(2, 2, 2, 64, BF16), _q(2, 2, 4, 64, BF16, 2)
    ops = torch.ops.flash_attn_v100
    calls = [(ops.paged_fwd.default, (q, *c.args(), c.seqused_k, None, c.k_scale, c.v_scale, 0.125, True), {}),
             (ops.paged_read.default, (*c.args(), c.seqused_k, 41, c.k_scale, c.v_scale), {"dtype": BF16})]
    calls.append((ops.paged_write.default, (x, x, *c.args(), c.seqused_k, None, c.k_scale, c.v_scale), {}))
    utils = ("test_faketensor", "test_autograd_registration") + (() if e4m3 else ("test_schema",))  # (which multiplies 8-bit types)
    for op, args, kwargs in calls:
        torch.library.opcheck(op, args, kwargs, test_utils=utils)


def test_traced_below_autograd():
    """A step through AOT tracing (functionalised, in-place writes among it) is the eager step."""
    from flash_attn_v100 import flash_attn_paged_func, paged_cache_write

    def step(q, k, v, k_cache, v_cache, table, lengths):
        paged_cache_write(k, v, k_cache, v_cache, table, lengths)
        return flash_attn_paged_func(q, k_cache, v_cache, table, lengths + 1, causal=True)

    outs = []
    for run in (step, torch.compile(step, fullgraph=True, backend="aot_eager")):
        c = Cache([40, 9], 2, 64, 16, BF16, False, room=4)
        with torch.no_grad():
            outs.append((run(_q(2, 1, 4, 64, BF16), _q(2, 1, 2, 64, BF16, 2), _q(2, 1, 2, 64, BF16, 3), *c.args(), c.seqused_k),
                         c.k_cache.nan_to_num(7.0)))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
