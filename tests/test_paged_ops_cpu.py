"""CPU tests of the paged ops called directly (``torch.ops.flash_attn_v100``): what autograd would have to know is refused at the
call, as the functions refuse it, not in a backward pass later."""
import pytest
import torch


def _tensors():
    cache = torch.zeros(2, 16, 1, 64, dtype=torch.float16)
    return [torch.zeros(1, 1, 1, 64, dtype=torch.float16), cache, cache.clone(), torch.zeros(1, 2, dtype=torch.int32),
            torch.zeros(1, dtype=torch.int32)]


CALLS = {
    "paged_fwd": lambda x, k, v, t, n: torch.ops.flash_attn_v100.paged_fwd(x, k, v, t, n, None, None, None, 0.1, False),
    "paged_write": lambda x, k, v, t, n: torch.ops.flash_attn_v100.paged_write(x, x, k, v, t, n),
    "paged_read": lambda x, k, v, t, n: torch.ops.flash_attn_v100.paged_read(k, v, t, n, 16, dtype=torch.float16),
}


@pytest.mark.parametrize("op", CALLS)
@pytest.mark.parametrize("which", [0, 1, 2])
def test_gradients_are_refused_at_the_call(built_library, op, which):
    import torch.autograd.forward_ad as fw

    import flash_attn_v100  # noqa: F401  (registers the ops)

    if op == "paged_read" and which == 0:
        return
    a = _tensors()
    a[which].requires_grad_()
    with pytest.raises(RuntimeError, match="no derivative"):
        CALLS[op](*a)
    assert all(t.is_leaf and t._version == 0 for t in a)
    with torch.no_grad(), pytest.raises(NotImplementedError, match="CPU"):  # as far as the missing device
        CALLS[op](*a)
    a = _tensors()
    with fw.dual_level():
        a[which] = fw.make_dual(a[which], torch.ones_like(a[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            CALLS[op](*a)
