"""CPU tests of the paged attention's size query: what the call itself refuses has a workspace of no size, and neither
ends the process."""
import ctypes

import pytest

GOOD = dict(batch=2, heads_q=4, heads_k=2, seqlen_q=5, head_dim=128)
BAD = [dict(dtype=-1), dict(dtype=2), dict(head_dim=32), dict(head_dim=0), dict(heads_q=5), dict(heads_q=0), dict(heads_q=1),
       dict(heads_q=-4), dict(heads_k=0), dict(heads_k=-2), dict(heads_q=258), dict(heads_q=1 << 30, heads_k=1),
       dict(seqlen_q=-1), dict(batch=-1), dict(seqlen_q=0x7fffffff), dict(heads_q=2, seqlen_q=0x7fffffff),
       dict(heads_q=1, heads_k=1, batch=0x7fffffff, seqlen_q=0x7fffffff), dict(batch=0x7fffffff, seqlen_q=200),
       dict(batch=1 << 20, heads_q=128, heads_k=1, seqlen_q=1 << 10)]


def _params(cabi, **kw):
    p = cabi.FmhaPagedFwdParams()
    c = p.cache
    c.k, c.v, c.block_table = 0x1000, 0x2000, 0x3000  # never dereferenced
    c.num_pages, c.page_size, c.max_pages, c.block_table_stride = 10, 32, 4, 4
    for s in (c.k_strides, c.v_strides):
        s.batch, s.row, s.head = 32 * 2 * 128, 2 * 128, 128
    p.q, p.o, p.lse, p.seqused_k, p.scale = 0x6000, 0x7000, 0x9000, 0x8000, 0.1
    for s in (p.q_strides, p.o_strides):
        s.batch, s.row, s.head = 5 * 4 * 128, 4 * 128, 128
    for name, value in dict(GOOD, **kw).items():
        setattr(p, name, value)
    return p


@pytest.mark.parametrize("change", BAD)
def test_refused_sizes_need_no_workspace(built_library, change):
    from flash_attn_v100 import cabi

    lib, p = cabi.load_library(), _params(cabi, **change)
    assert lib.fmha_paged_fwd_workspace_bytes(ctypes.byref(p)) == 0
    assert lib.fmha_paged_fwd(ctypes.byref(p), None, 0, None) in (2, 3, 10, 11)


def test_sizes_that_are_taken(built_library):
    from flash_attn_v100 import cabi

    query = lambda **kw: cabi.load_library().fmha_paged_fwd_workspace_bytes(ctypes.byref(_params(cabi, **kw)))  # noqa: E731
    assert query(batch=0) == query(seqlen_q=0) == 0 == cabi.load_library().fmha_paged_fwd_workspace_bytes(None)
    # two slots of partial rows per SM, fp32, and their log-sum-exps; beside them two words per item
    assert query() >= 2 * 148 * 16 * (128 + 1) * 4 + 2 * 2 * 8
    for group in (1, 7, 65, 127, 128):  # (from 65 on a row tile of 128 has one token)
        tokens = 2 * (128 // group)
        items = query(heads_q=2 * group, seqlen_q=100 * tokens) - query(heads_q=2 * group, seqlen_q=99 * tokens)
        assert items == 2 * 2 * 8
