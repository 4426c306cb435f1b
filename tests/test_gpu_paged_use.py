"""GPU tests of the paged cache as it is used: written, read and attended to in one program, in captured graphs, on other
streams, next to memory that is not its own, with values at the ends of their types."""
import ctypes
import math

import pytest
import torch

from tests.paged_helpers import Cache, attend64, check_attention

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _q(z, n, h, d, dtype, seed=1, size=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((z, n, h, d), generator=g) * size).to(dtype).cuda()


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Server:
    """Entries that grow: new tokens are written, then attended to with all that came before."""

    def __init__(self, z, heads, d, dtype, e4m3, page=32, room=512):
        self.dtype, self.d, self.heads, self.e4m3, self.page = dtype, d, heads, e4m3, page
        pages = room // page
        order = torch.randperm(z * pages, generator=torch.Generator().manual_seed(5))
        self.table = order.to(torch.int32).reshape(z, pages).cuda()
        shape = (z * pages, page, heads, d)
        kind = torch.float8_e4m3fn if e4m3 else dtype
        self.k, self.v = (torch.empty(shape, dtype=torch.uint8 if e4m3 else dtype, device="cuda").view(kind) for _ in range(2))
        self.scales = {}
        if e4m3:
            self.scales = {n: torch.empty(shape[:3], dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
                           for n in ("k_scale", "v_scale")}
        self.length = torch.zeros(z, dtype=torch.int32, device="cuda")

    def step(self, q, k, v, new=None, causal=True):
        from flash_attn_v100 import flash_attn_paged_func, paged_cache_write

        paged_cache_write(k, v, self.k, self.v, self.table, self.length, new, **self.scales)
        self.length += k.shape[1] if new is None else new
        return flash_attn_paged_func(q, self.k, self.v, self.table, self.length, new, causal=causal, return_lse=True, **self.scales)

    def read(self):
        from flash_attn_v100 import paged_cache_read

        n = int(self.length.max())
        return paged_cache_read(self.k, self.v, self.table, self.length, n, dtype=self.dtype, **self.scales)


class Held:
    """What ``check_attention`` has to know of a cache whose rows were read back."""

    def __init__(self, k, v, lens, e4m3):
        self.k, self.v = ([x[z, :n].double() for z, n in enumerate(lens)] for x in (k, v))
        self.lens, self.heads, self.e4m3 = lens, k.shape[2], e4m3


@pytest.mark.parametrize("dtype,d,e4m3", [(BF16, 128, False), (BF16, 128, True), (F16, 64, True), (F16, 96, False)])
def test_prompts_then_tokens(dtype, d, e4m3):
    """Unequal prompts in unequal chunks, then tokens one at a time; every step against the rows that were read back,
    and for 16 bits the rows against what was written."""
    z, hk, group = 3, 2, 4
    s = Server(z, hk, d, dtype, e4m3)
    written = [[], [], []]
    for step, new in enumerate(([150, 33, 70], [64, 1, 0], [1, 1, 1], [1, 1, 1], [5, 5, 5])):
        n = max(new)
        q, k, v = _q(z, n, hk * group, d, dtype, 10 + step), _q(z, n, hk, d, dtype, 20 + step), _q(z, n, hk, d, dtype, 30 + step)
        with torch.no_grad():
            got = s.step(q, k, v, None if min(new) == n else _i32(new))
        for i in range(z):
            written[i].append(k[i, :new[i]])
        kr, vr = s.read()
        lens = s.length.tolist()
        if not e4m3:
            for i in range(z):
                assert torch.equal(kr[i, :lens[i]], torch.cat(written[i]))
        check_attention(got, q, Held(kr, vr, lens, e4m3), d ** -0.5, True, new)


@pytest.mark.parametrize("n", [32, 160, 512])
def test_a_prompt_at_once_is_the_ordinary_attention(n):
    from flash_attn_v100 import flash_attn_func

    d, h, dtype = 128, 3, BF16
    q, k, v = (_q(2, n, h, d, dtype, i) for i in range(3))
    s = Server(2, h, d, dtype, False)
    with torch.no_grad():
        out, lse = s.step(q, k, v)
        ref = flash_attn_func(q, k, v, causal=True)
    # both are within u (a + |o|) of the definition (P and O rounded to bf16): within twice that of one another
    held = Held(k, v, [n, n], False)
    o, _, a, _, _ = attend64(q, held, d ** -0.5, True)
    assert ((out.double() - ref.double()).abs() <= 2 ** -7 * (a + o.abs()) * 1.01 + 1e-6).all()


def test_captured_graphs_follow_lengths_and_share_nothing():
    """Two captured steps of two servers, replayed in turn and side by side on two streams, against steps that were
    not captured."""
    z, hk, group, d = 4, 2, 4, 128
    servers = [Server(z, hk, d, BF16, True), Server(z, hk, d, BF16, False)]
    plain = [Server(z, hk, d, BF16, True), Server(z, hk, d, BF16, False)]
    inputs = [tuple(_q(z, 1, h, d, BF16, 40 + i) for i, h in enumerate((hk * group, hk, hk))) for _ in servers]
    prompt = tuple(_q(z, 200, h, d, BF16, 50 + i) for i, h in enumerate((hk * group, hk, hk)))
    with torch.no_grad():
        for s in servers + plain:
            s.step(*prompt, new=_i32([200, 3, 77, 128]))
        warm = [s.step(*x) for s, x in zip(servers, inputs)]
        for s in servers:
            s.length -= 1  # (the warm-up's token is written again)
        graphs, outs = [], []
        for s, x in zip(servers, inputs):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append(s.step(*x))
            graphs.append(g)
        streams = [torch.cuda.Stream() for _ in graphs]
        for step in range(6):
            for i, x in enumerate(inputs):
                for j, t in enumerate(x):
                    t.copy_(_q(*t.shape, BF16, 100 * step + 10 * i + j))
            torch.cuda.synchronize()
            if step % 2:
                for g, st in zip(graphs, streams):
                    with torch.cuda.stream(st):
                        g.replay()
            else:
                for g in graphs:
                    g.replay()
            torch.cuda.synchronize()
            for p, x, (o, lse) in zip(plain, inputs, outs):
                r = p.step(*x)
                assert torch.equal(o, r[0]) and torch.equal(lse, r[1])
    assert len(warm) == 2


def test_two_streams_at_once():
    from flash_attn_v100 import flash_attn_paged_func

    a = Cache([3000, 500, 1900], 2, 128, 64, BF16, False, seed=1)
    b = Cache([700, 2500], 2, 64, 16, F16, True, seed=2)
    qa, qb = _q(3, 1, 8, 128, BF16), _q(2, 70, 4, 64, F16)
    call_a = lambda: flash_attn_paged_func(qa, *a.args(), a.seqused_k, causal=True, return_lse=True)  # noqa: E731
    call_b = lambda: flash_attn_paged_func(qb, *b.args(), b.seqused_k, causal=True, return_lse=True, **b.scales())  # noqa: E731
    ref = call_a(), call_b()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(20):
        for st, call in zip(streams, (call_a, call_b)):
            with torch.cuda.stream(st):
                got.append(call())
    torch.cuda.synchronize()
    for i, (o, lse) in enumerate(got):
        assert torch.equal(o, ref[i % 2][0]) and torch.equal(lse, ref[i % 2][1])


# ------------------------------------------------------------------------------------------ values
@pytest.mark.parametrize("n", [1, 4, 40])
@pytest.mark.parametrize("dtype,e4m3", [(BF16, True), (F16, True), (BF16, False)])
def test_rows_of_very_unequal_size(n, dtype, e4m3):
    """Rows of K and V of sizes from 2^-30 to 2^12 (fp16: 2^-12 to 2^9) next to one another: scales beyond what fp16 can
    take among them."""
    from flash_attn_v100 import flash_attn_paged_func, paged_cache_write

    low, high = (-30, 12) if dtype == BF16 else (-12, 9)
    c = Cache([0, 0], 2, 128, 32, dtype, e4m3, room=700)
    g = torch.Generator().manual_seed(9)
    size = torch.exp2(torch.randint(low, high, (2, 700, 2, 1), generator=g).float())
    size[:, 300:] = torch.exp2(torch.full((2, 400, 2, 1), float(low)))  # and whole tiles of the smallest
    k, v = ((torch.randn((2, 700, 2, 128), generator=g) * size).to(dtype).cuda() for _ in range(2))
    k = (k.float() * 2.0 ** -6).to(dtype)
    paged_cache_write(k, v, *c.args(), _i32([0, 0]), **c.scales())
    from flash_attn_v100 import paged_cache_read

    kr, vr = paged_cache_read(*c.args(), _i32([700, 690]), 700, dtype=dtype, **c.scales())
    held = Held(kr, vr, [700, 690], e4m3)
    q = _q(2, n, 8, 128, dtype, 4, 0.5)
    got = flash_attn_paged_func(q, *c.args(), _i32([700, 690]), causal=True, return_lse=True, **c.scales())
    check_attention(got, q, held, 128 ** -0.5, True)


@pytest.mark.parametrize("n", [1, 3, 50])
@pytest.mark.parametrize("e4m3", [False, True])
def test_scores_that_leap_and_signs(n, e4m3):
    """Keys whose norm grows by 1.2 every 16 tokens make the running reference grow; a negative scale, large queries."""
    from flash_attn_v100 import flash_attn_paged_func, paged_cache_write

    d, length = 64, 900
    c = Cache([0], 2, d, 16, F16, e4m3, room=length)
    grow = 1.2 ** (torch.arange(length) // 16).float().reshape(1, -1, 1, 1) / 2.0 ** 8
    k = (_q(1, length, 2, d, F16, 6).float().cpu() * grow).to(F16).cuda()
    v = _q(1, length, 2, d, F16, 7)
    paged_cache_write(k, v, *c.args(), _i32([0]), **c.scales())
    from flash_attn_v100 import paged_cache_read

    held = Held(*paged_cache_read(*c.args(), _i32([length]), length, dtype=F16, **c.scales()), [length], e4m3)
    q = _q(1, n, 4, d, F16, 8, 3.0)
    for scale in (0.3, -0.3):
        got = flash_attn_paged_func(q, *c.args(), _i32([length]), softmax_scale=scale, causal=True, return_lse=True, **c.scales())
        check_attention(got, q, held, scale, True)


@pytest.mark.parametrize("n", [1, 6, 80])
@pytest.mark.parametrize("e4m3", [False, True])
def test_not_finite_stays_in_its_rows(n, e4m3):
    """A NaN in a key makes NaN of every row that sees the key, one in a value of the value's element; what does not see
    them, other entries and heads, is as it was."""
    from flash_attn_v100 import flash_attn_paged_func

    c = Cache([300, 200], 2, 128, 32, BF16, e4m3, seed=3)
    q = _q(2, n, 8, 128, BF16)
    call = lambda: flash_attn_paged_func(q, *c.args(), c.seqused_k, causal=True, return_lse=True, **c.scales())  # noqa: E731
    o0, l0 = call()
    page, slot = c.where(0, [297, 298])  # seen by the last 3 and the last 2 new tokens
    nan = 0x7F if e4m3 else float("nan")
    kv, vv = (x.view(torch.uint8) if e4m3 else x for x in (c.k_cache, c.v_cache))
    kv[page[0], slot[0], 1, 5] = nan
    vv[page[1], slot[1], 0, 7] = nan
    o, lse = call()
    assert torch.equal(o[1], o0[1]) and torch.equal(lse[1], l0[1])
    first_k, first_v = max(0, n - 3), max(0, n - 2)
    assert torch.isnan(o[0, first_k:, 4:]).all() and torch.isnan(lse[0, 4:, first_k:]).all()
    assert torch.equal(lse[0, :4], l0[0, :4])
    assert torch.isnan(o[0, first_v:, :4, 7]).all()
    o[0, first_v:, :4, 7] = o0[0, first_v:, :4, 7]
    assert torch.equal(o[0, :, :4].isnan().sum(), torch.tensor(0, device="cuda")) or first_v > 0
    # (a value's NaN spreads to the tokens of its tile that do not see it yet: 0 times it is NaN, as in any product)
    seen = slice(first_v, None)
    assert torch.equal(o[0, seen, :4], o0[0, seen, :4])


@pytest.mark.parametrize("n", [1, 6, 80])
@pytest.mark.parametrize("dtype,e4m3", [(BF16, False), (BF16, True), (F16, False), (F16, True)])
def test_an_infinite_score_is_no_answer(n, dtype, e4m3):
    """An infinite element of a query makes scores of infinity, and inf / inf is NaN: in the whole row, and in no other."""
    from flash_attn_v100 import flash_attn_paged_func

    c = Cache([700, 90], 2, 64, 32, dtype, e4m3, seed=11)
    clean = _q(2, n, 8, 64, dtype, 12)
    call = lambda q: flash_attn_paged_func(q, *c.args(), c.seqused_k, causal=True, return_lse=True, **c.scales())  # noqa: E731
    o0, l0 = call(clean)
    q = clean.clone()
    rows = [(0, n - 1, 1), (0, n // 2, 6), (1, n - 1, 0)]
    for i, (z, t, h) in enumerate(rows):
        q[z, t, h, 9 + i] = math.inf if i % 2 else -math.inf
    o, lse = call(q)
    for z, t, h in rows:
        assert torch.isnan(o[z, t, h]).all() and not torch.isfinite(lse[z, h, t]) and lse[z, h, t] != -math.inf
        o[z, t, h], lse[z, h, t] = o0[z, t, h], l0[z, h, t]
    check_attention((o, lse), clean, c, 0.125, True)


@pytest.mark.parametrize("n", [1, 6, 80])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_scores_of_minus_infinity_have_no_weight(n, dtype):
    """Keys of -inf in one element (16 bits): to queries that are positive there they are as good as absent, over whole tiles
    too; queries that are negative there have no answer."""
    from flash_attn_v100 import flash_attn_paged_func

    gone = 150
    c = Cache([700], 2, 64, 32, dtype, False, seed=13)
    page, slot = c.where(0, range(gone))
    c.k_cache[page, slot, :, 5] = -math.inf
    q = _q(1, n, 8, 64, dtype, 14)
    q[..., 5] = q[..., 5].abs() + 0.125
    clean, bad = q.clone(), [(n - 1, 2), (n // 2, 7)]
    for t, h in bad:
        q[0, t, h, 5] *= -1
    o0, l0 = flash_attn_paged_func(clean, *c.args(), c.seqused_k, causal=True, return_lse=True)
    o, lse = flash_attn_paged_func(q, *c.args(), c.seqused_k, causal=True, return_lse=True)
    for t, h in bad:
        assert torch.isnan(o[0, t, h]).all() and not torch.isfinite(lse[0, h, t]) and lse[0, h, t] != -math.inf
        o[0, t, h], lse[0, h, t] = o0[0, t, h], l0[0, h, t]
    c.k, c.v, c.lens = [c.k[0][gone:]], [c.v[0][gone:]], [c.lens[0] - gone]
    check_attention((o, lse), clean, c, 0.125, True)


def test_missing_pages_are_keys_of_zero():
    from flash_attn_v100 import flash_attn_paged_func, paged_cache_read

    for e4m3 in (False, True):
        c = Cache([400, 160], 2, 64, 32, BF16, e4m3, seed=4)
        table = c.table.clone()
        table[0, 3], table[0, 7], table[1, 0] = -1, c.k_cache.shape[0], 1 << 30
        kr, vr = paged_cache_read(c.k_cache, c.v_cache, table, c.seqused_k, 400, dtype=BF16, **c.scales())
        held = Held(kr, vr, [400, 160], e4m3)
        for n in (1, 40):
            q = _q(2, n, 8, 64, BF16)
            got = flash_attn_paged_func(q, c.k_cache, c.v_cache, table, c.seqused_k, causal=True, return_lse=True, **c.scales())
            check_attention(got, q, held, 0.125, True)


# ------------------------------------------------------------------------------------------ shapes and memory
@pytest.mark.parametrize("n", [15, 16, 17, 32, 33, 47, 48, 49, 64, 65, 127, 128, 129])
@pytest.mark.parametrize("d,dtype,e4m3", [(128, BF16, False), (64, F16, True), (96, BF16, True), (128, F16, True), (64, BF16, False)])
def test_numbers_of_rows_at_the_kernels_ends(n, d, dtype, e4m3):
    from flash_attn_v100 import flash_attn_paged_func

    c = Cache([700, 260, 128], 2, d, 32, dtype, e4m3, seed=n)
    q = _q(3, n, 2, d, dtype, n)
    new = [n, n // 2, 1]
    for causal in (True, False):
        got = flash_attn_paged_func(q, *c.args(), c.seqused_k, _i32(new), causal=causal, return_lse=True, **c.scales())
        check_attention(got, q, c, d ** -0.5, causal, new)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("n", [1, 33])
def test_many_entries_and_lengths_beyond_their_pages(e4m3, n):
    """300 entries of 0 to 299 tokens; lengths that say more than the table has room for are what it has room for."""
    lens = list(range(300))
    c = Cache(lens, 1, 64, 16, F16, e4m3, seed=5)
    q = _q(300, n, 4, 64, F16)
    from flash_attn_v100 import flash_attn_paged_func

    got = flash_attn_paged_func(q, *c.args(), c.seqused_k, causal=False, return_lse=True, **c.scales())
    check_attention(got, q, c, 0.125, False)
    one = Cache([64], 1, 64, 16, F16, e4m3, seed=6)
    q = q[:1]
    a = flash_attn_paged_func(q, one.k_cache, one.v_cache, one.table[:, :4].contiguous(), _i32([64]), return_lse=True, **one.scales())
    b = flash_attn_paged_func(q, one.k_cache, one.v_cache, one.table[:, :4].contiguous(), _i32([1 << 30]), return_lse=True, **one.scales())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("e4m3", [False, True])
def test_offsets_beyond_32_bits(e4m3):
    """A pool of 5 GB whose pages in use lie at its end."""
    from flash_attn_v100 import flash_attn_paged_func, paged_cache_read, paged_cache_write

    page, h, d, dtype = 64, 8, 128, BF16
    row = page * h * d * (1 if e4m3 else 2)
    pages = 5 * 2 ** 30 // row
    kind = torch.uint8 if e4m3 else dtype
    k_cache, v_cache = (torch.empty((pages, page, h, d), dtype=kind, device="cuda") for _ in range(2))
    scales = {}
    if e4m3:
        k_cache, v_cache = k_cache.view(torch.float8_e4m3fn), v_cache.view(torch.float8_e4m3fn)
        scales = {n: torch.empty((pages, page, h), dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for n in ("k_scale", "v_scale")}
    table = _i32([[pages - 1, pages - 3, 0], [pages - 2, pages // 2 + 1, 5]])
    k, v = _q(2, 150, h, d, dtype, 1), _q(2, 150, h, d, dtype, 2)
    paged_cache_write(k, v, k_cache, v_cache, table, _i32([0, 0]), **scales)
    kr, vr = paged_cache_read(k_cache, v_cache, table, _i32([150, 150]), 150, dtype=dtype, **scales)
    if not e4m3:
        assert torch.equal(kr, k) and torch.equal(vr, v)
    held = Held(kr, vr, [150, 150], e4m3)
    for n in (1, 40):
        q = _q(2, n, 16, d, dtype, 3)
        got = flash_attn_paged_func(q, k_cache, v_cache, table, _i32([150, 150]), causal=True, return_lse=True, **scales)
        check_attention(got, q, held, d ** -0.5, True)


@pytest.mark.parametrize("n", [1, 5, 70])
@pytest.mark.parametrize("e4m3", [False, True])
def test_nothing_around_the_outputs_is_written(n, e4m3):
    """Outputs, log-sum-exps and workspace inside larger buffers; strided q and o."""
    from flash_attn_v100 import cabi

    d, hk, group = 96, 2, 3
    c = Cache([500, 90], hk, d, 48, BF16, e4m3, seed=8)
    base = _q(2, n, 2 * hk * group, 2 * d, BF16)
    q = base[:, :, ::2, :d]
    pad = torch.full((2, n + 3, hk * group + 2, d + 16), 7.0, dtype=BF16, device="cuda")
    o = pad[:, :n, 1:-1, 8:d + 8]
    lse_pad = torch.full((2 * hk * group * n + 64,), 7.0, device="cuda")
    lse = lse_pad[32:-32].view(2, hk * group, n)
    cc = cabi.paged_cache(c.k_cache, c.v_cache, c.table, c.k_scale, c.v_scale)
    p = cabi.FmhaPagedFwdParams()
    p.cache, p.batch, p.heads_q, p.heads_k, p.seqlen_q, p.head_dim, p.dtype = cc, 2, hk * group, hk, n, d, 1
    need = cabi.load_library().fmha_paged_fwd_workspace_bytes(ctypes.byref(p))
    ws = torch.full((need + 512,), 0xFF, dtype=torch.uint8, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cabi.paged_fwd(q, cc, hk, c.seqused_k, d ** -0.5, True, status=status, workspace=ws[256:-256], out=o, lse=lse)
    check_attention((o, lse), q, c, d ** -0.5, True)
    inside = torch.zeros_like(pad, dtype=torch.bool)
    inside[:, :n, 1:-1, 8:d + 8] = True
    assert (pad[~inside] == 7).all() and (lse_pad[:32] == 7).all() and (lse_pad[-32:] == 7).all()
    assert (ws[:256] == 0xFF).all() and (ws[-256:] == 0xFF).all()
    assert int(status) == 0


@pytest.mark.parametrize("n", [1, 100])
def test_a_set_status_word_leaves_the_outputs_alone(n):
    from flash_attn_v100 import cabi

    c = Cache([700, 300], 2, 128, 64, BF16, False)
    q = _q(2, n, 4, 128, BF16)
    cc = cabi.paged_cache(c.k_cache, c.v_cache, c.table)
    out, lse = torch.full_like(q, 3.0), torch.full((2, 4, n), 3.0, device="cuda")
    status = _i32([77])
    cabi.paged_fwd(q, cc, 2, c.seqused_k, 0.1, True, status=status, out=out, lse=lse)
    torch.cuda.synchronize()
    assert (out == 3).all() and (lse == 3).all() and int(status) == 77
    status.zero_()
    cabi.paged_fwd(q, cc, 2, c.seqused_k, 128 ** -0.5, True, status=status, out=out, lse=lse)
    check_attention((out, lse), q, c, 128 ** -0.5, True)
    assert int(status) == 0


def test_nothing_to_do():
    from flash_attn_v100 import flash_attn_paged_func, paged_cache_read, paged_cache_write

    c = Cache([10], 2, 64, 16, F16, False)
    empty = torch.empty((1, 0, 4, 64), dtype=F16, device="cuda")
    out, lse = flash_attn_paged_func(empty, *c.args(), c.seqused_k, return_lse=True)
    assert out.shape == (1, 0, 4, 64) and lse.shape == (1, 4, 0)
    paged_cache_write(empty[:, :, :2], empty[:, :, :2], *c.args(), c.seqused_k)
    k, v = paged_cache_read(*c.args(), c.seqused_k, 0)
    assert k.shape == v.shape == (1, 0, 2, 64)
    none = _i32([]).reshape(0, 3)
    out = flash_attn_paged_func(torch.empty((0, 5, 4, 64), dtype=F16, device="cuda"), c.k_cache, c.v_cache, none, _i32([]))
    assert out.shape == (0, 5, 4, 64)


def test_traced_and_under_inference_mode():
    from flash_attn_v100 import flash_attn_paged_func, paged_cache_read, paged_cache_write

    with torch.inference_mode():
        c = Cache([40, 9], 2, 64, 16, BF16, True, room=4)

        def step(q, k, v, k_cache, v_cache, table, lengths, k_scale, v_scale):
            paged_cache_write(k, v, k_cache, v_cache, table, lengths, None, k_scale, v_scale)
            out = flash_attn_paged_func(q, k_cache, v_cache, table, lengths + 1, None, k_scale, v_scale, causal=True)
            return out, paged_cache_read(k_cache, v_cache, table, lengths + 1, 41, k_scale, v_scale, torch.bfloat16)[0]

        args = (_q(2, 1, 4, 64, BF16), _q(2, 1, 2, 64, BF16, 2), _q(2, 1, 2, 64, BF16, 3), *c.args(), c.seqused_k, c.k_scale, c.v_scale)
        want = step(*args)
    with torch.no_grad():
        args = tuple(a.clone() if a.dtype.itemsize > 1 else a.view(torch.uint8).clone().view(a.dtype) for a in args)
        got = torch.compile(step, fullgraph=True, backend="eager")(*args)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals_of_tensors():
    from flash_attn_v100 import flash_attn_paged_func, paged_cache_write

    c = Cache([20], 2, 64, 16, F16, False)
    e = Cache([20], 2, 64, 16, F16, True)
    q = _q(1, 1, 4, 64, F16)
    bad = [
        lambda: flash_attn_paged_func(q.to(BF16), *c.args(), c.seqused_k),                              # another type
        lambda: flash_attn_paged_func(_q(1, 1, 5, 64, F16), *c.args(), c.seqused_k),                    # heads
        lambda: flash_attn_paged_func(q, *e.args(), e.seqused_k),                                       # no scales
        lambda: flash_attn_paged_func(q, *c.args(), c.seqused_k, None, e.k_scale, e.v_scale),           # scales of nothing
        lambda: flash_attn_paged_func(q, c.k_cache, c.v_cache[:1], c.table, c.seqused_k),               # pools unlike
        lambda: flash_attn_paged_func(q, *c.args(), c.seqused_k.long()),                                # lengths of 64 bits
        lambda: flash_attn_paged_func(q, c.k_cache, c.v_cache, c.table.cpu(), c.seqused_k),             # a table on the host
        lambda: flash_attn_paged_func(q, c.k_cache[:, :8], c.v_cache[:, :8], c.table, c.seqused_k),     # pages of 8
        lambda: flash_attn_paged_func(q, *c.args(), c.seqused_k, softmax_scale=math.inf),
        lambda: paged_cache_write(q, q, *c.args(), c.seqused_k),                                        # four heads into two
        lambda: paged_cache_write(q[:, :, :2], q[:, :, :2].to(BF16), *c.args(), c.seqused_k),
    ]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
