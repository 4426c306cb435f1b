"""A paged cache made by hand, and the definitions of its operators in 64 bits."""
import math

import torch

#: half a step of each type, relative to the value
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
EXPONENTS = {torch.float16: (-15, 8), torch.bfloat16: (-120, 120)}


def nearest_e4m3(y):
    """The e4m3 number nearest to y, halves to even (|y| <= 464): three bits behind the point, steps of 2^-9 at least."""
    _, ex = torch.frexp(y)  # y = m 2^ex, m in [1/2, 1)
    step = torch.exp2(torch.clamp(ex.double() - 4, min=-9.0))
    return torch.round(y / step) * step


def encode64(x):
    """(codes, exponents) of rows of a 16-bit tensor by the format's definition, in 64 bits."""
    low, high = EXPONENTS[x.dtype]
    y = x.double()
    finite = torch.isfinite(y)
    top = torch.where(finite, y, 0.0).abs().amax(-1)
    e = torch.full_like(top, low)
    for k in range(low, high):  # the least e with top <= 448 * 2^e, high at most
        e = torch.where(top > 448.0 * 2.0 ** k, float(k + 1), e)
    codes = nearest_e4m3(torch.where(finite, y, 0.0) * torch.exp2(-e).unsqueeze(-1))
    codes = torch.where((e == high).unsqueeze(-1), codes.clamp(-240.0, 240.0), codes)
    return torch.where(finite, codes, float("nan")), e


class Cache:
    """Pools of pages in shuffled order with `lens` tokens per entry; what no entry holds is junk (NaN), and so are
    the block table's entries behind an entry's last page."""

    def __init__(self, lens, heads, d, page, dtype, e4m3, seed=0, room=0, device="cuda", layout="nhd", spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.page, self.dtype, self.e4m3, self.heads, self.d = list(lens), page, dtype, e4m3, heads, d
        need = [-(-(n + room) // page) for n in lens]
        total, width = sum(need) + 2, max(max(need), 1)
        order = torch.randperm(total, generator=g).tolist()
        table = torch.full((len(lens), width + 1), 0x7fffffff, dtype=torch.int32)
        table[:, 1::2] = -5
        at = 0
        for z, n in enumerate(need):
            table[z, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        self.host_table = table.clone()
        self.table = table.to(device)[:, :width] if width > 0 else table.to(device)
        shape = {"nhd": (total, page, heads, d), "hnd": (total, heads, page, d)}[layout]
        byte = torch.uint8

        def pool():
            if e4m3:
                p = torch.full(shape, 0x7F, dtype=byte, device=device).view(torch.float8_e4m3fn)
            else:
                p = torch.full(shape, float("nan"), dtype=dtype, device=device)
            return p if layout == "nhd" else p.transpose(1, 2)

        self.k_cache, self.v_cache = pool(), pool()
        self.k_scale = self.v_scale = None
        if e4m3:
            self.k_scale, self.v_scale = (torch.full(shape[:-1], 255, dtype=byte, device=device).view(torch.float8_e8m0fnu)
                                          for _ in range(2))
            if layout == "hnd":
                self.k_scale, self.v_scale = (s.view(byte).transpose(1, 2).view(torch.float8_e8m0fnu)
                                              for s in (self.k_scale, self.v_scale))
        # what the entries hold: rows of unequal size
        self.k, self.v = [], []
        for z, n in enumerate(lens):
            for rows, cache, scale in ((self.k, self.k_cache, self.k_scale), (self.v, self.v_cache, self.v_scale)):
                x = torch.randn((n, heads, d), generator=g) * spread * torch.exp2(torch.randn((n, heads, 1), generator=g))
                rows.append(self.put(z, 0, x.to(dtype).to(device), cache, scale))
        self.seqused_k = torch.tensor(self.lens, dtype=torch.int32, device=device)

    def where(self, z, tokens):
        t = torch.tensor(list(tokens), dtype=torch.int64)
        pages = self.host_table[z, t // self.page].long()
        return pages.to(self.k_cache.device), (t % self.page).to(self.k_cache.device)

    def put(self, z, first, x, cache, scale):
        """Writes rows by the definition; returns what they stand for, in 64 bits."""
        page, slot = self.where(z, range(first, first + x.shape[0]))
        if not self.e4m3:
            cache[page, slot] = x
            return x.double()
        codes, e = encode64(x)
        cache.view(torch.uint8)[page, slot] = codes.float().to(torch.float8_e4m3fn).view(torch.uint8)
        scale.view(torch.uint8)[page, slot] = (e + 127).to(torch.uint8)
        return codes * torch.exp2(e).unsqueeze(-1)

    def args(self):
        return self.k_cache, self.v_cache, self.table

    def scales(self):
        return {"k_scale": self.k_scale, "v_scale": self.v_scale}


def attend64(q, cache, scale, causal, new=None):
    """(o, lse, sum of p |v|, sum of |v| over the keys seen, the largest sum of |q k| of a row) of the definition, in 64
    bits."""
    z_, n, hq, d = q.shape
    group = hq // cache.heads
    o = torch.zeros((z_, n, hq, d), dtype=torch.float64, device=q.device)
    a, b = torch.zeros_like(o), torch.zeros_like(o)
    lse = torch.full((z_, hq, n), -math.inf, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(lse)
    for z in range(z_):
        sq, sk = n if new is None else min(max(new[z], 0), n), cache.lens[z]
        if sq == 0 or sk == 0:
            continue
        k, v = (x[z].repeat_interleave(group, 1).permute(1, 0, 2) for x in (cache.k, cache.v))
        x = q[z, :sq].double().permute(1, 0, 2)
        s = scale * x @ k.transpose(1, 2)
        i, j = torch.arange(sq, device=q.device)[:, None], torch.arange(sk, device=q.device)[None, :]
        seen = (j <= sk - sq + i) if causal else (j >= 0).expand(sq, sk)
        s = torch.where(seen, s, -math.inf)
        some = seen.any(-1)
        p = torch.where(some[:, None], torch.softmax(s, -1), 0.0)
        lse[z, :, :sq] = torch.logsumexp(s, -1)
        o[z, :sq] = (p @ v).permute(1, 0, 2)
        a[z, :sq] = (p @ v.abs()).permute(1, 0, 2)
        b[z, :sq] = (seen.double() @ v.abs()).permute(1, 0, 2)
        size[z, :, :sq] = (abs(scale) * x.abs() @ k.abs().transpose(1, 2)).amax(-1)
    return o, lse, a, b, size


def check_attention(got, q, cache, scale, causal, new=None):
    """A score is a sum of D products, exact in fp32, whose additions are off by 2^-23 each of what they add
    (truncation included): D 2^-23 size.  The exponent's argument is rounded twice more in units of a score, and the
    exponential is off by 2^-22: e = 2^-23 ((D + 4) size + 8) in all, for every p and for the row sum.  So the LSE is
    off by e, and by its own rounding; P is rounded to the type (u), O too: |O - o| <= u (a + |o|) (1 + u) + 4 e a.

    fp16 has steps of 2^-24 at least, so a P in fp16 is off by up to 2^-25 where u P is less than that.  P is the exponential
    of a score over a reference that is no more than the row's largest score, so the row sum is 1 or more, and O is off by
    2^-25 b at most for it, b the sum of |v| over the keys seen.  (P is fp16 for fp16 tensors, and for 8-bit caches of few
    rows.)  Seen where a first key has p = 1 and v = 4.6e-5 and 254 others, of p = 1.4e-5 and less, have v of 1: by the
    formula without this term 1.001 of what is allowed."""
    o, lse = got
    u = UNIT[q.dtype]
    r_o, r_lse, a, b, size = attend64(q, cache, scale, causal, new)
    e = 2.0 ** -23 * ((q.shape[-1] + 4) * size + 8)
    seen = torch.isfinite(r_lse)
    assert torch.equal(torch.isfinite(lse), seen) and torch.equal(lse[~seen].double(), r_lse[~seen])
    off = (lse.double() - r_lse).abs()[seen]
    assert (off <= (e + 2.0 ** -22 * r_lse.abs())[seen]).all(), f"LSE off by {off.max():.2e}"
    e = e.permute(0, 2, 1).unsqueeze(-1)
    limit = u * (1 + u) * (a + r_o.abs()) + 4 * e * a + 2.0 ** -24  # (2^-24: the least fp16)
    if q.dtype == torch.float16 or cache.e4m3:
        limit = limit + 2.0 ** -25 * b
    off = (o.double() - r_o).abs()
    assert (off <= limit).all(), f"O off by {off.max():.2e}, {(off / limit).max():.2f} of the limit"
    none = ~seen.permute(0, 2, 1)
    assert (o[none] == 0).all()
