"""The packed key / value cache on the GPU: block tables, append and read, attention, and a run of them together,
against plain implementations (the pure-path oracle of the quantizer; loops and fp64)."""
import math

import pytest
import torch

from helpers import assert_bits_equal
from microxcaling_amd import _lib
from microxcaling_amd import custom_extensions as ce
from microxcaling_amd.kv_cache import (PackedKVCache, kv_append, kv_attention, kv_block_tables, kv_read, new_kv_cache)
from oracle import mx_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    return torch.Generator().manual_seed(seed)


def quantized(x, round="nearest"):
    """What the cache holds for rows x: the quantizer's pure path."""
    return O.quantize_mx(x.cpu(), 8, "fp4_e2m1", axes=[-1], block_size=32, round=round).float()


def rows_like(shape, dtype, seed):
    x = torch.randn(shape, generator=gen(seed)) * torch.exp(2 * torch.randn(shape[0], 1, 1, generator=gen(seed + 1)))
    return x.to(dtype)


# ---- append and read -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,heads,page,tokens,round", [
    (128, 2, 16, 37, "nearest"), (80, 3, 48, 21, "even"), (1, 1, 16, 5, "nearest"), (31, 2, 32, 9, "floor"),
    (256, 1, 16, 18, "nearest"), (64, 5, 16, 1, "floor"), (96, 2, 80, 33, "even"), (200, 1, 16, 16, "nearest")])
def test_append_then_read(dtype, dim, heads, page, tokens, round):
    """Rows at scattered slots, and untouched bytes everywhere else."""
    pages = -(-tokens // page) + 2
    cache = new_kv_cache(pages, page, heads, dim, DEV)
    cache.data.fill_(0x5A)
    before = cache.data.clone()
    both = rows_like((tokens, 2 * heads, dim), dtype, 1).to(DEV)
    k, v = both[:, :heads], both[:, heads:]                      # slices of one projection
    slots = torch.randperm(pages * page, generator=gen(2))[:tokens]
    if tokens > 4:
        slots[1], slots[3] = -1, pages * page                    # outside the cache
    kv_append(cache, k, v, slots.to(DEV), round=round)
    got_k, got_v = kv_read(cache, slots.to(DEV))
    live = (slots >= 0) & (slots < pages * page)
    for got, x in ((got_k, k), (got_v, v)):
        want = quantized(x, round)
        want[~live] = 0
        assert_bits_equal(got.cpu(), want, "rows")
    others = torch.tensor([s for s in range(pages * page) if s not in set(slots[live].tolist())], device=DEV)
    a, b = kv_read(cache, others), kv_read(PackedKVCache(before, page, dim), others)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # bytes: what changed is at most 34 NB a row and head
    changed = (cache.data != before).sum().item()
    assert changed <= int(live.sum()) * heads * -(-dim // 32) * 34


@pytest.mark.parametrize("first,tokens", [(0, 64), (0, 61), (3, 30), (16, 5), (7, 1)])
def test_append_of_consecutive_tokens(first, tokens):
    """Whole groups of four tokens, groups cut at either end, across pages."""
    heads, dim, page = 2, 96, 16
    cache = new_kv_cache(6, page, heads, dim, DEV)
    k, v = (rows_like((tokens, heads, dim), torch.bfloat16, s) for s in (3, 4))
    slots = torch.arange(first, first + tokens, device=DEV)
    kv_append(cache, k.to(DEV), v.to(DEV), slots)
    for got, x in zip(kv_read(cache, slots), (k, v)):
        assert_bits_equal(got.cpu(), quantized(x), "rows")
    flipped = slots.flip(0)
    for got, x in zip(kv_read(cache, flipped, torch.bfloat16), (k, v)):
        assert_bits_equal(got.cpu(), quantized(x).flip(0).bfloat16(), "bf16 rows, another order")
    rest = kv_read(cache, torch.arange(first + tokens, 96, device=DEV))
    assert not rest[0].any() and not rest[1].any()


def unpack_record(data, page, dim):
    """The documented layout, byte by byte: values (pages, heads, page, 32 NB) of K and V."""
    P, H, _ = data.shape
    NB = -(-dim // 32)
    mag = [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    lut = torch.tensor(mag + [-m for m in mag])
    k, v = torch.empty(P, H, page, 32 * NB), torch.empty(P, H, page, 32 * NB)
    d = data.cpu().long()
    for t in range(page):
        for e in range(32 * NB):
            kb, ks = d[:, :, t * 16 * NB + e // 2], d[:, :, page * 32 * NB + t * NB + e // 32]
            b, i = e // 32, e % 32 // 2
            vb = d[:, :, page * 16 * NB + t // 4 * 64 * NB + (i * NB + b) * 4 + t % 4]
            vs = d[:, :, page * 33 * NB + t // 4 * 4 * NB + 4 * b + t % 4]
            k[:, :, t, e] = lut[(kb >> 4 * (e % 2)) & 15] * 2.0 ** (ks - 127).float()
            v[:, :, t, e] = lut[(vb >> 4 * (e % 2)) & 15] * 2.0 ** (vs - 127).float()
    return k, v


@pytest.mark.parametrize("dim,page", [(64, 16), (72, 32)])
def test_layout_of_a_record(dim, page):
    heads, tokens = 2, 2 * page
    cache = new_kv_cache(2, page, heads, dim, DEV)
    k, v = (rows_like((tokens, heads, dim), torch.float32, s) for s in (5, 6))
    kv_append(cache, k.to(DEV), v.to(DEV), torch.arange(tokens, device=DEV))
    for got, x in zip(unpack_record(cache.data, page, dim), (k, v)):
        want = torch.zeros(tokens, heads, got.shape[-1])
        want[..., :dim] = quantized(x)
        assert torch.equal(got, want.view(2, page, heads, -1).transpose(1, 2))


def test_special_values_and_fp16_rows():
    """Inf and NaN make their block NaN; zeros stay zero; fp16 rows in the exact exponent mode only."""
    cache = new_kv_cache(1, 16, 1, 64, DEV)
    x = torch.randn(4, 1, 64, generator=gen(7))
    x[0, 0, 3], x[1, 0, 40], x[2] = float("inf"), float("nan"), 0.0
    x[3, 0, :32] = -0.0
    s = torch.arange(4, device=DEV)
    kv_append(cache, x.to(DEV), (2 * x).to(DEV), s)
    for got, y in zip(kv_read(cache, s), (x, 2 * x)):
        assert_bits_equal(got.cpu(), quantized(y), "specials")
    h = torch.randn(4, 1, 64, generator=gen(8)).half().to(DEV)
    with pytest.raises(RuntimeError, match="fp16"):
        kv_append(cache, h, h, s)
    ce.set_exponent_mode("exact")
    try:
        kv_append(cache, h, h, s)
        from microxcaling_amd.mx_ops import _quantize_mx
        got, want = kv_read(cache, s, torch.float16)[0], _quantize_mx(h, 8, "fp4_e2m1", axes=[-1], block_size=32)
    finally:
        ce.set_exponent_mode("torch")
    assert_bits_equal(got, want, "fp16, exact exponents")


@pytest.mark.parametrize("round", ["nearest", "even", "floor"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_values_at_and_next_to_every_border(dtype, round):
    """Every finite bf16 code beside block maxima that put it at every place of the grid (fp32: the borders between
    codes and their neighbours), maxima at both ends of the range and in the zone where log2 rounds up."""
    if dtype == torch.bfloat16:
        codes = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).float()
        codes = codes[torch.isfinite(codes)]
    else:
        edges = torch.tensor([0, 0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7, 2.0 ** -126, 2.0 ** -149, 1e-3])
        bits = edges.view(torch.int32)[:, None] + torch.arange(-3, 4, dtype=torch.int32)
        codes = bits.clamp(min=0).view(torch.float32).flatten()
        codes = torch.cat([codes, -codes, codes * 2.0 ** -30, codes * 2.0 ** 20])
    maxima = torch.tensor([4.0, 5.0, 6.5, 7.96875, 1.0, 2.0 ** -126, 2.0 ** -130, 3e38, 2.0 ** 127, 0.0078125]).to(dtype).float()
    x = torch.zeros(len(maxima) * -(-len(codes) // 31), 1, 32)
    n = -(-len(codes) // 31)
    padded = torch.cat([codes, codes.new_zeros(n * 31 - len(codes))]).view(n, 31)
    for i, m in enumerate(maxima):
        part = x[i * n:(i + 1) * n, 0]
        part[:, 0], part[:, 1:] = m, torch.where(padded.abs() <= m, padded, torch.zeros(()))
    x = x.to(dtype)
    cache = new_kv_cache(-(-len(x) // 16), 16, 1, 32, DEV)
    slots = torch.arange(len(x), device=DEV)
    kv_append(cache, x.to(DEV), (-x).to(DEV), slots, round=round)
    for got, y in zip(kv_read(cache, slots), (x, -x)):
        assert_bits_equal(got.cpu(), quantized(y, round), "codes")


# ---- block tables ----------------------------------------------------------------------------------------------------
def tables_by_loops(ctx, new, table, free, start, page, rows):
    table, R, C = [list(r) for r in table], len(ctx), len(table[0]) if table else 0
    slots, positions, owners, starts, lens = [], [], [], [0], []
    for r in range(R):
        c, n = max(0, ctx[r]), max(0, new[r])
        for j in range(-(-c // page), min(-(-(c + n) // page), C)):
            table[r][j] = free[start] if 0 <= start < len(free) else -1
            start += 1
        for i in range(n):
            j = (c + i) // page
            p = table[r][j] if j < C else -1
            slots.append(p * page + (c + i) % page if p >= 0 else -1)
            positions.append(c + i)
            owners.append(r)
        starts.append(starts[-1] + n)
        lens.append(c + n)
    pad = [-1] * max(0, rows - len(slots))
    return (table, (slots + pad)[:rows], (positions + pad)[:rows], (owners + pad)[:rows], [min(s, rows) for s in starts], lens, start)


@pytest.mark.parametrize("requests,most,new,page,width,pad,free_slack", [
    (1, 100, 1, 16, 8, 0, 2), (5, 60, 30, 16, 7, 9, 2), (40, 200, 3, 48, 6, 0, 0), (300, 90, 2, 16, 7, 13, 5),
    (7, 80, 700, 64, 14, 0, 1), (6, 60, 40, 16, 4, 3, 4), (6, 60, 40, 16, 8, 0, -6), (600, 40, 1, 32, 3, 50, 3)])
def test_block_tables(requests, most, new, page, width, pad, free_slack):
    """Mixed lengths with empty, negative and padded requests; tables and lists of free pages that are too short;
    more requests than a workgroup scans at once; more tokens than a workgroup writes."""
    g = gen(requests)
    ctx = torch.randint(0, most + 1, (requests,), generator=g)
    fresh = torch.randint(0, new + 1, (requests,), generator=g)
    if requests > 4:
        ctx[1], fresh[1], fresh[2], ctx[3], fresh[3] = -5, 0, -3, page, 1
    pages = torch.randperm(requests * width + 40, generator=g).int()
    table = torch.full((requests, width), -7, dtype=torch.int32)
    used = 0
    for r in range(requests):
        n = min(max(0, -(-int(ctx[r]) // page)), width)
        table[r, :n] = pages[used:used + n]
        used += n
    need = sum(max(0, min(-(-(max(0, int(c)) + max(0, int(n))) // page), width) - -(-max(0, int(c)) // page))
               for c, n in zip(ctx, fresh))
    skip = 3
    free = torch.cat([pages.new_full((skip,), 99999), pages[used:used + max(0, need + free_slack)]])
    rows = int(fresh.clamp(min=0).sum()) + pad
    want = tables_by_loops(ctx.tolist(), fresh.tolist(), table.tolist(), free.tolist(), skip, page, rows)
    wide = torch.full((requests, width + 3), -9, dtype=torch.int32, device=DEV)      # rows further apart
    wide[:, :width] = table.to(DEV)
    t = wide[:, :width]
    for _ in range(2):                                                               # the same again: the same
        got = kv_block_tables(ctx.int().to(DEV), fresh.int().to(DEV), t, free.to(DEV), torch.tensor([skip], dtype=torch.int32, device=DEV),
                              page, rows)
        assert got.block_table is t
        for name, w in zip(("block_table", "slots", "positions", "requests", "starts", "seq_lens"), want):
            assert getattr(got, name).tolist() == w, name
        assert got.free_start.tolist() == [want[6]]
    assert (wide[:, width:] == -9).all()


def test_block_tables_of_nothing():
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    one = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = kv_block_tables(none, none, torch.empty(0, 4, dtype=torch.int32, device=DEV), none, one, 16, 5)
    assert got.slots.tolist() == [-1] * 5 and got.starts.tolist() == [0] and got.free_start.tolist() == [0]
    got = kv_block_tables(one, one, torch.full((1, 4), -1, dtype=torch.int32, device=DEV), none, one, 16, 0)
    assert got.slots.numel() == 0 and got.starts.tolist() == [0, 0] and got.seq_lens.tolist() == [0]


# ---- attention -------------------------------------------------------------------------------------------------------
class Setup:
    """Requests with `lens` tokens, the last new[r] of which are queried; pages in random order, the cache filled with
    0xFF (NaN) where no token is."""

    def __init__(self, lens, new, heads, group, dim, page, dtype=torch.bfloat16, seed=0, spare=0, kv_scale=1.0):
        self.page, self.dim, self.heads, self.group, self.lens, self.new = page, dim, heads, group, lens, new
        g = gen(seed)
        need = [-(-n // page) for n in lens]
        width, pages = max(need + [1]) + spare, sum(need) + 3
        order = torch.randperm(pages, generator=g).int()
        self.table = torch.full((len(lens), width), -1, dtype=torch.int32)
        used = 0
        for r, n in enumerate(need):
            self.table[r, :n] = order[used:used + n]
            used += n
        cache = new_kv_cache(pages, page, heads, dim, DEV)
        cache.data.fill_(0xFF)
        self.k, self.v, slots = [], [], []
        for r, n in enumerate(lens):
            t = torch.arange(n)
            slots.append(self.table[r].long()[t // page] * page + t % page)
            self.k.append(torch.randn(n, heads, dim, generator=g).mul(kv_scale).bfloat16())
            self.v.append((torch.randn(n, heads, dim, generator=g) + 0.3).mul(kv_scale).bfloat16())
        self.slots = slots
        if sum(lens):
            kv_append(cache, torch.cat(self.k).to(DEV), torch.cat(self.v).to(DEV), torch.cat(slots).to(DEV))
        self.cache = cache
        self.starts = torch.tensor([0] + new).cumsum(0).int()
        rows = int(self.starts[-1])
        self.q = torch.randn(rows, heads * group, dim, generator=g).to(dtype)
        self.seq = torch.tensor(lens, dtype=torch.int32)

    def call(self, q=None, **kw):
        single = kw.pop("single", False)
        q = self.q.to(DEV) if q is None else q
        return kv_attention(q, self.cache, self.table.to(DEV), self.seq.to(DEV),
                            None if single else self.starts.to(DEV), return_lse=True, **kw)

    def want(self, scale=None, causal=True, seen=None, terms=2):
        """(out, lse, tolerance of out, tolerance of lse) in fp64.  seen(r): which tokens of a request can be seen."""
        scale = self.dim ** -0.5 if scale is None else scale
        H, G, rows = self.heads, self.group, self.q.shape[0]
        out = torch.zeros(rows, H * G, self.dim, dtype=torch.float64)
        lse = torch.full((rows, H * G), -math.inf, dtype=torch.float64)
        tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
        for r, n in enumerate(self.lens):
            k, v = (quantized(x).double() for x in (self.k[r], self.v[r]))
            for i in range(self.new[r]):
                sees = min(n, n - self.new[r] + i + 1) if causal else n
                keep = torch.arange(n) < sees
                if seen is not None:
                    keep &= seen(r)
                if not keep.any():
                    continue
                row = int(self.starts[r]) + i
                for h in range(H * G):
                    kk, vv, x = k[keep, h // G], v[keep, h // G], self.q[row, h].double()
                    z = kk @ x * scale
                    lse[row, h] = z.logsumexp(0)
                    p = (z - lse[row, h]).exp()
                    out[row, h] = p @ vv
                    # a score's error: sums of head_dim products in fp32, the factor, the subtraction of the maximum;
                    # 2^x itself is good to 2 units in the last place
                    off = (self.dim + 4) * 2.0 ** -24 * (kk.abs() @ x.abs() * abs(scale)).max() + 2.0 ** -22 * (1 + z.abs().max())
                    weight = (p[:, None] * vv.abs()).sum(0)
                    # fp32 sums over the tokens; the probabilities in one bf16 term (half a step: 2^-8) or two (2^-16);
                    # the output's own rounding
                    part = 2 * off + (keep.sum() + 16) * 2.0 ** -24 + 2.0 ** (-8 if terms == 1 else -16)
                    tol[row, h] = torch.finfo(self.q.dtype).eps / 2 * out[row, h].abs() * (1 + 2.0 ** -7) + part * weight + 1e-30
                    ltol[row, h] = off + (keep.sum() + 16) * 2.0 ** -24 + 2.0 ** -22 * lse[row, h].abs()
        return out, lse, tol, ltol

    def check(self, got, **kw):
        out, lse, tol, ltol = self.want(**kw)
        o, l = got[0].double().cpu(), got[1].double().cpu()
        rows = out.shape[0]
        assert torch.isfinite(o[:rows]).all()
        worst = ((o[:rows] - out).abs() - tol).max() if rows else torch.tensor(-1.0)
        assert worst <= 0, "out is off by %g more than allowed" % worst
        assert torch.equal(torch.isinf(l[:rows]), torch.isinf(lse)) and not torch.isnan(l[:rows]).any()
        f = torch.isfinite(lse)
        assert ((l[:rows] - lse)[f].abs() <= ltol[f]).all(), "lse"


DECODE = [  # lens, heads, group, dim, page
    ([1], 1, 1, 32, 16), ([33, 0, 7], 2, 4, 128, 16), ([130, 16, 95], 1, 8, 64, 48), ([40], 1, 16, 128, 32),
    ([70, 31], 1, 17, 96, 16), ([200], 1, 3, 80, 16), ([65], 2, 1, 256, 64), ([50, 129], 1, 5, 33, 16),
    ([47], 1, 2, 160, 16), ([90], 1, 2, 192, 48), ([35], 1, 2, 224, 16), ([300], 1, 40, 64, 16)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,heads,group,dim,page", DECODE)
def test_attention_of_single_tokens(lens, heads, group, dim, page, dtype):
    s = Setup(lens, [1] * len(lens), heads, group, dim, page, dtype, seed=dim)
    s.check(s.call(single=True))


@pytest.mark.parametrize("lens,new,heads,group,dim,page,causal", [
    ([40, 19, 64], [3, 1, 5], 1, 4, 64, 16, True), ([40, 19, 0], [3, 0, 0], 2, 2, 128, 16, False),
    ([130, 9], [9, 9], 1, 6, 96, 48, True), ([20, 5], [2, 7], 1, 3, 32, 16, True)])
def test_attention_of_some_tokens(lens, new, heads, group, dim, page, causal):
    """A few rows a request (drafted tokens); rows without any token before them see nothing."""
    s = Setup(lens, new, heads, group, dim, page, seed=3)
    s.check(s.call(causal=causal, max_new=max(new)), causal=causal)
    s.check(s.call(causal=causal), causal=causal, terms=1)       # without the hint


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,new,heads,group,dim,page", [
    ([100, 35, 0, 64], [70, 1, 0, 64], 2, 2, 64, 16), ([150], [101], 1, 4, 128, 48), ([140], [130], 1, 1, 80, 16),
    ([90, 77], [70, 77], 1, 1, 256, 16), ([90], [35], 1, 3, 96, 32), ([80], [80], 1, 1, 33, 16), ([81], [66], 1, 2, 200, 16)])
def test_attention_of_prompt_chunks(lens, new, heads, group, dim, page, dtype):
    """Many rows for some requests, one or none for others."""
    s = Setup(lens, new, heads, group, dim, page, dtype, seed=4)
    s.check(s.call(max_new=max(new)), terms=1 if dtype == torch.bfloat16 else 2)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0])
def test_scales(scale):
    s = Setup([70, 33], [1, 1], 1, 4, 64, 16)
    s.check(s.call(single=True, scale=scale), scale=scale)


@pytest.mark.parametrize("lens,spare", [([700, 3, 0, 1025], 0), ([1500], 40), ([129] * 5 + [900], 100)])
def test_requests_shared_by_workgroups(lens, spare):
    """Tables long enough for the tokens to be shared out over the grid and the parts to be joined."""
    s = Setup(lens, [1] * len(lens), 2, 2, 64, 16, seed=9, spare=spare)
    first = s.call(single=True)
    s.check(first)
    second = s.call(single=True)
    assert torch.equal(first[0], second[0]) and torch.equal(first[1], second[1])


@pytest.mark.parametrize("width_spare", [0, 40])
def test_more_requests_than_a_workgroup_scans(width_spare):
    lens = [(7 * r) % 41 for r in range(290)]
    s = Setup(lens, [1] * 290, 1, 1, 32, 16, seed=10, spare=width_spare)
    s.check(s.call(single=True))
    new = [min(n, r % 3) for r, n in enumerate(lens)]
    s = Setup(lens, new, 1, 1, 32, 16, seed=11, spare=width_spare)
    s.check(s.call(max_new=2))


@pytest.mark.parametrize("new", [1, 40])
def test_tokens_on_missing_pages_are_not_seen(new):
    """Table entries that are negative or beyond the cache, a whole request without pages, lengths beyond the table."""
    s = Setup([100, 64, 50], [new] * 3, 1, 2, 64, 16, seed=12)
    s.table[0, 2], s.table[0, 4], s.table[1] = -1, 2 ** 31 - 1, s.cache.data.shape[0]
    missing = torch.zeros(100, dtype=torch.bool)
    missing[32:48] = missing[64:80] = True
    s.seq[2] = 50
    s.table[2, 3:] = -5
    seen = {0: ~missing, 1: torch.zeros(64, dtype=torch.bool), 2: torch.arange(50) < 48}
    s.check(s.call(max_new=new), seen=lambda r: seen[r], terms=1 if new > 1 else 2)
    # a length that the table cannot hold: the tokens it can name are seen by rows behind them
    t = Setup([48], [1], 1, 2, 64, 16, seed=13)
    t.seq[0] = 1000
    t.check(t.call())
    t.seq[0] = -4
    assert not t.call()[0].any()


@pytest.mark.parametrize("dim,at", [(64, 21), (128, 90)])
def test_a_token_with_nan_reaches_the_rows_that_see_it_only(dim, at):
    """Inf in a value (its block becomes NaN) and in a key: earlier rows of the prompt are untouched."""
    for what in ("v", "k"):
        s = Setup([120], [110], 1, 1, dim, 16, seed=14)
        (s.v if what == "v" else s.k)[0][at, 0, 5] = float("inf")
        kv_append(s.cache, s.k[0].to(DEV), s.v[0].to(DEV), s.slots[0].to(DEV))
        out, lse = (t.cpu() for t in s.call(max_new=110))
        clean = Setup([120], [110], 1, 1, dim, 16, seed=14)
        cout, clse = (t.cpu() for t in clean.call(max_new=110))
        before = at - 10                                          # rows 0 .. see 11 .. tokens
        assert torch.equal(out[:before], cout[:before]) and torch.equal(lse[:before], clse[:before])
        if what == "v":
            assert torch.isnan(out[before:, 0, :32]).all() and torch.equal(out[before:, 0, 32:], cout[before:, 0, 32:])
            assert torch.equal(lse, clse)
        else:
            assert torch.isnan(out[before:]).all() and torch.isnan(lse[before:]).all()


def test_queries_with_inf_or_nan():
    s = Setup([40, 40], [1, 1], 1, 2, 64, 16, seed=15)
    want = s.call(single=True)
    q = s.q.clone()
    q[0, 0, 3] = float("nan")
    q[0, 1, 3] = float("inf")
    out, lse = s.call(q=q.to(DEV), single=True)
    assert torch.isnan(out[0]).all() and torch.isnan(lse[0]).all()
    assert torch.equal(out[1], want[0][1]) and torch.equal(lse[1], want[1][1])


def test_large_scores_and_small_values():
    """Scores of hundreds (the maximum moves by much), values near the ends of the range."""
    s = Setup([150, 37], [1, 1], 1, 2, 64, 16, seed=16, kv_scale=40.0)
    s.check(s.call(single=True))
    s = Setup([70], [1], 1, 2, 64, 16, seed=17, kv_scale=2.0 ** -100)
    s.check(s.call(single=True))


def test_rows_behind_the_last_request_and_given_outputs():
    s = Setup([40, 19], [3, 2], 1, 4, 72, 16, seed=18)
    q = torch.cat([s.q, torch.full((4, 4, 72), float("nan"), dtype=s.q.dtype)]).to(DEV)
    for hint in (3, 200):
        got = s.call(q=q, max_new=hint)
        s.check((got[0][:5], got[1][:5]), terms=1)
        assert not got[0][5:].any() and (got[1][5:] == -math.inf).all()
        out = torch.full((9, 4, 80), 7.0, dtype=s.q.dtype, device=DEV)
        into = out[:, :, 3:75]                                    # rows that are not 16-byte aligned
        res = s.call(q=q, max_new=hint, out=into)
        assert res[0] is into and torch.equal(into[:5], got[0][:5])
        assert (out[5:] == 7).all() and (out[:, :, :3] == 7).all() and (out[:, :, 75:] == 7).all()
    # queries as a slice of a projection, heads before rows
    proj = torch.zeros(4, 5, 145, dtype=s.q.dtype, device=DEV)
    proj[:, :, 73:] = s.q.to(DEV).transpose(0, 1)
    again = s.call(q=proj[:, :, 73:].transpose(0, 1), max_new=3)
    assert torch.equal(again[0], s.call(max_new=3)[0])


def wide_table(new, q_heads, page):
    """Table entries behind the tokens, as of a server with a long context: what a call could read decides whether
    requests with many columns take the prompt kernel, and short ones alone would not."""
    return min(-(-60_000_000 // (sum(new) * q_heads * page)), (1 << 29) // page)


def takes_prompt_kernel(s, hint):
    size = lambda n: _lib.gpu().mxq_kv_attention_workspace_bytes(len(s.lens), s.q.shape[0], s.q.shape[1], n, s.table.shape[1], s.heads,
                                                                 s.page, s.dim, ce._DTYPE[s.q.dtype])
    return size(hint) > size(16 // s.group + 1)                   # parts of prompts and a plan


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,new,heads,group,dim,page,causal", [
    ([100, 35, 0, 64], [70, 1, 0, 64], 2, 2, 64, 16, True), ([150], [101], 1, 4, 128, 48, True), ([140], [130], 1, 1, 80, 16, False),
    ([90, 77], [70, 77], 1, 1, 256, 16, True), ([90, 8], [60, 8], 1, 3, 96, 32, False), ([180, 140], [150, 140], 1, 1, 33, 16, True),
    ([81], [66], 1, 2, 200, 16, True), ([70, 300], [70, 1], 1, 3, 160, 16, True)])
def test_prompt_chunks_in_wide_tables(lens, new, heads, group, dim, page, causal, dtype):
    s = Setup(lens, new, heads, group, dim, page, dtype, seed=4, spare=wide_table(new, heads * group, page))
    assert takes_prompt_kernel(s, max(new))
    first = s.call(max_new=max(new), causal=causal)
    s.check(first, terms=1 if dtype == torch.bfloat16 else 2, causal=causal)
    again = s.call(max_new=max(new), causal=causal)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("scale", [-0.3, 0.0])
def test_scales_of_prompt_chunks_in_wide_tables(scale):
    s = Setup([90, 33], [80, 20], 1, 4, 64, 16, spare=wide_table([100], 4, 16))
    assert takes_prompt_kernel(s, 80)
    s.check(s.call(max_new=80, scale=scale), scale=scale, terms=1)


def test_prompt_chunks_on_missing_pages_in_wide_tables():
    s = Setup([130, 96, 90], [70] * 3, 1, 2, 64, 16, seed=12, spare=wide_table([210], 2, 16))
    assert takes_prompt_kernel(s, 70)
    s.table[0, 2], s.table[0, 4], s.table[1] = -1, 2 ** 31 - 1, s.cache.data.shape[0]
    s.table[2, 3:] = -5
    missing = torch.zeros(130, dtype=torch.bool)
    missing[32:48] = missing[64:80] = True
    seen = {0: ~missing, 1: torch.zeros(96, dtype=torch.bool), 2: torch.arange(90) < 48}
    s.check(s.call(max_new=70), seen=lambda r: seen[r], terms=1)


@pytest.mark.parametrize("dim,at", [(64, 41), (128, 130)])
def test_a_token_with_nan_in_prompt_chunks_in_wide_tables(dim, at):
    for what in ("v", "k"):
        runs = []
        for bad in (False, True):
            s = Setup([180], [170], 1, 1, dim, 16, seed=14, spare=wide_table([170], 1, 16))
            assert takes_prompt_kernel(s, 170)
            if bad:
                (s.v if what == "v" else s.k)[0][at, 0, 5] = float("inf")
                kv_append(s.cache, s.k[0].to(DEV), s.v[0].to(DEV), s.slots[0].to(DEV))
            runs.append([t.cpu() for t in s.call(max_new=170)])
        (cout, clse), (out, lse) = runs
        before = at - 10                                          # rows 0 .. see 11 .. tokens
        assert torch.equal(out[:before], cout[:before]) and torch.equal(lse[:before], clse[:before])
        if what == "v":
            assert torch.isnan(out[before:, 0, :32]).all() and torch.equal(out[before:, 0, 32:], cout[before:, 0, 32:])
            assert torch.equal(lse, clse)
        else:
            assert torch.isnan(out[before:]).all() and torch.isnan(lse[before:]).all()


def test_rows_and_outputs_of_prompt_chunks_in_wide_tables():
    """Rows of no request, outputs that are not aligned, queries as a slice with heads before rows."""
    s = Setup([90, 60, 45], [80, 2, 40], 1, 4, 72, 16, seed=18, spare=wide_table([122], 4, 16))
    assert takes_prompt_kernel(s, 80)
    q = torch.cat([s.q, torch.full((4, 4, 72), float("nan"), dtype=s.q.dtype)]).to(DEV)
    got = s.call(q=q, max_new=80)
    s.check((got[0][:122], got[1][:122]), terms=1)
    assert not got[0][122:].any() and (got[1][122:] == -math.inf).all()
    out = torch.full((126, 4, 80), 7.0, dtype=s.q.dtype, device=DEV)
    res = s.call(q=q, max_new=80, out=out[:, :, 3:75])
    assert torch.equal(res[0][:122], got[0][:122]) and torch.equal(res[1], got[1])
    assert (out[122:] == 7).all() and (out[:, :, :3] == 7).all() and (out[:, :, 75:] == 7).all()
    proj = torch.zeros(4, 122, 145, dtype=s.q.dtype, device=DEV)
    proj[:, :, 73:] = s.q.to(DEV).transpose(0, 1)
    assert torch.equal(s.call(q=proj[:, :, 73:].transpose(0, 1), max_new=80)[0], got[0][:122])
    none, table = torch.zeros(0, dtype=torch.int32, device=DEV), torch.zeros((0, s.table.shape[1]), dtype=torch.int32, device=DEV)
    got, lse = kv_attention(q, s.cache, table, none, torch.zeros(1, dtype=torch.int32, device=DEV), max_new=80, return_lse=True)
    assert not got.any() and (lse == -math.inf).all()


def test_rows_of_no_request():
    """Steps without requests, rows before the first request and behind the last one: zero in a new output, as they were
    in a given one; their lse is -inf in both."""
    s = Setup([40, 19], [3, 2], 1, 4, 72, 16, seed=19)
    q = torch.cat([torch.full((2, 4, 72), float("nan"), dtype=s.q.dtype), s.q, s.q[:3]]).to(DEV)
    starts, want = (s.starts + 2).to(DEV), s.call(max_new=3)
    for hint in (3, 200):
        for out in (None, torch.full_like(q, 7.0)):
            got, lse = kv_attention(q, s.cache, s.table.to(DEV), s.seq.to(DEV), starts, max_new=hint, out=out, return_lse=True)
            rest = torch.cat([got[:2], got[7:]])
            assert (rest == (0 if out is None else 7)).all() and (torch.cat([lse[:2], lse[7:]]) == -math.inf).all()
            if hint == 3:
                assert torch.equal(got[2:7], want[0]) and torch.equal(lse[2:7], want[1])
    none, table = torch.zeros(0, dtype=torch.int32, device=DEV), torch.zeros((0, 100), dtype=torch.int32, device=DEV)
    for hint in (None, 1, 200):
        got, lse = kv_attention(q, s.cache, table, none, torch.zeros(1, dtype=torch.int32, device=DEV), max_new=hint, return_lse=True)
        assert not got.any() and (lse == -math.inf).all()
    got, lse = kv_attention(q[:0], s.cache, table, none, return_lse=True)
    assert got.shape == (0, 4, 72) and lse.shape == (0, 4)
    # requests whose tables have no columns see nothing
    got, lse = s.call(max_new=3)[0] * 0, kv_attention(q[2:7], s.cache, s.table.to(DEV)[:, :0].contiguous(), s.seq.to(DEV), s.starts.to(DEV), return_lse=True)
    assert torch.equal(lse[0], got) and (lse[1] == -math.inf).all()


@pytest.mark.parametrize("starts", [[0, 300, 0, 300, 0, 300], [-5, 300, 7, 2 ** 31 - 1, -2 ** 31, 280], [400, 300, 200, 100, 50, 0]])
@pytest.mark.parametrize("hint,spare", [(1, 30), (300, 30), (300, 60000)])
def test_starts_that_are_not_in_order_stay_in_bounds(starts, hint, spare):
    """Rows named twice get one of the requests' results; nothing outside the tensors and the workspace is written."""
    s = Setup([300, 20, 90, 260, 5], [1] * 5, 1, 4, 32, 16, seed=20, spare=spare)
    q = torch.randn(300, 4, 32, generator=gen(21)).to(s.q.dtype).to(DEV)
    lib, st = _lib.gpu(), torch.tensor(starts, dtype=torch.int32).to(DEV)
    table, seq = s.table.to(DEV), s.seq.to(DEV)
    need = lib.mxq_kv_attention_workspace_bytes(5, 300, 4, hint, table.shape[1], 1, 16, 32, ce._DTYPE[q.dtype])
    pad = 1 << 16
    ws = torch.full((need + 2 * pad,), 0xA5, dtype=torch.uint8, device=DEV)
    out = torch.zeros((302, 4, 32), dtype=q.dtype, device=DEV)
    rc = lib.mxq_kv_attention_mx(q.data_ptr(), 128, 32, out[1:].data_ptr(), 128, 32, None, ce._DTYPE[q.dtype], 300, 4, table.data_ptr(),
                                 table.stride(0), table.shape[1], seq.data_ptr(), st.data_ptr(), 5, 0.2, 1, hint, 0,
                                 s.cache.data.data_ptr(), s.cache.data.shape[0], 1, 16, 32, ws[pad:].data_ptr(), need, None)
    assert rc == 0
    torch.cuda.synchronize()
    assert (ws[:pad] == 0xA5).all() and (ws[pad + need:] == 0xA5).all()
    assert not out[0].any() and not out[-1].any()


def test_refusals():
    s = Setup([20, 20], [1, 1], 2, 2, 64, 16)
    q, t, n = s.q.to(DEV), s.table.to(DEV), s.seq.to(DEV)
    slots = torch.arange(3, device=DEV)
    k = torch.randn(3, 2, 64, device=DEV)
    one = torch.zeros(1, dtype=torch.int32, device=DEV)
    two = torch.zeros(2, dtype=torch.int32, device=DEV)
    bad = [
        lambda: new_kv_cache(4, 20, 2, 64, DEV), lambda: new_kv_cache(4, 16, 2, 257, DEV), lambda: new_kv_cache(0, 16, 2, 64, DEV),
        lambda: kv_append(s.cache._replace(page_size=32), k, k, slots), lambda: kv_append(s.cache, k[:2], k, slots),
        lambda: kv_append(s.cache, k.double(), k.double(), slots), lambda: kv_append(s.cache, k, k.bfloat16(), slots),
        lambda: kv_append(s.cache, k, k, slots.int()), lambda: kv_append(s.cache, k, k, slots[:2]),
        lambda: kv_append(s.cache, k[:, :1], k[:, :1], slots), lambda: kv_append(s.cache, k, k, slots, round="dither"),
        lambda: kv_append(s.cache, k, k, slots, scale_bits=9), lambda: kv_append(s.cache, k, k, slots.repeat(2)[::2]),
        lambda: kv_append(s.cache, k.requires_grad_(True), k, slots), lambda: kv_append(s.cache, k.mT.contiguous().mT, k, slots),
        lambda: kv_read(s.cache, slots.int()), lambda: kv_read(s.cache, slots, torch.float64),
        lambda: kv_read(s.cache._replace(data=s.cache.data[:, :, 1:]), slots),
        lambda: kv_attention(q.float(), s.cache, t, n), lambda: kv_attention(q[:, :3], s.cache, t, n),
        lambda: kv_attention(q, s.cache, t.long(), n), lambda: kv_attention(q, s.cache, t[:1], n),
        lambda: kv_attention(q, s.cache, t, n.long()), lambda: kv_attention(q[:1], s.cache, t, n),
        lambda: kv_attention(q, s.cache, t, n, starts=two), lambda: kv_attention(q, s.cache, t.repeat(1, 2)[:, ::2], n),
        lambda: kv_attention(q, s.cache, t, n, scale=float("nan")), lambda: kv_attention(q, s.cache, t, n, out=q[:1]),
        lambda: kv_attention(q, s.cache, t, n, out=q[:1].expand(2, 4, 64)), lambda: kv_attention(q, s.cache, t, n, out=q.half()),
        lambda: kv_attention(q.detach().clone().requires_grad_(True), s.cache, t, n),
        lambda: kv_block_tables(two, two, t, one, one, 24, 4), lambda: kv_block_tables(two, one, t, one, one, 16, 4),
        lambda: kv_block_tables(two, two, t, one, two, 16, 4), lambda: kv_block_tables(two.long(), two, t, one, one, 16, 4),
        lambda: kv_block_tables(two, two, t, one, one, 16, -1), lambda: kv_block_tables(two, two, t[0], one, one, 16, 4),
    ]
    before = s.cache.data.clone()
    for n_bad, call in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError)):
            call()
            pytest.fail("call %d was not refused" % n_bad)
    assert torch.equal(before, s.cache.data)


def test_calls_with_their_arguments_in_an_array():
    lib = _lib.gpu()
    for which in (-1, 4):
        assert lib.mxq_kv_call(which, bytes(8 * 25), None, 0, None) != 0 and b"unknown call" in lib.mxq_last_error()
    for which in range(4):                                        # zeros are refused by the calls themselves, before any launch
        assert lib.mxq_kv_call(which, None, None, 0, None) != 0
        assert lib.mxq_kv_call(which, bytes(8 * 25), None, 0, None) != 0


# ---- the operators together ------------------------------------------------------------------------------------------
def serve(steps, heads, group, dim, page, capture=False):
    """Requests grow step by step through tables, append and attention; every step's rows against the plain form."""
    R, width, g = 4, 12, gen(21)
    cache = new_kv_cache(40, page, heads, dim, DEV)
    table = torch.full((R, width), -1, dtype=torch.int32, device=DEV)
    free, start = torch.randperm(40, generator=g).int().to(DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    s = Setup([0] * R, [0] * R, heads, group, dim, page)
    s.cache, s.k, s.v = cache, [torch.empty(0, heads, dim).bfloat16() for _ in range(R)], [torch.empty(0, heads, dim).bfloat16() for _ in range(R)]
    for new in steps:
        rows = sum(new) + 2
        k, v = (torch.randn(rows, heads, dim, generator=g).bfloat16() for _ in range(2))
        q = torch.randn(rows, heads * group, dim, generator=g).bfloat16()
        held = torch.tensor(s.lens, dtype=torch.int32, device=DEV)
        t = kv_block_tables(held, torch.tensor(new, dtype=torch.int32, device=DEV), table, free, start, page, rows)
        start = t.free_start
        kv_append(cache, k.to(DEV), v.to(DEV), t.slots)
        got = kv_attention(q.to(DEV), cache, t.block_table, t.seq_lens, t.starts, max_new=max(new), return_lse=True)
        at = 0
        for r, n in enumerate(new):
            s.k[r], s.v[r] = torch.cat([s.k[r], k[at:at + n]]), torch.cat([s.v[r], v[at:at + n]])
            at += n
        s.lens, s.new, s.q = [a + b for a, b in zip(s.lens, new)], new, q[:at]
        s.starts = torch.tensor([0] + new).cumsum(0).int()
        s.check((got[0][:at], got[1][:at]), terms=1)
        assert not got[0][at:].any() and t.slots[at:].tolist() == [-1, -1]


def test_a_run_of_steps():
    serve([[33, 5, 0, 1], [1, 1, 40, 1], [1, 1, 1, 1], [2, 3, 1, 0], [1, 0, 1, 1]], 2, 2, 64, 16)


def test_another_stream():
    s = Setup([300, 45], [1, 1], 2, 4, 128, 16, seed=22, spare=60)
    want = s.call(single=True)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = s.call(single=True)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_captured_steps_replay_with_new_lengths():
    """Two graphs of a whole step over the same cache, replayed in turns with lengths that change in place, the
    program's own eager calls between them; every replay against the eager result."""
    heads, group, dim, page, R = 2, 4, 64, 16, 3
    cache = new_kv_cache(64, page, heads, dim, DEV)
    table = torch.full((R, 16), -1, dtype=torch.int32, device=DEV)
    free = torch.randperm(64, generator=gen(23)).int().to(DEV)
    start, held, new = (torch.zeros(n, dtype=torch.int32, device=DEV) for n in (1, R, R))

    def step(q, k, v):
        t = kv_block_tables(held, new, table, free, start, page, q.shape[0])
        kv_append(cache, k, v, t.slots)
        return kv_attention(q, cache, table, t.seq_lens, t.starts, max_new=4, return_lse=True) + (t.free_start,)

    sets = []
    for seed in (24, 25):
        g = gen(seed)
        sets.append((torch.randn(8, heads * group, dim, generator=g).bfloat16().to(DEV),
                     *(torch.randn(8, heads, dim, generator=g).bfloat16().to(DEV) for _ in range(2))))
    step(*sets[0])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(*x))
        graphs.append(graph)
    cache.data.zero_()
    table.fill_(-1)
    for n in range(6):
        new.copy_(torch.tensor([[1, 3, 4], [4, 0, 1], [2, 2, 2]][n % 3], dtype=torch.int32))
        which = n % 2
        graphs[which].replay()
        got = [t.clone() for t in outs[which]]
        torch.cuda.synchronize()
        eager = step(*sets[which])
        for a, b in zip(got, eager):
            assert torch.equal(a, b)
        held += new
        start.copy_(eager[2])


def test_offsets_beyond_32_bits():
    """A cache of more than 4 GiB: the last pages are written, read and attended to."""
    heads, dim, page = 8, 128, 128
    pages = (1 << 32) // (heads * page * 4 * 34) + 3
    data = torch.empty(pages, heads, page * 4 * 34, dtype=torch.uint8, device=DEV)
    data[-2:] = 0xFF
    data[:2] = 0xFF
    cache = PackedKVCache(data, page, dim)
    s = Setup([150], [1], heads, 1, dim, page, seed=26)
    s.table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32)
    t = torch.arange(150)
    slots = (s.table[0].long()[t // page] * page + t % page).to(DEV)
    kv_append(cache, s.k[0].to(DEV), s.v[0].to(DEV), slots)
    for got, x in zip(kv_read(cache, slots), (s.k[0], s.v[0])):
        assert_bits_equal(got.cpu(), quantized(x), "rows")
    s.cache = cache
    s.check(s.call(single=True))
    assert (data[:2] == 0xFF).all()
