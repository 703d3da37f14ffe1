"""The packed key / value cache at its edges: what the shapes of test_zy_kv_cache.py, whose Setup and tolerances serve here
too, do not reach."""
import math

import pytest
import torch

from microxcaling_amd import _lib
from microxcaling_amd import custom_extensions as ce
from microxcaling_amd.kv_cache import kv_append, kv_attention, kv_read, new_kv_cache
from test_zy_kv_cache import DEV, Setup, gen, takes_prompt_kernel, wide_table

pytestmark = pytest.mark.gpu


# ---- prompt chunks whose output rows are not 16-byte aligned, several items in a workgroup's stretch --------------------
# 64 kv heads of more than 6 blocks share the prompt kernel's 256 workgroups: four stretches a head, and an item has 64
# columns (16 query heads a kv head: four rows).  So 40 rows are 10 items, and two stretches hold an item from its first
# tile to its last between parts of two others.
SEVERAL = [([40], [40], 64, 16, 225, 16, True), ([33, 33, 33, 33], [8, 9, 10, 11], 64, 16, 230, 16, True),
           ([60], [40], 64, 16, 241, 48, False)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,new,heads,group,dim,page,causal", SEVERAL)
def test_rows_of_any_length_with_several_items_in_a_stretch(lens, new, heads, group, dim, page, causal, dtype):
    s = Setup(lens, new, heads, group, dim, page, dtype, seed=30, spare=50)
    assert takes_prompt_kernel(s, max(new))
    s.check(s.call(max_new=max(new), causal=causal), causal=causal, terms=1 if dtype == torch.bfloat16 else 2)


def test_given_outputs_that_are_not_aligned_with_several_items_in_a_stretch():
    s = Setup([40], [40], 64, 16, 256, 16, seed=31, spare=50)
    assert takes_prompt_kernel(s, 40)
    out = torch.full((40, 1024, 264), 7.0, dtype=s.q.dtype, device=DEV)
    got = s.call(max_new=40, out=out[:, :, 3:259])
    s.check(got, terms=1)
    assert (out[:, :, :3] == 7).all() and (out[:, :, 259:] == 7).all()
    want = s.call(max_new=40)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def attention_in_64_bits(q, k, v, scale):
    """(out, lse, a bound on what a kernel may be off by: Setup.want's, with the probabilities as one bf16 term) of one
    request whose rows are its last tokens; k, v as the cache holds them."""
    n, new, H = k.shape[0], q.shape[0], k.shape[1]
    G = q.shape[1] // H
    hidden = torch.arange(n, device=q.device)[None] > torch.arange(n - new, n, device=q.device)[:, None]
    outs, lses, tols, ltols = [], [], [], []
    for h in range(H):
        kh, vh = k[:, h].double(), v[:, h].double()
        for g in range(h * G, h * G + G):
            x = q[:, g].double()
            z = (x @ kh.T * scale).masked_fill_(hidden, -math.inf)
            lse = z.logsumexp(-1)
            top = z.masked_fill_(hidden, 0).abs().amax(-1)
            off = (k.shape[2] + 4) * 2.0 ** -24 * (x.abs() @ kh.abs().T * abs(scale)).amax(-1) + 2.0 ** -22 * (1 + top)
            p = (z - lse[:, None]).exp_().masked_fill_(hidden, 0)
            out = p @ vh
            part = 2 * off + (n + 16) * 2.0 ** -24 + 2.0 ** -8
            outs.append(out)
            lses.append(lse)
            tols.append(torch.finfo(q.dtype).eps / 2 * out.abs() * (1 + 2.0 ** -7) + part[:, None] * (p @ vh.abs()) + 1e-30)
            ltols.append(off + (n + 16) * 2.0 ** -24 + 2.0 ** -22 * lse.abs())
    return (torch.stack(t, 1) for t in (outs, lses, tols, ltols))


@pytest.mark.parametrize("context,new,heads,group,dim,page", [(0, 2048, 8, 4, 100, 16), (700, 4001, 8, 4, 100, 64), (0, 4096, 32, 1, 127, 32)])
def test_long_prompts_with_rows_of_any_length(context, new, heads, group, dim, page):
    """Hundreds of rows in a stretch, at sizes of ordinary prompts (their fp64 result is worked out on the GPU)."""
    n = context + new
    g = torch.Generator(DEV).manual_seed(32)
    k, v = (torch.randn(n, heads, dim, generator=g, device=DEV).bfloat16() for _ in range(2))
    q = torch.randn(new, heads * group, dim, generator=g, device=DEV).bfloat16()
    pages = -(-n // page)
    cache = new_kv_cache(pages + 1, page, heads, dim, DEV)
    table = torch.randperm(pages + 1, generator=gen(33))[None, :pages].int().to(DEV)
    t = torch.arange(n, device=DEV)
    slots = table[0].long()[t // page] * page + t % page
    kv_append(cache, k, v, slots)
    lens, starts = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([n], [0, new]))
    want, lse, tol, ltol = attention_in_64_bits(q, *kv_read(cache, slots), dim ** -0.5)
    wide = torch.empty(new, heads * group, dim + 9, dtype=q.dtype, device=DEV)
    for out in (None, wide[:, :, 5:5 + dim]):
        got, got_lse = kv_attention(q, cache, table, lens, starts, max_new=new, out=out, return_lse=True)
        assert ((got.double() - want).abs() <= tol).all()
        assert ((got_lse.double() - lse).abs() <= ltol).all()


# ---- rows of no request, more of them than the decode kernel has workgroups -----------------------------------------------
def call_into(s, q, out, lse, hint, zero_tail=1, starts=None):
    """The C call with buffers that hold something already."""
    lib, table, seq = _lib.gpu(), s.table.to(DEV), s.seq.to(DEV)
    st = (s.starts if starts is None else starts).to(DEV)
    rows, heads = q.shape[0], q.shape[1]
    need = lib.mxq_kv_attention_workspace_bytes(len(s.lens), rows, heads, hint, table.shape[1], s.heads, s.page, s.dim, ce._DTYPE[q.dtype])
    ws = torch.full((need,), 0xA5, dtype=torch.uint8, device=DEV)
    data = s.cache.data
    rc = lib.mxq_kv_attention_mx(q.data_ptr(), q.stride(0), q.stride(1), out.data_ptr(), out.stride(0), out.stride(1), lse.data_ptr(),
                                 ce._DTYPE[q.dtype], rows, heads, table.data_ptr(), table.stride(0), table.shape[1], seq.data_ptr(),
                                 st.data_ptr(), len(s.lens), s.dim ** -0.5, 1, hint, zero_tail, data.data_ptr(), data.shape[0], s.heads,
                                 s.page, s.dim, ws.data_ptr(), need, None)
    _lib.check(rc, lib)
    torch.cuda.synchronize()


@pytest.mark.parametrize("new,heads,group,dim,before,behind", [(80, 1, 4, 32, 0, 400), (70, 8, 4, 128, 37, 60), (40, 8, 4, 256, 1, 200)])
def test_many_rows_of_no_request_beside_prompt_chunks(new, heads, group, dim, before, behind):
    s = Setup([new], [new], heads, group, dim, 16, seed=34, spare=wide_table([new], heads * group, 16))
    assert takes_prompt_kernel(s, new)
    rows, q_heads = before + new + behind, heads * group
    q = torch.full((rows, q_heads, dim), math.nan, dtype=s.q.dtype)
    q[before:before + new] = s.q
    nobody = torch.ones(rows, dtype=torch.bool)
    nobody[before:before + new] = False
    for zero_tail in (1, 0):
        out, lse = torch.full((rows, q_heads, dim), 7.0, dtype=s.q.dtype, device=DEV), torch.full((rows, q_heads), 7.0, device=DEV)
        call_into(s, q.to(DEV), out, lse, new, zero_tail, s.starts + before)
        assert (out.cpu()[nobody] == (0 if zero_tail else 7)).all()
        assert (lse.cpu()[nobody] == -math.inf).all()
        s.check((out[before:before + new], lse[before:before + new]), terms=1)


# ---- more rows and heads than a launch has workgroups (2^32 threads of 256 a workgroup) -----------------------------------
@pytest.mark.parametrize("rows,heads,group,width,long", [(132000, 1, 128, 65, 600), (131500, 128, 1, 1, 0)])
def test_more_rows_than_a_launch_has_workgroups(rows, heads, group, width, long):
    """Requests that share their pages, most of them short; the last ones, beyond the first launch of the join, long
    enough to be cut.  Or (width 1) more items than workgroups that take a whole one."""
    dim, page = 1, 16
    g = torch.Generator(DEV).manual_seed(35)
    cache = new_kv_cache(width, page, heads, dim, DEV)
    slots = torch.arange(width * page, device=DEV)
    kv_append(cache, *(torch.randn(width * page, heads, dim, generator=g, device=DEV).bfloat16() for _ in range(2)), slots)
    k, v = (t.double()[..., 0] for t in kv_read(cache, slots))                       # (tokens, heads)
    lens = torch.randint(0, 6, (rows,), generator=g, device=DEV, dtype=torch.int32)
    lens[rows - long:] = width * page - 3
    q = torch.randn(rows, heads * group, dim, generator=g, device=DEV).bfloat16()
    table = torch.arange(width, dtype=torch.int32, device=DEV).expand(rows, width).contiguous()
    out, lse = kv_attention(q, cache, table, lens, scale=0.7, out=torch.full_like(q, 7.0), return_lse=True)
    for r0, r1 in ((0, rows - long), (rows - long, rows)):
        n = int(lens[r0:r1].max()) if r1 > r0 else 0
        for a in range(r0, r1, 20000):
            b = min(a + 20000, r1)
            z = q[a:b].double().view(b - a, heads, group, 1) * k[:n].T[None, :, None] * 0.7
            z = z.masked_fill(torch.arange(n, device=DEV) >= lens[a:b, None, None, None], -math.inf)
            want_lse = z.logsumexp(-1)
            p = torch.where(torch.isfinite(want_lse)[..., None], (z - want_lse[..., None]).exp(), 0.0)
            want, weight = ((p * x[:n].T[None, :, None]).sum(-1).view(b - a, -1, 1) for x in (v, v.abs()))
            top = z.masked_fill(z == -math.inf, 0).abs().amax(-1)
            off = (dim + 4) * 2.0 ** -24 * top + 2.0 ** -22 * (1 + top)
            tol = 2.0 ** -8 * want.abs() * (1 + 2.0 ** -7) + (2 * off.view(b - a, -1, 1) + (n + 16) * 2.0 ** -24 + 2.0 ** -16) * weight + 1e-30
            assert ((out[a:b].double() - want).abs() <= tol).all()
            want_lse = want_lse.view(b - a, -1)
            assert torch.equal(torch.isinf(lse[a:b]), torch.isinf(want_lse))
            near = (lse[a:b].double() - want_lse).abs() <= off.view(b - a, -1) + (n + 16) * 2.0 ** -24 + 2.0 ** -22 * want_lse.abs()
            assert (near | torch.isinf(want_lse)).all()


# ---- values whose rounding overflows -------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("prompt,dim,lens,new,at", [(False, 64, [40], [30], 21), (False, 128, [70, 33], [1, 1], 20), (True, 64, [180], [170], 41),
                                                    (True, 160, [150], [140], 130)])
def test_a_value_that_overflows_reaches_the_rows_that_see_it_only(prompt, dim, lens, new, at, dtype):
    """3.3e38 is rounded to 4 * 2^126, which is Inf, as quantize_mx has it.  Rows before the token are untouched, and so are
    the other blocks of the rows that see it."""
    runs = []
    for bad in (False, True):
        s = Setup(lens, new, 1, 2, dim, 16, dtype, seed=36, spare=wide_table(new, 2, 16) if prompt else 0)
        assert takes_prompt_kernel(s, max(new)) == prompt
        if bad:
            s.v[0][at, 0, 37] = 3.3e38
            kv_append(s.cache, s.k[0].to(DEV), s.v[0].to(DEV), s.slots[0].to(DEV))
            assert kv_read(s.cache, s.slots[0][at:at + 1].to(DEV))[1][0, 0, 37] == math.inf
        runs.append([t.cpu() for t in s.call(max_new=max(new))])
    (want, want_lse), (out, lse) = runs
    first = max(0, at - (lens[0] - new[0]))                       # the first row that sees the token
    last = new[0]
    assert torch.equal(lse, want_lse)
    assert torch.equal(out[:first], want[:first]) and torch.equal(out[last:], want[last:])
    assert not torch.isfinite(out[first:last, :, 37]).any()
    others = torch.ones(dim, dtype=torch.bool)
    others[32:64] = False
    assert torch.equal(out[..., others], want[..., others])


# ---- given outputs -------------------------------------------------------------------------------------------------------
def test_outputs_whose_rows_overlap_are_refused():
    s = Setup([20, 20], [1, 1], 2, 2, 64, 16)
    room = torch.zeros(2 * 4 * 64, dtype=s.q.dtype, device=DEV)
    for strides in ((256, 32, 1), (64, 64, 1), (1, 64, 1), (255, 64, 1), (0, 64, 1)):
        with pytest.raises(RuntimeError, match="share memory"):
            s.call(single=True, out=room.as_strided((2, 4, 64), strides))
    want = s.call(single=True)
    for out in (room.view(4, 2, 64).transpose(0, 1), room.as_strided((2, 4, 64), (256, 64, 1)), torch.zeros(4, 3, 70, dtype=s.q.dtype, device=DEV)[:, :2, 1:65].transpose(0, 1)):
        got = s.call(single=True, out=out)
        assert got[0] is out and torch.equal(out, want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("lens,new,heads,group,dim,spare", [([33, 0, 7], [1, 1, 1], 2, 4, 128, 0), ([700, 30], [3, 5], 1, 4, 64, 60), ([90, 33], [80, 33], 1, 4, 64, 6000),
                                                           ([90, 33], [80, 33], 1, 4, 66, 6000)])
def test_the_queries_as_output(lens, new, heads, group, dim, spare):
    """Every result replaces the query it belongs to: one workgroup, shared-out requests, the prompt kernel."""
    s = Setup(lens, new, heads, group, dim, 16, seed=37, spare=spare)
    assert takes_prompt_kernel(s, max(new)) == (spare == 6000)
    want, q = s.call(max_new=max(new)), s.q.to(DEV)
    got = s.call(q=q, max_new=max(new), out=q)
    assert got[0] is q and torch.equal(q, want[0]) and torch.equal(got[1], want[1])


def test_scales_that_are_too_large_are_refused():
    """Scores are taken to base 2: |scale| * log2(e) has to be an fp32 number too."""
    s = Setup([20, 20], [1, 1], 2, 2, 64, 16)
    for scale in (2.4e38, -2.4e38, 3.4e38, 1e39, -math.inf):
        with pytest.raises(RuntimeError, match="scale"):
            s.call(single=True, scale=scale)
    s.check(s.call(single=True, scale=100.0), scale=100.0)


# ---- several rows a request in the decode kernel, whose probabilities are two bf16 terms ----------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,new,heads,group,dim,page,causal,hint", [
    ([100, 35, 0, 64], [70, 1, 0, 64], 2, 2, 64, 16, True, 70), ([150], [101], 1, 4, 128, 48, True, 101), ([140], [130], 1, 1, 80, 16, True, 130),
    ([90, 77], [70, 77], 1, 1, 256, 16, True, 77), ([90], [35], 1, 3, 96, 32, False, 35), ([80], [80], 1, 1, 33, 16, True, 80),
    ([81], [66], 1, 2, 200, 16, True, 66), ([40, 19, 64], [3, 1, 5], 1, 4, 64, 16, True, None), ([130, 9], [9, 9], 1, 6, 96, 48, False, 1),
    ([20, 5], [2, 7], 1, 3, 32, 16, True, None), ([700, 90], [9, 40], 2, 2, 64, 16, True, 4)])
def test_chunks_in_the_decode_kernel_keep_both_terms(lens, new, heads, group, dim, page, causal, hint, dtype):
    """Within 2^-16 of each probability: one term alone is off by up to 2^-8."""
    s = Setup(lens, new, heads, group, dim, page, dtype, seed=38, spare=40 if max(lens) == 700 else 0)
    assert not takes_prompt_kernel(s, sum(new) if hint is None else hint)
    s.check(s.call(causal=causal, max_new=hint), causal=causal, terms=2)


@pytest.mark.parametrize("new", [2, 40])
def test_missing_pages_in_the_decode_kernel_keep_both_terms(new):
    s = Setup([100, 64, 50], [new] * 3, 1, 2, 64, 16, seed=39)
    assert not takes_prompt_kernel(s, new)
    s.table[0, 2], s.table[0, 4], s.table[1] = -1, 2 ** 31 - 1, s.cache.data.shape[0]
    missing = torch.zeros(100, dtype=torch.bool)
    missing[32:48] = missing[64:80] = True
    seen = {0: ~missing, 1: torch.zeros(64, dtype=torch.bool), 2: torch.ones(50, dtype=torch.bool)}
    s.check(s.call(max_new=new), seen=lambda r: seen[r], terms=2)


# ---- the prompt kernel, its plan and its parts in graphs and on streams ----------------------------------------------------
def test_captured_prompt_chunks_replay_with_new_lengths():
    """Two graphs over the same cache, aligned and unaligned rows, padding behind; lengths and starts change in place and the
    program's own calls come between the replays."""
    s = Setup([300, 260], [200, 150], 2, 4, 72, 16, seed=40, spare=wide_table([360], 8, 16))
    assert takes_prompt_kernel(s, 200)
    table, seq, starts = s.table.to(DEV), s.seq.to(DEV), s.starts.to(DEV)
    qs = [torch.randn(400, 8, 72, generator=gen(seed)).bfloat16().to(DEV) for seed in (41, 42)]
    call = lambda n: kv_attention(qs[n], s.cache, table, seq, starts, max_new=200, return_lse=True,
                                  out=None if n == 0 else torch.zeros(400, 8, 80, dtype=torch.bfloat16, device=DEV)[:, :, 3:75])
    call(0), call(1)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for n in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(n))
        graphs.append(graph)
    for step in range(6):
        seq.copy_(torch.tensor([[300, 260], [200, 7], [1, 260]][step % 3], dtype=torch.int32))
        starts.copy_(torch.tensor([[0, 200, 350], [0, 200, 200], [3, 3, 160]][step % 3], dtype=torch.int32))
        graphs[step % 2].replay()
        got = [t.clone() for t in outs[step % 2]]
        torch.cuda.synchronize()
        for a, b in zip(got, call(step % 2)):
            assert torch.equal(a, b)


def test_calls_on_two_streams_at_once():
    sets = [Setup([300, 260], [200, 150], 2, 4, 72, 16, seed=43, spare=wide_table([350], 8, 16)),
            Setup([900, 45, 2000], [1, 3, 2], 2, 4, 128, 16, seed=44, spare=60)]
    args = [(s.q.to(DEV), s.cache, s.table.to(DEV), s.seq.to(DEV), s.starts.to(DEV)) for s in sets]
    want = [kv_attention(*a, max_new=max(s.new), return_lse=True) for a, s in zip(args, sets)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], []
    for _ in range(10):
        for n, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got.append((n, kv_attention(*args[n], max_new=max(sets[n].new), return_lse=True)))
    torch.cuda.synchronize()
    for n, (out, lse) in got:
        assert torch.equal(out, want[n][0]) and torch.equal(lse, want[n][1])
