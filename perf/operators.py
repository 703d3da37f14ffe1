"""Measured cases of the packed key/value cache: block tables, writing and reading the cache, attention over it.

A cache is one uint8 tensor (pages, kv heads, record).  The record of a page and head holds, for page_size tokens
(a multiple of 16) of NB = ceil(head_dim / 32) blocks of 32 elements,

    K codes   [page_size][NB * 16]          e2m1 nibbles, the lower element in the low nibble
    V codes   [page_size / 4][16][NB][4]    byte (i, b, t): elements 32 b + 2 i (low nibble) and 32 b + 2 i + 1 of token t
    K scales  [page_size][NB]               E8M0
    V scales  [page_size / 4][NB][4]        E8M0

and slot page * page_size + offset names a token's place.  With `own` false, `run` computes everything in elementary
torch operations; with `own` true it makes the calls a user makes."""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---- the cases -------------------------------------------------------------------------------------------------------
def _tables(requests, most_context, most_new, page, **more):
    return dict(op="tables", requests=requests, most_context=most_context, most_new=most_new, page=page, **more)


def _append(tokens, heads, dim, page, dtype, **more):
    return dict(op="append", tokens=tokens, heads=heads, dim=dim, page=page, dtype=dtype, **more)


def _attend(requests, most_context, most_new, heads, group, dim, page, dtype, **more):
    return dict(op="attend", requests=requests, most_context=most_context, most_new=most_new, heads=heads, group=group,
                dim=dim, page=page, dtype=dtype, **more)


def listed():
    return [
        # one decoding step of a large batch: one token a request (a padded one has none), a new page for one in 16
        _tables(256, 8192, 1, 16, name="tables_step"),
        # prompts admitted beside running requests: up to 2048 new tokens each, rows of padding behind them
        _tables(48, 4096, 2048, 64, name="tables_prompts"),
        # keys and values of one decoding step, as one layer writes them
        _append(128, 8, 128, 16, "bf16", name="append_step"),
        # keys and values of a step of prompts
        _append(16384, 8, 128, 64, "bf16", name="append_prompts"),
        # an odd number of tokens and heads, rows that end inside a block of 32, fp32 tensors, pages of 48
        _append(777, 5, 80, 48, "fp32", name="append_odd_fp32"),
        # one request shortly after its start: latency
        _attend(1, 300, 1, 8, 4, 128, 16, "bf16", name="decode_one_short"),
        # an ordinary serving batch: lengths from empty to thousands of tokens
        _attend(64, 8192, 1, 8, 4, 128, 16, "bf16", name="decode_batch"),
        # few requests with a long context: one axis has to be split
        _attend(2, 131072, 1, 8, 8, 128, 64, "bf16", name="decode_long"),
        # every head with its own keys, smaller heads, fp16
        _attend(32, 2048, 1, 12, 1, 64, 32, "fp16", name="decode_own_heads_fp16"),
        # a few drafted tokens for each request, checked at once
        _attend(16, 4096, 5, 4, 6, 96, 48, "bf16", name="drafted_tokens"),
        # a mixed step: prompt chunks of several requests beside short ones
        _attend(4, 4096, 1024, 8, 4, 128, 16, "bf16", name="prompt_chunks"),
        # a long chunk behind a long context
        _attend(1, 12000, 4001, 8, 4, 128, 64, "bf16", name="long_prompt_chunk"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    page = 16 * rng.randint(1, 8)
    kind = rng.choice(["tables", "append", "attend", "attend", "attend"])
    if kind == "tables":
        requests = _spread(rng, 1, 512)
        return _tables(requests, _spread(rng, 1, 16384), min(_spread(rng, 1, 2048), 98304 // requests), page)
    dim = rng.choice([64, 128, 128, rng.randint(8, 256)])
    if kind == "append":
        heads = rng.randint(1, 12)
        return _append(min(_spread(rng, 1, 16384), 16384 * 1024 // (heads * dim)), heads, dim, page, rng.choice(["bf16", "bf16", "fp32"]))
    heads, group, dtype = rng.choice([1, 2, 4, 8, rng.randint(1, 12)]), rng.choice([1, 4, 8, rng.randint(1, 16)]), rng.choice(["bf16", "bf16", "fp16"])
    most_new = rng.choice([1, 1, rng.randint(2, 8), _spread(rng, 9, 2048)])
    blocks = -(-dim // 32)
    # no more than the largest listed cases move and multiply
    requests = _spread(rng, 1, 64)
    if most_new > 8:
        requests = max(1, min(requests, 4096 // most_new))
    room = min(2 * 131072 * 8 * 4 // (requests * heads * blocks), 14000 * 4001 * 32 // (requests * most_new * heads * group))
    return _attend(requests, _spread(rng, 16, max(17, min(131072, room))), most_new, heads, group, dim, page, dtype)


# ---- sizes that follow from a case -----------------------------------------------------------------------------------
def _lengths(case):
    """(tokens held, new tokens) of each request.  Contexts are spread over their logarithm, and one request of a batch
    is a padded one with nothing at all; the requests with short contexts bring the most new tokens."""
    R, top, new = case["requests"], case["most_context"], case["most_new"]
    if R == 1:
        return [top], [new]
    held = [int(round(max(1, top / 64) * (top / max(1, top / 64)) ** (i / (R - 1)))) for i in range(R)]
    fresh = [max(1, int(round(new * (R - i) / R))) for i in range(R)]
    if R > 2:
        held[R // 2], fresh[R // 2] = 0, 0
    return held, fresh


def _blocks(dim):
    return -(-dim // 32)


def _rows(case):
    """Rows of queries or of slots that the call is made with: those of the new tokens and, in a step with several tokens
    a request, some padding behind them."""
    fresh = sum(_lengths(case)[1])
    if case["most_new"] == 1:
        return case["requests"]
    return fresh if case["requests"] == 1 else fresh + 7


# ---- MXFP4 in elementary operations ----------------------------------------------------------------------------------
def _codes(x):
    """(codes 0..15 as (..., NB, 32), E8M0 bytes (..., NB)) of rows x, rounded half away from zero, saturated at 6.  Where
    x has 16 bits, log2 of a block's maximum and the sum with one half are rounded to them: values next to a border go
    where that type's own arithmetic sends them."""
    half = x.dtype == torch.bfloat16
    pad = _blocks(x.shape[-1]) * 32 - x.shape[-1]
    x = torch.nn.functional.pad(x.float(), (0, pad)).unflatten(-1, (-1, 32))
    top = x.abs().amax(-1)
    log = torch.where(top == 0, torch.tensor(2.0 ** -126, dtype=torch.float64, device=x.device), top.double()).log2().float()
    log = log.bfloat16().float() if half else log
    e = (log.floor() - 2).clamp(min=-127)
    scale = torch.exp2(e.double())
    a = (x.abs().double() / scale[..., None])
    p = torch.where(a >= 4, 2.0, torch.where(a >= 2, 1.0, 0.0))
    s = a / torch.exp2(p) * 2 + 0.5
    s = (s.float().bfloat16() if half else s.float()).floor()
    v = (s * torch.exp2(p.float()) / 2).clamp(max=6)
    code = (v > 0.25).to(torch.uint8) + (v > 0.75) + (v > 1.25) + (v > 1.75) + (v > 2.5) + (v > 3.5) + (v > 5)
    return torch.where(x < 0, code + 8, code), (e + 127).to(torch.uint8)


def _value(codes, scales, table):
    """The values that codes (..., 32 a block) and E8M0 bytes (...) stand for, as fp32."""
    factor = torch.exp2(scales.double() - 127).float()
    return table[codes.long()] * torch.where(scales == 255, torch.nan, factor)[..., None]


def _table(device):
    v = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    return torch.tensor(v + [-x for x in v], device=device)


def _pack(k, v, page):
    """Pages (P, H, record) of rows k, v (P, page, H, D)."""
    (kc, ks), (vc, vs) = _codes(k), _codes(v)
    P, S, H, NB = ks.shape
    kc = kc.view(P, S, H, NB * 16, 2)
    kb = (kc[..., 0] | kc[..., 1] << 4).permute(0, 2, 1, 3).reshape(P, H, -1)
    vc = vc.view(P, S // 4, 4, H, NB, 16, 2)
    vb = (vc[..., 0] | vc[..., 1] << 4).permute(0, 3, 1, 5, 4, 2).reshape(P, H, -1)
    sb = ks.permute(0, 2, 1, 3).reshape(P, H, -1)
    tb = vs.view(P, S // 4, 4, H, NB).permute(0, 3, 1, 4, 2).reshape(P, H, -1)
    return torch.cat([kb, vb, sb, tb], -1)


def _unpack(data, page, dim):
    """(K, V) as fp32 (P, H, page, dim) of pages (P, H, record)."""
    P, H, NB = data.shape[0], data.shape[1], _blocks(dim)
    kb, vb, sb, tb = data.split([page * NB * 16, page * NB * 16, page * NB, page * NB], -1)
    table = _table(data.device)
    kc = torch.stack([kb & 15, kb >> 4], -1).view(P, H, page, NB, 32)
    k = _value(kc, sb.reshape(P, H, page, NB), table)
    vb = vb.reshape(P, H, page // 4, 16, NB, 4).permute(0, 1, 2, 5, 4, 3)
    vc = torch.stack([vb & 15, vb >> 4], -1).reshape(P, H, page, NB, 32)
    v = _value(vc, tb.reshape(P, H, page // 4, NB, 4).transpose(-1, -2).reshape(P, H, page, NB), table)
    return k.flatten(-2)[..., :dim], v.flatten(-2)[..., :dim]


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _normal(shape, gen, device, dtype=torch.float32):
    """Activations: normal, with channels of different size."""
    x = torch.randn(shape, generator=gen, device=device)
    gain = torch.exp(0.5 * torch.randn(shape[-1], generator=gen, device=device))
    return (x * gain).to(dtype)


def _tables_of(held, page, width, pages, gen, device):
    """A table in which every request holds the pages of its tokens, and the pages that nobody holds, in random order."""
    R = len(held)
    need = (held + page - 1) // page
    order = torch.randperm(pages, generator=gen, device=device).int()
    at = torch.arange(width, device=device)
    first = need.cumsum(0) - need
    mine = at[None] < need[:, None]
    table = torch.where(mine, order[(first[:, None] + at[None]).clamp(max=pages - 1)], -1).int()
    return table.contiguous(), order, int(sum(-(-int(h) // page) for h in held.tolist()))


def prepare(case, seed):
    device = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    gen = torch.Generator(device=device).manual_seed(seed)
    state = {"case": case}
    if case["op"] == "append":
        T, H, D, S = case["tokens"], case["heads"], case["dim"], case["page"]
        pages = -(-T // S) + 3
        # projections of queries, keys and values are one tensor: keys and values are slices of it
        both = _normal((T, 2, H, D), gen, device, _TYPES[case["dtype"]])
        slots = torch.randperm(pages * S, generator=gen, device=device)[:T]
        if T > 4:
            slots[T // 2] = -1  # a row of padding
        data = torch.zeros(pages, H, S * _blocks(D) * 34, dtype=torch.uint8, device=device)
        return dict(state, k=both[:, 0], v=both[:, 1], slots=slots, data=data)
    held, fresh = _lengths(case)
    order = torch.randperm(case["requests"], generator=gen, device=device)
    held, fresh = (torch.tensor(x, device=device)[order] for x in (held, fresh))
    S = case["page"]
    width = -(-(case["most_context"] + case["most_new"]) // S) + 1
    if case["op"] == "tables":
        pages = int(sum(-(-(int(h) + int(n)) // S) for h, n in zip(held.tolist(), fresh.tolist()))) + 5
        table, order, used = _tables_of(held, S, width, pages, gen, device)
        free = order[used:].contiguous()
        return dict(state, held=held.int(), fresh=fresh.int(), table=table, free=free,
                    free_start=torch.zeros(1, dtype=torch.int32, device=device))
    H, G, D = case["heads"], case["group"], case["dim"]
    pages = int(sum(-(-(int(h) + int(n)) // S) for h, n in zip(held.tolist(), fresh.tolist()))) + 2
    table, _, _ = _tables_of(held + fresh, S, width, pages, gen, device)
    data = torch.empty(pages, H, S * _blocks(D) * 34, dtype=torch.uint8, device=device)
    step = max(1, (1 << 25) // (S * H * D))
    for at in range(0, pages, step):
        n = min(step, pages - at)
        data[at:at + n] = _pack(_normal((n, S, H, D), gen, device), _normal((n, S, H, D), gen, device), S)
    q = _normal((_rows(case), H * G, D), gen, device, _TYPES[case["dtype"]])
    starts = torch.cat([fresh.new_zeros(1), fresh.cumsum(0)]).int()
    single = case["most_new"] == 1
    if single:  # one row a request, also for a request of padding
        starts = None
    return dict(state, q=q, data=data, table=table, seq_lens=(held + fresh).int(), starts=starts, scale=D ** -0.5)


# ---- one pass --------------------------------------------------------------------------------------------------------
def _plain_tables(s):
    held, fresh, table, free, S = s["held"].long(), s["fresh"].long(), s["table"], s["free"], s["case"]["page"]
    R, width, rows = held.numel(), table.shape[1], _rows(s["case"])
    first, last = (held + S - 1) // S, ((held + fresh + S - 1) // S).clamp(max=width)
    need = (last - first).clamp(min=0)
    from_ = s["free_start"].long() + need.cumsum(0) - need
    at = torch.arange(width, device=held.device)[None]
    pick = from_[:, None] + at - first[:, None]
    page = torch.where(pick < free.numel(), free[pick.clamp(0, max(0, free.numel() - 1))], -1)
    table.copy_(torch.where((at >= first[:, None]) & (at < last[:, None]), page, table))
    ends = fresh.cumsum(0)
    row = torch.arange(rows, device=held.device)
    r = (row[:, None] >= ends[None]).sum(1)
    live = r < R
    q = r.clamp(max=R - 1)
    pos = held[q] + row - (ends - fresh)[q]
    page = table[q, (pos // S).clamp(max=width - 1)].long()
    slot = torch.where(live & (page >= 0) & (pos // S < width), page * S + pos % S, -1)
    none = torch.tensor(-1, device=held.device)
    starts = torch.cat([ends.new_zeros(1), ends]).int()
    return {"table": table, "slots": slot, "positions": torch.where(live, pos, none).int(), "requests": torch.where(live, r, none).int(),
            "starts": starts, "seq_lens": (held + fresh).int(), "free_start": (s["free_start"] + need.sum()).int()}


def _plain_append(s):
    k, v, slots, data = s["k"], s["v"], s["slots"], s["data"]
    S, D = s["case"]["page"], s["case"]["dim"]
    P, H, _ = data.shape
    NB = _blocks(D)
    live = slots >= 0
    at = slots.clamp(min=0)
    page, off = at // S, at % S
    (kc, ks), (vc, vs) = _codes(k), _codes(v)
    T = k.shape[0]
    kb = kc.view(T, H, NB * 16, 2)
    kb = kb[..., 0] | kb[..., 1] << 4
    vb = vc.view(T, H, NB, 16, 2)
    vb = (vb[..., 0] | vb[..., 1] << 4).transpose(-1, -2).reshape(T, H, NB * 16)
    n = torch.arange(NB * 16, device=k.device)
    m = torch.arange(NB, device=k.device)
    base = (page[:, None] * H + torch.arange(H, device=k.device)) * data.shape[2]
    o, tile, t = off[:, None, None], (off // 4)[:, None, None], (off % 4)[:, None, None]
    where = torch.cat([o * NB * 16 + n, S * NB * 16 + (tile * NB * 16 + n) * 4 + t,
                       S * NB * 32 + o * NB + m, S * NB * 33 + (tile * NB + m) * 4 + t], -1) + base[..., None]
    flat = data.view(-1)
    flat[where[live].view(-1)] = torch.cat([kb, vb, ks, vs], -1)[live].view(-1)
    got = flat[where.view(-1)].view(T, H, -1)  # and back again
    kb, vb, ks, vs = got.split([NB * 16, NB * 16, NB, NB], -1)
    table = _table(k.device)
    kq = _value(torch.stack([kb & 15, kb >> 4], -1).view(T, H, NB, 32), ks, table)
    vb = vb.view(T, H, 16, NB).transpose(-1, -2)
    vq = _value(torch.stack([vb & 15, vb >> 4], -1).view(T, H, NB, 32), vs, table)
    keep = live[:, None, None]
    return tuple(torch.where(keep, x.flatten(-2)[..., :D], 0.0) for x in (kq, vq))


def _plain_attend(s):
    case, q, seq = s["case"], s["q"], s["seq_lens"].long()
    H, G, D, S = case["heads"], case["group"], case["dim"], case["page"]
    R, N, rows = case["requests"], case["most_new"], q.shape[0]
    L = -(-(case["most_context"] + N) // S) * S
    table = s["table"][:, :L // S].long().clamp(min=0)
    k, v = _unpack(s["data"], S, D)
    k, v = (x[table].transpose(1, 2).reshape(R, H, L, D) for x in (k, v))
    if s["starts"] is None:
        start, new = torch.arange(R, device=q.device), torch.ones(R, dtype=torch.long, device=q.device)
    else:
        start = s["starts"][:-1].long()
        new = s["starts"][1:].long() - start
    i = torch.arange(N, device=q.device)
    row = (start[:, None] + i).clamp(max=rows - 1)
    x = q[row].float().view(R, N, H, G, D).permute(0, 2, 3, 1, 4).reshape(R * H, G * N, D)
    score = torch.bmm(x, k.reshape(R * H, L, D).transpose(1, 2)).mul_(s["scale"]).view(R, H, G, N, L)
    sees = (seq - new)[:, None] + i + 1  # keys that the i-th new token sees
    score.masked_fill_(torch.arange(L, device=q.device) >= sees[:, None, None, :, None], -torch.inf)
    top = score.amax(-1, keepdim=True)
    safe = torch.where(top == -torch.inf, 0.0, top)
    p = score.sub_(safe).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.bmm(p.view(R * H, G * N, L), v.reshape(R * H, L, D)).view(R, H, G, N, D) / torch.where(total == 0, 1.0, total)
    lse = (safe + total.log()).squeeze(-1)
    out = torch.zeros(rows + 1, H * G, D, device=q.device)
    lses = torch.full((rows + 1, H * G), -torch.inf, device=q.device)
    to = torch.where(i < new[:, None], start[:, None] + i, rows).view(-1)
    out[to] = o.permute(0, 3, 1, 2, 4).reshape(R * N, H * G, D)
    lses[to] = lse.permute(0, 3, 1, 2).reshape(R * N, H * G)
    return out[:rows].to(q.dtype), lses[:rows]


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"tables": _plain_tables, "append": _plain_append, "attend": _plain_attend}[op](state)
    from microxcaling_amd import kv_cache
    case = state["case"]
    if op == "tables":
        t = kv_cache.kv_block_tables(state["held"], state["fresh"], state["table"], state["free"], state["free_start"],
                                     case["page"], _rows(case))
        return {"table": t.block_table, "slots": t.slots, "positions": t.positions, "requests": t.requests,
                "starts": t.starts, "seq_lens": t.seq_lens, "free_start": t.free_start}
    cache = kv_cache.PackedKVCache(state["data"], case["page"], case["dim"])
    if op == "append":
        kv_cache.kv_append(cache, state["k"], state["v"], state["slots"])
        return kv_cache.kv_read(cache, state["slots"])
    return kv_cache.kv_attention(state["q"], cache, state["table"], state["seq_lens"], state["starts"], scale=state["scale"],
                                 max_new=case["most_new"], return_lse=True)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    if case["op"] == "append":
        T, H, D = case["tokens"], case["heads"], case["dim"]
        rows = T * H
        return {"bytes": rows * (2 * D * _SIZES[case["dtype"]] + 2 * 34 * _blocks(D) + 2 * 4 * D) + 8 * T, "flops": 0}
    held, fresh = _lengths(case)
    S, R = case["page"], case["requests"]
    if case["op"] == "tables":
        new_pages = sum(-(-(h + n) // S) - -(-h // S) for h, n in zip(held, fresh))
        width = -(-(case["most_context"] + case["most_new"]) // S) + 1
        touched = min(R * width, sum(-(-(h + n) // S) - h // S for h, n in zip(held, fresh)))
        return {"bytes": 8 * R + 4 * touched + 8 * new_pages + 16 * _rows(case) + 8 * R + 12, "flops": 0}
    H, G, D, NB = case["heads"], case["group"], case["dim"], _blocks(case["dim"])
    if case["most_new"] == 1:
        fresh_rows = [1] * R
        sees = [h + n for h, n in zip(held, fresh)]
    else:
        fresh_rows = fresh
        sees = [n * h + n * (n + 1) // 2 for h, n in zip(held, fresh)]
    tokens = sum(h + n for h, n in zip(held, fresh))
    rows = sum(fresh_rows)
    return {"bytes": tokens * H * NB * 34 + rows * H * G * (D * 4 + 4) + 4 * sum(-(-(h + n) // S) for h, n in zip(held, fresh)) + 4 * R,
            "flops": 4 * H * G * D * sum(sees)}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------
def _exact_rounded(x):
    """MXFP4 values of rows x as fp64, from the nearest of the fifteen values of e2m1."""
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    edges = (grid[1:] + grid[:-1]) / 2  # half away from zero: a border belongs to the upper value
    half = x.dtype == torch.bfloat16
    D = x.shape[-1]
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for at in range(0, D, 32):
        b = x[..., at:at + 32].double()
        top = b.abs().amax(-1, keepdim=True)
        log = torch.where(top == 0, 2.0 ** -126, top).log2()
        log = log.bfloat16().double() if half else log.float().double()
        scale = 2.0 ** torch.clamp(log.floor() - 2, min=-127)
        a = b.abs() / scale
        # bfloat16 has no value between the last one below the first border, 0.25 - 2^-10, plus a border and two borders
        a = torch.where((a == 0.25 - 2.0 ** -10) & half, 0.25, a)
        out[..., at:at + 32] = grid[torch.bucketize(a.contiguous(), edges, right=True)] * b.sign() * scale
    return out


def _exact_rows(data, page, dim, slots, head):
    """(K, V) of the tokens at `slots` of one head, fp64, byte by byte."""
    NB = _blocks(dim)
    value = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64, device=data.device)
    record = data[:, head].reshape(-1)
    base, off = slots // page * data.shape[2], slots % page
    d = torch.arange(dim, device=data.device)
    block, shift = d // 32, (d % 2 * 4)[None]
    kb = record[(base + off * NB * 16)[:, None] + (d // 2)[None]]
    ks = record[(base + page * NB * 32 + off * NB)[:, None] + block[None]]
    quad, lane = off // 4, off % 4
    vb = record[(base + page * NB * 16 + quad * NB * 64 + lane)[:, None] + ((d % 32 // 2) * NB * 4 + block * 4)[None]]
    vs = record[(base + page * NB * 33 + quad * NB * 4 + lane)[:, None] + (block * 4)[None]]
    return tuple(value[(c.long() >> shift) & 15] * 2.0 ** (e.double() - 127) for c, e in ((kb, ks), (vb, vs)))


def exact(case, seed):
    if case["op"] == "tables":
        return None
    s = prepare(case, seed)
    if case["op"] == "append":
        live = (s["slots"] >= 0).double()[:, None, None]
        return _exact_rounded(s["k"]) * live, _exact_rounded(s["v"]) * live
    H, G, D, S = case["heads"], case["group"], case["dim"], case["page"]
    q, rows = s["q"], s["q"].shape[0]
    out = torch.zeros(rows, H * G, D, dtype=torch.float64, device=q.device)
    lse = torch.full((rows, H * G), -math.inf, dtype=torch.float64, device=q.device)
    lens = s["seq_lens"].tolist()
    starts = s["starts"].tolist() if s["starts"] is not None else list(range(len(lens) + 1))
    for r, n in enumerate(lens):
        a, b = starts[r], starts[r + 1]
        if n == 0 or a == b:
            continue
        t = torch.arange(n, device=q.device)
        slots = s["table"][r].long()[t // S] * S + t % S
        hidden = t[None] > (n - (b - a) + torch.arange(b - a, device=q.device))[:, None]
        for h in range(H):
            k, v = _exact_rows(s["data"], S, D, slots, h)
            for g in range(h * G, h * G + G):
                z = (q[a:b, g].double() @ k.T * s["scale"]).masked_fill(hidden, -math.inf)
                lse[a:b, g] = z.logsumexp(-1)
                out[a:b, g] = (z - lse[a:b, g, None]).exp() @ v
    return out, lse
