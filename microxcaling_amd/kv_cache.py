"""A paged key / value cache held in MXFP4, and attention that reads it (include/mxq.h: mxq_kv_*; no counterpart in
the reference, whose attention multiplies whole sequences: mx/bmm.py:20-67, mx/softmax.py:20-88).

    cache = new_kv_cache(num_pages, page_size=16, num_heads=8, head_dim=128, device="cuda")
    step = kv_block_tables(context_lens, new_lens, block_table, free_pages, free_start, 16, num_tokens)
    kv_append(cache, k, v, step.slots)                       # (num_tokens, 8, 128) each
    out = kv_attention(q, cache, block_table, step.seq_lens, step.starts, max_new=1)

Keys and values are quantized along head_dim in blocks of 32 with the arithmetic of pack_mx (fp4_e2m1, 4.25 bits an
element): what kv_read returns is bit for bit what quantize_mx returns for the same rows.  Lengths, tables, slots and
starts stay on the GPU, no call waits for it, and every call can be captured into a graph.  Indexes in those tensors
are checked by the kernels: a slot or a page outside the cache is neither written nor read."""
import struct
from typing import NamedTuple

import torch

from . import _lib
from .custom_extensions import _DTYPE, _flags_value, _stream
from .formats import RoundingMode

MAX_HEAD_DIM = 256
_ROUNDINGS = {name: int(RoundingMode[name]) for name in RoundingMode.string_enums()}
_TOKEN_BYTES = 34                 # K and V of a token, for each block of 32: 2 x (16 bytes of codes + 1 scale)


class PackedKVCache(NamedTuple):
    """data: uint8 (num_pages, num_heads, page_size * ceil(head_dim / 32) * 34), contiguous; the layout of a record is
    described in include/mxq.h.  A slot is page * page_size + place in the page."""
    data: torch.Tensor
    page_size: int
    head_dim: int


class KVBlockTables(NamedTuple):
    """What kv_block_tables returns (rows = its num_tokens)."""
    block_table: torch.Tensor     # the table that was passed, with the new pages entered
    slots: torch.Tensor           # int64 (rows): where each new token goes, -1 for none
    positions: torch.Tensor       # int32 (rows): its position in its request, -1 behind the last request
    requests: torch.Tensor        # int32 (rows): its request, -1 behind the last request
    starts: torch.Tensor          # int32 (requests + 1): first row of each request
    seq_lens: torch.Tensor        # int32 (requests): lengths with the new tokens
    free_start: torch.Tensor      # int32 (1): first free page left; beyond len(free_pages): the list ran out


def _record_bytes(page_size, head_dim):
    return page_size * (-(-head_dim // 32)) * _TOKEN_BYTES


def _check_sizes(page_size, head_dim, who):
    if not 1 <= head_dim <= MAX_HEAD_DIM:
        raise RuntimeError("%s: head_dim must be 1 to %d, got %d" % (who, MAX_HEAD_DIM, head_dim))
    if page_size < 16 or page_size % 16 != 0 or page_size > 65536:
        raise RuntimeError("%s: page_size must be a multiple of 16 up to 65536, got %d" % (who, page_size))


def new_kv_cache(num_pages, page_size, num_heads, head_dim, device="cuda"):
    """A cache of zeros."""
    who = "new_kv_cache"
    _check_sizes(page_size, head_dim, who)
    if num_pages < 1 or num_heads < 1:
        raise RuntimeError("%s: needs at least one page and one head" % who)
    data = torch.zeros((num_pages, num_heads, _record_bytes(page_size, head_dim)), dtype=torch.uint8, device=device)
    return PackedKVCache(data, page_size, head_dim)


def _check_cache(cache, who):
    data, page_size, head_dim = cache
    _check_sizes(page_size, head_dim, who)
    if data.dtype != torch.uint8 or data.dim() != 3 or data.shape[2] != _record_bytes(page_size, head_dim):
        raise RuntimeError("%s: a cache of pages of %d tokens and head_dim %d is uint8 (pages, heads, %d), got %s %s"
                           % (who, page_size, head_dim, _record_bytes(page_size, head_dim), data.dtype, tuple(data.shape)))
    if data.shape[0] < 1 or data.shape[1] < 1:
        raise RuntimeError("%s: the cache needs at least one page and one head" % who)
    if not data.is_contiguous():
        raise RuntimeError("%s: the cache must be contiguous" % who)
    _check_on(data, data, "the cache", who)


def _check_on(t, first, name, who):
    if not t.is_cuda:
        raise RuntimeError("%s: %s must be a CUDA tensor" % (who, name))
    if t.get_device() != first.get_device():
        raise RuntimeError("%s: %s is on %s, not on %s" % (who, name, t.device, first.device))


# (a torch without GPU support lacks the two; its tensors are refused before a call gets to them)
_current_device, _raw_stream = (getattr(torch._C, name, None) for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"))


# mxq_kv_call's numbers of the calls, and their arguments packed as it takes them (a double among the attention's)
_TABLES, _APPEND, _READ, _ATTENTION = range(4)
_tables_args, _append_args, _read_args = (struct.Struct("%dq" % n).pack for n in (17, 18, 10))
_attention_args = struct.Struct("16qd8q").pack


def _call(t, which, args, ws=None, ws_bytes=0):
    """The call on t's device and its current stream.  Where that device is the current one already, as it nearly always
    is, the context of torch.cuda.device and the stream object (3.5 us of a call of 10) are not needed."""
    index = t.get_device()
    if index >= 0 and index == _current_device():
        rc = _lib.gpu().mxq_kv_call(which, args, ws, ws_bytes, _raw_stream(index))
    else:
        with torch.cuda.device(t.device):
            rc = _lib.gpu().mxq_kv_call(which, args, ws, ws_bytes, _stream(t))
    if rc != 0:
        _lib.check(rc, _lib.gpu())


def _check_index(t, shape, dtype, first, name, who):
    """An index tensor: dtype, shape (None: any size), contiguous."""
    if t.dtype != dtype or t.dim() != len(shape) or any(n is not None and n != m for n, m in zip(shape, t.shape)):
        raise RuntimeError("%s: %s must be %s of shape (%s), got %s %s"
                           % (who, name, dtype, ", ".join("any" if n is None else str(n) for n in shape), t.dtype, tuple(t.shape)))
    if not t.is_contiguous():
        raise RuntimeError("%s: %s must be contiguous" % (who, name))
    _check_on(t, first, name, who)


def _check_table(t, first, requests, page_size, who):
    if t.dtype != torch.int32 or t.dim() != 2 or (requests is not None and t.shape[0] != requests):
        raise RuntimeError("%s: block_table must be int32 (requests, pages of a request), got %s %s"
                           % (who, t.dtype, tuple(t.shape)))
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise RuntimeError("%s: the entries of a block_table row must be contiguous, and the rows apart" % who)
    if t.shape[1] * page_size > 1 << 30:
        raise RuntimeError("%s: a row of block_table names too many tokens" % who)
    _check_on(t, first, "block_table", who)


def _check_rows(t, name, who):
    """(rows, heads, head_dim) with contiguous elements."""
    if t.dim() != 3:
        raise RuntimeError("%s: %s must be (rows, heads, head_dim), got %s" % (who, name, tuple(t.shape)))
    if t.shape[2] > 1 and t.stride(2) != 1:
        raise RuntimeError("%s: the elements of a row of %s must be contiguous" % (who, name))


def _check_no_grad(who, *tensors):
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError("%s: has no gradient (the cache holds rounded values): call it under torch.no_grad()" % who)


def _check_block_tables(context_lens, new_lens, block_table, free_pages, free_start, page_size, num_tokens):
    who = "kv_block_tables"
    if page_size < 16 or page_size % 16 != 0 or page_size > 65536:
        raise RuntimeError("%s: page_size must be a multiple of 16 up to 65536, got %d" % (who, page_size))
    if num_tokens < 0 or num_tokens > 0x7FFFFF00:
        raise RuntimeError("%s: bad number of tokens %d" % (who, num_tokens))
    _check_table(block_table, block_table, None, page_size, who)
    R = block_table.shape[0]
    _check_index(context_lens, (R,), torch.int32, block_table, "context_lens", who)
    _check_index(new_lens, (R,), torch.int32, block_table, "new_lens", who)
    _check_index(free_pages, (None,), torch.int32, block_table, "free_pages", who)
    _check_index(free_start, (1,), torch.int32, block_table, "free_start", who)


def kv_block_tables(context_lens, new_lens, block_table, free_pages, free_start, page_size, num_tokens):
    """Pages, slots and positions of a step's new tokens, from the requests' lengths (KVBlockTables).

    Request r has context_lens[r] tokens in the pages of row r of block_table and gets new_lens[r] more (int32,
    negative counts as zero).  The pages it lacks are taken from free_pages (int32) at free_start[0] on (int32, one
    element), in the order of the requests, and entered into block_table in place.  num_tokens is the number of rows
    that the step's tensors have: at least the sum of new_lens, rows behind it are marked -1, so that a padded batch
    keeps its shapes.  Where the free pages or the row of the table end, tokens have slot -1: kv_append leaves them
    out, kv_attention does not see them.  Repeating a call gives the same results; the returned free_start is what the
    next step passes.  (Pages of a finished request go back to the list with free_pages[...] = block_table[r, :n].)"""
    table, R, int32 = block_table.shape, context_lens.numel(), torch.int32
    at = block_table.get_device()
    if not (len(table) == 2 and table[0] == R and context_lens.shape == new_lens.shape == table[:1] and free_start.shape == (1,) and
            free_pages.dim() == 1 and block_table.dtype is int32 and context_lens.dtype is int32 and new_lens.dtype is int32 and
            free_pages.dtype is int32 and free_start.dtype is int32 and block_table.is_cuda and
            at == context_lens.get_device() == new_lens.get_device() == free_pages.get_device() == free_start.get_device() and
            block_table.is_contiguous() and context_lens.is_contiguous() and new_lens.is_contiguous() and free_pages.is_contiguous() and
            page_size % 16 == 0 and 16 <= page_size <= 65536 and 0 <= num_tokens <= 0x7FFFFF00 and table[1] * page_size <= 1 << 30):
        _check_block_tables(context_lens, new_lens, block_table, free_pages, free_start, page_size, num_tokens)
    slots = block_table.new_empty(num_tokens, dtype=torch.int64)
    # the int32 results share one allocation
    ints = block_table.new_empty(2 * num_tokens + 2 * R + 2)
    positions, requests, starts, seq_lens, free_next = ints.split_with_sizes((num_tokens, num_tokens, R + 1, R, 1))
    first = ints.data_ptr()
    _call(block_table, _TABLES, _tables_args(
        context_lens.data_ptr(), new_lens.data_ptr(), block_table.data_ptr(), block_table.stride(0), table[1],
        free_pages.data_ptr(), free_pages.numel(), free_start.data_ptr(), R, page_size, num_tokens, slots.data_ptr(), first,
        first + 4 * num_tokens, first + 8 * num_tokens, first + 8 * num_tokens + 4 * (R + 1),
        first + 8 * num_tokens + 4 * (2 * R + 1)))
    return KVBlockTables(block_table, slots, positions, requests, starts, seq_lens, free_next)


def _check_append(cache, k, v, slots, round):
    who = "kv_append"
    _check_cache(cache, who)
    data, _, head_dim = cache
    for t, name in ((k, "k"), (v, "v")):
        _check_rows(t, name, who)
        _check_on(t, data, name, who)
        if tuple(t.shape[1:]) != (data.shape[1], head_dim):
            raise RuntimeError("%s: %s %s does not fit a cache of %d heads of %d" % (who, name, tuple(t.shape), data.shape[1], head_dim))
    if k.dtype != v.dtype or k.dtype not in _DTYPE:
        raise RuntimeError("%s: k and v must be float32, bfloat16 or float16, both the same (got %s, %s)" % (who, k.dtype, v.dtype))
    if k.shape[0] != v.shape[0]:
        raise RuntimeError("%s: k has %d rows, v has %d" % (who, k.shape[0], v.shape[0]))
    _check_index(slots, (k.shape[0],), torch.int64, data, "slots", who)
    if round not in _ROUNDINGS:
        raise RuntimeError("%s: unknown rounding %r" % (who, round))
    _check_no_grad(who, k, v)


def kv_append(cache, k, v, slots, scale_bits=8, round="nearest", flush_fp32_subnorms=False):
    """Quantizes rows k, v (rows, heads, head_dim; any strides with contiguous elements) as pack_mx does and stores them
    at `slots` (int64, one a row) of the cache, in place.  Rows whose slot is negative or beyond the cache are left out.
    No slot may be named twice in a call: what it would then hold is not defined.  fp16 rows need
    custom_extensions.set_exponent_mode('exact'), as for pack_mx."""
    who = "kv_append"
    data, page_size, head_dim = cache
    at, shape, rows, ks, vs = data.get_device(), data.shape, k.shape, k.stride(), v.stride()
    # one look at what has to hold (2 us less of a call); what is wrong is named by the checks one by one
    if not (len(shape) == 3 and len(rows) == 3 and rows == v.shape and rows[1] == shape[1] and rows[2] == head_dim and
            shape[2] == _record_bytes(page_size, head_dim) and ks[2] == 1 and vs[2] == 1 and slots.shape == rows[:1] and
            k.dtype in _DTYPE and v.dtype is k.dtype and data.dtype is torch.uint8 and slots.dtype is torch.int64 and
            at == k.get_device() == v.get_device() == slots.get_device() and k.is_cuda and data.is_contiguous() and
            slots.is_contiguous() and round in _ROUNDINGS and not (k.requires_grad or v.requires_grad) and
            page_size % 16 == 0 and 16 <= page_size <= 65536 and 1 <= head_dim <= MAX_HEAD_DIM and shape[0] > 0 and shape[1] > 0):
        _check_append(cache, k, v, slots, round)
    _call(data, _APPEND, _append_args(
        k.data_ptr(), v.data_ptr(), _DTYPE[k.dtype], rows[0], ks[0], ks[1], vs[0], vs[1], slots.data_ptr(), data.data_ptr(),
        shape[0], shape[1], page_size, head_dim, scale_bits, 1 if flush_fp32_subnorms else 0, _ROUNDINGS[round], _flags_value()))


def kv_read(cache, slots, dtype=torch.float32):
    """(k, v): the values stored at `slots` (int64), each (rows, heads, head_dim) of `dtype`; zeros for slots outside the
    cache.  A block that held Inf or NaN when it was stored is NaN, as with quantize_mx."""
    data, page_size, head_dim = cache
    sizes, n = data.shape, slots.shape
    if not (len(sizes) == 3 and len(n) == 1 and sizes[2] == _record_bytes(page_size, head_dim) and dtype in _DTYPE and
            data.dtype is torch.uint8 and slots.dtype is torch.int64 and data.get_device() == slots.get_device() and data.is_cuda and
            data.is_contiguous() and slots.is_contiguous() and page_size % 16 == 0 and 16 <= page_size <= 65536 and
            1 <= head_dim <= MAX_HEAD_DIM and sizes[0] > 0 and sizes[1] > 0):
        who = "kv_read"
        _check_cache(cache, who)
        _check_index(slots, (None,), torch.int64, data, "slots", who)
        if dtype not in _DTYPE:
            raise RuntimeError("%s: Tensor dtype not supported (%s)" % (who, dtype))
    shape = (n[0], sizes[1], head_dim)
    k, v = data.new_empty(shape, dtype=dtype), data.new_empty(shape, dtype=dtype)
    _call(data, _READ, _read_args(k.data_ptr(), v.data_ptr(), _DTYPE[dtype], shape[0], slots.data_ptr(), data.data_ptr(), sizes[0],
                                  sizes[1], page_size, head_dim))
    return k, v


def _check_attention(q, cache, block_table, seq_lens, starts, out):
    who = "kv_attention"
    _check_cache(cache, who)
    data, page_size, head_dim = cache
    _check_rows(q, "q", who)
    _check_on(q, data, "q", who)
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise RuntimeError("%s: q must be bfloat16 or float16, got %s" % (who, q.dtype))
    heads = data.shape[1]
    if q.shape[2] != head_dim or q.shape[1] < 1 or q.shape[1] % heads != 0:
        raise RuntimeError("%s: q %s does not fit a cache of %d heads of %d" % (who, tuple(q.shape), heads, head_dim))
    _check_index(seq_lens, (None,), torch.int32, data, "seq_lens", who)
    R = seq_lens.shape[0]
    _check_table(block_table, data, R, page_size, who)
    if starts is not None:
        _check_index(starts, (R + 1,), torch.int32, data, "starts", who)
    elif q.shape[0] != R:
        raise RuntimeError("%s: without starts every request has one row: %d rows, %d requests" % (who, q.shape[0], R))
    if q.shape[0] * q.shape[1] > 0x7FFFFF00:
        raise RuntimeError("%s: q has too many rows" % who)
    _check_no_grad(who, q, *(() if out is None else (out,)))
    if out is not None:
        _check_rows(out, "out", who)
        _check_on(out, data, "out", who)
        if out.shape != q.shape or out.dtype != q.dtype:
            raise RuntimeError("%s: out must be %s %s, got %s %s" % (who, q.dtype, tuple(q.shape), out.dtype, tuple(out.shape)))
        reach = 1                                        # from the narrowest stride to the widest: each passes what is inside it
        for step, n in sorted((step, n) for n, step in zip(out.shape, out.stride()) if n > 1):
            if step < reach:
                raise RuntimeError("%s: rows of out share memory" % who)
            reach += step * (n - 1)


def kv_attention(q, cache, block_table, seq_lens, starts=None, scale=None, causal=True, max_new=None, out=None,
                 return_lse=False):
    """softmax(scale * q K^T) V over the cached tokens of each row's request; q (rows, query heads, head_dim), bf16 or
    fp16, any strides with contiguous elements.  Query head h reads kv head h // (query heads // kv heads).

    seq_lens (int32): tokens of each request, the new ones (already appended) included.  starts (int32, requests + 1):
    request r has the rows starts[r] .. starts[r + 1] - 1, which are its last tokens; None: one row a request.  With
    causal a row sees the tokens up to its own, otherwise all of its request.  Tokens whose page is not in the cache are
    not seen.  NaN or Inf in the cache reaches the rows that see its token (in a value: some or all of its block of 32), no
    others.  A row that sees no token gets zeros (lse -inf).  Rows of no request (before the first one's and behind the
    last one's) are zero in a new output and left as they are in a given `out`; their lse is -inf.  scale defaults to
    head_dim ** -0.5.  out may be q itself, but may not overlap it, or itself, in another way.

    max_new: the most rows that a request has, if known.  A hint: the result is right whatever it is, but it and the table's
    width choose the kernels, and bits and error are theirs.  Accumulation, maxima and sums are fp32 in all of them.  The
    probabilities enter the second product as two bf16 terms (off by up to 2^-17 of each); in the kernel for large chunks with
    bf16 queries as one (2^-8).  return_lse: also the logarithm of the sum of exponentials, fp32 (rows, query heads)."""
    data, page_size, head_dim = cache
    at, shape, table, q_shape, R = data.get_device(), data.shape, block_table.shape, q.shape, seq_lens.numel()
    qs, heads = q.stride(), shape[1] if len(shape) == 3 else 0
    # one look at what has to hold; what is wrong, or only unusual, is for the checks one by one
    if not (out is None and len(q_shape) == 3 and len(table) == 2 and q_shape[2] == head_dim and qs[2] == 1 and
            heads > 0 and shape[0] > 0 and q_shape[1] > 0 and q_shape[1] % heads == 0 and seq_lens.shape == table[:1] and
            shape[2] == _record_bytes(page_size, head_dim) and (q.dtype is torch.bfloat16 or q.dtype is torch.float16) and
            data.dtype is torch.uint8 and seq_lens.dtype is torch.int32 and block_table.dtype is torch.int32 and
            (q_shape[0] == R if starts is None else starts.dtype is torch.int32 and starts.shape == (R + 1,) and
             starts.get_device() == at and starts.is_contiguous()) and
            at == q.get_device() == block_table.get_device() == seq_lens.get_device() and q.is_cuda and data.is_contiguous() and
            block_table.is_contiguous() and seq_lens.is_contiguous() and not q.requires_grad and q_shape[0] * q_shape[1] < 1 << 30 and
            page_size % 16 == 0 and 16 <= page_size <= 65536 and 1 <= head_dim <= MAX_HEAD_DIM and table[1] * page_size <= 1 << 30):
        _check_attention(q, cache, block_table, seq_lens, starts, out)
    scale = head_dim ** -0.5 if scale is None else float(scale)
    new = out is None
    if new:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(q_shape)
    rows, q_heads, width = q_shape[0], q_shape[1], table[1]
    lse = q.new_empty((rows, q_heads), dtype=torch.float32) if return_lse else None
    max_new = (1 if starts is None else rows) if max_new is None else max(1, int(max_new))
    outs = out.stride()
    args = _attention_args(
        q.data_ptr(), qs[0], qs[1], out.data_ptr(), outs[0], outs[1], 0 if lse is None else lse.data_ptr(), _DTYPE[q.dtype], rows, q_heads,
        block_table.data_ptr(), block_table.stride(0), width, seq_lens.data_ptr(), 0 if starts is None else starts.data_ptr(), R, scale,
        1 if causal else 0, max_new, 1 if new else 0, data.data_ptr(), shape[0], heads, page_size, head_dim)
    ws_bytes = _lib.gpu().mxq_kv_attention_args_workspace_bytes(args)
    if ws_bytes:
        ws = data.new_empty(ws_bytes)
        _call(data, _ATTENTION, args, ws.data_ptr(), ws_bytes)
    else:
        _call(data, _ATTENTION, args)
    return (out, lse) if return_lse else out
