// C ABI of libmxq_gfx950.so, continued: the paged MXFP4 key / value cache.
#include <cstring>

#include "mxq_capi_kv.h"
#include "mxq_kv_rows.h"

namespace mxq_kv {
void launch_decode(int dtype, const void* args, const Plan& p, hipStream_t s);
void launch_prompt(int dtype, const void* args, const Plan& p, hipStream_t s);
void launch_join(int dtype, const void* args, const Plan& p, hipStream_t s);
}  // namespace mxq_kv

namespace {

using mxq_kv::Plan;

// tokens that a table row may name: positions stay far from the end of int32
constexpr int64_t kMaxTokens = (int64_t)1 << 30;

int make_cache(void* data, int64_t num_pages, int heads, int page_size, int head_dim, KvCache* c, const char* who) {
    if (head_dim < 1 || head_dim > 32 * KV_MAX_NB)
        return fail(MXQ_ERR_ARGUMENT, "%s: head_dim must be 1 to %d, got %d", who, 32 * KV_MAX_NB, head_dim);
    if (page_size < 16 || page_size % 16 != 0 || page_size > 65536)
        return fail(MXQ_ERR_ARGUMENT, "%s: page_size must be a multiple of 16 up to 65536, got %d", who, page_size);
    if (heads < 1 || heads > 65535) return fail(MXQ_ERR_ARGUMENT, "%s: bad number of heads %d", who, heads);
    if (num_pages < 1 || num_pages > 0x7FFFFFFF) return fail(MXQ_ERR_ARGUMENT, "%s: the cache has no pages, or too many", who);
    if (!data) return fail(MXQ_ERR_ARGUMENT, "%s: null pointer", who);
    if (!aligned16(data)) return fail(MXQ_ERR_ARGUMENT, "%s: the cache must be 16-byte aligned", who);
    c->data = reinterpret_cast<unsigned char*>(data);
    c->num_pages = num_pages;
    c->heads = heads;
    c->page_size = page_size;
    c->head_dim = head_dim;
    c->nb = (head_dim + 31) / 32;
    c->record = (int64_t)page_size * c->nb * KV_TOKEN_BYTES;
    c->by_page = kv_divide((uint32_t)page_size);
    int64_t total;
    if (mul_overflows(num_pages, heads, c->record, &total)) return fail(MXQ_ERR_ARGUMENT, "%s: size overflows int64", who);
    return MXQ_OK;
}

template <int DT, int RMODE, bool ZE, bool LEAN>
struct LaunchAppend {
    static void run(KvRowsArgs a, MxParams p, uint32_t max_code, int grid, hipStream_t s) {
        kv_append_kernel<DT, RMODE, ZE><<<grid, kThreads, 0, s>>>(a, p, max_code);
    }
};

// workgroups of the row kernels: each has 16 of the units (head, K or V, block) of a group of four tokens and goes through
// the groups; enough of them to fill the chip
int rows_grid(const KvCache& c, int64_t tokens) {
    const int64_t unit_blocks = ceil_div((int64_t)c.heads * 2 * c.nb, 16), quads = ceil_div(tokens, 4);
    const int64_t most = ceil_div(kMaxBlocks, unit_blocks);
    return (int)(unit_blocks * (quads < most ? quads : most));
}

// Which kernels a call runs, and with what shares.  max_new: tokens that a request brings at most (a hint: every
// choice made with it is right for any number).  room: tokens that a table row can name.  It stands for the lengths, which
// the host does not know: short prompts in wide tables take the prompt kernel too.  What is measured here is bf16.
Plan make_plan(int64_t requests, int64_t rows, int group, int64_t max_new, int64_t room, int heads, int nb, int terms) {
    Plan p;
    p.nb = nb;
    if (max_new > rows) max_new = rows;
    if (max_new < 1) max_new = 1;
    const int64_t columns = max_new * group;
    const int most_ct = kv_decode_most_ct(nb, terms);
    // 30 columns of 96 with two tiles of them for each reading of the tokens 35.9 us, with one 42.6 (16 requests of 4096)
    p.ct = columns <= 16 ? 1 : most_ct;
    // The prompt kernel multiplies at up to four times the decode kernel's rate, but takes a plan and a join of many
    // columns, 20 us of launches.  8 x 4 heads of 128, us with decode and prompt kernel: 4 requests of 2048 with 128, 192,
    // 256, 384 columns each 32 : 42, 40 : 45, 47 : 48, 62 : 54; 16 of them with 128 and 192 51 : 62, 92 : 67; one of 4096
    // with 512 39 : 53; one of 16384 with 256 48 : 69; new prompts alone, 512 tokens 18 : 39, 1024 60 : 59.
    const double work = (double)rows * group * heads * (room + 3 * KV_UNIT) * (2.0 / most_ct);
    p.prompt = columns > 64 * most_ct && work > 28e6;
    p.decode_columns = p.prompt ? 64 * most_ct : 0x7FFFFFFF;
    const int64_t units = ceil_div(room, KV_UNIT) > 0 ? ceil_div(room, KV_UNIT) : 1;
    p.decode_items = rows * group / (16 * p.ct) + (requests > 0 ? requests : 1);
    // A workgroup for each item, and no join: 32 requests of 500, 760, 1000, 1500 tokens (8 x 4 heads of 128) 11.3, 13.7, 16.3,
    // 20.7 us, against 16.6, 17.0, 19.3, 21.8 with the units dealt out; 8 requests 12.2, 13.9, 17.7 against 13.0, 13.9, 14.9
    // from 760 on; one request 10.5, 12.1, 13.7 against 11.5, 11.7, 11.7.
    p.whole = (units <= 4 || (units <= 8 && requests * heads >= 64)) && p.decode_items * heads < mxq_kv::kMostWorkgroups;
    const int64_t chip = 256 * kv_decode_waves(nb, p.ct, terms);
    p.shares = ceil_div(chip, heads) < KV_MAX_SHARES ? ceil_div(chip, heads) : KV_MAX_SHARES;
    if (p.shares > p.decode_items * units) p.shares = p.decode_items * units;
    const int64_t cols = 64 * kv_prompt_ct(nb, terms);
    p.prompt_items = rows * group / cols + (requests > 0 ? requests : 1);
    p.prompt_shares = 256 * (nb <= 4 ? 2 : 1) / heads > 1 ? 256 * (nb <= 4 ? 2 : 1) / heads : 1;
    return p;
}

// pieces of the workspace, each a multiple of 16 bytes
int64_t decode_part_bytes(const Plan& p, int heads) {
    return p.whole ? 0 : p.shares * heads * 2 * (16 * p.ct) * (32 * p.nb + 2) * (int64_t)sizeof(float);
}
int64_t span_bytes(const Plan& p) { return p.whole ? 0 : ceil_div(p.decode_items, 2) * 16; }
int64_t prompt_part_bytes(const Plan& p, int heads, int terms) {
    return p.prompt ? p.prompt_shares * heads * 2 * (64 * kv_prompt_ct(p.nb, terms)) * (32 * p.nb + 2) * (int64_t)sizeof(float) : 0;
}
int64_t part_bytes(const Plan& p, int heads, int terms, int64_t requests) {
    return decode_part_bytes(p, heads) + span_bytes(p) + prompt_part_bytes(p, heads, terms) +
           (p.prompt ? kv_plan_bytes(p.prompt_items, p.prompt_shares, requests) : 0);
}

}  // namespace

#pragma GCC visibility push(default)
extern "C" {

int mxq_kv_block_tables(const int* context_lens, const int* new_lens, int* block_table, int64_t table_stride, int64_t width,
                        const int* free_pages, int64_t free_count, const int* free_start, int64_t requests, int page_size,
                        int64_t tokens, int64_t* slots, int* positions, int* owners, int* starts, int* seq_lens,
                        int* free_next, void* hip_stream) {
    const char* who = "mxq_kv_block_tables";
    if (requests < 0 || width < 0 || free_count < 0 || tokens < 0) return fail(MXQ_ERR_ARGUMENT, "%s: negative size", who);
    if (page_size < 16 || page_size % 16 != 0 || page_size > 65536)
        return fail(MXQ_ERR_ARGUMENT, "%s: page_size must be a multiple of 16 up to 65536, got %d", who, page_size);
    if (requests > 0x7FFFFF00 || tokens > 0x7FFFFF00) return fail(MXQ_ERR_ARGUMENT, "%s: size too large", who);
    if (width * page_size > kMaxTokens) return fail(MXQ_ERR_ARGUMENT, "%s: a table row names too many tokens", who);
    if (requests > 0 && (!context_lens || !new_lens || !seq_lens || (width > 0 && !block_table)))
        return fail(MXQ_ERR_ARGUMENT, "%s: null pointer", who);
    if ((free_count > 0 && !free_pages) || !free_start || !free_next || !starts ||
        (tokens > 0 && (!slots || !positions || !owners)))
        return fail(MXQ_ERR_ARGUMENT, "%s: null pointer", who);
    KvTablesArgs a;
    a.context = context_lens;
    a.fresh = new_lens;
    a.table = block_table;
    a.table_stride = table_stride;
    a.width = (int)width;
    a.free_pages = free_pages;
    a.free_count = free_count;
    a.free_start = free_start;
    a.requests = (int)requests;
    a.page_size = page_size;
    a.tokens = tokens;
    a.slots = slots;
    a.positions = positions;
    a.owners = owners;
    a.starts = starts;
    a.seq_lens = seq_lens;
    a.free_next = free_next;
    const int64_t grid = ceil_div(tokens, KV_TABLE_TOKENS) > 0 ? ceil_div(tokens, KV_TABLE_TOKENS) : 1;
    kv_block_tables_kernel<KV_TABLE_TOKENS><<<(unsigned)grid, kThreads, 0, (hipStream_t)hip_stream>>>(a);
    return check_launch(who);
}

int mxq_kv_append_mx(const void* k, const void* v, int dtype, int64_t tokens, int64_t k_token_stride, int64_t k_head_stride,
                     int64_t v_token_stride, int64_t v_head_stride, const int64_t* slots, void* cache, int64_t num_pages,
                     int heads, int page_size, int head_dim, int scale_bits, int flush_fp32_subnorms, int rmode, int flags,
                     void* hip_stream) {
    const char* who = "mxq_kv_append_mx";
    if (f16_ops(dtype, flags))
        return fail(MXQ_ERR_ARGUMENT, "%s: fp16 tensors have a packed form under MXQ_FLAG_EXACT_EXPONENT only "
                    "(the op-by-op fp16 arithmetic of the default mode has no packing kernel)", who);
    MxParams p;
    bool ze;
    int rc = make_mx_params(dtype, scale_bits, 2, 3, 6.0f, flush_fp32_subnorms, rmode, flags, &p, &ze, who);
    if (rc) return rc;
    KvRowsArgs a;
    rc = make_cache(cache, num_pages, heads, page_size, head_dim, &a.c, who);
    if (rc) return rc;
    if (tokens < 0) return fail(MXQ_ERR_ARGUMENT, "%s: negative size", who);
    if (tokens == 0) return MXQ_OK;
    if (!k || !v || !slots) return fail(MXQ_ERR_ARGUMENT, "%s: null pointer", who);
    a.k = k;
    a.v = v;
    a.k_token = k_token_stride;
    a.k_head = k_head_stride;
    a.v_token = v_token_stride;
    a.v_head = v_head_stride;
    a.slots = slots;
    a.tokens = tokens;
    const int per16 = 16 / elem_size(dtype);             // elements in 16 bytes
    a.wide = aligned16(k) && aligned16(v) && head_dim % 8 == 0 && k_token_stride % per16 == 0 && k_head_stride % per16 == 0 &&
             v_token_stride % per16 == 0 && v_head_stride % per16 == 0;
    dispatch<LaunchAppend>(dtype, rmode, ze, true, a, p, mxq_max_code(p.fmt), rows_grid(a.c, tokens), (hipStream_t)hip_stream);
    return check_launch(who);
}

int mxq_kv_read_mx(void* k, void* v, int dtype, int64_t tokens, const int64_t* slots, const void* cache, int64_t num_pages,
                   int heads, int page_size, int head_dim, void* hip_stream) {
    const char* who = "mxq_kv_read_mx";
    if (dtype < 0 || dtype > 2) return fail(MXQ_ERR_ARGUMENT, "%s: unknown dtype code %d", who, dtype);
    KvReadArgs a;
    int rc = make_cache(const_cast<void*>(cache), num_pages, heads, page_size, head_dim, &a.c, who);
    if (rc) return rc;
    if (tokens < 0) return fail(MXQ_ERR_ARGUMENT, "%s: negative size", who);
    if (tokens == 0) return MXQ_OK;
    if (!k || !v || !slots) return fail(MXQ_ERR_ARGUMENT, "%s: null pointer", who);
    a.k = k;
    a.v = v;
    a.slots = slots;
    a.tokens = tokens;
    const int wide = aligned16(k) && aligned16(v) && head_dim % 8 == 0;
    const int grid = rows_grid(a.c, tokens);
    hipStream_t s = (hipStream_t)hip_stream;
    if (dtype == MXQ_DTYPE_F32) kv_read_kernel<MXQ_F32><<<grid, kThreads, 0, s>>>(a, wide);
    else if (dtype == MXQ_DTYPE_BF16) kv_read_kernel<MXQ_BF16><<<grid, kThreads, 0, s>>>(a, wide);
    else kv_read_kernel<MXQ_F16><<<grid, kThreads, 0, s>>>(a, wide);
    return check_launch(who);
}

int64_t mxq_kv_attention_workspace_bytes(int64_t requests, int64_t rows, int q_heads, int64_t max_new, int64_t width, int heads,
                                         int page_size, int head_dim, int dtype) {
    if (requests < 0 || rows <= 0 || heads <= 0 || q_heads < heads || width < 0 || page_size <= 0 || head_dim < 1 ||
        head_dim > 32 * KV_MAX_NB)
        return 0;
    const int terms = dtype == MXQ_DTYPE_F16 ? 2 : 1;
    return part_bytes(make_plan(requests, rows, q_heads / heads, max_new, width * page_size, heads, (head_dim + 31) / 32, terms),
                      heads, terms, requests);
}

int mxq_kv_attention_mx(const void* q, int64_t q_token_stride, int64_t q_head_stride, void* out, int64_t out_token_stride,
                        int64_t out_head_stride, float* lse, int dtype, int64_t rows, int q_heads, const int* block_table,
                        int64_t table_stride, int64_t width, const int* seq_lens, const int* starts, int64_t requests,
                        float scale, int causal, int64_t max_new, int zero_tail, const void* cache, int64_t num_pages,
                        int heads, int page_size, int head_dim, void* workspace, int64_t workspace_bytes, void* hip_stream) {
    const char* who = "mxq_kv_attention_mx";
    if (dtype != MXQ_DTYPE_BF16 && dtype != MXQ_DTYPE_F16)
        return fail(MXQ_ERR_ARGUMENT, "%s: queries must be bf16 or fp16 (dtype code %d)", who, dtype);
    KvAttnArgs a;
    int rc = make_cache(const_cast<void*>(cache), num_pages, heads, page_size, head_dim, &a.c, who);
    if (rc) return rc;
    if (q_heads < 1 || q_heads % heads != 0)
        return fail(MXQ_ERR_ARGUMENT, "%s: %d query heads do not share %d kv heads evenly", who, q_heads, heads);
    if (rows < 0 || requests < 0 || width < 0) return fail(MXQ_ERR_ARGUMENT, "%s: negative size", who);
    const float scale_log2 = (scale < 0 ? -scale : scale) * 1.4426950408889634f;
    if (!(scale_log2 < __builtin_inff())) return fail(MXQ_ERR_ARGUMENT, "%s: scale must be finite, also times log2(e)", who);
    if (rows == 0) return MXQ_OK;
    if (requests == 0 && !starts) return fail(MXQ_ERR_ARGUMENT, "%s: rows without requests", who);
    if (!starts && rows != requests) return fail(MXQ_ERR_ARGUMENT, "%s: without starts every request has one row", who);
    if (requests > 0x7FFFFF00 || rows * q_heads > 0x7FFFFF00 || width * page_size > kMaxTokens)
        return fail(MXQ_ERR_ARGUMENT, "%s: size too large", who);
    if (!q || !out || (requests > 0 && (!seq_lens || (width > 0 && !block_table))))
        return fail(MXQ_ERR_ARGUMENT, "%s: null pointer", who);
    const int terms = dtype == MXQ_DTYPE_F16 ? 2 : 1;
    const Plan p = make_plan(requests, rows, q_heads / heads, max_new, width * page_size, heads, a.c.nb, terms);
    const int64_t needed = part_bytes(p, heads, terms, requests);
    // units and items are numbered in 32 bits
    const int64_t most_units = (requests + ceil_div(rows * q_heads / heads, 16)) * (ceil_div(width * page_size, KV_UNIT) + 1 + KV_ITEM_UNITS);
    // .. and so are the join's workgroups
    const int64_t most_joins = p.prompt ? p.prompt_items * heads * 16 + (int64_t)128 * requests * heads : rows * q_heads;
    if (most_units > 0x7FFFFFFF || most_joins > 0x7FFFFFFF) return fail(MXQ_ERR_ARGUMENT, "%s: size too large", who);
    if (workspace_bytes < needed || (needed > 0 && !workspace))
        return fail(MXQ_ERR_ARGUMENT, "%s: the workspace is too small", who);
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return fail(MXQ_ERR_ARGUMENT, "%s: the workspace must be 16-byte aligned", who);
    a.q = reinterpret_cast<const unsigned short*>(q);
    a.q_token = q_token_stride;
    a.q_head = q_head_stride;
    a.out = reinterpret_cast<unsigned short*>(out);
    a.out_token = out_token_stride;
    a.out_head = out_head_stride;
    a.lse = lse;
    a.table = block_table;
    a.table_stride = table_stride;
    a.width = (int)width;
    a.seq_lens = seq_lens;
    a.starts = starts;
    a.requests = (int)requests;
    a.group = q_heads / heads;
    a.by_group = kv_divide((uint32_t)a.group);
    a.by_heads = kv_divide((uint32_t)heads);
    a.by_q_heads = kv_divide((uint32_t)q_heads);
    a.rows = rows;
    a.scale_log2 = scale_log2;
    if (a.scale_log2 < 1.17549435e-38f) a.scale_log2 = 1.17549435e-38f;      // 0 times a masked score of -inf would be NaN
    a.negative = scale < 0 ? 1 : 0;
    a.causal = causal ? 1 : 0;
    a.q_wide = aligned16(q) && head_dim % 8 == 0 && q_token_stride % 8 == 0 && q_head_stride % 8 == 0;
    a.out_wide = aligned16(out) && head_dim % 8 == 0 && out_token_stride % 8 == 0 && out_head_stride % 8 == 0;
    a.zero_tail = zero_tail ? 1 : 0;
    a.item_shift = p.ct == 1 ? 4 : 5;
    a.decode_columns = p.decode_columns;
    a.whole = p.whole ? 1 : 0;
    a.direct = p.whole && !starts && a.group <= 16 * p.ct ? 1 : 0;
    a.shares = (int)p.shares;
    a.by_shares = kv_divide((uint32_t)a.shares);
    a.join_rows = p.prompt ? p.decode_columns / a.group : 0;
    a.part = reinterpret_cast<float*>(workspace);
    unsigned char* behind = reinterpret_cast<unsigned char*>(workspace) + decode_part_bytes(p, heads);
    a.spans = reinterpret_cast<int*>(behind);
    behind += span_bytes(p);
    a.prompt_part = p.prompt ? reinterpret_cast<float*>(behind) : nullptr;
    a.plan = p.prompt ? behind + prompt_part_bytes(p, heads, terms) : nullptr;
    a.prompt_shares = (int)p.prompt_shares;
    a.prompt_items = (int)p.prompt_items;
    // requests with few columns have few rows where the others are the prompt kernel's
    const int64_t join = p.whole ? 0 : (p.prompt ? a.join_rows * requests : rows) * q_heads;
    a.join_blocks = (int)join;
    a.join_first = 0;
    hipStream_t s = (hipStream_t)hip_stream;
    mxq_kv::launch_decode(dtype, &a, p, s);
    if ((rc = check_launch(who))) return rc;
    if (p.prompt) {
        mxq_kv::launch_prompt(dtype, &a, p, s);
        if ((rc = check_launch(who))) return rc;
    }
    mxq_kv::launch_join(dtype, &a, p, s);
    return check_launch(who);
}

int mxq_kv_call(int which, const int64_t* a, void* workspace, int64_t workspace_bytes, void* hip_stream) {
    if (!a) return fail(MXQ_ERR_ARGUMENT, "mxq_kv_call: null pointer");
    const auto ints = [&](int n) { return reinterpret_cast<int*>(a[n]); };
    const auto at = [&](int n) { return reinterpret_cast<void*>(a[n]); };
    const auto number = [&](int n) { return (int)a[n]; };
    switch (which) {
        case MXQ_KV_BLOCK_TABLES:
            return mxq_kv_block_tables(ints(0), ints(1), ints(2), a[3], a[4], ints(5), a[6], ints(7), a[8], number(9), a[10],
                                       reinterpret_cast<int64_t*>(a[11]), ints(12), ints(13), ints(14), ints(15), ints(16), hip_stream);
        case MXQ_KV_APPEND:
            return mxq_kv_append_mx(at(0), at(1), number(2), a[3], a[4], a[5], a[6], a[7], reinterpret_cast<const int64_t*>(a[8]), at(9),
                                    a[10], number(11), number(12), number(13), number(14), number(15), number(16), number(17), hip_stream);
        case MXQ_KV_READ:
            return mxq_kv_read_mx(at(0), at(1), number(2), a[3], reinterpret_cast<const int64_t*>(a[4]), at(5), a[6], number(7), number(8),
                                  number(9), hip_stream);
        case MXQ_KV_ATTENTION: {
            double scale;
            memcpy(&scale, &a[16], sizeof scale);
            return mxq_kv_attention_mx(at(0), a[1], a[2], at(3), a[4], a[5], reinterpret_cast<float*>(a[6]), number(7), a[8], number(9),
                                       ints(10), a[11], a[12], ints(13), ints(14), a[15], (float)scale, number(17), a[18], number(19),
                                       at(20), a[21], number(22), number(23), number(24), workspace, workspace_bytes, hip_stream);
        }
    }
    return fail(MXQ_ERR_ARGUMENT, "mxq_kv_call: unknown call %d", which);
}

int64_t mxq_kv_attention_args_workspace_bytes(const int64_t* a) {
    return mxq_kv_attention_workspace_bytes(a[15], a[8], (int)a[9], a[18], a[12], (int)a[22], (int)a[23], (int)a[24], (int)a[7]);
}

}  // extern "C"
#pragma GCC visibility pop
