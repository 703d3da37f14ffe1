// Kernels around the packed key / value cache of mxq_kv.h that deal with rows of tokens: block tables and slots from
// request lengths, quantize-and-store, read-back.
#pragma once
#include "mxq_kv.h"

namespace {

// ================================================================================================================
// block tables and slots
// ================================================================================================================
// Request r holds ctx_r tokens and gets new_r more.  Its pages behind ceil(ctx_r / ps) come from the list of free
// pages, in the order of the requests: an exclusive prefix sum.  A thread owns a new token: it finds its request
// by bisection in the prefix sums of the workgroup's share, its page either in the old part of the table or in the
// free list (so no thread waits for another one's table entry), and the first token of a page writes the entry.
// One launch, bound by latency: 4.0 us for a decoding step of one workgroup, 7.1 us for 50000 new tokens; every workgroup
// repeats the sums over all requests, which are a few kilobytes.
struct KvTablesArgs {
    const int* context;
    const int* fresh;
    int* table;
    int64_t table_stride;
    int width;                                           // entries of a table row
    const int* free_pages;
    int64_t free_count;
    const int* free_start;
    int requests, page_size;
    int64_t tokens;                                      // rows of slots / positions / owners
    int64_t* slots;
    int* positions;
    int* owners;
    int* starts;
    int* seq_lens;
    int* free_next;
};

struct KvRequest {
    int64_t ctx, fresh, held, fresh_pages;
};
__device__ __forceinline__ KvRequest kv_request(const KvTablesArgs& a, int r) {
    KvRequest q;
    q.ctx = a.context[r] > 0 ? a.context[r] : 0;
    q.fresh = a.fresh[r] > 0 ? a.fresh[r] : 0;
    q.held = (q.ctx + a.page_size - 1) / a.page_size;
    int64_t last = (q.ctx + q.fresh + a.page_size - 1) / a.page_size;
    last = last < a.width ? last : a.width;
    q.fresh_pages = last > q.held ? last - q.held : 0;
    return q;
}

constexpr int KV_TABLE_TOKENS = 1024;                    // tokens of a workgroup

template <int TOKENS>
__global__ __launch_bounds__(TPB) void kv_block_tables_kernel(KvTablesArgs a) {
    __shared__ int64_t s_wave[TPB / 64];
    // the requests that have tokens in this workgroup's share: at most one for each token
    __shared__ int64_t s_start[TOKENS];
    __shared__ int64_t s_page[TOKENS];
    __shared__ int s_owner[TOKENS];
    __shared__ int s_count;
    const int64_t t0 = (int64_t)blockIdx.x * TOKENS, t1 = t0 + TOKENS;
    const bool first_block = blockIdx.x == 0;
    if (threadIdx.x == 0) s_count = 0;
    int64_t tokens = 0, pages = a.free_start[0], listed = 0;
    for (int r0 = 0; r0 < a.requests; r0 += TPB) {
        const int r = r0 + threadIdx.x;
        KvRequest q{0, 0, 0, 0};
        if (r < a.requests) q = kv_request(a, r);
        int64_t token_sum, page_sum, list_sum;
        const int64_t start = tokens + block_scan(q.fresh, s_wave, &token_sum) - q.fresh;
        const int64_t page = pages + block_scan(q.fresh_pages, s_wave, &page_sum) - q.fresh_pages;
        const bool here = q.fresh > 0 && start < t1 && start + q.fresh > t0;
        const int64_t at = listed + block_scan((int64_t)(here ? 1 : 0), s_wave, &list_sum) - 1;
        if (here) {
            s_start[at] = start;
            s_page[at] = page;
            s_owner[at] = r;
        }
        if (first_block && r < a.requests) {
            a.starts[r] = (int)(start < a.tokens ? start : a.tokens);
            const int64_t len = q.ctx + q.fresh;
            a.seq_lens[r] = len < 0x7FFFFFFF ? (int)len : 0x7FFFFFFF;
        }
        tokens += token_sum;
        pages += page_sum;
        listed += list_sum;
    }
    if (first_block && threadIdx.x == 0) {
        a.starts[a.requests] = (int)(tokens < a.tokens ? tokens : a.tokens);
        a.free_next[0] = pages < 0x7FFFFFFF ? (int)pages : 0x7FFFFFFF;
    }
    if (threadIdx.x == 0) s_count = (int)listed;
    __syncthreads();
    const int count = s_count;
    for (int64_t t = t0 + threadIdx.x; t < t1 && t < a.tokens; t += TPB) {
        int64_t slot = -1;
        int pos32 = -1, owner = -1;
        if (t < tokens) {
            int lo = 0, hi = count;                      // the last listed request that starts at or before t
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (s_start[mid] <= t) lo = mid;
                else hi = mid;
            }
            owner = s_owner[lo];
            const KvRequest q = kv_request(a, owner);
            const int64_t pos = q.ctx + (t - s_start[lo]);
            const int64_t j = pos / a.page_size, off = pos % a.page_size;
            pos32 = pos < 0x7FFFFFFF ? (int)pos : 0x7FFFFFFF;
            if (j < a.width) {
                int* entry = a.table + (int64_t)owner * a.table_stride + j;
                int page;
                if (j < q.held) {
                    page = *entry;
                } else {
                    const int64_t at = s_page[lo] + (j - q.held);
                    page = at >= 0 && at < a.free_count ? a.free_pages[at] : -1;
                    if (off == 0) *entry = page;
                }
                if (page >= 0) slot = (int64_t)page * a.page_size + off;
            }
        }
        a.slots[t] = slot;
        a.positions[t] = pos32;
        a.owners[t] = owner;
    }
}

// ================================================================================================================
// quantize and store; read back
// ================================================================================================================
// A lane owns 8 elements of a block (a dword of codes): lane bits 0-1 the token of four, 2-3 the quarter j of the
// block; a group of 16 lanes keeps its head, K or V, and block, and goes through the groups of four tokens.  K's dword
// goes out as it is.  Of V the four lanes of a quad hold the bytes (i = 4 j .. 4 j + 3) of four tokens; where these
// tokens are the four of one V tile (every tile of a prompt), they trade bytes and store a dword each, otherwise
// (decoding steps) four bytes.  Bound by memory for prompts (16384 rows of 8 heads of 128 in bf16 at random slots: 36 us, 66 MB
// read and 41 MB written for 18, since the bytes of a V tile come at different times; reading them back as fp32 40 us,
// 4.5 TB/s), by latency for single tokens (3.8 and 3.6 us for a step of 128 rows).
//
// Rounding half away from zero with v_cvt_scalef32_pk_fp4_f32, which rounds half to even: values are moved a little
// further from zero first, so that what lies on a border between two codes lies above it, and nothing else crosses one.
//   bf16: times 1 + 2^-8 + 2^-15.  A border is half of a 2-bit significand's step; the largest bf16 below one of them is
//     2^-7 of it or more below (2^-8 above a power of two: all but the first border are), except below the first
//     border 1/4, where 1/4 - 2^-10 is the very value that the bf16 sum with one half carries over it.
//   fp32 (and fp16 widened): the low 8 bits become 0x80, which puts a border above itself and keeps everything below it
//     below; 2^-26 is added first, which lets the one value do the same that the fp32 sum with one half carries over.
// That replaces 14 instructions an element by 3 or 6: 16384 rows of 8 heads of 128 took 46 us with them.
template <int DT>
struct KvNudge {
    static __device__ __forceinline__ float inverse(float inv_scale) { return inv_scale; }
    static __device__ __forceinline__ float apply(float x, float inv) {
        const float a = x * inv;
        const uint32_t away = (mxq_bits(__builtin_fabsf(a) + 1.4901161193847656e-08f) & 0xFFFFFF00u) | 0x80u;
        return mxq_float(away | (mxq_bits(a + 0.0f) & 0x80000000u));         // (-0 is +0)
    }
};
template <>
struct KvNudge<MXQ_BF16> {
    static __device__ __forceinline__ float inverse(float inv_scale) { return inv_scale * 1.003936767578125f; }
    // + 1.004 x 2^-134: what bf16 would round to zero, -0 among it, becomes +0
    static __device__ __forceinline__ float apply(float x, float inv) { return __builtin_fmaf(x, inv, 4.610e-41f); }
};

struct KvRowsArgs {
    const void* k;
    const void* v;
    int64_t k_token, k_head, v_token, v_head;            // strides in elements
    const int64_t* slots;
    int64_t tokens;
    int wide;                                            // rows can be read / written 16 bytes at a time
    KvCache c;
};

struct KvPlace {
    bool live;
    unsigned char* record;
    int off;
};
__device__ __forceinline__ KvPlace kv_place(const KvCache& c, int64_t slot, int head) {
    KvPlace p{false, nullptr, 0};
    if (slot < 0) return p;
    int64_t page;
    if (slot < 0x100000000LL) {
        page = kv_page_of(c, (uint32_t)slot);
        p.off = (int)((uint32_t)slot - (uint32_t)page * (uint32_t)c.page_size);
    } else {
        page = slot / c.page_size;
        p.off = (int)(slot - page * c.page_size);
    }
    if (page >= c.num_pages) return p;
    p.live = true;
    p.record = c.data + (page * c.heads + head) * c.record;
    return p;
}

// quad lane t's value of v, for t = 0 .. 3
template <int T>
__device__ __forceinline__ uint32_t quad_lane(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, T * 0x55, 0xF, 0xF, false);
}
// byte `me` of the dwords of the quad's four lanes: a 4 x 4 byte transpose over the quad
__device__ __forceinline__ uint32_t quad_transpose(uint32_t v, int me) {
    const int s = 8 * me;
    return ((quad_lane<0>(v) >> s) & 255u) | (((quad_lane<1>(v) >> s) & 255u) << 8) |
           (((quad_lane<2>(v) >> s) & 255u) << 16) | (((quad_lane<3>(v) >> s) & 255u) << 24);
}
// are the quad's four tokens one V tile?
__device__ __forceinline__ bool quad_is_tile(int64_t slot, int me) {
    const uint32_t lo = (uint32_t)slot, hi = (uint32_t)((uint64_t)slot >> 32);
    const int64_t first = (int64_t)(((uint64_t)quad_lane<0>(hi) << 32) | quad_lane<0>(lo));
    const uint32_t ok = slot >= 0 && first >= 0 && (first & 3) == 0 && slot == first + me ? 1u : 0u;
    return (quad_lane<0>(ok) & quad_lane<1>(ok) & quad_lane<2>(ok) & quad_lane<3>(ok)) != 0u;
}

// the unit of a group of 16 lanes, and the groups of four tokens that it goes through: neighbouring ones, so that the
// lines that their scales share are completed in one L2
struct KvUnit {
    int head, is_v, b;
    int64_t quad, end;
};
__device__ __forceinline__ KvUnit kv_unit(const KvCache& c, int64_t tokens) {
    const int units = c.heads * 2 * c.nb, blocks = (units + 15) / 16;
    const int at = (int)blockIdx.x % blocks * 16 + (threadIdx.x >> 4);
    KvUnit u;
    u.head = at / (2 * c.nb);
    u.is_v = at - u.head * 2 * c.nb >= c.nb;
    u.b = at - u.head * 2 * c.nb - u.is_v * c.nb;
    const int64_t quads = (tokens + 3) / 4;
    const int shares = gridDim.x / blocks, share = blockIdx.x / blocks;
    const int64_t each = (quads + shares - 1) / shares;
    u.quad = each * share;
    u.end = at < units ? (u.quad + each < quads ? u.quad + each : quads) : 0;
    return u;
}

template <int DT, int RMODE, bool ZONE_ELEM>
__global__ __launch_bounds__(TPB) void kv_append_kernel(KvRowsArgs a, MxParams p, uint32_t max_code) {
    constexpr int ADT = Arith<DT>::DT_;
    constexpr int ZS = (ADT == MXQ_BF16) ? 16 : 0;
    __shared__ unsigned char zone[ZONE_PAD];
    load_zone(zone, g_zone_tables[p.zone_row]);
    const int NB = a.c.nb, me = threadIdx.x & 3, j = (threadIdx.x >> 2) & 3;
    const KvUnit u = kv_unit(a.c, a.tokens);
    const int head = u.head, is_v = u.is_v, b = u.b;
    for (int64_t quad = u.quad; quad < u.end; ++quad) {
        const int64_t token = quad * 4 + me;
        const bool row = token < a.tokens;
        const int64_t slot = row ? a.slots[token] : -1;
        const int e0 = 32 * b + 8 * j;                   // first element of the lane
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = 0.0f;
        if (row && e0 < a.c.head_dim) {
            const int64_t at = is_v ? token * a.v_token + head * a.v_head + e0 : token * a.k_token + head * a.k_head + e0;
            const void* src = is_v ? a.v : a.k;
            if (a.wide) {                                // head_dim a multiple of 8, rows 16-byte aligned
                if constexpr (DT == MXQ_F32) {
                    const u32x4* s = reinterpret_cast<const u32x4*>(reinterpret_cast<const float*>(src) + at);
                    const u32x4 lo = s[0], hi = s[1];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[e] = mxq_float(lo[e]);
                        x[e + 4] = mxq_float(hi[e]);
                    }
                } else {
                    const u32x4 w = *reinterpret_cast<const u32x4*>(reinterpret_cast<const unsigned short*>(src) + at);
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = Pack<DT>::get(w[e / 2], e & 1);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e0 + e < a.c.head_dim) x[e] = load_scalar<DT>(src, at + e);
            }
        }
        uint32_t um = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) um = max(um, abs_bits(x[e]));
        // the block's four lanes are 4 apart: rotations by 8 and 4 inside the row of 16 lanes
        um = max(um, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)um, 0x128, 0xF, 0xF, false));
        um = max(um, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)um, 0x124, 0xF, 0xF, false));
        const MxqScale sc = mxq_block_scale(um, p.emax, p.scale_emax, p.flush != 0, zone, ZS);
        const uint32_t sb = mxq_encode_e8m0(sc.scale);
        uint32_t codes = 0;
        if constexpr (RMODE == MXQ_NEAREST && !ZONE_ELEM) {
            using Nudge = KvNudge<ADT>;
            const float inv = Nudge::inverse(sc.inv_scale);
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = Nudge::apply(x[e], inv);
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, y[0], y[1], 1.0f, 0);
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, y[2], y[3], 1.0f, 1);
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, y[4], y[5], 1.0f, 2);
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, y[6], y[7], 1.0f, 3);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                uint32_t c;
                if constexpr (!ZONE_ELEM) c = mxq_quant_mx_code<RMODE, ADT, 3>(x[e], sc, p.fmt, max_code);
                else c = mxq_encode_e2m1(mxq_quant_mx_elem_unscaled<RMODE, ADT, ZONE_ELEM>(x[e], sc, p.fmt, zone, ZS));
                codes |= c << (4 * e);
            }
        }
        const KvPlace pl = kv_place(a.c, slot, head);
        const int ps = a.c.page_size;
        const bool tile = quad_is_tile(pl.live ? slot : -1, me);
        const uint32_t turned = quad_transpose(codes, me);           // by every lane: an exchange
        const uint32_t scales4 = quad_transpose(sb, 0);
        if (!pl.live) continue;
        if (!is_v) {
            *reinterpret_cast<uint32_t*>(pl.record + (int64_t)pl.off * (16 * NB) + 16 * b + 4 * j) = codes;
            if (j == 0) pl.record[(int64_t)ps * (32 * NB) + (int64_t)pl.off * NB + b] = (unsigned char)sb;
            continue;
        }
        unsigned char* vt = pl.record + (int64_t)ps * (16 * NB) + (int64_t)(pl.off >> 2) * (64 * NB) + 4 * b;
        unsigned char* st = pl.record + (int64_t)ps * (33 * NB) + (int64_t)(pl.off >> 2) * (4 * NB) + 4 * b;
        if (tile) {
            *reinterpret_cast<uint32_t*>(vt + (4 * j + me) * 4 * NB) = turned;
            if (j == 0 && me == 0) *reinterpret_cast<uint32_t*>(st) = scales4;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) vt[(4 * j + i) * 4 * NB + (pl.off & 3)] = (unsigned char)(codes >> (8 * i));
            if (j == 0) st[pl.off & 3] = (unsigned char)sb;
        }
    }
}

template <int SEL>
__device__ __forceinline__ void kv_decode_floats(uint32_t codes, float scale, float* y) {
    const kv_f32x2 v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, SEL);
    y[2 * SEL] = v[0];
    y[2 * SEL + 1] = v[1];
}

// The rows at `slots` as values: codes times scale, rounded once to the output type; rows without a slot are zero.
struct KvReadArgs {
    void* k;
    void* v;                                             // (tokens, heads, head_dim), contiguous
    const int64_t* slots;
    int64_t tokens;
    KvCache c;
};
template <int DT>
__global__ __launch_bounds__(TPB) void kv_read_kernel(KvReadArgs a, int wide) {
    // fp32 rows: a lane takes the elements 4 j .. and 16 + 4 j .. of the block instead of 8 j .., so that each of its two
    // 16-byte stores lies next to its neighbours'
    constexpr bool HALVES = DT == MXQ_F32;
    const int NB = a.c.nb, me = threadIdx.x & 3, j = (threadIdx.x >> 2) & 3;
    const auto pair = [&](int i) { return !HALVES ? 4 * j + i : i < 2 ? 2 * j + i : 6 + 2 * j + i; };   // of elements
    const KvUnit u = kv_unit(a.c, a.tokens);
    const int head = u.head, is_v = u.is_v, b = u.b;
    for (int64_t quad = u.quad; quad < u.end; ++quad) {
        const int64_t token = quad * 4 + me;
        const int64_t slot = token < a.tokens ? a.slots[token] : -1;
        const KvPlace pl = kv_place(a.c, slot, head);
        const int ps = a.c.page_size;
        const bool tile = quad_is_tile(pl.live ? slot : -1, me);
        uint32_t codes = 0, sb = 127;
        if (pl.live) {
            if (!is_v) {
                const unsigned char* kr = pl.record + (int64_t)pl.off * (16 * NB) + 16 * b;
                if constexpr (HALVES)
                    codes = *reinterpret_cast<const unsigned short*>(kr + 2 * j) |
                            (uint32_t)*reinterpret_cast<const unsigned short*>(kr + 8 + 2 * j) << 16;
                else codes = *reinterpret_cast<const uint32_t*>(kr + 4 * j);
                sb = pl.record[(int64_t)ps * (32 * NB) + (int64_t)pl.off * NB + b];
            } else {
                const unsigned char* vt = pl.record + (int64_t)ps * (16 * NB) + (int64_t)(pl.off >> 2) * (64 * NB) + 4 * b;
                sb = pl.record[(int64_t)ps * (33 * NB) + (int64_t)(pl.off >> 2) * (4 * NB) + 4 * b + (pl.off & 3)];
                if (tile) {
                    codes = *reinterpret_cast<const uint32_t*>(vt + pair(me) * 4 * NB);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) codes |= (uint32_t)vt[pair(i) * 4 * NB + (pl.off & 3)] << (8 * i);
                }
            }
        }
        const uint32_t turned = quad_transpose(codes, me);
        if (is_v && tile) codes = turned;
        const int e0 = 32 * b + (HALVES ? 4 * j : 8 * j);
        if (token >= a.tokens || e0 >= a.c.head_dim) continue;
        float y[8];
        const float scale = mxq_float(sb << 23);         // (the exponent field counts: 255 is NaN, 0 is 2^-127)
        kv_decode_floats<0>(codes, scale, y);
        kv_decode_floats<1>(codes, scale, y);
        kv_decode_floats<2>(codes, scale, y);
        kv_decode_floats<3>(codes, scale, y);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = pl.live ? mxq_round_dt<Arith<DT>::DT_>(y[e]) : 0.0f;
        const int64_t at = (token * a.c.heads + head) * (int64_t)a.c.head_dim + e0;
        void* dst = is_v ? a.v : a.k;
        if (wide) {
            if constexpr (DT == MXQ_F32) {
                u32x4* o = reinterpret_cast<u32x4*>(reinterpret_cast<float*>(dst) + at);
                o[0] = u32x4{mxq_bits(y[0]), mxq_bits(y[1]), mxq_bits(y[2]), mxq_bits(y[3])};
                if (e0 + 16 < a.c.head_dim) o[4] = u32x4{mxq_bits(y[4]), mxq_bits(y[5]), mxq_bits(y[6]), mxq_bits(y[7])};
            } else {
                *reinterpret_cast<u32x4*>(reinterpret_cast<unsigned short*>(dst) + at) =
                    u32x4{Pack<DT>::put(y[0], y[1]), Pack<DT>::put(y[2], y[3]), Pack<DT>::put(y[4], y[5]), Pack<DT>::put(y[6], y[7])};
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int d = HALVES && e >= 4 ? e + 12 : e;
                if (e0 + d < a.c.head_dim) store_scalar<DT>(dst, at + d, y[e]);
            }
        }
    }
}

}  // namespace
