// Attention over the packed cache of mxq_kv.h: one pass over keys and values with the running maximum and sum of
// the softmax, K and V decoded in registers.
//
// The columns of a request are its new tokens times the query heads of a kv head: column c is token c / G, head
// c % G.  A wave multiplies 32 tokens at a time with CT tiles of 16 columns:
//   S^T (tokens x columns) = K q^T          2 NB CT instructions of 16 x 16 x 32
//   p = 2^(s - m)                           a lane holds 8 tokens of one column in each tile
//   O^T (elements x columns) += V^T p^T     2 NB CT instructions, the probabilities straight from the lane
// m is raised only when a score passes it by 8 (a factor of 256, which fp32 sums carry easily), so the accumulators
// are rarely rescaled.  q enters as bf16 (fp16 queries as two bf16 terms, exactly: 11 bits in 8 + 8); the
// probabilities as one bf16 term (half a step is 2^-8 of each, which averages over the tokens) or as two (2^-17).
// Sums, maxima and accumulators are fp32.
//
// Two kernels share this body.  kv_decode_kernel (few columns): the waves of a workgroup take turns over the
// tokens, and the whole grid shares all tokens of all requests evenly: a request that crosses workgroups leaves
// partial results that kv_join_kernel adds in the order of the workgroups.  kv_prompt_kernel (many columns): every
// wave has its own columns and walks over all the tokens they see.
#pragma once
#include "mxq_kv.h"

namespace {

struct KvAttnArgs {
    const unsigned short* q;
    int64_t q_token, q_head;                             // strides in elements
    unsigned short* out;
    int64_t out_token, out_head;
    float* lse;                                          // (rows, query heads), or null
    const int* table;
    int64_t table_stride;
    int width;                                           // entries of a table row
    const int* seq_lens;
    const int* starts;                                   // (requests + 1), or null: one row a request
    int requests, group;                                 // query heads of a kv head
    int64_t rows;                                        // rows of q and out
    float scale_log2;                                    // |scale| log2(e)
    unsigned q_sign;                                     // 0x80008000 where scale is negative
    int causal, q_wide, out_wide, zero_tail;
    int tile_columns;                                    // decode: columns of an item, 16 CT
    int decode_columns;                                  // requests with more columns belong to the prompt kernel
    int whole;                                           // decode: a workgroup for each item, nothing to join
    int shares;                                          // decode: workgroups of a kv head
    float* part;                                         // decode: partial results, two places for each workgroup
    KvCache c;
};

// a request as the attention sees it
struct KvSeq {
    int64_t row0;                                        // its first row of q
    int fresh;                                           // its rows
    int len;                                             // tokens, unlimited
    int keys;                                            // tokens that the table can name
};
__device__ __forceinline__ KvSeq kv_seq(const KvAttnArgs& a, int r) {
    KvSeq s;
    if (a.starts) {
        int64_t s0 = a.starts[r], s1 = a.starts[r + 1];
        s0 = s0 < 0 ? 0 : (s0 < a.rows ? s0 : a.rows);
        s1 = s1 < s0 ? s0 : (s1 < a.rows ? s1 : a.rows);
        s.row0 = s0;
        s.fresh = (int)(s1 - s0);
    } else {
        s.row0 = r;
        s.fresh = 1;
    }
    s.len = a.seq_lens[r] > 0 ? a.seq_lens[r] : 0;
    const int64_t room = (int64_t)a.width * a.c.page_size;
    s.keys = s.len < room ? s.len : (int)room;
    return s;
}
// keys that new token i sees (0 or less: none)
__device__ __forceinline__ int kv_limit(const KvAttnArgs& a, const KvSeq& s, int i) {
    if (!a.causal) return s.keys;
    const int64_t n = (int64_t)s.len - s.fresh + i + 1;
    return n < s.keys ? (int)(n > 0 ? n : 0) : s.keys;
}

constexpr int KV_UNIT = 128;                             // tokens of a unit of work: a tile of 32 for each wave

// units and column groups of a request in the decode kernel; a request without keys still has one unit, whose
// workgroup writes the zeros
struct KvWork {
    int units, groups;
};
__device__ __forceinline__ KvWork kv_work(const KvAttnArgs& a, const KvSeq& s) {
    const int64_t columns = (int64_t)s.fresh * a.group;
    if (columns == 0 || columns > a.decode_columns) return KvWork{0, 0};
    const int units = (s.keys + KV_UNIT - 1) / KV_UNIT;
    return KvWork{units > 0 ? units : 1, (int)((columns + a.tile_columns - 1) / a.tile_columns)};
}

// ---- loads -------------------------------------------------------------------------------------------------------
// N dwords from an address that is aligned to min(4 N, 16) bytes where N is a power of two, to 4 otherwise
template <int N>
__device__ __forceinline__ void load_dwords(const unsigned char* p, uint32_t* d) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const u32x4 w = reinterpret_cast<const u32x4*>(p)[i];
#pragma unroll
            for (int e = 0; e < 4; ++e) d[4 * i + e] = w[e];
        }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const u32x2 w = reinterpret_cast<const u32x2*>(p)[i];
            d[2 * i] = w[0];
            d[2 * i + 1] = w[1];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) d[i] = reinterpret_cast<const uint32_t*>(p)[i];
    }
}

// Lane group g's K elements 8 NB g + 8 s .. + 7 of step s lie in block (NB g + s) / 4: the scale bytes of the
// blocks from NB g / 4 on, as many as its steps can touch
template <int NB>
constexpr int kv_k_scales() { return NB % 4 == 0 ? NB / 4 : NB <= 2 ? 1 : (NB + 2) / 4 + 1; }
template <int NB>
__device__ __forceinline__ uint32_t kv_k_scale(const uint32_t* ks, int g, int s) {
    constexpr int N = kv_k_scales<NB>();
    if constexpr (N == 1) return ks[0];
    if constexpr (NB % 4 == 0) return ks[s / 4];
    const int at = (NB * g + s) / 4 - NB * g / 4;
    uint32_t v = ks[0];
#pragma unroll
    for (int k = 1; k < N; ++k) v = at == k ? ks[k] : v;
    return v;
}

template <int NB>
struct KvTile {                                          // what a lane holds of 32 tokens
    uint32_t k[2][NB], ks[2][kv_k_scales<NB>()];
    uint32_t v[2][NB], vs[2][NB];
    bool there[2];                                       // the two pages exist (uniform over the wave)
};

// the scale operand of v_cvt_scalef32_*: only the exponent field counts (255: NaN, 0: 2^-127)
template <int SEL>
__device__ __forceinline__ uint32_t kv_decode2(uint32_t codes, uint32_t scale_bits) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, mxq_float(scale_bits), SEL));
}
__device__ __forceinline__ kv_bf16x8 kv_operand(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(kv_bf16x8, u32x4{a, b, c, d});
}
template <int SEL>                                       // exponent field of byte SEL of four E8M0 bytes
__device__ __forceinline__ uint32_t kv_scale_bits(uint32_t four) {
    return SEL == 3 ? four >> 1 : four << (23 - 8 * SEL);
}

template <int NB, int CT, int NT, int NP>
struct KvWave {
    kv_f32x4 acc[CT][NB][2];                             // element 32 b + 2 (4 g + r) + n of the lane's column
    float m[CT], l[CT];                                  // l: this lane's tokens only
    kv_bf16x8 q[CT][NT][NB];
    int limit[CT];                                       // keys that the lane's column sees
    int min_limit, max_limit;                            // over the wave's columns
    const unsigned char* base;                           // of the kv head
    int lane, i16, g;

    // columns c0 .. c0 + 16 CT - 1 of request s
    __device__ __forceinline__ void begin(const KvAttnArgs& a, const KvSeq& s, int head, int c0) {
        lane = threadIdx.x & 63;
        i16 = lane & 15;
        g = lane >> 4;
        base = a.c.data + (int64_t)head * a.c.record;
        const int columns = s.fresh * a.group;
        const int last = (c0 + 16 * CT < columns ? c0 + 16 * CT : columns) - 1;
        min_limit = kv_limit(a, s, c0 / a.group);
        max_limit = kv_limit(a, s, last / a.group);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            m[ct] = -__builtin_inff();
            l[ct] = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b) acc[ct][b][0] = acc[ct][b][1] = kv_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            const int c = c0 + 16 * ct + i16, token = c / a.group;
            const bool live = c < columns;
            limit[ct] = live ? kv_limit(a, s, token) : max_limit;
            const unsigned short* row = a.q + (s.row0 + (live ? token : 0)) * a.q_token +
                                        ((int64_t)head * a.group + (live ? c - token * a.group : 0)) * a.q_head;
#pragma unroll
            for (int st = 0; st < NB; ++st) {
                const int e0 = 8 * NB * g + 8 * st;
                u32x4 w = {0, 0, 0, 0};
                if (live && e0 < a.c.head_dim) {
                    if (a.q_wide) {
                        w = *reinterpret_cast<const u32x4*>(row + e0);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (e0 + e < a.c.head_dim) w[e / 2] |= (uint32_t)row[e0 + e] << (16 * (e & 1));
                    }
                    w ^= a.q_sign;
                }
                if constexpr (NT == 1) {
                    q[ct][0][st] = __builtin_bit_cast(kv_bf16x8, w);
                } else {                                 // fp16: 11 bits as 8 + the rest, both exact
                    u32x4 hi, lo;
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        const float x0 = Pack<MXQ_F16>::get(w[d], 0), x1 = Pack<MXQ_F16>::get(w[d], 1);
                        const uint32_t h = Pack<MXQ_BF16>::put(x0, x1);
                        const float r0 = x0 - Pack<MXQ_BF16>::get(h, 0), r1 = x1 - Pack<MXQ_BF16>::get(h, 1);
                        hi[d] = h;
                        lo[d] = Pack<MXQ_BF16>::put(r0, r1);
                    }
                    q[ct][0][st] = __builtin_bit_cast(kv_bf16x8, hi);
                    q[ct][NT - 1][st] = __builtin_bit_cast(kv_bf16x8, lo);
                }
            }
        }
    }

    // tokens 16 sub .. of page `page` (negative: none), as sub-tile j
    __device__ __forceinline__ void load_half(const KvAttnArgs& a, KvTile<NB>& t, int j, int page, int sub) const {
        t.there[j] = page >= 0;
        const int ps = a.c.page_size;
        const unsigned char* rec = base + (int64_t)(page >= 0 ? page : 0) * ((int64_t)a.c.heads * a.c.record);
        const int off = 16 * (page >= 0 ? sub : 0);
        load_dwords<NB>(rec + (off + i16) * (16 * NB) + g * (4 * NB), t.k[j]);
        const unsigned char* vt = rec + ps * (16 * NB) + (off / 4 + g) * (64 * NB);
        load_dwords<NB>(vt + i16 * (4 * NB), t.v[j]);
        const unsigned char* ks = rec + ps * (32 * NB) + (off + i16) * NB;
#pragma unroll
        for (int k = 0; k < kv_k_scales<NB>(); ++k) {
            const int b = NB * g / 4 + k;
            t.ks[j][k] = ks[b < NB ? b : NB - 1];
        }
        load_dwords<NB>(rec + ps * (33 * NB) + (off / 4 + g) * (4 * NB), t.vs[j]);
    }

    // tokens t0 .. t0 + 31
    __device__ __forceinline__ void step(const KvAttnArgs& a, KvTile<NB>& t, int t0) {
        kv_f32x4 sc[CT][2];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) sc[ct][0] = sc[ct][1] = kv_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int st = 0; st < NB; ++st) {
                const uint32_t bits = kv_k_scale<NB>(t.ks[j], g, st) << 23, w = t.k[j][st];
                const kv_bf16x8 k8 = kv_operand(kv_decode2<0>(w, bits), kv_decode2<1>(w, bits), kv_decode2<2>(w, bits),
                                                kv_decode2<3>(w, bits));
#pragma unroll
                for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        sc[ct][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k8, q[ct][nt][st], sc[ct][j], 0, 0, 0);
            }
        // a tile that every column sees entirely needs no mask
        const bool masked = t0 + 32 > min_limit || !t.there[0] || !t.there[1];
        uint32_t nan_of[NB];                             // masked tiles: which of the 32 tokens have a NaN block b of V
        bool any_nan = false;
        if (masked) {
            uint32_t mine = 0;
#pragma unroll
            for (int b = 0; b < NB; ++b) nan_of[b] = 0;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int token = t0 + 16 * j + 4 * g + r;
                    const bool seen = t.there[j] && token < max_limit;
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const uint32_t byte = (t.vs[j][b] >> (8 * r)) & 255u;
                        const bool nan = byte == 255u;
                        if (nan && seen) nan_of[b] |= 1u << (16 * j + 4 * g + r);
                        if (nan || !seen) t.vs[j][b] &= ~(255u << (8 * r));     // 0 x NaN must not reach a column that
                    }                                                           // does not see the token
                }
#pragma unroll
            for (int b = 0; b < NB; ++b) mine |= nan_of[b];
            any_nan = any_lane(mine != 0u);
        }
        uint32_t p_hi[CT][4], p_lo[CT][NP == 2 ? 4 : 1];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            float p[8];
            if (masked) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const bool seen = t.there[e >> 2] && t0 + 16 * (e >> 2) + 4 * g + (e & 3) < limit[ct];
                    p[e] = seen ? sc[ct][e >> 2][e & 3] * a.scale_log2 : -__builtin_inff();
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) p[e] = sc[ct][e >> 2][e & 3] * a.scale_log2;
            }
            float mx = p[0];
#pragma unroll
            for (int e = 1; e < 8; ++e) mx = __builtin_fmaxf(mx, p[e]);
            mx = max_over_groups(mx);
            if (any_lane(mx > m[ct] + 8.0f)) {           // -inf at first
                const float up = mx > m[ct] + 8.0f ? mx : m[ct];
                const float f = up > m[ct] ? __builtin_amdgcn_exp2f(m[ct] - up) : 1.0f;
                m[ct] = up;
                l[ct] *= f;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[ct][b][n][r] *= f;
            }
            const float mm = m[ct] == -__builtin_inff() ? 0.0f : m[ct];      // nothing seen yet: 2^-inf = 0
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(p[e] - mm);
            l[ct] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                p_hi[ct][d] = Pack<MXQ_BF16>::put(p[2 * d], p[2 * d + 1]);
                if constexpr (NP == 2)
                    p_lo[ct][d] = Pack<MXQ_BF16>::put(p[2 * d] - Pack<MXQ_BF16>::get(p_hi[ct][d], 0),
                                                      p[2 * d + 1] - Pack<MXQ_BF16>::get(p_hi[ct][d], 1));
            }
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            uint32_t cv[8];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                cv[4 * j + 0] = kv_decode2<0>(t.v[j][b], kv_scale_bits<0>(t.vs[j][b]));
                cv[4 * j + 1] = kv_decode2<1>(t.v[j][b], kv_scale_bits<1>(t.vs[j][b]));
                cv[4 * j + 2] = kv_decode2<2>(t.v[j][b], kv_scale_bits<2>(t.vs[j][b]));
                cv[4 * j + 3] = kv_decode2<3>(t.v[j][b], kv_scale_bits<3>(t.vs[j][b]));
            }
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const uint32_t sel = n ? 0x07060302u : 0x05040100u;          // the upper or lower halves of two dwords
                const kv_bf16x8 v8 = kv_operand(
                    __builtin_amdgcn_perm(cv[1], cv[0], sel), __builtin_amdgcn_perm(cv[3], cv[2], sel),
                    __builtin_amdgcn_perm(cv[5], cv[4], sel), __builtin_amdgcn_perm(cv[7], cv[6], sel));
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
                    acc[ct][b][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        v8, kv_operand(p_hi[ct][0], p_hi[ct][1], p_hi[ct][2], p_hi[ct][3]), acc[ct][b][n], 0, 0, 0);
                    if constexpr (NP == 2)
                        acc[ct][b][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            v8, kv_operand(p_lo[ct][0], p_lo[ct][1], p_lo[ct][2], p_lo[ct][3]), acc[ct][b][n], 0, 0, 0);
                }
            }
        }
        if (any_nan) {                                   // rare: the NaN blocks reach the columns that see them
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const uint32_t of = or_over_groups(nan_of[b]);
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
                    const int n = limit[ct] - t0;
                    const uint32_t sees = n >= 32 ? 0xFFFFFFFFu : n > 0 ? (1u << n) - 1u : 0u;
                    if (of & sees) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[ct][b][0][r] = acc[ct][b][1][r] = mxq_float(MXQ_QNAN_BITS);
                    }
                }
            }
        }
    }

    // the tiles first, first + stride, .. of 32 tokens below tile `end`: the pages of 32 tiles at a time sit in the
    // lanes (lane: tile lane / 2, half lane % 2), and a tile's codes are on their way while the one before is multiplied
    __device__ __forceinline__ void walk(const KvAttnArgs& a, int r, int first, int end, int stride) {
        const int subs = a.c.page_size / 16;
        const int seen_end = (max_limit + 31) / 32;      // uniform: nothing behind it is seen
        if (end > seen_end) end = seen_end;
        const int* row = a.table + (int64_t)r * a.table_stride;
        for (int chunk = first; chunk < end; chunk += 32 * stride) {
            const int sub = 2 * (chunk + (lane >> 1) * stride) + (lane & 1);
            int page = -1, in_page = 0;
            const int at = sub / subs;
            if (at < a.width && sub * 16 < max_limit) {
                page = row[at];
                in_page = sub - at * subs;
                if (page >= a.c.num_pages) page = -1;
            }
            KvTile<NB> next;
            load_half(a, next, 0, __builtin_amdgcn_readlane(page, 0), __builtin_amdgcn_readlane(in_page, 0));
            load_half(a, next, 1, __builtin_amdgcn_readlane(page, 1), __builtin_amdgcn_readlane(in_page, 1));
            int tiles = (end - chunk + stride - 1) / stride;
            if (tiles > 32) tiles = 32;
            for (int n = 0; n < tiles; ++n) {
                KvTile<NB> now = next;
                if (n + 1 < tiles) {
                    load_half(a, next, 0, __builtin_amdgcn_readlane(page, 2 * n + 2), __builtin_amdgcn_readlane(in_page, 2 * n + 2));
                    load_half(a, next, 1, __builtin_amdgcn_readlane(page, 2 * n + 3), __builtin_amdgcn_readlane(in_page, 2 * n + 3));
                }
                step(a, now, 32 * (chunk + n * stride));
            }
        }
    }
};

// rounds to the output type and stores elements e0 .. e0 + 7 of a row
template <int DT>
__device__ __forceinline__ void kv_store8(const KvAttnArgs& a, unsigned short* row, int e0, const float* y) {
    if (e0 >= a.c.head_dim) return;
    if (a.out_wide) {
        *reinterpret_cast<u32x4*>(row + e0) = u32x4{Pack<DT>::put(y[0], y[1]), Pack<DT>::put(y[2], y[3]),
                                                    Pack<DT>::put(y[4], y[5]), Pack<DT>::put(y[6], y[7])};
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e0 + e < a.c.head_dim) row[e0 + e] = (unsigned short)Pack<DT>::put(y[e], y[e]);
}
__device__ __forceinline__ unsigned short* kv_out_row(const KvAttnArgs& a, int64_t row, int64_t q_head) {
    return a.out + row * a.out_token + q_head * a.out_head;
}
// natural logarithm of the sum of exponentials; -inf where nothing was seen
__device__ __forceinline__ float kv_lse(float m, float l) {
    return l == 0.0f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
}

// where the partial results of a workgroup's first (0) or last (1) item lie: columns x (maximum, sum, elements)
template <int NB>
__device__ __forceinline__ float* kv_part(const KvAttnArgs& a, int64_t share, int head, int place, int column) {
    return a.part + (((share * a.c.heads + head) * 2 + place) * a.tile_columns + column) * (32 * NB + 2);
}

// ---- few columns -----------------------------------------------------------------------------------------------
// Units of all requests (each 128 tokens of one column group) are numbered through; workgroup w of W of a head
// takes the units from floor(w U / W) to floor((w + 1) U / W).
__device__ __forceinline__ int64_t kv_share_begin(int64_t w, int64_t units, int64_t shares) { return w * units / shares; }
__device__ __forceinline__ int64_t kv_share_of(int64_t unit, int64_t units, int64_t shares) {
    return ((unit + 1) * shares - 1) / units;
}

template <int DT, int NB, int CT>
__global__ __launch_bounds__(TPB, NB * CT <= 8 ? 2 : 1)
void kv_decode_kernel(KvAttnArgs a) {
    constexpr int NT = DT == MXQ_F16 ? 2 : 1, PB = NB < 4 ? NB : 4, PITCH = 32 * PB + 4;
    constexpr int CAP = 256;                             // requests scanned at a time
    static_assert(CAP == TPB, "a thread scans a request");
    __shared__ int64_t s_wave[TPB / 64];
    __shared__ int64_t s_begin[CAP];                     // first unit of each request of the scanned stretch
    __shared__ float s_ml[4][16][2];
    __shared__ __attribute__((aligned(16))) float s_acc[4][16][PITCH];
    const int head = blockIdx.x % a.c.heads, share = blockIdx.x / a.c.heads;
    const int wave = threadIdx.x >> 6;

    if (a.zero_tail && a.starts) {                       // rows behind the last request of a new output
        int64_t tail = a.starts[a.requests];
        tail = tail < 0 ? 0 : tail;
        const int heads = a.c.heads * a.group;
        for (int64_t e = tail * heads + blockIdx.x; e < a.rows * heads; e += gridDim.x) {
            unsigned short* o = kv_out_row(a, e / heads, e % heads);
            for (int d = threadIdx.x; d < a.c.head_dim; d += TPB) o[d] = 0;
            if (a.lse && threadIdx.x == 0) a.lse[e] = -__builtin_inff();
        }
    }

    int64_t total = 0;
    if (!a.whole && a.requests > CAP) {                  // with fewer, the one scan below tells it
        int64_t mine = 0;
        for (int r = threadIdx.x; r < a.requests; r += TPB) {
            const KvWork w = kv_work(a, kv_seq(a, r));
            mine += (int64_t)w.units * w.groups;
        }
        total = block_sum(mine, s_wave);
    }
    int64_t before = 0, begin = 0, end = 0;
    bool known = false;
    for (int r0 = 0; r0 < a.requests; r0 += CAP) {
        KvWork w{0, 0};
        if (r0 + (int)threadIdx.x < a.requests) w = kv_work(a, kv_seq(a, r0 + threadIdx.x));
        // with a workgroup for each item the numbers run over the items, whatever their units
        const int64_t count = a.whole ? (int64_t)w.groups : (int64_t)w.units * w.groups;
        int64_t sum;
        const int64_t upto = block_scan(count, s_wave, &sum);
        __syncthreads();
        s_begin[threadIdx.x] = before + upto - count;
        __syncthreads();
        if (!known) {
            if (a.requests <= CAP) total = sum;
            begin = a.whole ? share : kv_share_begin(share, total, a.shares);
            end = a.whole ? share + 1 : kv_share_begin(share + 1, total, a.shares);
            known = true;
        }
        const int64_t stretch_end = before + sum;
        int64_t at = begin > before ? begin : before;
        // the request of unit `at`: the last one that begins at or before it (those without units share its number
        // with the next one, so the last is the one that has it)
        int lo = 0, hi = CAP;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s_begin[mid] <= at && r0 + mid < a.requests) lo = mid;
            else hi = mid;
        }
        for (int k = lo; at < end && at < stretch_end; ++k) {
            const int r = r0 + k;
            const KvSeq s = kv_seq(a, r);
            const KvWork wk = kv_work(a, s);
            if (wk.groups == 0) continue;
            const int64_t req0 = s_begin[k];
            const int per = a.whole ? 1 : wk.units;
            for (; at < end && at < req0 + (int64_t)per * wk.groups;) {
                const int grp = (int)((at - req0) / per);
                const int64_t item0 = req0 + (int64_t)grp * per;
                const int64_t stop = end < item0 + per ? end : item0 + per;
                const int u0 = a.whole ? 0 : (int)(at - item0), u1 = a.whole ? wk.units : (int)(stop - item0);
                const bool complete = u0 == 0 && u1 == wk.units;
                const int place = item0 > begin ? 1 : 0;
                const int c0 = grp * 16 * CT, columns = s.fresh * a.group;
                KvWave<NB, CT, NT, 2> wv;
                wv.begin(a, s, head, c0);
                wv.walk(a, r, 4 * u0 + wave, 4 * u1, 4);
                // join the four waves: one tile of columns and up to four blocks at a time
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
                    const float l = sum_over_groups(wv.l[ct]);
#pragma unroll
                    for (int b0 = 0; b0 < NB; b0 += PB) {
                        const int nb = NB - b0 < PB ? NB - b0 : PB;
                        __syncthreads();                 // what was there has been read
                        if (b0 == 0 && wv.g == 0) {
                            s_ml[wave][wv.i16][0] = wv.m[ct];
                            s_ml[wave][wv.i16][1] = l;
                        }
#pragma unroll
                        for (int b = 0; b < PB; ++b)
                            if (b < nb) {
                                const kv_f32x4 even = wv.acc[ct][b0 + b][0], odd = wv.acc[ct][b0 + b][1];
                                float* dst = &s_acc[wave][wv.i16][32 * b + 8 * wv.g];
                                *reinterpret_cast<kv_f32x4*>(dst) = kv_f32x4{even[0], odd[0], even[1], odd[1]};
                                *reinterpret_cast<kv_f32x4*>(dst + 4) = kv_f32x4{even[2], odd[2], even[3], odd[3]};
                            }
                        __syncthreads();
                        // a thread takes 8 elements of a column at a time
                        for (int e = threadIdx.x; e < 64 * nb; e += TPB) {
                            const int col = e / (4 * nb), d0 = e % (4 * nb) * 8, c = c0 + 16 * ct + col;
                            if (c >= columns) continue;
                            float top = -__builtin_inff();
#pragma unroll
                            for (int w4 = 0; w4 < 4; ++w4) top = __builtin_fmaxf(top, s_ml[w4][col][0]);
                            float sum_l = 0.0f, y[8];
#pragma unroll
                            for (int x = 0; x < 8; ++x) y[x] = 0.0f;
#pragma unroll
                            for (int w4 = 0; w4 < 4; ++w4) {
                                const float mw = s_ml[w4][col][0];
                                const float f = mw == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(mw - top);
                                sum_l += s_ml[w4][col][1] * f;
#pragma unroll
                                for (int x = 0; x < 8; ++x) y[x] += s_acc[w4][col][d0 + x] * f;
                            }
                            if (complete) {
                                const float inv = sum_l == 0.0f ? 0.0f : 1.0f / sum_l;
#pragma unroll
                                for (int x = 0; x < 8; ++x) y[x] *= inv;
                                const int64_t row = s.row0 + c / a.group;
                                const int64_t qh = (int64_t)head * a.group + c % a.group;
                                kv_store8<DT>(a, kv_out_row(a, row, qh), 32 * b0 + d0, y);
                                if (a.lse && b0 == 0 && d0 == 0) a.lse[row * a.c.heads * a.group + qh] = kv_lse(top, sum_l);
                            } else {
                                float* part = kv_part<NB>(a, share, head, place, 16 * ct + col);
                                if (b0 == 0 && d0 == 0) {
                                    part[0] = top;
                                    part[1] = sum_l;
                                }
#pragma unroll
                                for (int x = 0; x < 8; ++x) part[2 + 32 * b0 + d0 + x] = y[x];
                            }
                        }
                    }
                }
                at = stop;
            }
        }
        before = stretch_end;
        if (before >= end) break;                        // uniform over the workgroup
    }
}

// One workgroup for each row and query head: adds the parts of requests that crossed workgroups, in their order.
template <int DT, int NB>
__global__ __launch_bounds__(TPB) void kv_join_kernel(KvAttnArgs a) {
    constexpr int DP = 32 * NB, LANES = DP / 4, ROWS = TPB / LANES;          // 4 elements a thread, ROWS parts at a time
    __shared__ int64_t s_wave[TPB / 64];
    __shared__ int s_request;
    __shared__ float s_ml[ROWS][2];
    __shared__ float s_acc[ROWS][DP];
    const int q_heads = a.c.heads * a.group;
    const int64_t row = blockIdx.x / q_heads;
    const int qh = blockIdx.x % q_heads, head = qh / a.group;
    int r = (int)row;
    if (a.starts) {
        if (threadIdx.x == 0) s_request = -1;
        __syncthreads();
        for (int k = threadIdx.x; k < a.requests; k += TPB) {
            const KvSeq s = kv_seq(a, k);
            if (s.row0 <= row && row < s.row0 + s.fresh) s_request = k;
        }
        __syncthreads();
        r = s_request;
        if (r < 0) return;
    }
    const KvSeq s = kv_seq(a, r);
    const KvWork wk = kv_work(a, s);
    if (wk.groups == 0) return;                          // the prompt kernel's
    int64_t mine = 0, mine_before = 0;
    for (int k = threadIdx.x; k < a.requests; k += TPB) {
        const KvWork w = kv_work(a, kv_seq(a, k));
        const int64_t n = (int64_t)w.units * w.groups;
        mine += n;
        if (k < r) mine_before += n;
    }
    const int64_t total = block_sum(mine, s_wave), before = block_sum(mine_before, s_wave);
    const int c = (int)(row - s.row0) * a.group + qh % a.group, grp = c / a.tile_columns, col = c % a.tile_columns;
    const int64_t item0 = before + (int64_t)grp * wk.units, item1 = item0 + wk.units;
    const int64_t w0 = kv_share_of(item0, total, a.shares), w1 = kv_share_of(item1 - 1, total, a.shares);
    if (w0 == w1) return;                                // written by the workgroup that had all of it
    const int lane = threadIdx.x % LANES, part_row = threadIdx.x / LANES;
    float m = -__builtin_inff(), l = 0.0f, y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (part_row < ROWS) {
        for (int64_t w = w0 + part_row; w <= w1; w += ROWS) {
            const int64_t begin = kv_share_begin(w, total, a.shares);
            if (begin == kv_share_begin(w + 1, total, a.shares)) continue;   // more workgroups than units: left nothing
            const int place = item0 > begin ? 1 : 0;
            const float* part = kv_part<NB>(a, w, head, place, col);
            const float pm = part[0], pl = part[1];
            if (pm == -__builtin_inff()) continue;       // nothing seen there
            const float up = __builtin_fmaxf(m, pm);
            const float f = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - up), fp = __builtin_amdgcn_exp2f(pm - up);
            l = l * f + pl * fp;
#pragma unroll
            for (int x = 0; x < 4; ++x) y[x] = y[x] * f + part[2 + 4 * lane + x] * fp;
            m = up;
        }
        if (lane == 0) {
            s_ml[part_row][0] = m;
            s_ml[part_row][1] = l;
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) s_acc[part_row][4 * lane + x] = y[x];
    }
    __syncthreads();
    float top = -__builtin_inff(), sum_l = 0.0f;
    for (int k = 0; k < ROWS; ++k) top = __builtin_fmaxf(top, s_ml[k][0]);
    for (int k = 0; k < ROWS; ++k)
        if (s_ml[k][0] != -__builtin_inff()) sum_l += s_ml[k][1] * __builtin_amdgcn_exp2f(s_ml[k][0] - top);
    const float inv = sum_l == 0.0f ? 0.0f : 1.0f / sum_l;
    unsigned short* o = kv_out_row(a, row, qh);
    for (int d = threadIdx.x; d < a.c.head_dim; d += TPB) {
        float v = 0.0f;
        for (int k = 0; k < ROWS; ++k)
            if (s_ml[k][0] != -__builtin_inff()) v += s_acc[k][d] * __builtin_amdgcn_exp2f(s_ml[k][0] - top);
        o[d] = (unsigned short)Pack<DT>::put(v * inv, 0.0f);
    }
    if (a.lse && threadIdx.x == 0) a.lse[row * q_heads + qh] = kv_lse(top, sum_l);
}

// ---- many columns ----------------------------------------------------------------------------------------------
// A workgroup takes 4 x 16 CT columns of a request, a quarter for each wave; the waves do not meet.
constexpr int kv_prompt_ct(int nb) { return nb <= 4 ? 4 : 2; }
template <int DT, int NB, int CT>
__global__ __launch_bounds__(TPB, NB * CT <= 8 ? 2 : 1) void kv_prompt_kernel(KvAttnArgs a) {
    constexpr int NT = DT == MXQ_F16 ? 2 : 1, NP = DT == MXQ_F16 ? 2 : 1, COLS = 64 * CT;
    __shared__ int64_t s_wave[TPB / 64];
    __shared__ int s_request, s_tile;
    const int head = blockIdx.x % a.c.heads;
    const int64_t want = blockIdx.x / a.c.heads;
    if (threadIdx.x == 0) s_request = -1;
    int64_t before = 0;
    for (int r0 = 0; r0 < a.requests; r0 += TPB) {
        int64_t n = 0, sum;
        const int r = r0 + threadIdx.x;
        if (r < a.requests) {
            const int64_t columns = (int64_t)kv_seq(a, r).fresh * a.group;
            if (columns > a.decode_columns) n = (columns + COLS - 1) / COLS;
        }
        const int64_t upto = before + block_scan(n, s_wave, &sum);
        if (want < upto && want >= upto - n) {
            s_request = r;
            s_tile = (int)(want - (upto - n));
        }
        before += sum;
    }
    __syncthreads();
    const int r = s_request;
    if (r < 0) return;
    const KvSeq s = kv_seq(a, r);
    const int columns = s.fresh * a.group;
    // the tiles that see the most come first
    const int c0 = ((columns + COLS - 1) / COLS - 1 - s_tile) * COLS + (threadIdx.x >> 6) * (16 * CT);
    if (c0 >= columns) return;
    KvWave<NB, CT, NT, NP> wv;
    wv.begin(a, s, head, c0);
    wv.walk(a, r, 0, 0x7FFFFFFF / 32, 1);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        const float l = sum_over_groups(wv.l[ct]);
        const int c = c0 + 16 * ct + wv.i16;
        if (c >= columns) continue;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const int64_t row = s.row0 + c / a.group, qh = (int64_t)head * a.group + c % a.group;
        unsigned short* o = kv_out_row(a, row, qh);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float y[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) y[x] = wv.acc[ct][b][x & 1][x >> 1] * inv;
            kv_store8<DT>(a, o, 32 * b + 8 * wv.g, y);
        }
        if (a.lse && wv.g == 0) a.lse[row * a.c.heads * a.group + qh] = kv_lse(wv.m[ct], l);
    }
}

}  // namespace
