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
// What bounds it, measured at 8 kv heads of 128 with 4 query heads each: reading the cache for single tokens (64 requests of
// 128 - 8192 tokens, 135 MB: 33.4 us, 5.6 TB/s while the waves walk; 131072 + 2048 tokens 31.8 us), instruction issue for
// prompts (4001 tokens behind 12000: a call 1.00 ms, 917 TFLOP/s, matrix instructions 39 % and vector instructions 47 %
// of the cycles).  A tile of 32 tokens costs 257 vector instructions, 64 of them conversions from fp4.  The 4-bit scaled matrix
// instruction, which would take K as it lies, is not used: its sums are off by 2^-13.5 of their absolute terms.
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
    KvDivide by_group, by_heads, by_q_heads, by_shares;
    int64_t rows;                                        // rows of q and out
    float scale_log2;                                    // |scale| log2(e)
    int negative;                                        // scale is
    int causal, q_wide, out_wide, zero_tail;
    int item_shift;                                      // decode: an item has 2^item_shift = 16 CT columns
    int decode_columns;                                  // requests with more columns belong to the prompt kernel
    int whole;                                           // decode: a workgroup for each item, nothing to join
    int direct;                                          // .. and one item for each request
    int shares;                                          // decode: workgroups of a kv head, at most KV_MAX_SHARES
    int join_rows;                                       // join: so many rows of each request, or 0: every row
    int* spans;                                          // decode: where the parts of each item lie (two numbers, KvShares)
    float* part;                                         // decode: partial results, two places for each workgroup
    int join_blocks;                                     // join: workgroups for decode rows, the others for prompt items
    int join_first;                                      // join: the first workgroup of this launch
    int prompt_shares, prompt_items;                     // prompt: workgroups of a kv head and items of it, at most
    float* prompt_part;
    void* plan;                                          // null: no prompt kernel
    KvCache c;
};

// a request as the attention sees it
struct KvSeq {
    int row0;                                            // its first row of q
    int fresh;                                           // its rows
    int len;                                             // tokens, unlimited
    int keys;                                            // tokens that the table can name
};
__device__ __forceinline__ KvSeq kv_seq(const KvAttnArgs& a, int r) {
    KvSeq s;
    if (a.starts) {
        const int rows = (int)a.rows;                    // (below 2^31)
        int s0 = a.starts[r], s1 = a.starts[r + 1];
        s0 = s0 < 0 ? 0 : (s0 < rows ? s0 : rows);
        s1 = s1 < s0 ? s0 : (s1 < rows ? s1 : rows);
        s.row0 = s0;
        s.fresh = s1 - s0;
    } else {
        s.row0 = r;
        s.fresh = 1;
    }
    s.len = a.seq_lens[r] > 0 ? a.seq_lens[r] : 0;
    const int room = a.width * a.c.page_size;            // (at most 2^30)
    s.keys = s.len < room ? s.len : room;
    return s;
}
// keys that new token i sees (0 or less: none)
__device__ __forceinline__ int kv_limit(const KvAttnArgs& a, const KvSeq& s, int i) {
    if (!a.causal) return s.keys;
    const int64_t n = (int64_t)s.len - s.fresh + i + 1;
    return n < s.keys ? (int)(n > 0 ? n : 0) : s.keys;
}

// the running maximum before anything has been seen: below every score, but finite, so that neither a difference of two
// of them nor one with a masked score's -inf is NaN
constexpr float KV_NOTHING = -3.0e38f;
constexpr int KV_MAX_SHARES = 1024;
constexpr int KV_UNIT = 128;                             // tokens of a unit of work: a tile of 32 for each wave
constexpr int KV_ITEM_UNITS = 3;                         // what beginning and ending an item counts for when work is dealt out

// units and column groups of a request in the decode kernel; a request without keys still has one unit, whose
// workgroup writes the zeros
struct KvWork {
    int units, groups;
    __device__ __forceinline__ int per() const { return units + KV_ITEM_UNITS; }
    __device__ __forceinline__ int count() const { return per() * groups; }  // (all of them together: below 2^31)
};
__device__ __forceinline__ KvWork kv_work(const KvAttnArgs& a, const KvSeq& s) {
    const int columns = s.fresh * a.group;
    if (columns == 0 || columns > a.decode_columns) return KvWork{0, 0};
    const int units = (s.keys + KV_UNIT - 1) / KV_UNIT;
    return KvWork{units > 0 ? units : 1, (columns + (1 << a.item_shift) - 1) >> a.item_shift};
}

// ---- loads -------------------------------------------------------------------------------------------------------
// Memory that is named by a uniform address, a uniform distance from it and an offset of the lane's own: buffer loads take
// the three as they are, without arithmetic in vector registers.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t kv_buffer(const unsigned char* base) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(base), 0, 0xFFFFFFFF, 0x00027000);
}
// N dwords from an address that is aligned to min(4 N, 16) bytes where N is a power of two, to 4 otherwise
template <int N>
__device__ __forceinline__ void load_dwords(__amdgpu_buffer_rsrc_t from, int lane_offset, int offset, uint32_t* d) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const u32x4 w = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(from, lane_offset + 16 * i, offset, 0));
#pragma unroll
            for (int e = 0; e < 4; ++e) d[4 * i + e] = w[e];
        }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(from, lane_offset + 8 * i, offset, 0));
            d[2 * i] = w[0];
            d[2 * i + 1] = w[1];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) d[i] = __builtin_amdgcn_raw_buffer_load_b32(from, lane_offset + 4 * i, offset, 0);
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
    uint32_t all = ks[0];                                // bytes side by side, picked by a shift
#pragma unroll
    for (int k = 1; k < N; ++k) all |= ks[k] << (8 * k);
    return all >> (8 * ((NB * g + s) / 4 - NB * g / 4));  // what is above the byte is shifted out or ignored
}

// A copy of a value that the compiler takes for a new one.  What rarely taken branches work out from a lane's number would
// otherwise be worked out before the loops around them and occupy registers throughout (16 of them for the masks).
__device__ __forceinline__ int here_only(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

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
// eight K elements of a lane as an operand
__device__ __forceinline__ kv_bf16x8 kv_k_operand(uint32_t codes, uint32_t scale) {
    const uint32_t bits = scale << 23;
    return kv_operand(kv_decode2<0>(codes, bits), kv_decode2<1>(codes, bits), kv_decode2<2>(codes, bits),
                      kv_decode2<3>(codes, bits));
}
// the two V operands of a block from a lane's codes and scales of two groups of four tokens
__device__ __forceinline__ void kv_v_operands(const uint32_t codes[2], const uint32_t scales[2], kv_bf16x8 out[2]) {
    uint32_t cv[8];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        cv[4 * j + 0] = kv_decode2<0>(codes[j], kv_scale_bits<0>(scales[j]));
        cv[4 * j + 1] = kv_decode2<1>(codes[j], kv_scale_bits<1>(scales[j]));
        cv[4 * j + 2] = kv_decode2<2>(codes[j], kv_scale_bits<2>(scales[j]));
        cv[4 * j + 3] = kv_decode2<3>(codes[j], kv_scale_bits<3>(scales[j]));
    }
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const uint32_t sel = n ? 0x07060302u : 0x05040100u;                  // the upper or lower halves of two dwords
        out[n] = kv_operand(__builtin_amdgcn_perm(cv[1], cv[0], sel), __builtin_amdgcn_perm(cv[3], cv[2], sel),
                            __builtin_amdgcn_perm(cv[5], cv[4], sel), __builtin_amdgcn_perm(cv[7], cv[6], sel));
    }
}

// The V scales of a masked tile of 32 tokens (t0 ..; a lane: tokens 4 g + r of halves j): tokens behind `end` or on
// missing pages and elements that are NaN or Inf get the scale 2^-127, since even a probability of 0 times one of them is NaN.
// Returns in which of the 32 tokens the block has such an element; their columns are told by spread_nan.  (A code of 2^2 and
// more times 2^126, or of 2 and more times 2^127, is Inf: the quantizer gets there with bf16 values from 2^127 * 1.75 on.)
__device__ __forceinline__ uint32_t kv_mend_scales(uint32_t scales[2], const uint32_t codes[2], const bool there[2], int t0, int g,
                                                   int end) {
    uint32_t high = 0;                                   // has a byte from 253 on
    g = here_only(g);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (!(there[j] && t0 + 16 * j + 4 * g + r < end)) scales[j] &= ~(255u << (8 * r));
        high |= ((scales[j] & 0x7F7F7F7Fu) + 0x03030303u) & scales[j] & 0x80808080u;
    }
    if (!any_lane(high != 0u)) return 0;
    uint32_t bad = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint32_t scale = (scales[j] >> (8 * r)) & 255u, pair = codes[j] >> (8 * r);
            const uint32_t least = scale == 255u ? 0u : scale == 254u ? 4u : 6u;
            if (scale >= 253u && ((pair & 7u) >= least || ((pair >> 4) & 7u) >= least)) {
                bad |= 1u << (16 * j + 4 * g + r);
                scales[j] &= ~(255u << (8 * r));
            }
        }
    for (int d = 1; d < 16; d <<= 1) bad |= (uint32_t)__shfl_xor((int)bad, d, 64);           // (a lane has two elements of the block)
    return or_over_groups(bad);
}

// Eight 16-bit elements e0 .. of a row that ends at `end`, where rows are not aligned.  A loop, not unrolled: unrolled,
// its conditions would occupy scalar registers through the kernels' main loops.
__device__ __forceinline__ void kv_store8_unaligned(unsigned short* row, int e0, int end, u32x4 w) {
    const uint64_t half[2] = {(uint64_t)w[1] << 32 | w[0], (uint64_t)w[3] << 32 | w[2]};
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma nounroll
        for (int e = 0; e < 4; ++e)
            if (e0 + 4 * h + e < end) row[e0 + 4 * h + e] = (unsigned short)(half[h] >> (16 * e));
}

template <int NB>
struct KvKeys {                                          // what a lane holds of 32 tokens' keys ..
    uint32_t k[2][NB], ks[2][kv_k_scales<NB>()];
};
template <int NB>
struct KvValues {                                        // .. and values
    uint32_t v[2][NB], vs[2][NB];
};

// Waves that share a SIMD take their turns by priority, then by age: left to age alone, the oldest workgroup of a compute
// unit is done long before the youngest, which then has nobody to hide its waits behind.  So a wave lowers its priority
// with every quarter of its work (64 requests with 1900 tokens on average, 8 x 4 heads of 128: 36.7 -> 34.6 us; the
// prompts below: 84.0 -> 75.5).
struct KvPace {
    int left, quarter;                                   // units of work, a tile of the wave each
    __device__ __forceinline__ void at(int units_left) {
        left = units_left;
        if (left > 3 * quarter) __builtin_amdgcn_s_setprio(3);
        else if (left > 2 * quarter) __builtin_amdgcn_s_setprio(2);
        else if (left > quarter) __builtin_amdgcn_s_setprio(1);
        else __builtin_amdgcn_s_setprio(0);
    }
    __device__ __forceinline__ void tile() {
        --left;
        if (left == 3 * quarter) __builtin_amdgcn_s_setprio(2);
        else if (left == 2 * quarter) __builtin_amdgcn_s_setprio(1);
        else if (left == quarter) __builtin_amdgcn_s_setprio(0);
    }
};

// the columns of a wave
template <int NB, int CT, int NT, int NP>
struct KvWave {
    kv_f32x4 acc[CT][NB][2];                             // element 32 b + 2 (4 g + r) + n of the lane's column
    float m[CT], l[CT];                                  // l: this lane's tokens only
    kv_bf16x8 q[CT][NT][NB];
    uint32_t limits;                                     // keys that the lane's columns see beyond min_limit: 8 bits each
    bool started;                                        // every column has seen a token (uniform)
    int min_limit, max_limit;                            // over the wave's columns
    int lane, i16, g;

    // Columns c0 .. c0 + 16 CT - 1 of request s.  Called by all waves of the workgroup; stage: 32 NB x 16 16-bit elements
    // of LDS for each wave, which q passes through where its rows are not aligned.
    __device__ __forceinline__ void begin(const KvAttnArgs& a, const KvSeq& s, int head, int c0, unsigned short* stage) {
        lane = threadIdx.x & 63;
        i16 = lane & 15;
        g = lane >> 4;
        const int columns = s.fresh * a.group;
        const int last = (c0 + 16 * CT < columns ? c0 + 16 * CT : columns) - 1;
        min_limit = kv_limit(a, s, a.by_group.of(c0));
        max_limit = kv_limit(a, s, a.by_group.of(last));
        started = false;
        limits = 0;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            m[ct] = KV_NOTHING;
            l[ct] = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b) acc[ct][b][0] = acc[ct][b][1] = kv_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            const int c = c0 + 16 * ct + i16, token = a.by_group.of(c);
            const bool live = c < columns;
            limits |= (uint32_t)((live ? kv_limit(a, s, token) : max_limit) - min_limit) << (8 * ct);   // (at most 16 CT tokens apart)
            const unsigned short* row = a.q + (int64_t)(s.row0 + (live ? token : 0)) * a.q_token +
                                        ((int64_t)head * a.group + (live ? c - token * a.group : 0)) * a.q_head;
            if (!a.q_wide) {
                __syncthreads();                         // what was there has been read
#pragma nounroll
                for (int e = here_only(lane); e < 16 * 32 * NB; e += 64) {
                    const int x = c0 + 16 * ct + e / (32 * NB), d = e % (32 * NB), t = a.by_group.of(x);
                    unsigned short v = 0;
                    if (x < columns && d < a.c.head_dim)
                        v = a.q[(int64_t)(s.row0 + t) * a.q_token + ((int64_t)head * a.group + (x - t * a.group)) * a.q_head + d];
                    stage[e] = v;
                }
                __syncthreads();
            }
#pragma unroll
            for (int st = 0; st < NB; ++st) {
                const int e0 = 8 * NB * g + 8 * st;
                u32x4 w = {0, 0, 0, 0};
                if (!a.q_wide) w = *reinterpret_cast<const u32x4*>(stage + i16 * (32 * NB) + e0);
                else if (live && e0 < a.c.head_dim) w = *reinterpret_cast<const u32x4*>(row + e0);
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

    __device__ __forceinline__ int limit(int ct) const { return min_limit + (int)(limits >> (8 * ct) & 255u); }

    // sc (+)= (operand of half j, step st) x q
    __device__ __forceinline__ void multiply_keys(const kv_bf16x8& k8, int j, int st, kv_f32x4 sc[CT][2]) const {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                sc[ct][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    k8, q[ct][nt][st], st == 0 && nt == 0 ? kv_f32x4{0.0f, 0.0f, 0.0f, 0.0f} : sc[ct][j], 0, 0, 0);
    }

    // scores of 32 tokens from t0 to probabilities, in place of which the maximum and the sums follow
    __device__ __forceinline__ void probabilities(const KvAttnArgs& a, kv_f32x4 sc[CT][2], bool masked, const bool there[2], int t0,
                                                  uint32_t p_hi[CT][4], uint32_t p_lo[CT][4]) {
        if (a.negative) {
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                sc[ct][0] = -sc[ct][0];
                sc[ct][1] = -sc[ct][1];
            }
        }
        if (masked) {
            const int first = t0 + 4 * here_only(g);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const bool seen = there[e >> 2] && first + 16 * (e >> 2) + (e & 3) < limit(ct);
                    sc[ct][e >> 2][e & 3] = seen ? sc[ct][e >> 2][e & 3] : -__builtin_inff();
                }
        }
        if (!started) {                                  // columns that have not seen a token yet begin with this tile's maximum
            bool waiting = false;
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                float mx = sc[ct][0][0];
#pragma unroll
                for (int e = 1; e < 8; ++e) mx = __builtin_fmaxf(mx, sc[ct][e >> 2][e & 3]);
                mx = max_over_groups(mx) * a.scale_log2; // (a scale of 0 is passed as the smallest normal number)
                if (m[ct] == KV_NOTHING) m[ct] = mx > KV_NOTHING ? mx : KV_NOTHING;
                waiting |= m[ct] == KV_NOTHING;
            }
            started = !any_lane(waiting);
        }
        // s - m; m is raised, and only then do the lane groups compare, after a jump by more than 8
        bool jump = false;
        float over[CT];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                sc[ct][e >> 2][e & 3] = __builtin_fmaf(sc[ct][e >> 2][e & 3], a.scale_log2, -m[ct]);
            over[ct] = sc[ct][0][0];
#pragma unroll
            for (int e = 1; e < 8; ++e) over[ct] = __builtin_fmaxf(over[ct], sc[ct][e >> 2][e & 3]);
            jump |= over[ct] > 8.0f;
        }
        if (any_lane(jump)) {
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                const float top = max_over_groups(over[ct]), up = top > 8.0f ? top : 0.0f;
                const float f = __builtin_amdgcn_exp2f(-up);                 // 1 where m stays
                m[ct] += up;
                l[ct] *= f;
#pragma unroll
                for (int e = 0; e < 8; ++e) sc[ct][e >> 2][e & 3] -= up;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[ct][b][n][r] *= f;
            }
        }
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(sc[ct][e >> 2][e & 3]);
            l[ct] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                p_hi[ct][d] = Pack<MXQ_BF16>::put(p[2 * d], p[2 * d + 1]);
                if constexpr (NP == 2)
                    p_lo[ct][d] = Pack<MXQ_BF16>::put(p[2 * d] - Pack<MXQ_BF16>::get(p_hi[ct][d], 0),
                                                      p[2 * d + 1] - Pack<MXQ_BF16>::get(p_hi[ct][d], 1));
            }
        }
    }

    // acc += (V operand n of block b) x probabilities
    __device__ __forceinline__ void multiply_values(const kv_bf16x8& v8, int b, int n, const uint32_t p_hi[CT][4],
                                                    const uint32_t p_lo[CT][4]) {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            acc[ct][b][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                v8, kv_operand(p_hi[ct][0], p_hi[ct][1], p_hi[ct][2], p_hi[ct][3]), acc[ct][b][n], 0, 0, 0);
            if constexpr (NP == 2)
                acc[ct][b][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    v8, kv_operand(p_lo[ct][0], p_lo[ct][1], p_lo[ct][2], p_lo[ct][3]), acc[ct][b][n], 0, 0, 0);
        }
    }

    // block b has NaN or Inf in the tokens `of` (of 32 from t0): it is NaN in the columns that see one of them
    __device__ __forceinline__ void spread_nan(int b, uint32_t of, int t0) {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            const int n = limit(ct) - t0;
            const uint32_t sees = n >= 32 ? 0xFFFFFFFFu : n > 0 ? (1u << n) - 1u : 0u;
            if (of & sees) {
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[ct][b][0][r] = acc[ct][b][1][r] = mxq_float(MXQ_QNAN_BITS);
            }
        }
    }

    // ---- straight from memory (the decode kernel) ----
    // a lane's constant offsets into the halves of a tile
    int at_k, at_v, at_ks[kv_k_scales<NB>()], at_vs;
    __device__ __forceinline__ void place(const KvAttnArgs& a) {
        const int ps = a.c.page_size;
        at_k = i16 * (16 * NB) + g * (4 * NB);
        at_v = ps * (16 * NB) + g * (64 * NB) + i16 * (4 * NB);
        at_vs = ps * NB + g * (4 * NB);
#pragma unroll
        for (int k = 0; k < kv_k_scales<NB>(); ++k) {
            const int b = NB * g / 4 + k;
            at_ks[k] = i16 * NB + (b < NB ? b : NB - 1);
        }
    }
    // 16 tokens in the cache, for the loads of a wave: where their K codes lie (V's are a page's K codes further), how far
    // it is from there to their K scales (V's are a page's K scales further), and whether the page exists (else: the
    // first tokens of the cache, whose scores are masked)
    struct Spot {
        int64_t codes;
        int scales;
        bool there;
    };
    __device__ __forceinline__ static Spot spot(const KvAttnArgs& a, const int* row, int head, int sub, int end) {
        const int subs = a.c.page_size / 16, at = (int)kv_page_of(a.c, 16u * (uint32_t)sub);
        int page = -1, in_page = 0;
        if (at < a.width && sub < end) {
            page = row[at];
            if (page >= a.c.num_pages) page = -1;
            if (page >= 0) in_page = sub - at * subs;
        }
        Spot p;
        p.there = page >= 0;
        p.codes = ((int64_t)(page >= 0 ? page : 0) * a.c.heads + head) * a.c.record + in_page * (256 * NB);
        p.scales = a.c.page_size * (32 * NB) - in_page * (240 * NB);
        return p;
    }
    __device__ __forceinline__ static __amdgpu_buffer_rsrc_t lane_codes(const KvAttnArgs& a, const Spot& p, int l) {
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)p.codes, l);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)p.codes >> 32), l);
        return kv_buffer(a.c.data + (((uint64_t)hi << 32) | lo));
    }
    __device__ __forceinline__ void fetch_keys(const KvAttnArgs& a, KvKeys<NB>& t, const Spot& p, int n) const {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const __amdgpu_buffer_rsrc_t from = lane_codes(a, p, 2 * n + j);
            const int scales = __builtin_amdgcn_readlane(p.scales, 2 * n + j);
            load_dwords<NB>(from, at_k, 0, t.k[j]);
#pragma unroll
            for (int k = 0; k < kv_k_scales<NB>(); ++k) t.ks[j][k] = __builtin_amdgcn_raw_buffer_load_b8(from, at_ks[k], scales, 0);
        }
    }
    __device__ __forceinline__ void fetch_values(const KvAttnArgs& a, KvValues<NB>& t, const Spot& p, int n) const {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const __amdgpu_buffer_rsrc_t from = lane_codes(a, p, 2 * n + j);
            load_dwords<NB>(from, at_v, 0, t.v[j]);
            load_dwords<NB>(from, at_vs, __builtin_amdgcn_readlane(p.scales, 2 * n + j), t.vs[j]);
        }
    }

    // The tiles first, first + stride, .. of 32 tokens below tile `end`.  The places of 32 tiles sit in the lanes (lane:
    // tile lane / 2, half lane % 2).  A tile's keys are loaded as soon as the last one's, in the same registers, have been
    // multiplied, its values likewise.
    __device__ __forceinline__ void walk(const KvAttnArgs& a, int r, int head, int first, int end, int stride, KvPace& pace) {
        const int seen_end = (max_limit + 31) / 32;      // uniform: nothing behind it is seen
        if (end > seen_end) end = seen_end;
        place(a);
        const int* row = a.table + (int64_t)r * a.table_stride;
        for (int chunk = first; chunk < end; chunk += 32 * stride) {
            const Spot p = spot(a, row, head, 2 * (chunk + (lane >> 1) * stride) + (lane & 1), (max_limit + 15) / 16);
            const uint64_t there = __ballot(p.there);
            int tiles = (end - chunk + stride - 1) / stride;
            if (tiles > 32) tiles = 32;
            KvKeys<NB> keys;
            KvValues<NB> values;
            // no load is conditional: behind the last tile it is loaded again.  The waits count the loads under way, and a
            // branch around one would make them wait for more than needed.  They are issued in the loop's order, on which
            // the waits rely.
            const int last = tiles - 1;
            fetch_keys(a, keys, p, 0);
            __builtin_amdgcn_sched_barrier(0);
            fetch_values(a, values, p, 0);
            __builtin_amdgcn_sched_barrier(0);
            for (int n = 0; n < tiles; ++n) {
                pace.tile();
                step(a, keys, values, p, (int)(there >> (2 * n)) & 3, n < last ? n + 1 : last, 32 * (chunk + n * stride));
            }
        }
    }
    // the tokens t0 .. (there_bits: which halves exist) from their registers, which then take tile `after`
    __device__ __forceinline__ void step(const KvAttnArgs& a, KvKeys<NB>& keys, KvValues<NB>& values, const Spot& p, int there_bits,
                                         int after, int t0) {
        kv_f32x4 sc[CT][2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int st = 0; st < NB; ++st)
                multiply_keys(kv_k_operand(keys.k[j][st], kv_k_scale<NB>(keys.ks[j], g, st)), j, st, sc);
        fetch_keys(a, keys, p, after);
        // a tile that every column sees entirely needs no mask
        const bool there[2] = {(there_bits & 1) != 0, (there_bits & 2) != 0};
        const bool masked = t0 + 32 > min_limit || there_bits != 3;
        uint32_t p_hi[CT][4], p_lo[CT][4];
        probabilities(a, sc, masked, there, t0, p_hi, p_lo);
        uint32_t nan_of[NB];
        bool any_nan = false;
        if (masked) {
            uint32_t all = 0;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                uint32_t scales[2] = {values.vs[0][b], values.vs[1][b]};
                const uint32_t codes[2] = {values.v[0][b], values.v[1][b]};
                nan_of[b] = kv_mend_scales(scales, codes, there, t0, g, max_limit);
                values.vs[0][b] = scales[0];
                values.vs[1][b] = scales[1];
                all |= nan_of[b];
            }
            any_nan = uniform((int)all) != 0;
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const uint32_t codes[2] = {values.v[0][b], values.v[1][b]}, scales[2] = {values.vs[0][b], values.vs[1][b]};
            kv_bf16x8 v8[2];
            kv_v_operands(codes, scales, v8);
#pragma unroll
            for (int n2 = 0; n2 < 2; ++n2) multiply_values(v8[n2], b, n2, p_hi, p_lo);
        }
        fetch_values(a, values, p, after);
        if (any_nan) {                                   // rare
#pragma unroll
            for (int b = 0; b < NB; ++b) spread_nan(b, nan_of[b], t0);
        }
    }
};

// rounds to the output type and stores elements e0 .. e0 + 7 of a row
template <int DT, bool WIDE = false>
__device__ __forceinline__ void kv_store8(const KvAttnArgs& a, unsigned short* row, int e0, const float* y) {
    if (e0 >= a.c.head_dim) return;
    const u32x4 w = {Pack<DT>::put(y[0], y[1]), Pack<DT>::put(y[2], y[3]), Pack<DT>::put(y[4], y[5]), Pack<DT>::put(y[6], y[7])};
    if (WIDE || a.out_wide) *reinterpret_cast<u32x4*>(row + e0) = w;
    else kv_store8_unaligned(row, e0, a.c.head_dim, w);
}
__device__ __forceinline__ unsigned short* kv_out_row(const KvAttnArgs& a, int64_t row, int64_t q_head) {
    return a.out + row * a.out_token + q_head * a.out_head;
}
// natural logarithm of the sum of exponentials; -inf where nothing was seen
__device__ __forceinline__ float kv_lse(float m, float l) {
    return l == 0.0f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
}

// where the partial results of a workgroup's first (0) or last (1) item lie, by column: elements, and behind all of
// them maximum and sum
__device__ __forceinline__ int64_t kv_part_row(const KvAttnArgs& a, int64_t share, int head, int place, int column) {
    return ((((share * a.c.heads + head) * 2 + place) << a.item_shift) + column);
}
template <int NB>
__device__ __forceinline__ float* kv_part(const KvAttnArgs& a, int64_t row) { return a.part + row * (32 * NB); }
template <int NB>
__device__ __forceinline__ float* kv_part_ml(const KvAttnArgs& a, int64_t row) {
    return a.part + ((int64_t)a.shares * a.c.heads * 2 << a.item_shift) * (32 * NB) + 2 * row;
}

template <int DT>
constexpr int kv_terms() { return DT == MXQ_F16 ? 2 : 1; }
// columns of a wave, in tiles of 16: accumulators and q fill about 160 of the 256 registers that leave two waves a SIMD
constexpr int kv_prompt_ct(int nb, int terms) {
    return nb * (8 + 4 * terms) * 4 <= 120 ? 4 : nb * (8 + 4 * terms) * 3 <= (terms == 1 ? 144 : 120) ? 3 : nb * (8 + 4 * terms) * 2 <= 160 ? 2 : 1;
}

// Items (a request's columns, COLS at a time) differ in the tokens they see, and a grid of items rarely fills the chip
// evenly.  So the work is numbered through -- an item counts the tokens it sees, in units of 1 / G -- and every workgroup
// of a head takes an equal stretch of the numbers: an item that a stretch ends in is cut between two of its tiles of 64
// tokens, and the join kernel adds its parts.  Numbers are closed forms of the group, so a place is found without a table.
// One workgroup of the decode kernel's launch, which comes first, works the stretches out (kv_plan), the same for every
// head: in the prompt kernel itself their arithmetic in 64 bits would hold registers that its loop needs.
// Tokens that beginning and ending an item counts for (three requests of 1024, 768 and 256 tokens behind 64, 256 and 4096,
// 8 x 4 heads of 128: 82.6 us with 64, 75.5 with 192, 78.1 with 320).
constexpr int KV_PROMPT_BEGIN = 192;
struct KvPrompt {
    int groups;
    int64_t first;                                       // what group 0 counts; a later one `step` more than the one before
    int64_t step;
    __device__ __forceinline__ int64_t begin(int64_t g) const { return g * first + step * (g * (g - 1) / 2); }
    __device__ __forceinline__ int group_of(int64_t number) const {          // number < begin(groups)
        int lo = 0, hi = groups;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (begin(mid) <= number) lo = mid;
            else hi = mid;
        }
        return lo;
    }
};
__device__ __forceinline__ KvPrompt kv_prompt(const KvAttnArgs& a, const KvSeq& s, int cols) {
    const int columns = s.fresh * a.group;
    if (columns == 0 || columns <= a.decode_columns) return KvPrompt{0, 0, 0};
    const int64_t seen = a.causal ? (s.len > s.fresh ? s.len - s.fresh : 0) : s.keys;
    return KvPrompt{(columns + cols - 1) / cols, (seen + KV_PROMPT_BEGIN) * a.group + (a.causal ? cols / 2 : 0), a.causal ? cols : 0};
}
struct KvStretch {
    int64_t each, more;
    int shares;
    // no stretch is shorter than 256 tokens for an item
    __device__ __forceinline__ KvStretch(const KvAttnArgs& a, int64_t total) {
        const int64_t most = total / (256 * a.group);
        shares = most < 1 ? 1 : most < a.prompt_shares ? (int)most : a.prompt_shares;
        each = total / shares;
        more = total - each * shares;
    }
    __device__ __forceinline__ int64_t begin(int64_t w) const { return w * each + (w < more ? w : more); }
    __device__ __forceinline__ int of(int64_t number) const {
        const int64_t big = more * (each + 1);
        return number < big ? (int)(number / (each + 1)) : (int)(more + (number - big) / each);
    }
};
// tiles of group g and the first one behind number x (x inside the group's numbers or beyond)
__device__ __forceinline__ int kv_prompt_tiles(const KvAttnArgs& a, const KvSeq& s, int g, int cols) {
    const int columns = s.fresh * a.group;
    const int last = ((g + 1) * cols < columns ? (g + 1) * cols : columns) - 1;
    return (kv_limit(a, s, a.by_group.of(last)) + 63) / 64;
}
__device__ __forceinline__ int kv_prompt_cut(const KvPrompt& p, int g, int tiles, int64_t x) {
    const int64_t b = p.begin(g), e = p.begin(g + 1);
    if (x <= b) return 0;
    if (x >= e) return tiles;
    return (int)((double)(x - b) / (double)(e - b) * tiles);
}

// what kv_plan leaves in the workspace
struct KvPiece {                                         // of an item, for a workgroup: tiles tile0 .. tile1 - 1
    int request, group_flags, tile0, tile1;              // flags: 2 the whole item, 1 its second place for parts
};
struct KvPlanView {
    int* head;                                           // items, shares
    int* items;                                          // of each item: first and last share that it lies in
    int* shares;                                         // of each share: its first piece, number of pieces, tiles of them all
    KvPiece* pieces;                                     // of item i in share w: at i + w
    int64_t* first;                                      // of each request: its first number
    int* item;                                           // .. and its first item
};
// (items + shares pieces; 16-byte pieces first)
__host__ __device__ __forceinline__ int64_t kv_plan_bytes(int64_t items, int64_t shares, int64_t requests) {
    return 16 * (items + shares) + 8 * requests + 4 * (2 + 2 * items + 3 * shares + requests);
}
__device__ __forceinline__ KvPlanView kv_plan_view(const KvAttnArgs& a) {
    KvPlanView v;
    v.pieces = reinterpret_cast<KvPiece*>(a.plan);
    v.first = reinterpret_cast<int64_t*>(v.pieces + a.prompt_items + a.prompt_shares);
    v.head = reinterpret_cast<int*>(v.first + a.requests);
    v.items = v.head + 2;
    v.shares = v.items + 2 * (int64_t)a.prompt_items;
    v.item = v.shares + 3 * (int64_t)a.prompt_shares;
    return v;
}
__device__ __forceinline__ void kv_plan(const KvAttnArgs& a, int cols, int64_t* s_wave64, int* s_wave) {
    const KvPlanView v = kv_plan_view(a);
    int64_t total = 0;
    int items = 0;
    for (int r0 = 0; r0 < a.requests; r0 += TPB) {
        const int r = r0 + threadIdx.x;
        KvPrompt p{0, 0, 0};
        if (r < a.requests) p = kv_prompt(a, kv_seq(a, r), cols);
        int64_t sum;
        int group_sum;
        const int64_t count = p.begin(p.groups), upto = block_scan(count, s_wave64, &sum);
        const int group_upto = block_scan(p.groups, s_wave, &group_sum);
        if (r < a.requests) {
            v.first[r] = total + upto - count;
            v.item[r] = items + group_upto - p.groups;
        }
        total += sum;
        items += group_sum;
    }
    __syncthreads();
    const KvStretch deal(a, total);
    if (threadIdx.x == 0) {
        v.head[0] = items < 0 || items > a.prompt_items ? a.prompt_items : items;
        v.head[1] = total > 0 ? deal.shares : 0;
    }
    if (total == 0) return;
    for (int w = threadIdx.x; w < deal.shares; w += TPB) {
        const int64_t from = deal.begin(w), to = deal.begin(w + 1);
        int lo = 0, hi = a.requests;                     // the last request that begins at or before `from` has it
        while (hi - lo > 1) {
            const int mid = lo + (hi - lo) / 2;
            if (v.first[mid] <= from) lo = mid;
            else hi = mid;
        }
        int begun = -1, count = 0, all_tiles = 0;
        for (int r = lo; r < a.requests; ++r) {
            const int64_t number = v.first[r];
            if (number >= to) break;
            const KvSeq s = kv_seq(a, r);
            const KvPrompt p = kv_prompt(a, s, cols);
            if (p.groups == 0) continue;
            for (int g = from > number ? p.group_of(from - number) : 0; g < p.groups && number + p.begin(g) < to; ++g) {
                const int tiles = kv_prompt_tiles(a, s, g, cols), item = v.item[r] + g;
                if ((uint32_t)item >= (uint32_t)a.prompt_items) break;       // (starts that are not in order name rows twice)
                const int tile0 = kv_prompt_cut(p, g, tiles, from - number), tile1 = kv_prompt_cut(p, g, tiles, to - number);
                const bool begins = number + p.begin(g) >= from;
                const bool whole = tile1 - tile0 == tiles && (tiles > 0 || begins);
                v.pieces[item + w] = KvPiece{r, 4 * g + (whole ? 2 : 0) + (number + p.begin(g) > from ? 1 : 0), tile0, tile1};
                if (begins) {
                    v.items[2 * item] = w;
                    v.items[2 * item + 1] = deal.of(number + p.begin(g + 1) - 1);
                }
                if (begun < 0) begun = item + w;
                ++count;
                all_tiles += tile1 - tile0;
            }
        }
        v.shares[3 * w] = begun;
        v.shares[3 * w + 1] = count;
        v.shares[3 * w + 2] = all_tiles;
    }
}

// ---- few columns -----------------------------------------------------------------------------------------------
// Units of all requests (each 128 tokens of one column group) are numbered through and dealt out to the workgroups of a
// head in order, as evenly as it goes: the first `more` of them have one number more than `each`.  Beginning and ending
// an item (its q, the first loads, the sum over four waves) takes as long as some units, so every item has KV_ITEM_UNITS
// numbers before its units: without them a workgroup with four short requests ended long after the others (64 requests of
// 128 to 8192 tokens: 39.1 us; with 2, 3, 4 of them 34.3, 34.6, 35.7; 32 requests of 32 to 2048: 16.0 and 14.2, 13.7, 13.8).
struct KvShares {
    int each = 0, more = 0;
    KvShares() = default;
    __device__ __forceinline__ KvShares(const KvAttnArgs& a, int units) : each(a.by_shares.of(units)), more(units - each * a.shares) {}
    __device__ __forceinline__ int begin(int w) const { return w * each + (w < more ? w : more); }
};

// The first item (16 CT columns of a request) of request r, in an order that needs no sums over requests: every item has a
// number of its own, below rows G / (16 CT) + requests.
__device__ __forceinline__ int kv_item(const KvAttnArgs& a, const KvSeq& s, int r) { return ((s.row0 * a.group) >> a.item_shift) + r; }

// Waves that share a SIMD, from the registers of a wave: accumulators, q, the tile under way and the rest (as the compiler
// needs them; 7 blocks, and 6 with fp16 queries, would spill at two waves).  More waves than fit lose more to spills than they
// hide: 4 blocks at four waves 49.6 us instead of 41.8 (64 requests of 128 - 8192 tokens, 8 x 4 heads of 128).
constexpr int kv_decode_registers(int nb, int ct, int terms) { return nb * (8 * ct + 4 * ct * terms + 7) + 72 + 18 * ct + 10 * (terms - 1); }
constexpr int kv_decode_waves(int nb, int ct, int terms) {
    const int n = kv_decode_registers(nb, ct, terms);
    return n <= 126 ? 4 : n <= 168 ? 3 : n <= 245 && nb != 7 && (nb != 6 || terms == 1) ? 2 : 1;
}
// two tiles of columns for one reading of the tokens, where the registers allow it
constexpr int kv_decode_most_ct(int nb, int terms) { return nb * (23 + 8 * terms) + 100 <= 240 ? 2 : 1; }

template <int DT, int NB, int CT>
__global__ __launch_bounds__(TPB, kv_decode_waves(NB, CT, DT == MXQ_F16 ? 2 : 1))
void kv_decode_kernel(KvAttnArgs a) {
    constexpr int NT = kv_terms<DT>(), PB = NB < 4 ? NB : 4, PITCH = 32 * PB + 4;
    __shared__ int s_wave[TPB / 64];
    __shared__ int s_found[2];                           // the request that the workgroup's units begin in, its first number
    __shared__ float s_ml[4][16][2];
    __shared__ __attribute__((aligned(16))) float s_acc[4][16][PITCH];
    if (a.plan && blockIdx.x == gridDim.x - 1) {
        __shared__ int64_t s_wave64[TPB / 64];
        kv_plan(a, 64 * kv_prompt_ct(NB, NT), s_wave64, s_wave);
        return;
    }
    const int share = a.by_heads.of((int)blockIdx.x), head = (int)blockIdx.x - share * a.c.heads;
    const int wave = uniform(threadIdx.x >> 6);

    if ((a.zero_tail || a.lse) && a.starts) {            // rows before the first request and behind the last one
        const int rows = (int)a.rows;
        int head_rows = a.starts[0], tail = a.starts[a.requests];
        head_rows = head_rows < 0 ? 0 : (head_rows < rows ? head_rows : rows);
        tail = tail < head_rows ? head_rows : (tail < rows ? tail : rows);
        const int heads = a.c.heads * a.group, nobodys = (head_rows + rows - tail) * heads;
        const uint32_t workgroups = gridDim.x - (a.plan ? 1u : 0u);          // (kv_plan's has left)
        for (uint32_t x = blockIdx.x; x < (uint32_t)nobodys; x += workgroups) {  // (rows x heads and the grid: below 2^31 each)
            const int e = (int)x < head_rows * heads ? (int)x : (int)x + (tail - head_rows) * heads;
            unsigned short* o = kv_out_row(a, e / heads, e % heads);
            if (a.zero_tail)
                for (int d = threadIdx.x; d < a.c.head_dim; d += TPB) o[d] = 0;
            if (a.lse && threadIdx.x == 0) a.lse[e] = -__builtin_inff();
        }
    }

    // the workgroup's numbers at .. end - 1: units, or with a workgroup for each item (whole) items
    int at = share, end = share + 1, window = share, number = share, k0 = 0;
    // 64 requests at a time sit in the lanes
    const int lane = threadIdx.x & 63;
    KvSeq in_lane{0, 0, 0, 0};
    KvWork work_in_lane{0, 0};
    const auto look = [&](int r) {
        in_lane = KvSeq{0, 0, 0, 0};
        work_in_lane = KvWork{0, 0};
        if (r < a.requests) {
            in_lane = kv_seq(a, r);
            work_in_lane = kv_work(a, in_lane);
        }
        return a.whole ? work_in_lane.groups : work_in_lane.count();
    };
    const bool few = a.requests <= 64;
    KvShares deal;
    if (!a.direct && few) {                              // every wave finds its place by itself
        const int mine = look(lane);
        int upto = mine;
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(upto, d, 64);
            if (lane >= d) upto += o;
        }
        const int total = __builtin_amdgcn_readlane(upto, 63);
        if (!a.whole) {
            deal = KvShares(a, total);
            at = deal.begin(share);
            end = deal.begin(share + 1);
        }
        if (at >= end || at >= total) return;
        k0 = uniform(__builtin_ctzll(__ballot(at < upto)));                  // the first request that ends behind `at`
        number = __builtin_amdgcn_readlane(upto - mine, k0);
        window = 0;
    } else if (!a.direct) {                              // (direct: one item a request, a workgroup for each)
        int mine = look(threadIdx.x), sum, upto = block_scan(mine, s_wave, &sum), total = sum;
        if (a.requests > TPB) {
            int rest = 0;
            for (int r = TPB + threadIdx.x; r < a.requests; r += TPB) rest += look(r);
            total += block_sum(rest, s_wave);
        }
        if (!a.whole) {
            deal = KvShares(a, total);
            at = deal.begin(share);
            end = deal.begin(share + 1);
        }
        if (at >= end || at >= total) return;
        int before = 0;
        for (int r0 = 0;; r0 += TPB) {                   // one round for up to 256 requests
            const int first = before + upto - mine;
            if (first <= at && at < first + mine) {
                s_found[0] = r0 + threadIdx.x;
                s_found[1] = first;
            }
            before += sum;
            if (at < before) break;
            mine = look(r0 + TPB + threadIdx.x);
            upto = block_scan(mine, s_wave, &sum);
        }
        __syncthreads();
        window = uniform(s_found[0]);
        number = uniform(s_found[1]);
    }
    const int first_number = at;
    KvPace pace{0, a.whole ? 0 : (end - at) / 4};
    for (; at < end && window < a.requests; window += 64, k0 = 0) {
        if (a.direct || !few) look(window + lane);
        const int last_lane = 63 < a.requests - 1 - window ? 63 : a.requests - 1 - window;
        for (int k = k0; k <= last_lane && at < end; ++k) {
            const KvWork wk{__builtin_amdgcn_readlane(work_in_lane.units, k), __builtin_amdgcn_readlane(work_in_lane.groups, k)};
            if (wk.groups == 0) continue;
            const int r = window + k;
            const KvSeq s{__builtin_amdgcn_readlane(in_lane.row0, k), __builtin_amdgcn_readlane(in_lane.fresh, k),
                          __builtin_amdgcn_readlane(in_lane.len, k), __builtin_amdgcn_readlane(in_lane.keys, k)};
            const int per = a.whole ? 1 : wk.per();
            for (int grp = wk.groups > 1 ? max((at - number) / per, 0) : 0; grp < wk.groups && at < end; ++grp) {
                const int item0 = number + grp * per;
                const int stop = end < item0 + per ? end : item0 + per;
                // an item's first numbers are its beginning, those behind them its units
                const int before = item0 + KV_ITEM_UNITS;
                // (between 0 and the item's units also where starts that are not in order let the numbers overflow)
                const int u0 = a.whole ? 0 : max(at - before, 0), u1 = a.whole ? wk.units : min(stop - before, wk.units);
                if (u1 <= u0) {
                    at = stop;
                    continue;
                }
                const bool complete = u0 == 0 && u1 == wk.units;
                const int place = u0 == 0 && !complete && at != first_number ? 1 : 0;
                const int c0 = grp * 16 * CT, columns = s.fresh * a.group;
                pace.at(a.whole ? u1 : end - at);
                KvWave<NB, CT, NT, 2> wv;
                wv.begin(a, s, head, c0, reinterpret_cast<unsigned short*>(&s_acc[wave][0][0]));
                wv.walk(a, r, head, 4 * u0 + wave, 4 * u1, 4, pace);
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
                                const int at_b = b0 + b < NB ? b0 + b : 0;
                                const kv_f32x4 even = wv.acc[ct][at_b][0], odd = wv.acc[ct][at_b][1];
                                float* dst = &s_acc[wave][wv.i16][32 * b + 8 * wv.g];
                                *reinterpret_cast<kv_f32x4*>(dst) = kv_f32x4{even[0], odd[0], even[1], odd[1]};
                                *reinterpret_cast<kv_f32x4*>(dst + 4) = kv_f32x4{even[2], odd[2], even[3], odd[3]};
                            }
                        __syncthreads();
                        // a thread takes 8 elements of a column at a time
                        for (int e = threadIdx.x; e < 64 * nb; e += TPB) {
                            const int col = e / (4 * nb), d0 = e % (4 * nb) * 8, c = c0 + 16 * ct + col;
                            if (c >= columns) continue;
                            float top = KV_NOTHING;
#pragma unroll
                            for (int w4 = 0; w4 < 4; ++w4) top = __builtin_fmaxf(top, s_ml[w4][col][0]);
                            float sum_l = 0.0f, y[8];
#pragma unroll
                            for (int x = 0; x < 8; ++x) y[x] = 0.0f;
#pragma unroll
                            for (int w4 = 0; w4 < 4; ++w4) {
                                const float f = __builtin_amdgcn_exp2f(s_ml[w4][col][0] - top);
                                sum_l += s_ml[w4][col][1] * f;
#pragma unroll
                                for (int x = 0; x < 8; ++x) y[x] += s_acc[w4][col][d0 + x] * f;
                            }
                            if (complete) {
                                const float inv = sum_l == 0.0f ? 0.0f : 1.0f / sum_l;
#pragma unroll
                                for (int x = 0; x < 8; ++x) y[x] *= inv;
                                const int token = a.by_group.of(c);
                                const int64_t row = s.row0 + token;
                                const int64_t qh = (int64_t)head * a.group + (c - token * a.group);
                                kv_store8<DT>(a, kv_out_row(a, row, qh), 32 * b0 + d0, y);
                                if (a.lse && b0 == 0 && d0 == 0) a.lse[row * a.c.heads * a.group + qh] = kv_lse(top, sum_l);
                            } else {
                                const int64_t part = kv_part_row(a, share, head, place, 16 * ct + col);
                                if (b0 == 0 && d0 == 0)
                                    *reinterpret_cast<kv_f32x2*>(kv_part_ml<NB>(a, part)) = kv_f32x2{top, sum_l};
                                kv_f32x4* dst = reinterpret_cast<kv_f32x4*>(kv_part<NB>(a, part) + 32 * b0 + d0);
                                dst[0] = kv_f32x4{y[0], y[1], y[2], y[3]};
                                dst[1] = kv_f32x4{y[4], y[5], y[6], y[7]};
                            }
                        }
                    }
                }
                if (!a.whole && head == 0 && threadIdx.x == 0) {             // for the join kernel
                    int* span = a.spans + 2 * (kv_item(a, s, r) + grp);
                    if (u0 == 0) span[0] = 2 * share + place;
                    if (u1 == wk.units) span[1] = share;
                }
                at = stop;
            }
            number += per * wk.groups;
        }
    }
}

template <int NB>
__device__ __forceinline__ float* kv_prompt_part(const KvAttnArgs& a, int64_t row) { return a.prompt_part + row * (32 * NB); }
template <int NB, int COLS>
__device__ __forceinline__ float* kv_prompt_part_ml(const KvAttnArgs& a, int64_t row) {
    return a.prompt_part + (int64_t)a.prompt_shares * a.c.heads * 2 * COLS * (32 * NB) + 2 * row;
}

// 16 columns of an item: adds its parts, in their order, if it was cut.
template <int DT, int NB, int CT>
__device__ __forceinline__ void kv_prompt_join(const KvAttnArgs& a, int block) {
    constexpr int COLS = 64 * CT, DP = 32 * NB;
    const int of_head = a.by_heads.of(block), head = block - of_head * a.c.heads, sixteen = of_head % (4 * CT), item = of_head / (4 * CT);
    const KvPlanView plan = kv_plan_view(a);
    if (plan.head[1] == 0 || item >= plan.head[0]) return;
    const int w0 = plan.items[2 * item], w1 = plan.items[2 * item + 1];
    if (w0 == w1) return;                                // written by the workgroup that had all of it
    const KvPiece first = plan.pieces[item + w0];
    const int grp = first.group_flags >> 2;
    const KvSeq s = kv_seq(a, first.request);
    const int columns = s.fresh * a.group;
    for (int e = threadIdx.x; e < 16 * (DP / 8); e += TPB) {
        const int col = 16 * sixteen + e / (DP / 8), d0 = e % (DP / 8) * 8, c = grp * COLS + col;
        if (c >= columns) continue;
        float m = KV_NOTHING, l = 0.0f, y[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) y[x] = 0.0f;
        bool cut = false;
        for (int w = w0; w <= w1; ++w) {
            const KvPiece piece = plan.pieces[item + w];
            if ((piece.group_flags & 2) || piece.tile0 == piece.tile1) continue;                  // written already; nothing done
            cut = true;
            const int64_t part = (((int64_t)w * a.c.heads + head) * 2 + (piece.group_flags & 1)) * COLS + col;
            const kv_f32x2 ml = *reinterpret_cast<const kv_f32x2*>(kv_prompt_part_ml<NB, COLS>(a, part));
            const kv_f32x4* v = reinterpret_cast<const kv_f32x4*>(kv_prompt_part<NB>(a, part) + d0);
            const kv_f32x4 lo = v[0], hi = v[1];
            const float up = __builtin_fmaxf(m, ml[0]);
            const float f = __builtin_amdgcn_exp2f(m - up), fp = __builtin_amdgcn_exp2f(ml[0] - up);
            m = up;
            l = l * f + ml[1] * fp;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                y[x] = y[x] * f + lo[x] * fp;
                y[x + 4] = y[x + 4] * f + hi[x] * fp;
            }
        }
        if (!cut) continue;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int x = 0; x < 8; ++x) y[x] *= inv;
        const int token = a.by_group.of(c);
        const int64_t q_row = s.row0 + token, qh = (int64_t)head * a.group + (c - token * a.group);
        kv_store8<DT>(a, kv_out_row(a, q_row, qh), d0, y);
        if (a.lse && d0 == 0) a.lse[q_row * a.c.heads * a.group + qh] = kv_lse(m, l);
    }
}

// One workgroup for each row and query head: adds the parts of a request that crossed workgroups, in their order.  Bound by
// latency: 4.8 us for 64 requests of 32 heads (8.0 when it worked out by itself where the parts lie).
// Behind these workgroups: those of the prompt kernel's cut items.
template <int DT, int NB>
__global__ __launch_bounds__(TPB) void kv_join_kernel(KvAttnArgs a) {
    constexpr int DP = 32 * NB, LANES = DP / 4, ROWS = TPB / LANES;          // 4 elements a thread, ROWS parts at a time
    __shared__ int s_wave[TPB / 64];
    __shared__ int s_request;
    __shared__ float s_weight[KV_MAX_SHARES];
    __shared__ float s_top[TPB / 64], s_sum[TPB / 64];
    __shared__ kv_f32x4 s_acc[ROWS][LANES];
    const int block = a.join_first + (int)blockIdx.x;
    if (block >= a.join_blocks) {
        kv_prompt_join<DT, NB, kv_prompt_ct(NB, kv_terms<DT>())>(a, block - a.join_blocks);
        return;
    }
    const int q_heads = a.c.heads * a.group;
    int64_t row = a.by_q_heads.of(block);
    const int qh = block - (int)row * q_heads, head = a.by_group.of(qh);
    int r = (int)row;
    if (a.join_rows) {                                   // the first rows of each request: others are the prompt kernel's
        r = (int)(row / a.join_rows);
        row -= (int64_t)r * a.join_rows;
    } else if (a.starts) {
        if (threadIdx.x == 0) s_request = -1;
        __syncthreads();
        for (int k = threadIdx.x; k < a.requests; k += TPB) {
            const KvSeq s = kv_seq(a, k);
            if (s.row0 <= row && row < s.row0 + s.fresh) s_request = k;
        }
        __syncthreads();
        r = uniform(s_request);
        if (r < 0) return;
    }
    const KvSeq s = kv_seq(a, r);
    const KvWork wk = kv_work(a, s);
    if (wk.groups == 0) return;
    if (a.join_rows) {
        if (row >= s.fresh) return;
        row += s.row0;
    }
    const int c = (int)(row - s.row0) * a.group + (qh - head * a.group), grp = c >> a.item_shift, col = c & ((1 << a.item_shift) - 1);
    // as the workgroups left it that begin and end the item: twice the first share, plus which of its places; the last share
    const kv_i32x2 span = *reinterpret_cast<const kv_i32x2*>(a.spans + 2 * (kv_item(a, s, r) + grp));
    const int place0 = uniform(span[0]) & 1;
    const uint32_t last_share = (uint32_t)(a.shares - 1);                    // (in bounds also where starts are not in order)
    const int w0 = (int)min((uint32_t)uniform(span[0]) >> 1, last_share), w1 = (int)min((uint32_t)uniform(span[1]), last_share);
    if (w1 <= w0) return;                                // written by the workgroup that had all of it
    const int parts = w1 - w0 + 1;
    const auto part_row = [&](int k) { return kv_part_row(a, w0 + k, head, k == 0 ? place0 : 0, col); };
    // maxima and sums of all parts at once
    float m = KV_NOTHING;
    for (int k = threadIdx.x; k < parts; k += TPB) {
        const float pm = kv_part_ml<NB>(a, part_row(k))[0];                  // (none between w0 and w1 is without a unit)
        s_weight[k] = pm;
        m = __builtin_fmaxf(m, pm);
    }
    for (int d = 32; d; d >>= 1) m = __builtin_fmaxf(m, __shfl_xor(m, d, 64));
    if ((threadIdx.x & 63) == 0) s_top[threadIdx.x >> 6] = m;
    __syncthreads();
    const float top = __builtin_fmaxf(__builtin_fmaxf(s_top[0], s_top[1]), __builtin_fmaxf(s_top[2], s_top[3]));
    float l = 0.0f;
    for (int k = threadIdx.x; k < parts; k += TPB) {
        const float w = __builtin_amdgcn_exp2f(s_weight[k] - top);
        s_weight[k] = w;
        l += kv_part_ml<NB>(a, part_row(k))[1] * w;
    }
    for (int d = 32; d; d >>= 1) l += __shfl_xor(l, d, 64);
    if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = l;
    __syncthreads();
    const float sum_l = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
    const int lane = threadIdx.x % LANES, first = threadIdx.x / LANES;
    kv_f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
    if (first < ROWS) {
        int k = first;
        for (; k + 3 * ROWS < parts; k += 4 * ROWS) {    // four loads under way
            kv_f32x4 v[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) v[x] = reinterpret_cast<const kv_f32x4*>(kv_part<NB>(a, part_row(k + x * ROWS)))[lane];
#pragma unroll
            for (int x = 0; x < 4; ++x) y += v[x] * s_weight[k + x * ROWS];
        }
        for (; k < parts; k += ROWS) y += reinterpret_cast<const kv_f32x4*>(kv_part<NB>(a, part_row(k)))[lane] * s_weight[k];
        s_acc[first][lane] = y;
    }
    __syncthreads();
    const float inv = sum_l == 0.0f ? 0.0f : 1.0f / sum_l;
    unsigned short* o = kv_out_row(a, row, qh);
    for (int d = threadIdx.x; d < a.c.head_dim; d += TPB) {
        float v = 0.0f;
        for (int k = 0; k < ROWS; ++k) v += s_acc[k][d >> 2][d & 3];
        o[d] = (unsigned short)Pack<DT>::put(v * inv, 0.0f);
    }
    if (a.lse && threadIdx.x == 0) a.lse[row * q_heads + qh] = kv_lse(top, sum_l);
}

// ---- many columns ----------------------------------------------------------------------------------------------
// A workgroup takes 4 x 16 CT columns of a request (an item), a quarter for each wave, and walks over 64 tokens at a time: the
// waves decode their shares of K and V to bf16 once, into LDS and in the order of the operands (a lane reads its 16
// bytes next to its neighbours'), and all of them multiply from there.  Two buffers: the tile ahead is decoded, the
// one behind it loaded, while a tile is multiplied; one barrier a tile.  Decoded by every wave for itself, straight from
// memory, the same prompt took 1940 us instead of 1023 (4001 tokens behind 12000, 8 x 4 heads of 128).
template <int NB>
struct KvShare {                                         // what a lane loads of 64 tokens for its wave to decode
    static constexpr int VB = (NB + 1) / 2;
    uint32_t k[NB], ks[kv_k_scales<NB>()];               // K: 16 tokens, all blocks
    uint32_t v[VB][2], vs[VB][2];                        // V: 32 tokens, every other block
};

// WIDE: a.out_wide.  (Decided while running, the stores of both kinds cost the loop scalar registers: 4001 tokens behind 12000,
// 8 x 4 heads of 128, 1056 us instead of 1028.)
template <int DT, int NB, int CT, bool WIDE>
__global__ __launch_bounds__(TPB, 2) void kv_prompt_kernel(KvAttnArgs a) {
    constexpr int NT = kv_terms<DT>(), NP = kv_terms<DT>(), COLS = 64 * CT, VB = KvShare<NB>::VB;
    using Wave = KvWave<NB, CT, NT, NP>;
    __shared__ uint32_t s_nan[2][2][NB];                 // masked tiles: tokens with a NaN block, by half of 32 tokens
    __shared__ u32x4 s_k[2][4 * NB][64], s_v[2][4 * NB][64];                 // [buffer][operand][lane]
    const int w = a.by_heads.of((int)blockIdx.x), head = (int)blockIdx.x - w * a.c.heads;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, g4 = lane >> 4, i16 = lane & 15;
    const KvPlanView plan = kv_plan_view(a);
    if (w >= plan.head[1]) return;
    const int piece0 = uniform(plan.shares[3 * w]), piece1 = piece0 + uniform(plan.shares[3 * w + 1]);
    const int all_tiles = uniform(plan.shares[3 * w + 2]);
    KvPace pace{0, all_tiles / 4};
    pace.at(all_tiles);
    for (int at_piece = piece0; at_piece < piece1; ++at_piece) {
        const KvPiece piece = plan.pieces[at_piece];
        const int r = uniform(piece.request), flags = uniform(piece.group_flags), grp = flags >> 2;
        const int tile0 = uniform(piece.tile0), tile1 = uniform(piece.tile1);
        if (tile0 == tile1 && !(flags & 2)) continue;
        const bool complete = (flags & 2) != 0;
        const KvSeq in_lanes = kv_seq(a, r);
        const KvSeq s{uniform(in_lanes.row0), uniform(in_lanes.fresh), uniform(in_lanes.len), uniform(in_lanes.keys)};
        const int columns = s.fresh * a.group;
        const int wg_c0 = grp * COLS, c0 = wg_c0 + wave * (16 * CT);
        const int wg_last = (wg_c0 + COLS < columns ? wg_c0 + COLS : columns) - 1;
        const int wg_min = kv_limit(a, s, a.by_group.of(wg_c0)), wg_max = kv_limit(a, s, a.by_group.of(wg_last));
        const bool works = c0 < columns;         // uniform over the wave
        Wave wv;
        wv.begin(a, s, head, works ? c0 : wg_c0, reinterpret_cast<unsigned short*>(&s_k[0][0][0]) + wave * (16 * 32 * NB));
        const int half = wave & 1;
        const int* row = a.table + (int64_t)r * a.table_stride;
        typename Wave::Spot spots;                           // lane: 16 tokens of the next sixteen tiles
        uint64_t there_mask = 0;
        wv.place(a);
        KvShare<NB> share;
        int share_there = 0;                                 // which of the loaded tile's four pages exist
        const auto load = [&](int tile) {
            const int at = 4 * ((tile - tile0) & 15);
            if (at == 0) {
                spots = Wave::spot(a, row, head, 4 * tile + lane, (wg_max + 15) / 16);
                there_mask = __ballot(spots.there);
            }
            share_there = (int)(there_mask >> at) & 15;
            {
                const __amdgpu_buffer_rsrc_t source = Wave::lane_codes(a, spots, at + wave);
                const int scales = __builtin_amdgcn_readlane(spots.scales, at + wave);
                load_dwords<NB>(source, wv.at_k, 0, share.k);
#pragma unroll
                for (int k = 0; k < kv_k_scales<NB>(); ++k) share.ks[k] = __builtin_amdgcn_raw_buffer_load_b8(source, wv.at_ks[k], scales, 0);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int from = at + 2 * half + j;
                const __amdgpu_buffer_rsrc_t source = Wave::lane_codes(a, spots, from);
                const int scales = __builtin_amdgcn_readlane(spots.scales, from);
#pragma unroll
                for (int x = 0; x < VB; ++x) {
                    int b = (wave >> 1) + 2 * x;
                    if (b > NB - 1) b = NB - 1;              // (an odd NB: two waves have one block less)
                    share.v[x][j] = __builtin_amdgcn_raw_buffer_load_b32(source, wv.at_v, 4 * b, 0);
                    share.vs[x][j] = __builtin_amdgcn_raw_buffer_load_b32(source, wv.at_vs, scales + 4 * b, 0);
                }
            }
        };
        int there_bits[2] = {0, 0};                          // by buffer: which of the tile's four pages exist
        const auto decode = [&](int tile, int buffer) {
#pragma unroll
            for (int st = 0; st < NB; ++st)
                s_k[buffer][wave * NB + st][lane] =
                    __builtin_bit_cast(u32x4, kv_k_operand(share.k[st], kv_k_scale<NB>(share.ks, g4, st)));
            there_bits[buffer] = share_there;
            const bool masked = 64 * tile + 64 > wg_min || share_there != 15;
            const bool there2[2] = {(share_there >> (2 * half) & 1) != 0, (share_there >> (2 * half + 1) & 1) != 0};
#pragma unroll
            for (int x = 0; x < VB; ++x) {
                const int b = (wave >> 1) + 2 * x;
                if (b < NB) {
                    uint32_t scales[2] = {share.vs[x][0], share.vs[x][1]};
                    const uint32_t codes[2] = {share.v[x][0], share.v[x][1]};
                    if (masked) {
                        const uint32_t nan = kv_mend_scales(scales, codes, there2, 64 * tile + 32 * half, g4, wg_max);
                        if (lane == 0) s_nan[buffer][half][b] = nan;
                    }
                    kv_bf16x8 v8[2];
                    kv_v_operands(codes, scales, v8);
#pragma unroll
                    for (int n = 0; n < 2; ++n) s_v[buffer][(half * NB + b) * 2 + n][lane] = __builtin_bit_cast(u32x4, v8[n]);
                }
            }
        };

        if (tile0 < tile1) {
            load(tile0);
            decode(tile0, 0);
            if (tile0 + 1 < tile1) load(tile0 + 1);
        }
        __syncthreads();
        for (int tile = tile0; tile < tile1; ++tile) {
            const int buffer = (tile - tile0) & 1;
            pace.tile();
            if (tile + 1 < tile1) {
                decode(tile + 1, buffer ^ 1);
                if (tile + 2 < tile1) load(tile + 2);
            }
            if (works && 64 * tile < wv.max_limit) {
                const bool wg_masked = 64 * tile + 64 > wg_min || there_bits[buffer] != 15;
                // (a loop, not unrolled: both halves at once need registers that are not there)
#pragma nounroll
                for (int h = 0; h < 2; ++h) {
                    const int t0 = 64 * tile + 32 * h;
                    kv_f32x4 sc[CT][2];
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int st = 0; st < NB; ++st)
                            wv.multiply_keys(__builtin_bit_cast(kv_bf16x8, s_k[buffer][(2 * h + j) * NB + st][lane]), j, st, sc);
                    const bool there[2] = {(there_bits[buffer] >> (2 * h) & 1) != 0, (there_bits[buffer] >> (2 * h + 1) & 1) != 0};
                    const bool masked = t0 + 32 > wv.min_limit || !there[0] || !there[1];
                    uint32_t p_hi[CT][4], p_lo[CT][4];
                    wv.probabilities(a, sc, masked, there, t0, p_hi, p_lo);
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int n = 0; n < 2; ++n)
                            wv.multiply_values(__builtin_bit_cast(kv_bf16x8, s_v[buffer][(h * NB + b) * 2 + n][lane]), b, n, p_hi, p_lo);
                    if (wg_masked) {
#pragma unroll
                        for (int b = 0; b < NB; ++b) {
                            const uint32_t of = s_nan[buffer][h][b];
                            if (any_lane(of != 0u)) wv.spread_nan(b, of, t0);
                        }
                    }
                }
            }
            __syncthreads();
        }
        // addresses below are worked out here: known before, they would be kept in registers through the loop above
        const int g_out = here_only(g4), i_out = here_only(i16);
        if (!WIDE && complete) {
            // Rows that are not aligned go through LDS, 16 columns of each wave at a time.  (As parts they would need a
            // place for every item of the stretch; there are two, for the items that its ends cut.)
            unsigned short* stage = reinterpret_cast<unsigned short*>(&s_k[0][0][0]) + wave * (16 * 32 * NB);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                const float l = sum_over_groups(wv.l[ct]), inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const kv_f32x4 even = wv.acc[ct][b][0] * inv, odd = wv.acc[ct][b][1] * inv;
                    *reinterpret_cast<u32x4*>(stage + i_out * (32 * NB) + 32 * b + 8 * g_out) =
                        u32x4{Pack<DT>::put(even[0], odd[0]), Pack<DT>::put(even[1], odd[1]), Pack<DT>::put(even[2], odd[2]),
                              Pack<DT>::put(even[3], odd[3])};
                }
                const int c = c0 + 16 * ct + i_out, token = a.by_group.of(c);
                if (a.lse && g_out == 0 && c < columns)
                    a.lse[(int64_t)(s.row0 + token) * a.c.heads * a.group + (int64_t)head * a.group + (c - token * a.group)] = kv_lse(wv.m[ct], l);
                __syncthreads();
#pragma nounroll
                for (int e = here_only(lane); e < 16 * 32 * NB; e += 64) {
                    const int x = c0 + 16 * ct + e / (32 * NB), d = e % (32 * NB), t = a.by_group.of(x);
                    if (x < columns && d < a.c.head_dim)
                        kv_out_row(a, s.row0 + t, (int64_t)head * a.group + (x - t * a.group))[d] = stage[e];
                }
                __syncthreads();                             // what is there has been read
            }
            continue;
        }
        if (!works) continue;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            const float l = sum_over_groups(wv.l[ct]);
            const int c = c0 + 16 * ct + i_out;
            if (c >= columns) continue;
            if (complete) {
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                const int token = a.by_group.of(c);
        const int64_t q_row = s.row0 + token, qh = (int64_t)head * a.group + (c - token * a.group);
                unsigned short* o = kv_out_row(a, q_row, qh);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    float y[8];
#pragma unroll
                    for (int x = 0; x < 8; ++x) y[x] = wv.acc[ct][b][x & 1][x >> 1] * inv;
                    kv_store8<DT, true>(a, o, 32 * b + 8 * g_out, y);
                }
                if (a.lse && g_out == 0) a.lse[q_row * a.c.heads * a.group + qh] = kv_lse(wv.m[ct], l);
            } else {
                const int64_t part = (((int64_t)w * a.c.heads + head) * 2 + (flags & 1)) * COLS + (c - wg_c0);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    kv_f32x4* dst = reinterpret_cast<kv_f32x4*>(kv_prompt_part<NB>(a, part) + 32 * b + 8 * g_out);
                    const kv_f32x4 even = wv.acc[ct][b][0], odd = wv.acc[ct][b][1];
                    dst[0] = kv_f32x4{even[0], odd[0], even[1], odd[1]};
                    dst[1] = kv_f32x4{even[2], odd[2], even[3], odd[3]};
                }
                if (g_out == 0) *reinterpret_cast<kv_f32x2*>(kv_prompt_part_ml<NB, COLS>(a, part)) = kv_f32x2{wv.m[ct], l};
            }
        }
    }
}

}  // namespace
