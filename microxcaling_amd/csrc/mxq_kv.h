// A paged key / value cache held in MXFP4 and the kernels around it (gfx950): block tables and slots from
// request lengths, quantize-and-store, read-back, attention.
//
// The cache is (pages, kv heads, record) bytes.  With NB = ceil(head_dim / 32) blocks of 32 elements a token's row
// has 32 NB elements (zeros behind head_dim), and the record of a page of ps tokens (a multiple of 16) holds
//   K codes   [ps][16 NB]           e2m1 nibbles, the lower element in the low nibble (as in a packed tensor)
//   V codes   [ps / 4][16][NB][4]   byte (i, b, t): elements 32 b + 2 i (low) and 32 b + 2 i + 1 of token t of four
//   K scales  [ps][NB]              E8M0
//   V scales  [ps / 4][NB][4]       E8M0, byte (b, t)
// = 34 NB bytes a token.  One record is one contiguous piece, so the scales never cost memory lines of their own.
// Both code arrays are stored the way the matrix instruction v_mfma_f32_16x16x32_bf16 wants its first operand:
//   S^T = K q^T   lane (row i = lane % 16, g = lane / 16) of 16 tokens x 32 NB elements takes the 4 NB contiguous
//                 bytes at 4 NB g of token i: eight elements for each of the NB instructions.  Which elements meet in
//                 one instruction does not matter as long as q is dealt out alike.
//   O^T = V^T P^T lane (row i, g) takes, of the four tokens 4 g .. 4 g + 3, the bytes (i, b, .): elements 32 b + 2 i
//                 and + 1, i.e. row i of two instructions.  The scores arrive with the tokens 4 g + r in lane group
//                 g -- the very tokens whose V codes that lane has -- so the probabilities never change lanes.
// v_cvt_scalef32_pk_bf16_fp4 turns a byte of codes and an E8M0 scale into two bf16 values, exactly.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mxq_kernels.h"

namespace {

typedef float kv_f32x2 __attribute__((ext_vector_type(2)));
typedef int kv_i32x2 __attribute__((ext_vector_type(2)));
typedef float kv_f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 kv_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 kv_bf16x2 __attribute__((ext_vector_type(2)));

constexpr int KV_MAX_NB = 8;                             // head_dim up to 256
constexpr int KV_TOKEN_BYTES = 34;                       // bytes of a token's K and V for each block of 32

// Division of 32-bit numbers by one that the host knows (Granlund and Montgomery, Division by Invariant Integers using
// Multiplication, 1994): five instructions instead of forty.
struct KvDivide {
    uint32_t by, first, then;                            // n / d = (h + (n - h >> first)) >> then, h = high half of n by
    __device__ __forceinline__ uint32_t of(uint32_t n) const {
        const uint32_t h = (uint32_t)(((uint64_t)n * by) >> 32);
        return (h + ((n - h) >> first)) >> then;
    }
    __device__ __forceinline__ int of(int n) const { return (int)of((uint32_t)n); }          // n >= 0
};
inline KvDivide kv_divide(uint32_t d) {                  // exact: by = 2^32 (2^l - d) / d + 1 with l the first 2^l >= d
    int l = 0;
    while (((uint64_t)1 << l) < d) ++l;
    return KvDivide{(uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << l) - d)) / d + 1), l > 0 ? 1u : 0u, l > 0 ? (uint32_t)(l - 1) : 0u};
}

struct KvCache {
    unsigned char* data;
    int64_t num_pages;
    int64_t record;                                      // bytes of a (page, head)
    int heads, page_size, head_dim, nb;
    KvDivide by_page;                                    // by page_size
};
__device__ __forceinline__ uint32_t kv_page_of(const KvCache& c, uint32_t n) { return c.by_page.of(n); }

// ---- exchanges between the four lane groups of 16 -------------------------------------------------------------
// f(v of this lane, v of lane ^ 16), then the same with lane ^ 32: a reduction over the groups, in every lane
template <class F>
__device__ __forceinline__ float over_groups(float v, const F& f) {
    const auto a = __builtin_amdgcn_permlane16_swap(mxq_bits(v), mxq_bits(v), false, false);
    v = f(mxq_float(a[0]), mxq_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(mxq_bits(v), mxq_bits(v), false, false);
    return f(mxq_float(b[0]), mxq_float(b[1]));
}
__device__ __forceinline__ float max_over_groups(float v) {
    return over_groups(v, [](float a, float b) { return __builtin_fmaxf(a, b); });
}
__device__ __forceinline__ float sum_over_groups(float v) {
    return over_groups(v, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ uint32_t or_over_groups(uint32_t v) {
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = a[0] | a[1];
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return b[0] | b[1];
}
__device__ __forceinline__ bool any_lane(bool p) { return !__all(!p); }
// a value that is the same in every lane of the wave, told to the compiler: it goes to a scalar register, and branches
// and addresses that follow from it stay scalar too
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform64(int64_t v) {
    const uint32_t lo = (uint32_t)uniform((int)(uint32_t)v), hi = (uint32_t)uniform((int)(uint32_t)((uint64_t)v >> 32));
    return (int64_t)(((uint64_t)hi << 32) | lo);
}

template <class T>
__device__ __forceinline__ T uniform_any(T v) {
    if constexpr (sizeof(T) == 8) return uniform64(v);
    else return uniform(v);
}
// sum over the workgroup, in every thread (s: a value for each wave)
template <class T>
__device__ __forceinline__ T block_sum(T v, T* s) {
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < TPB / 64; ++w) v += s[w];
    return uniform_any(v);
}
// inclusive prefix sum over the workgroup's threads; *total: their sum
template <class T>
__device__ __forceinline__ T block_scan(T v, T* s, T* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int d = 1; d < 64; d <<= 1) {
        const T o = __shfl_up(v, d, 64);
        if (lane >= d) v += o;
    }
    __syncthreads();
    if (lane == 63) s[wave] = v;
    __syncthreads();
    T t = 0;
    for (int w = 0; w < TPB / 64; ++w) {
        if (w == wave) v += t;
        t += s[w];
    }
    *total = uniform_any(t);
    return v;
}

}  // namespace
