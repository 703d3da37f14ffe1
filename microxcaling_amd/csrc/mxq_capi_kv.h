// Shared by the translation units of the packed key / value cache: the launches of one tensor type, for every
// number of blocks, live in a unit of their own.
#pragma once
#include "mxq_capi_common.h"
#include "mxq_kv_attention.h"

namespace mxq_kv {
// workgroups of a launch: its threads are counted in 32 bits, and what is above them is left out without an error
constexpr int64_t kMostWorkgroups = 0xFFFFFFFF / kThreads;

// what a call of the attention runs
struct Plan {
    int nb, ct;                    // blocks of a row; column tiles of a decode item
    bool prompt, whole;
    int decode_columns;
    int64_t decode_items;          // whole: workgroups of a kv head
    int64_t shares;
    int64_t prompt_items, prompt_shares;
};
}  // namespace mxq_kv

#define MXQ_KV_CASES(NB_, ...)                  \
    switch (NB_) {                              \
        case 1: { constexpr int NB = 1; __VA_ARGS__; break; } \
        case 2: { constexpr int NB = 2; __VA_ARGS__; break; } \
        case 3: { constexpr int NB = 3; __VA_ARGS__; break; } \
        case 4: { constexpr int NB = 4; __VA_ARGS__; break; } \
        case 5: { constexpr int NB = 5; __VA_ARGS__; break; } \
        case 6: { constexpr int NB = 6; __VA_ARGS__; break; } \
        case 7: { constexpr int NB = 7; __VA_ARGS__; break; } \
        default: { constexpr int NB = 8; __VA_ARGS__; break; } \
    }
