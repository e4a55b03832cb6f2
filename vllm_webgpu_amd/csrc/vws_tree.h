// vws_tree.h -- argument blocks and shape constants of the drafted trees' kernels (vws_tree_kernel.h, vws_tree.hip),
// shared with their launcher (vws_capi.hip).
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "vws_cache.h"

namespace vws {

constexpr int kTrThreads = 256;   // four waves
constexpr int kTrWideThreads = 512, kTrWideRows = 128;  // eight, which share their keys
constexpr int kTrKeys = 32;       // keys of a wave's step
constexpr int kTrMaxSplits = 256;
constexpr int kAcThreads = 64;    // one wave a request
constexpr int kAcMaxNodes = 256;  // VWS_MAX_TREE_NODES

struct TreeArgs {
    CacheView c;
    int B, T, max_nodes;
    int group;          // query heads of a key head
    const uint16_t* q;
    int64_t qts, qhs;
    uint16_t* out;
    int64_t ots, ohs;
    const int32_t* table;
    int64_t table_stride;
    int max_pages;
    const int32_t* context;
    const int32_t* cu;
    const uint32_t* visible;  // or null: a chain
    int64_t visible_stride;
    int words;                // of a row that may be read
    float c2;                 // scale * log2(e)
    float back;               // 1 / c2
    int splits;               // parts of the longest request's keys
    int chunk;                // keys of a part: a multiple of every wave's step
    int blocks;               // workgroups that a part's rows need, at most
    int rows;                 // rows of a part's record (splits > 1)
    int longest_first;        // requests are served by their length (B <= kTrThreads)
    float* part;              // [B, splits, heads, rows, D] products, then
    float* stat;              // [B, splits, heads, rows, 2] references and sums
};

struct AcceptArgs {
    int B, T, width;
    const int32_t* sampled;
    const int32_t* tokens;
    const int32_t* parents;
    const int32_t* cu;
    int32_t* out;
    int32_t* path;
    int32_t* accepted;
};

}  // namespace vws
