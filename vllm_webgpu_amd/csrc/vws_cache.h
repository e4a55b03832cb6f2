// vws_cache.h -- argument blocks and shape constants of the paged cache's kernels (vws_cache.hip), shared with
// their launcher (vws_capi.hip), and the cache as the attention's kernel sees it too.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace vws {

constexpr int kCacheMinPage = 8, kCacheMaxPage = 256;
constexpr int kCacheMaxPosition = 0x7FFF0000;  // of a request: what a step's arithmetic adds fits 32 bits
constexpr int kApThreads = 256;    // threads of a workgroup, all three kernels
constexpr int kApValueTokens = 32;  // tokens of a workgroup that stores values (at most 64)
constexpr int kApGroup = 4;         // ... that rotates, at most

// One layer's cache (vws_kv_cache): 16-bit elements whatever their type.
struct CacheView {
    uint16_t* k;   // [pages, heads, P, D]
    uint16_t* v;   // [pages, heads, D, P]
    int64_t kps, vps;  // page strides
    int pages;
    int pshift;    // log2(P)
    int heads, D;
};

struct AppendArgs {
    CacheView c;
    int T;
    const uint16_t* k;
    int64_t kts, khs;  // token and head strides
    const uint16_t* v;
    int64_t vts, vhs;
    const int32_t* slots;
    const int32_t* positions;  // or null: nothing is rotated
    const float* inv_freq;
    int R;
    int interleaved;
    float scale;
    int Hq;
    const uint16_t* q;
    int64_t qts, qhs;
    uint16_t* qo;
    int64_t qots, qohs;
    int group;   // tokens of a workgroup that rotates
    int wgs;     // workgroups that rotate; the values' follow
};

struct CompactArgs {
    CacheView c;
    const int32_t* table;
    int64_t table_stride;
    int max_pages;
    const int32_t* context;
    const int32_t* path;
    int64_t path_stride;
    int width;
};

}  // namespace vws
