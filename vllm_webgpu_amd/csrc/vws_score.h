// vws_score.h -- argument block and shape constants of the log-probability kernels (vws_score.hip), shared with
// their launcher (vws_capi.hip).
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace vws {

constexpr int kScThreads = 256;
constexpr int kScMaxParts = 64;     // parts of a row: one lane each in the join
constexpr int kScMaxTopParts = 16;  // ... that keep a list of their largest logits
constexpr int kScMaxTop = 64;       // VWS_MAX_LOGPROBS
constexpr int kScSlots = 8;         // groups of a thread's logits whose maxima are kept
constexpr int kScGroups = 512;      // groups that may hold a row's largest logits
constexpr int kScCands = 1024;      // logits that may be among the largest
constexpr int kScRowStats = 8;      // floats of a row's statistics (ScoreStat)

// What the backward needs of a row: its maximum, the reciprocal of sum exp2((x - max) c), log2 of that sum, the
// entropy, and whether the row counts.
enum ScoreStat { kScMax = 0, kScInvTotal = 1, kScLog2Total = 2, kScEntropy = 3, kScLive = 4 };

struct ScoreRec { uint64_t ms, wn; };  // a part's maximum and sum, weighted sum and count

struct ScoreArgs {
    const void* x;       // [N, V] logits
    int64_t xstride;
    int N, V;
    const int32_t* ids;  // [N]
    float c;             // log2(e) / T
    float inv_T;
    int L;               // the largest logits that are listed, or -1
    int S, part_len;     // parts per row; elements per part (a multiple of 64)
    float* logprobs;     // [N]
    float* entropy;      // [N] or null
    int32_t* lp_ids;     // [N, L + 1]
    float* lp_vals;      // [N, L + 1]
    int32_t* ranks;      // [N]
    float* stats;        // [N, kScRowStats] or null
    ScoreRec* rec;       // [N * S], S > 1
    uint64_t* list;      // [N * S, L], S > 1
    uint32_t* ctr;       // [N] parts arrived (left at zero), S > 1
    const float* gl;     // [N] or null
    const float* gh;     // [N] or null
    void* grad;          // [N, V]
    int64_t gstride;
};

}  // namespace vws
