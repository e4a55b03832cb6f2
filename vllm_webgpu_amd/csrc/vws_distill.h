// vws_distill.h -- argument block and shape constants of the distillation kernels
// (vws_distill.hip), shared with their launcher (vws_capi.hip).
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace vws {

constexpr int kDsThreads = 256;     // threads of a part (forward and backward)
constexpr int kDsStepThreads = 512;   // threads of a row (step)
constexpr int kDsMaxK = 256;        // teacher entries of a row, one per thread of a part
constexpr int kDsMaxParts = 64;     // parts of a row: one lane each in the join
constexpr int kDsRowStats = 8;      // floats of a row's statistics (DistillStat)

// What the backward needs of a row, e(x) = exp2(x log2(e) / T): student elements outside the teacher's
// entries get e(x - ref) * coef, teacher entries e(x - max) * inv_total - P (P: DistillArgs::entry_p), both
// times weight * upstream / T.
enum DistillStat { kDsRef = 0, kDsCoef = 1, kDsMax = 2, kDsInvTotal = 3, kDsLive = 4 };

struct DistillArgs {
    const void* x;          // [N, V] student logits
    int64_t xstride;
    int N, V, K;
    const int32_t* ids;     // [N, K] teacher ids
    int64_t ids_stride;
    const float* lp;        // [N, K] teacher log-probabilities
    int64_t lp_stride;
    const float* weight;    // [N] or null
    float c;                // log2(e) / T
    float inv_T;
    int S;                  // parts per row
    int part_len;           // elements per part (a multiple of 64)
    const float* gout;      // [N] upstream gradient or null (1)
    void* grad;             // [N, V] or null
    int64_t gstride;
    float* loss;            // [N]
    float* stats;           // [N, kDsRowStats]
    float* entry_p;         // [N, K] probability of each id at its first entry, -1 elsewhere
    uint64_t* rec;          // [N * S] parts' ExpSum, S > 1
    uint32_t* ctr;          // [N] parts arrived (left at zero), S > 1
};

}  // namespace vws
