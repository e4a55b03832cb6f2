// vws_verify.h -- argument block, shape constants and workspace layout of draft verification
// (vws_verify.hip), shared with its launcher (vws_capi.hip).
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "vws_internal.h"

namespace vws {

constexpr int kVfThreads = 256;      // threads of a part (row statistics, race)
constexpr int kVfCutThreads = 1024;  // threads of a cut row
constexpr int kVfMaxParts = 64;      // parts of a row: one lane each in the join
constexpr int kVfMaxDrafts = 64;     // VWS_MAX_DRAFTS: one lane each in the decision
constexpr uint32_t kVfAcceptBase = 1u << 19;  // VWS_MAX_VOCAB: generated acceptance uniforms' tokens

// A row's statistics.  One per part for rows that nothing cuts (sum: of the part's exponentials relative to
// its own largest logit), or the row's own (part 0) once verify_cut_kernel has cut it (sum: of the kept
// exponentials).
struct VfRec {
    uint64_t top;   // key of the largest logit << 32 | 0x7FFFFFFF - its lowest index; 0: all NaN
    float sum;
    int32_t owner;  // the request whose parameters cut the row
};

constexpr int kVfBins = 2048;      // bins of a row's masses
constexpr int kVfFlat = 256;       // rows of a launch that verify_mass_kernel takes: a workgroup each, at least
constexpr int kVfMassWgs = 256;    // its workgroups, one of 1024 threads for each compute unit

// Rows or requests of a launch, at most: a workgroup of 1024 threads each stays below the 2^32 threads of
// a grid, from where a launch runs some of its workgroups only and reports nothing.
constexpr int kVfLaunchRows = 1 << 21;

struct VfFlat {
    int32_t row;
    uint32_t ctr;                  // parts arrived
    uint64_t rest;                 // the masses beyond the bins
    uint64_t hist[kVfBins];
};

struct VerifyArgs {
    const void* x;               // [R, V] target logits, n_b + 1 rows per request
    int64_t xstride;
    int R, V, B, D, K;           // K: columns of drafts in the outputs
    int r0;                      // first row (verify_token_kernel: request) of the launch
    const int32_t* drafts;       // [D]
    const int32_t* cu;           // [B + 1]
    const void* q;               // [D, V] draft probabilities or null
    int64_t qstride;
    int qdtype;
    const float* temperature;    // [B]; null: greedy
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    const float* au;             // [D] acceptance uniforms (when u is given)
    const float* u;              // [B, V] race uniforms or null
    int64_t ustride;
    const uint64_t* rng_seed;    // [B]
    const uint64_t* rng_offset;  // [B] or null
    uint64_t rng_key;
    int32_t* tokens;             // [B, K + 1]
    int32_t* accepted;           // [B]
    float* logprobs;             // [B, K + 1]
    int S, part_len;             // parts of a row in the statistics
    int S2, part2_len;           // parts of a row in the race
    VfRec* rec;                  // [R, S]
    float* gmax;                 // [R, groups] maxima of groups of vectors, of rows that are cut; or null
    int groups;                  // of a row
    uint64_t* cut;               // [R] kept: (key(y) << 32 | index) >= cut
    int32_t* kept;               // [R, 1 + kVfKept] of cut rows: how many are kept (-1: not listed), and they
    uint32_t* flat_n;            // rows whose masses verify_mass_kernel adds up; cleared by the statistics' launch
    VfFlat* flat;                // [kVfFlat]
    uint64_t* best;              // [B, S2] race: key bits << 32 | 0x7FFFFFFF - index
    uint32_t* ctr;               // [B] race parts arrived; cleared by the statistics' launch
};

constexpr int kVfGroup = 4;          // vectors whose maximum the first pass leaves together

// Groups of a row (their maxima's places): those of its parts, kVfThreads an iteration.
inline int vf_groups(int S, int part_len, int vec) {
    const int per = kVfGroup * kVfThreads * vec;
    return S * ((part_len + per - 1) / per) * kVfThreads;
}

constexpr int kVfKept = 511;         // tokens of a cut row that the race takes from a list

struct VfLayout {
    size_t rec, gmax, cut, kept, flat_n, flat, best, ctr, total;
};

inline VfLayout vf_layout(int R, int B, int S, int S2, int groups) {
    VfLayout w{};
    size_t off = align256(sizeof(CoopState));  // every workspace starts with the fixed region
    w.rec = off;   off = align256(off + sizeof(VfRec) * (size_t)R * S);
    w.gmax = off;  off = align256(off + sizeof(float) * (size_t)R * groups);
    w.cut = off;   off = align256(off + sizeof(uint64_t) * (size_t)R);
    w.kept = off;  off = align256(off + sizeof(int32_t) * (size_t)R * (1 + kVfKept));
    w.flat_n = off; off = align256(off + sizeof(uint32_t));
    w.flat = off;  off = align256(off + sizeof(VfFlat) * (size_t)(R < kVfFlat ? R : kVfFlat));
    w.best = off;  off = align256(off + sizeof(uint64_t) * (size_t)B * S2);
    w.ctr = off;   off = align256(off + sizeof(uint32_t) * (size_t)B);
    w.total = off;
    return w;
}

}  // namespace vws
