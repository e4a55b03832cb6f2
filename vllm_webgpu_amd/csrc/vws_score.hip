// vws_score.hip -- log-probabilities of given tokens with entropy, ranks and top alternatives, and the
// logits' gradient.
//
// A row: logits x [V], token t, temperature T; y = x log2(e) / T, m the maximum, e_j = exp2(y_j - y_m),
// S = sum e_j, W = sum e_j (y_j - y_m):
//   log p_t = (x_t - m) / T - ln S,   H = ln S - ln 2 W / S
//   dL/dx_j = (g_l (1{j = t} - p_j) - g_h p_j (log p_j + H)) / T = e_j (a + b (y_j - y_m)) + 1{j = t} g_l / T
// One read of the row for the forward, with the running reference of vws_expsum.h, and one for the
// backward, an fma and an exp2 for each logit.  W follows its sum's reference: relative to a reference
// higher by D it is (W - D S) exp2(-D).
//
// The L largest logits come from the same read: each thread keeps the maxima of a few groups of its
// logits.  At least L logits are as large as the L-th largest of the threads' maxima, and only groups whose own
// maximum reaches it hold any: a handful of groups is read again.
//
// HBM bounds both: 1999 x 151936 bf16 with entropy and 20 alternatives 135 us (4.5 TB/s of
// logits, 5.9 with the groups' lines; without alternatives 109), 4096 x 128256 bf16, a fifth of
// the rows padding, forward 150 (5.6 TB/s, reads alone) and backward 345 (5.5 TB/s read and written, some of the reads from the
// last-level cache).  Few rows are split over workgroups: 7 x 50257 fp32 with 5 alternatives 10.9 us, a part's read, its list and the join one after another.
#include "vws_device.h"
#include "vws_expsum.h"
#include "vws_sampler.h"
#include "vws_score.h"

namespace vws {

static_assert(kScMaxTop == VWS_MAX_LOGPROBS && kScMaxTopParts * kScMaxTop <= kScCands && kScMaxTop <= kScThreads,
              "the parts' lists are joined in one candidate list, the threshold is a thread's maximum");

constexpr float kScLn2 = 0x1.62e43p-1f;
// The least y - reference in a weighted sum: exp2 of it is 0, and so its product, -inf's among them.
constexpr float kScLeast = -16384.0f;

// Widened logits back to a row's words.
template <typename T> __device__ __forceinline__ void sc_pack(const float* v, uint32_t (&w)[4]);
template <> __device__ __forceinline__ void sc_pack<float>(const float* v, uint32_t (&w)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = f2u(v[i]);
}
template <> __device__ __forceinline__ void sc_pack<uint16_t>(const float* v, uint32_t (&w)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v[2 * i]) | ((uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v[2 * i + 1]) << 16);
}
template <> __device__ __forceinline__ void sc_pack<_Float16>(const float* v, uint32_t (&w)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * i]) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * i + 1]) << 16);
}
template <typename T> __device__ __forceinline__ T sc_narrow(float v);
template <> __device__ __forceinline__ float sc_narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ uint16_t sc_narrow<uint16_t>(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
template <> __device__ __forceinline__ _Float16 sc_narrow<_Float16>(float v) { return (_Float16)v; }

// (not temporal: what the forward has read stays in the last-level cache for the backward)
template <typename T>
__device__ __forceinline__ void sc_store(T* row, int vi, const uint32_t (&w)[4]) {
    typename RowVec<T>::U4 u;
    u[0] = w[0]; u[1] = w[1]; u[2] = w[2]; u[3] = w[3];
    __builtin_nontemporal_store(u, reinterpret_cast<typename RowVec<T>::U4*>(reinterpret_cast<char*>(row) + 16u * (uint32_t)vi));
}

// (maximum, sum, weighted sum) of some logits, relative to their maximum; the empty one is (-inf, 0, 0).
struct ScSum {
    float m = -kExpInf, s = 0.0f, w = 0.0f;
    __device__ __forceinline__ void merge(float om, float os, float ow, float c) {
        const float n = __builtin_fmaxf(m, om), ref = n == -kExpInf ? 0.0f : n;
        const float d = m == -kExpInf ? 0.0f : (m - ref) * c, od = om == -kExpInf ? 0.0f : (om - ref) * c;
        const float f = es_exp2(d), of = es_exp2(od);
        w = (w + s * __builtin_fmaxf(d, kScLeast)) * f + (ow + os * __builtin_fmaxf(od, kScLeast)) * of;
        s = s * f + os * of;
        m = n;
    }
    template <int O>
    __device__ __forceinline__ void lane_merge(float c) { merge(es_lane_xor(m, O), es_lane_xor(s, O), es_lane_xor(w, O), c); }
    __device__ __forceinline__ void wave_merge(float c) {
        lane_merge<32>(c);
        lane_merge<16>(c);
        lane_merge<8>(c);
        lane_merge<4>(c);
        lane_merge<2>(c);
        lane_merge<1>(c);
    }
};

// A logit as a 64-bit key that orders by value, then by the lower index; 0 is none (a NaN).
__device__ __forceinline__ uint64_t sc_key(float v, int i) {
    return v == v ? ((uint64_t)key_of(v + 0.0f) << 32) | (0xFFFFFFFFu - (uint32_t)i) : 0u;
}

struct ScShared {
    float m[kScThreads / 64], s[kScThreads / 64], w[kScThreads / 64];
    uint32_t n[kScThreads / 64];
    float t;               // threshold of the listed logits
    uint32_t groups, cands;
    uint16_t group[kScGroups];
    uint64_t top[kScMaxTop];
    union {
        float gmax[(kScSlots + 1) * kScThreads];  // [slot][thread], the last slot for a part's last few logits
        uint64_t cand[kScCands];
    };
};

__device__ __forceinline__ uint32_t sc_plus(uint32_t a, uint32_t b) { return a + b; }
__device__ __forceinline__ uint32_t sc_block_sum(ScShared& sh, uint32_t v) {
    VWS_BUTTERFLY(v, lane_xor, sc_plus);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.n[threadIdx.x >> 6] = v;
    __syncthreads();
    uint32_t t = 0u;
#pragma unroll
    for (int i = 0; i < kScThreads / 64; ++i) t += sh.n[i];
    return t;
}

// f(value, index) of every logit of a part, any order.
template <typename T, typename F>
__device__ __forceinline__ void sc_each(const T* row, int len, F f) {
    constexpr int VEC = Elem<T>::kVec;
    const int nvec = len / VEC, i = nvec * VEC + (int)threadIdx.x;
    for (int vi = threadIdx.x; vi < nvec; vi += kScThreads) {
        uint32_t w[4];
        row_load<T>(row, vi, w);
        float v[VEC];
        Elem<T>::from_words(w[0], w[1], w[2], w[3], v);
#pragma unroll
        for (int j = 0; j < VEC; ++j) f(v[j], vi * VEC + j);
    }
    if (i < len) f(Elem<T>::load1(row + i), i);
}

// Candidates that do not fit (many logits of the threshold's value, mostly: masked rows): what lies above the
// threshold, then what equals it by index.
template <typename T>
__device__ __attribute__((noinline)) void sc_ties(const T* row, int len, int lo, int L, ScShared& sh) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    float t = sh.t;
    auto above = [&](float v) {
        uint32_t n = 0u;
        sc_each<T>(row, len, [&](float x, int) { n += x > v ? 1u : 0u; });
        return sc_block_sum(sh, n);
    };
    if (above(t) >= (uint32_t)L) {
        // the L-th largest key: the largest that at least L logits reach
        uint32_t key = 0u;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t k = key | (1u << bit);
            uint32_t n = 0u;
            sc_each<T>(row, len, [&](float x, int) { n += x == x && key_of(x + 0.0f) >= k ? 1u : 0u; });
            if (sc_block_sum(sh, n) >= (uint32_t)L) key = k;
        }
        t = val_of(key);
    }
    __syncthreads();
    if (tid == 0) sh.cands = 0u;
    __syncthreads();
    sc_each<T>(row, len, [&](float x, int i) {
        if (x > t) {
            const uint32_t at = atomicAdd(&sh.cands, 1u);
            if (at < kScCands) sh.cand[at] = sc_key(x, lo + i);  // (fewer than L)
        }
    });
    __syncthreads();
    uint32_t have = sh.cands;
    for (int b = 0; b < len && have < (uint32_t)L; b += kScThreads) {
        const int i = b + tid;
        const float x = i < len ? Elem<T>::load1(row + i) : __builtin_nanf("");
        const uint64_t hit = wave_ballot(x == t);
        __syncthreads();
        if (lane == 0) sh.n[wave] = (uint32_t)__builtin_popcountll(hit);
        __syncthreads();
        uint32_t at = have + (uint32_t)lane_prefix(hit), all = 0u;
        for (int w = 0; w < kScThreads / 64; ++w) {
            if (w < wave) at += sh.n[w];
            all += sh.n[w];
        }
        if (x == t && at < (uint32_t)L) sh.cand[at] = sc_key(x, lo + i);
        have += all;
    }
    __syncthreads();
    if (tid == 0) sh.cands = min(have, (uint32_t)L);
    __syncthreads();
}

// The L largest of sh.cand (sh.cands of them), in order, to sh.top; none: 0.  After a barrier; ends with one.  A
// candidate's place is the number of larger ones, counted by eight neighbouring threads.
__device__ __forceinline__ void sc_sort(ScShared& sh, int L) {
    constexpr int kSide = 8;
    const int tid = threadIdx.x, side = tid % kSide, n = (int)sh.cands;
    if (tid < L) sh.top[tid] = 0u;
    __syncthreads();
    for (int i0 = 0; i0 < n; i0 += kScThreads / kSide) {
        const int i = i0 + tid / kSide;
        const uint64_t k = i < n ? sh.cand[i] : 0u;
        uint32_t at = 0u;
#pragma unroll 4
        for (int j = side; j < n; j += kSide) at += sh.cand[j] > k ? 1u : 0u;
        at += lane_xor(at, 1);
        at += lane_xor(at, 2);
        at += lane_xor(at, 4);
        if (side == 0 && at < (uint32_t)L && k) sh.top[at] = k;
    }
    __syncthreads();
}

// A part's L largest logits to sh.top, from its groups' maxima (`own`: this thread's largest).
template <typename T>
__device__ __forceinline__ void sc_top(const T* row, int len, int lo, int L, int per, float own, ScShared& sh) {
    constexpr int VEC = Elem<T>::kVec, U = 4;
    const int tid = threadIdx.x, nvec = len / VEC;
    // The L-th largest of the threads' maxima, or, where L is small, the largest of the waves' own L-th largest: as good a
    // bound, without looking at every thread's (L = 32: some 130 candidates in place of 32; L = 20, 1999 x 151936: 135 us, 141
    // with the threads' own).
    __shared__ float tops[kScThreads];
    if (tid == 0) sh.groups = sh.cands = 0u;
    if (L <= 32) {
        const uint32_t key = wave_mth_largest64_count(key_of(own), L);
        if ((tid & 63) == 0) tops[tid >> 6] = val_of(key);
        __syncthreads();
        if (tid == 0) {
            float t = tops[0];
#pragma unroll
            for (int i = 1; i < kScThreads / 64; ++i) t = __builtin_fmaxf(t, tops[i]);
            sh.t = t;
        }
    } else {
        tops[tid] = own;
        __syncthreads();
        int at = 0;
        const float4* q = reinterpret_cast<const float4*>(tops);
#pragma unroll 4
        for (int j = 0; j < kScThreads / 4; ++j) {
            const float4 v = q[j];
            at += v.x > own || (v.x == own && 4 * j < tid) ? 1 : 0;
            at += v.y > own || (v.y == own && 4 * j + 1 < tid) ? 1 : 0;
            at += v.z > own || (v.z == own && 4 * j + 2 < tid) ? 1 : 0;
            at += v.w > own || (v.w == own && 4 * j + 3 < tid) ? 1 : 0;
        }
        if (at == L - 1) sh.t = own;
    }
    __syncthreads();
    const float t = sh.t;
    if (own >= t) {
#pragma unroll
        for (int s = 0; s <= kScSlots; ++s)
            if (sh.gmax[s * kScThreads + tid] >= t) {
                const uint32_t at = atomicAdd(&sh.groups, 1u);
                if (at < kScGroups) sh.group[at] = (uint16_t)(s * kScThreads + tid);
            }
    }
    __syncthreads();
    const int groups = (int)sh.groups;
    if (groups <= kScGroups) {
        const int size = per * U;  // vectors of a group
        for (int i = tid; i < groups * size; i += kScThreads) {
            const int gi = i / size, u = i - gi * size, g = sh.group[gi], s = g / kScThreads, th = g - s * kScThreads;
            auto take = [&](float v, int idx) {
                if (v >= t) {
                    const uint32_t at = atomicAdd(&sh.cands, 1u);
                    if (at < kScCands) sh.cand[at] = sc_key(v, lo + idx);
                }
            };
            if (s == kScSlots) {
                if (u == 0) take(Elem<T>::load1(row + nvec * VEC + th), nvec * VEC + th);
                continue;
            }
            const int vi = (s * size + u) * kScThreads + th;
            if (vi >= nvec) continue;
            uint32_t w[4];
            row_load<T>(row, vi, w);
            float v[VEC];
            Elem<T>::from_words(w[0], w[1], w[2], w[3], v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) take(v[j], vi * VEC + j);
        }
    }
    __syncthreads();
    if (groups > kScGroups || sh.cands > kScCands) sc_ties<T>(row, len, lo, L, sh);  // (every thread alike)
    sc_sort(sh, L);
}

template <typename T, bool ENT, bool TOP>
__global__ __launch_bounds__(kScThreads) void score_kernel(ScoreArgs a) {
    constexpr int VEC = Elem<T>::kVec, U = 4, NW = kScThreads / 64;
    __shared__ ScShared sh;
    __shared__ uint32_t last;
    const int S = a.S, r = blockIdx.x / S, p = blockIdx.x - r * S, tid = threadIdx.x, L = a.L;
    const T* whole = static_cast<const T*>(a.x) + (size_t)r * a.xstride;
    const int lo = p * a.part_len, len = min(a.V, lo + a.part_len) - lo, nvec = len / VEC;
    const T* row = whole + lo;
    uint32_t next[U][4];
    auto fetch = [&](int b) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u) row_load<T>(row, min(b + u * kScThreads, nvec - 1), next[u]);
    };
    // (rows that are split are few: they need not wait for their token, which pads a row at the cost of these loads)
    if (S > 1 && nvec > 0) fetch(tid);
    const int token = a.ids[r];
    if (token < 0 || token >= a.V) {  // padding: not read
        if (p == 0) {
            if (tid == 0) {
                a.logprobs[r] = 0.0f;
                if (ENT) a.entropy[r] = 0.0f;
                if (TOP) a.ranks[r] = 0;
                if (a.stats) a.stats[(size_t)r * kScRowStats + kScLive] = 0.0f;
            }
            if (TOP && tid <= L) {
                a.lp_ids[(size_t)r * (L + 1) + tid] = -1;
                a.lp_vals[(size_t)r * (L + 1) + tid] = 0.0f;
            }
        }
        return;
    }
    const float c = a.c, xt = Elem<T>::load1(whole + token);
    const int batches = (nvec + U * kScThreads - 1) / (U * kScThreads), per = max(1, (batches + kScSlots - 1) / kScSlots);

    // the stream: the next four vectors' loads are issued before these are used
    ExpRun run(c);
    float wsum = 0.0f, own = -kExpInf;
    uint32_t rank = 0u;
    auto add = [&](float g, const auto& v) __attribute__((always_inline)) {
        constexpr int n = sizeof(v) / sizeof(float);
        const float was = run.ref, had = run.s, kept = run.raise(g, c);
        if (ENT) wsum = (wsum + had * (was - run.ref)) * es_exp2(was - run.ref);
        float s[4] = {kept, 0.0f, 0.0f, 0.0f}, w[4] = {wsum, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < n; ++j) {
            const float y = __builtin_fmaf(v[j], c, -run.ref), e = es_exp2(y);
            s[j & 3] += e;
            if (ENT) w[j & 3] = __builtin_fmaf(e, __builtin_fmaxf(y, kScLeast), w[j & 3]);
        }
        run.s = (s[0] + s[1]) + (s[2] + s[3]);
        if (ENT) wsum = (w[0] + w[1]) + (w[2] + w[3]);
    };
    if (S == 1 && nvec > 0) fetch(tid);
    if (TOP) {
#pragma unroll
        for (int s = 0; s <= kScSlots; ++s) sh.gmax[s * kScThreads + tid] = -kExpInf;
    }
    float gm = -kExpInf;
    int slot = 0, left = per;
    for (int b = tid; b < nvec; b += U * kScThreads) {
        float v[U * VEC];
#pragma unroll
        for (int u = 0; u < U; ++u) Elem<T>::from_words(next[u][0], next[u][1], next[u][2], next[u][3], v + u * VEC);
        const int now = b;
        if (b + U * kScThreads < nvec) fetch(b + U * kScThreads);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool in = now + u * kScThreads < nvec;
            uint32_t n = 0u;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                if (TOP) n += v[u * VEC + j] >= xt ? 1u : 0u;
                v[u * VEC + j] = in ? v[u * VEC + j] : -kExpInf;
            }
            if (TOP) rank += in ? n : 0u;
        }
        float g = v[0];
#pragma unroll
        for (int j = 1; j < U * VEC; ++j) g = __builtin_fmaxf(g, v[j]);
        add(g, v);
        if (TOP) {
            gm = __builtin_fmaxf(gm, g);
            if (--left == 0) {
                sh.gmax[slot * kScThreads + tid] = gm;
                own = __builtin_fmaxf(own, gm);
                gm = -kExpInf;
                ++slot;
                left = per;
            }
        }
    }
    if (TOP && left != per) {
        sh.gmax[slot * kScThreads + tid] = gm;
        own = __builtin_fmaxf(own, gm);
    }
    if (nvec * VEC + tid < len) {
        const float x = Elem<T>::load1(row + nvec * VEC + tid);
        const float one[1] = {x};
        add(x, one);
        if (TOP) {
            rank += x >= xt ? 1u : 0u;
            const float z = __builtin_fmaxf(x, -kExpInf);  // (a NaN is none)
            sh.gmax[kScSlots * kScThreads + tid] = z;
            own = __builtin_fmaxf(own, z);
        }
    }
    ScSum t;
    {
        // from the reference, whose product is rounded, to the maximum
        const float d = -__builtin_fmaf(__builtin_fmaxf(run.m, run.floor), c, -run.ref), f = es_exp2(d);
        t.m = run.m;
        t.s = run.s * f;
        t.w = (wsum + run.s * d) * f;
        // (logits below the floor alone: relative to it, not to their maximum; they add nothing to a sum that is not far)
    }
    t.wave_merge(c);
    if ((tid & 63) == 0) { sh.m[tid >> 6] = t.m; sh.s[tid >> 6] = t.s; sh.w[tid >> 6] = t.w; }
    __syncthreads();
    t = ScSum();
#pragma unroll
    for (int i = 0; i < NW; ++i) t.merge(sh.m[i], sh.s[i], sh.w[i], c);
    if (exp_far(t.m, c)) {  // (every thread alike: a second read of the part, from the caches)
        float s = 0.0f, w = 0.0f;
        sc_each<T>(row, len, [&](float x, int) {
            const float y = (x - t.m) * c, e = es_exp2(y);
            s += e;
            if (ENT) w = __builtin_fmaf(e, __builtin_fmaxf(y, kScLeast), w);
        });
        s = es_wave_sum(s);
        w = es_wave_sum(w);
        __syncthreads();
        if ((tid & 63) == 0) { sh.s[tid >> 6] = s; sh.w[tid >> 6] = w; }
        __syncthreads();
        t.s = t.w = 0.0f;
#pragma unroll
        for (int i = 0; i < NW; ++i) { t.s += sh.s[i]; t.w += sh.w[i]; }
    }
    if (TOP) {
        rank = sc_block_sum(sh, rank);
        if (L > 0) sc_top<T>(row, len, lo, L, per, own, sh);
    }
    if (S > 1) {
        // the part that arrives last joins them
        const size_t at = (size_t)r * S + p;
        if (TOP && tid < L) ag_store64(&a.list[at * L + tid], sh.top[tid]);
        if (tid == 0) {
            ag_store64(&a.rec[at].ms, ((uint64_t)f2u(t.m) << 32) | f2u(t.s));
            ag_store64(&a.rec[at].wn, ((uint64_t)f2u(t.w) << 32) | rank);
        }
        stores_complete();
        __syncthreads();
        if (tid == 0) last = ag_add32(&a.ctr[r], 1u) == (uint32_t)S - 1u ? 1u : 0u;
        __syncthreads();
        if (!last) return;
        if (tid == 0) ag_store32(&a.ctr[r], 0u);
        t = ScSum();
        rank = 0u;
        const int part = tid & 63;
        if (part < S) {  // (S <= 64: a lane each, in every wave)
            const uint64_t v = ag_load64(&a.rec[(size_t)r * S + part].ms), w = ag_load64(&a.rec[(size_t)r * S + part].wn);
            t.m = u2f((uint32_t)(v >> 32));
            t.s = u2f((uint32_t)v);
            t.w = u2f((uint32_t)(w >> 32));
            rank = (uint32_t)w;
        }
        t.wave_merge(c);
        if (TOP) {
            VWS_BUTTERFLY(rank, lane_xor, sc_plus);
            if (L > 0) {
                // every part's first ceil(L / S) reach the least of those parts' last: L together
                const uint64_t* list = a.list + (size_t)r * S * L;
                const int deep = (L + S - 1) / S;
                const uint32_t least = part < S ? (uint32_t)(ag_load64(list + (size_t)part * L + deep - 1) >> 32) : ~0u;
                const uint32_t t = wave_min_u32(least);
                if (tid == 0) sh.cands = 0u;
                __syncthreads();
                for (int i = tid; i < S * L; i += kScThreads) {
                    const uint64_t k = ag_load64(list + i);
                    if (k && (uint32_t)(k >> 32) >= t) sh.cand[atomicAdd(&sh.cands, 1u)] = k;
                }
                __syncthreads();
                sc_sort(sh, L);
            }
        }
    }
    const bool some = t.s > 0.0f || t.s != t.s;
    const float ln_s = some ? logf(t.s) : __builtin_nanf("");
    const float h = ln_s - kScLn2 * (t.w / t.s);
    if (tid == 0) {
        const float lp = (xt - t.m) * a.inv_T - ln_s;
        a.logprobs[r] = lp;
        if (ENT) a.entropy[r] = h;
        if (TOP) {
            a.ranks[r] = (int32_t)rank;
            a.lp_ids[(size_t)r * (L + 1)] = token;
            a.lp_vals[(size_t)r * (L + 1)] = lp;
        }
        if (a.stats) {
            float* st = a.stats + (size_t)r * kScRowStats;
            st[kScMax] = t.m;
            st[kScInvTotal] = some ? 1.0f / t.s : __builtin_nanf("");
            st[kScLog2Total] = some ? log2f(t.s) : __builtin_nanf("");
            st[kScEntropy] = ENT ? h : 0.0f;
            st[kScLive] = 1.0f;
        }
    }
    if (TOP && tid < L) {
        const uint64_t k = sh.top[tid];
        const size_t at = (size_t)r * (L + 1) + 1 + tid;
        a.lp_ids[at] = k ? (int32_t)(0xFFFFFFFFu - (uint32_t)k) : -1;
        a.lp_vals[at] = k ? (val_of((uint32_t)(k >> 32)) - t.m) * a.inv_T - ln_s : __builtin_nanf("");
    }
}

// The gradient of part p of row r.  Rows from the last to the first: those that the forward read last are still
// in the last-level cache; gradients are stored past it.
template <typename T>
__global__ __launch_bounds__(kScThreads) void score_backward_kernel(ScoreArgs a) {
    constexpr int VEC = Elem<T>::kVec, U = 4;
    const int S = a.S, block = gridDim.x - 1 - blockIdx.x, r = block / S, p = block - r * S, tid = threadIdx.x;
    const T* row = static_cast<const T*>(a.x) + (size_t)r * a.xstride;
    T* out = static_cast<T*>(a.grad) + (size_t)r * a.gstride;
    const int lo = p * a.part_len, len = min(a.V, lo + a.part_len) - lo, nvec = len / VEC, tail = nvec * VEC + tid;
    row += lo;
    out += lo;
    const float* st = a.stats + (size_t)r * kScRowStats;
    const float gl = (a.gl ? a.gl[r] : 0.0f) * a.inv_T, gh = (a.gh ? a.gh[r] : 0.0f) * a.inv_T;
    // (a row that is not a number has no total, and a gradient of NaN whatever its upstream)
    if (st[kScLive] == 0.0f || (gl == 0.0f && gh == 0.0f && st[kScLog2Total] == st[kScLog2Total])) {
        const uint32_t zero[4] = {0u, 0u, 0u, 0u};
        for (int vi = tid; vi < nvec; vi += kScThreads) sc_store<T>(out, vi, zero);
        if (tail < len) out[tail] = sc_narrow<T>(0.0f);
        return;
    }
    const int at = a.ids[r] - lo, tvec = at >= 0 && at < nvec * VEC ? at / VEC : -1;  // the token's vector here
    const float m = st[kScMax], c = a.c, ref = m * c;
    // log p_j = ln 2 (y_j - y_m - log2 S)
    const float a0 = -(gl + gh * (st[kScEntropy] - kScLn2 * st[kScLog2Total])), a1 = -gh * kScLn2;
    auto stream = [&](auto value) __attribute__((always_inline)) {
        for (int b = tid; b < nvec; b += U * kScThreads) {
            uint32_t w[U][4];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int vi = b + u * kScThreads;
                row_load<T>(row, vi < nvec ? vi : b, w[u]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int vi = b + u * kScThreads;
                float v[VEC];
                Elem<T>::from_words(w[u][0], w[u][1], w[u][2], w[u][3], v);
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] = value(v[j]);
                if (vi == tvec) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) v[j] += j == at - tvec * VEC ? gl : 0.0f;
                }
                sc_pack<T>(v, w[u]);
                if (vi < nvec) sc_store<T>(out, vi, w[u]);
            }
        }
        if (tail < len) out[tail] = sc_narrow<T>(value(Elem<T>::load1(row + tail)) + (tail == at ? gl : 0.0f));
    };
    const float inv = st[kScInvTotal];
    if (exp_far(m, c)) {
        stream([&](float x) __attribute__((always_inline)) {
            const float y = (x - m) * c;
            return es_exp2(y) * inv * __builtin_fmaf(a1, __builtin_fmaxf(y, kScLeast), a0);
        });
    } else {
        // (ref is off m c by its rounding, and so is every power)
        const float d = __builtin_fmaf(m, c, -ref), near = inv * es_exp2(-d);
        const float b0 = near * (a0 - a1 * d), b1 = near * a1;
        stream([&](float x) __attribute__((always_inline)) {
            const float y = __builtin_fmaf(x, c, -ref);
            return es_exp2(y) * __builtin_fmaf(b1, __builtin_fmaxf(y, kScLeast), b0);
        });
    }
}

#define VWS_SCORE(T)                                             \
    template __global__ void score_kernel<T, false, false>(ScoreArgs); \
    template __global__ void score_kernel<T, true, false>(ScoreArgs);  \
    template __global__ void score_kernel<T, false, true>(ScoreArgs);  \
    template __global__ void score_kernel<T, true, true>(ScoreArgs);   \
    template __global__ void score_backward_kernel<T>(ScoreArgs);
VWS_SCORE(float)
VWS_SCORE(uint16_t)
VWS_SCORE(_Float16)

}  // namespace vws
