// vws_distill.hip -- distillation from a teacher's top log-probabilities: loss, gradient, and
// both in one kernel.
//
// A row: student logits x [V], teacher entries (t_k, l_k), k < K, weight w, temperature T.
// With z = x / T, q = softmax(z):
//   renormalize: p = softmax_k(l / T);              L = w sum_k p_k (log p_k - log q_k)
//                                                   dL/dx_j = w / T (q_j - p_j)
//   bucket:      p = exp(l), r = 1 - sum p, s = sum of q outside the entries;
//                                                   L = w (sum_k ... + r log(r / s))
//                dL/dx_j = w / T (t q_j - p_j) at the entries, w / T q_j (t - r / s) elsewhere, t = r + sum p
//                (1, but where the entries' sum exceeds 1: r is 0 then, or the rest is no event).
// Exponentials are powers of two of x * log2(e) / T relative to a maximum; one fma and one exp2 per logit
// (vws_expsum.h).  Rows whose maximum is far from zero in those units (a mask's value, mostly) take
// differences from it instead.  s is the sum over the rest, never 1 - sum of the entries (which cancels when
// the student is sure), and the rest keeps its own maximum, so that log(s) and q_j / s stay finite
// however far the rest lies below the entries: q_j (t - r / s) = e_j (t s - r) / Z_rest with e_j and
// Z_rest relative to the rest's maximum.
#include "vws_device.h"
#include "vws_distill.h"
#include "vws_expsum.h"
#include "vws_sampler.h"

namespace vws {

constexpr float kLn2 = 0x1.62e43p-1f;

// Widened logits back to a row's words.
template <typename T> struct DsVec;
template <> struct DsVec<float> {
    static constexpr uint32_t kNegInf = 0xFF800000u;
    static __device__ __forceinline__ void set_neg_inf(uint32_t (&w)[4], int j) { w[j] = kNegInf; }
    static __device__ __forceinline__ void pack(const float* v, uint32_t (&w)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = f2u(v[i]);
    }
    static __device__ __forceinline__ float narrow(float v) { return v; }
};
template <> struct DsVec<uint16_t> {
    static constexpr uint32_t kNegInf = 0xFF80FF80u;
    static __device__ __forceinline__ void set_neg_inf(uint32_t (&w)[4], int j) {
        w[j >> 1] = (j & 1) ? (w[j >> 1] & 0xFFFFu) | 0xFF800000u : (w[j >> 1] & 0xFFFF0000u) | 0xFF80u;
    }
    static __device__ __forceinline__ uint16_t narrow(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
    static __device__ __forceinline__ void pack(const float* v, uint32_t (&w)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (uint32_t)narrow(v[2 * i]) | ((uint32_t)narrow(v[2 * i + 1]) << 16);
    }
};
template <> struct DsVec<_Float16> {
    static constexpr uint32_t kNegInf = 0xFC00FC00u;
    static __device__ __forceinline__ void set_neg_inf(uint32_t (&w)[4], int j) {
        w[j >> 1] = (j & 1) ? (w[j >> 1] & 0xFFFFu) | 0xFC000000u : (w[j >> 1] & 0xFFFF0000u) | 0xFC00u;
    }
    static __device__ __forceinline__ _Float16 narrow(float v) { return (_Float16)v; }
    static __device__ __forceinline__ void pack(const float* v, uint32_t (&w)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = (uint32_t)__builtin_bit_cast(uint16_t, narrow(v[2 * i])) |
                   ((uint32_t)__builtin_bit_cast(uint16_t, narrow(v[2 * i + 1])) << 16);
    }
};

// row_load for logits that are read once: they leave the caches to the gradients on their way out.
template <typename T>
__device__ __forceinline__ void ds_load_once(const T* row, int vi, uint32_t (&w)[4]) {
    const auto u = __builtin_nontemporal_load(
        reinterpret_cast<const typename RowVec<T>::U4*>(reinterpret_cast<const char*>(row) + 16u * (uint32_t)vi));
    w[0] = u[0]; w[1] = u[1]; w[2] = u[2]; w[3] = u[3];
}
// (not temporal: what the forward has read stays in the last-level cache for the backward)
template <typename T>
__device__ __forceinline__ void ds_store(T* row, int vi, const uint32_t (&w)[4]) {
    typename RowVec<T>::U4 u;
    u[0] = w[0]; u[1] = w[1]; u[2] = w[2]; u[3] = w[3];
    __builtin_nontemporal_store(u, reinterpret_cast<typename RowVec<T>::U4*>(reinterpret_cast<char*>(row) + 16u * (uint32_t)vi));
}

// Adds U vectors (widened) to a thread's running sum: their maximum first, then one exponential
// each and one for the rescaling.  NaN and +inf make the sum NaN, as log-softmax has it.
template <typename T, int U>
__device__ __forceinline__ void ds_add(ExpRun& t, const uint32_t (&w)[U][4], float c) {
    constexpr int VEC = Elem<T>::kVec;
    float v[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) Elem<T>::from_words(w[u][0], w[u][1], w[u][2], w[u][3], v[u]);
    float g = v[0][0];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < VEC; ++j) g = __builtin_fmaxf(g, v[u][j]);
    float a[4] = {t.raise(g, c), 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < VEC; ++j) a[j & 3] += es_exp2(__builtin_fmaf(v[u][j], c, -t.ref));
    t.s = (a[0] + a[1]) + (a[2] + a[3]);
}

__device__ __forceinline__ void ds_add1(ExpRun& t, float x, float c) {
    const float had = t.raise(x, c);
    t.s = had + es_exp2(__builtin_fmaf(x, c, -t.ref));
}

// Bitmap of a part's elements that are teacher entries, from its first element on.
__device__ __forceinline__ void ds_clear_bits(uint32_t* bm, int len) {
    for (int i = threadIdx.x; i < (len + 31) / 32; i += blockDim.x) bm[i] = 0u;
}
__device__ __forceinline__ void ds_set_bit(uint32_t* bm, int len, int d) {
    if (d >= 0 && d < len) atomicOr(&bm[d >> 5], 1u << (d & 31));
}
template <typename T>
__device__ __forceinline__ uint32_t ds_bits(const uint32_t* bm, int vi) {
    constexpr int VEC = Elem<T>::kVec;
    return (bm[(vi * VEC) >> 5] >> ((vi * VEC) & 31)) & ((1u << VEC) - 1u);
}

// Sets the elements of vector vi whose bit is set to -inf.
template <typename T>
__device__ __forceinline__ void ds_drop(const uint32_t* bm, int vi, uint32_t (&w)[4]) {
    constexpr int VEC = Elem<T>::kVec;
    const uint32_t b = ds_bits<T>(bm, vi);
    if (b) {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if ((b >> j) & 1u) DsVec<T>::set_neg_inf(w, j);
    }
}

// A part's running sum: elements [0, len) of `row`, without those whose bit is set (BUCKET).  The next
// four vectors' loads are issued before these are used; the first before `ready` (the bitmap).
template <typename T, bool BUCKET, typename F>
__device__ __forceinline__ ExpSum ds_stream(const T* row, int len, float c, const uint32_t* bm, F ready) {
    constexpr int VEC = Elem<T>::kVec, U = 4;
    const int nvec = len / VEC, tid = threadIdx.x;
    uint32_t next[U][4];
    auto fetch = [&](int b) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u) row_load<T>(row, min(b + u * kDsThreads, nvec - 1), next[u]);
    };
    if (nvec > 0) fetch(tid);
    ready();
    ExpRun t(c);
    for (int b = tid; b < nvec; b += U * kDsThreads) {
        uint32_t w[U][4];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < 4; ++k) w[u][k] = next[u][k];
        if (b + U * kDsThreads < nvec) fetch(b + U * kDsThreads);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int vi = b + u * kDsThreads;
            if (vi >= nvec) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) DsVec<T>::set_neg_inf(w[u], j);
            } else if (BUCKET) {
                ds_drop<T>(bm, vi, w[u]);
            }
        }
        ds_add<T, U>(t, w, c);
    }
    const int i = nvec * VEC + tid;
    if (i < len && !(BUCKET && ((bm[i >> 5] >> (i & 31)) & 1u))) ds_add1(t, Elem<T>::load1(row + i), c);
    return t.close(c);
}

// This thread's share of the sum of a part whose maximum m is far from zero, over differences from it.
template <typename T, bool BUCKET>
__device__ __forceinline__ float ds_far_sum(const T* row, int len, float c, const uint32_t* bm, float m) {
    constexpr int VEC = Elem<T>::kVec;
    const int nvec = len / VEC, i = nvec * VEC + (int)threadIdx.x;
    float s = 0.0f;
    for (int vi = threadIdx.x; vi < nvec; vi += kDsThreads) {
        uint32_t w[4];
        row_load<T>(row, vi, w);
        if (BUCKET) ds_drop<T>(bm, vi, w);
        float v[VEC];
        Elem<T>::from_words(w[0], w[1], w[2], w[3], v);
#pragma unroll
        for (int j = 0; j < VEC; ++j) s += es_exp2((v[j] - m) * c);
    }
    if (i < len && !(BUCKET && ((bm[i >> 5] >> (i & 31)) & 1u))) s += es_exp2((Elem<T>::load1(row + i) - m) * c);
    return s;
}

// A row's teacher entry k, one for each of a workgroup's first K threads (id -1: none).
struct DsEntry {
    int id;
    float l, x;  // its log-probability, the student's logit
};
__device__ __forceinline__ DsEntry ds_entry(const DistillArgs& a, int r) {
    const int k = threadIdx.x;
    DsEntry e{-1, -kExpInf, 0.0f};
    if (k < a.K) {
        e.id = a.ids[(size_t)r * a.ids_stride + k];
        e.l = a.lp[(size_t)r * a.lp_stride + k];
        if (e.id < 0 || e.id >= a.V) e.id = -1;
    }
    return e;
}

// The entries' ids, hashed: at most 256 of 512 places are taken.
struct DsHash {
    int32_t id[2 * kDsMaxK];
    uint32_t first[2 * kDsMaxK], count[2 * kDsMaxK];  // its first entry, its entries
    float value[2 * kDsMaxK];                         // its gradient (step)
    __device__ __forceinline__ void clear() {
        for (int i = threadIdx.x; i < 2 * kDsMaxK; i += blockDim.x) {
            id[i] = -1;
            first[i] = ~0u;
            count[i] = 0u;
        }
    }
    __device__ __forceinline__ int insert(int t) {
        int slot = (int)(((uint32_t)t * 2654435761u) >> 23);
        for (;;) {
            const int had = atomicCAS(&id[slot], -1, t);
            if (had == -1 || had == t) break;
            slot = (slot + 1) & (2 * kDsMaxK - 1);
        }
        atomicMin(&first[slot], threadIdx.x);
        atomicAdd(&count[slot], 1u);
        return slot;
    }
    __device__ __forceinline__ float of(int t) const {  // (t has been inserted)
        int slot = (int)(((uint32_t)t * 2654435761u) >> 23);
        while (id[slot] != t) slot = (slot + 1) & (2 * kDsMaxK - 1);
        return value[slot];
    }
};

struct DsShared {
    float wm[kDsStepThreads / 64], ws[kDsStepThreads / 64];  // the waves' sums
    float top[kDsMaxK / 64], sums[kDsMaxK / 64][5];          // the entries' maxima and sums, of four waves
    float p[kDsMaxK];
    int32_t id[kDsMaxK];
};

struct DsRow {
    float ref, coef, max, inv_total;  // DistillStat
    bool live;
    float p;                          // P of this thread's entry (-1: none)
};

// Each wave's merged sum, and all of them (after a barrier).
__device__ __forceinline__ void ds_put(DsShared& sh, const ExpSum& t) {
    if ((threadIdx.x & 63) == 0) { sh.wm[threadIdx.x >> 6] = t.m; sh.ws[threadIdx.x >> 6] = t.s; }
}
template <int NW>
__device__ __forceinline__ ExpSum ds_get(const DsShared& sh, float c) {
    ExpSum t;
#pragma unroll
    for (int i = 0; i < NW; ++i) t.m = __builtin_fmaxf(t.m, sh.wm[i]);
    const float ref = t.m == -kExpInf ? 0.0f : t.m;
#pragma unroll
    for (int i = 0; i < NW; ++i) t.s += sh.ws[i] * es_exp2((sh.wm[i] - ref) * c);
    return t;
}

// The entries' ids and their maxima, for ds_finish after a barrier: of the student over its entries
// (BUCKET), or of the teacher.
template <bool BUCKET>
__device__ __forceinline__ void ds_put_entries(const DistillArgs& a, const DsEntry& e, DsShared& sh) {
    const int k = threadIdx.x, wave = k >> 6;
    const float logp = e.l * a.inv_T;
    // (a NaN makes the row NaN by way of the sums)
    const float mine = e.id >= 0 ? (BUCKET ? e.x : (logp != logp ? kExpInf : logp)) : -kExpInf;
    if (wave < kDsMaxK / 64) {
        const float m = es_wave_max(mine);
        if ((k & 63) == 0) sh.top[wave] = m;
    }
    if (k < a.K) sh.id[k] = e.id;
}

// A row's loss and statistics, from its sum over the rest (BUCKET) or all of it and what ds_put_entries left.
// Every thread of the workgroup calls; `slot`: where this thread's entry was inserted, since the last
// barrier or before.  One barrier.
template <typename T, bool BUCKET>
__device__ __forceinline__ DsRow ds_finish(const DistillArgs& a, int r, const ExpSum& rest, float w, DsEntry e, int slot,
                                           const DsHash& hash, DsShared& sh) {
    constexpr int EW = kDsMaxK / 64;
    const int k = threadIdx.x, K = a.K, wave = k >> 6;
    const bool valid = e.id >= 0, lead = (k & 63) == 0;
    const float logp = BUCKET ? e.l : e.l * a.inv_T;
    const float ref = rest.m == -kExpInf ? 0.0f : rest.m;
    float top = -kExpInf;
#pragma unroll
    for (int i = 0; i < EW; ++i) top = __builtin_fmaxf(top, sh.top[i]);
    const float M = BUCKET ? __builtin_fmaxf(rest.m, top) : rest.m, mref = M == -kExpInf ? 0.0f : M;
    // entries that share an id: the first takes their probability together
    const bool first = valid && hash.first[slot] == (uint32_t)k, several = first && hash.count[slot] > 1u;
    // then the sums: p, p log p, p T (log q + log(total)) (scaled, so that up to 256 entries of the type's
    // lowest value do not overflow), the student's at the entries, the entries
    float p = 0.0f;
    if (valid) p = BUCKET ? expf(logp) : (top > -kExpInf ? expf(logp - top) : 0.0f);
    const float gap = e.x - mref;
    const bool on = valid && !(p <= 0.0f);
    float v[5] = {p, on ? p * (BUCKET ? logp : logp - top) : 0.0f, on ? p * (gap * 0x1p-10f) : 0.0f,
                  BUCKET && first ? es_exp2(gap * a.c) : 0.0f, valid ? 1.0f : 0.0f};
    if (k < K) sh.p[k] = p;
    if (wave < EW) {
#pragma unroll
        for (int i = 0; i < 5; ++i) {
            v[i] = es_wave_sum(v[i]);
            if (lead) sh.sums[wave][i] = v[i];
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 5; ++i) {
        v[i] = 0.0f;
#pragma unroll
        for (int q = 0; q < EW; ++q) v[i] += sh.sums[q][i];
    }
    if (several) {
        p = 0.0f;
        for (int i = 0; i < K; ++i)
            if (sh.id[i] == e.id) p += sh.p[i];
    }
    DsRow o;
    o.max = mref;
    o.ref = ref;
    const float Z = BUCKET ? (rest.s != 0.0f ? rest.s * es_exp2((ref - mref) * a.c) : 0.0f) + v[3] : rest.s;
    const bool some = Z > 0.0f || Z != Z;  // (no finite logit: every log q is -inf)
    const float lz = some ? log2f(Z) : 0.0f;
    o.inv_total = some ? 1.0f / Z : 0.0f;
    float L;
    if (BUCKET) {
        o.live = v[4] > 0.0f;
        const float sp = v[0], rr = 1.0f - sp;
        L = v[1] - v[2] * a.inv_T * 0x1p10f + lz * sp * kLn2;
        // a rest without a finite logit is no event
        const bool have = rest.s > 0.0f || rest.s != rest.s;
        const float rem = have && !(rr < 0.0f) ? rr : 0.0f;
        if (!(rem <= 0.0f)) L += rem * (logf(rem) - (rest.m - mref) * a.inv_T - (log2f(rest.s) - lz) * kLn2);
        // the teacher's events add up to tot, 1 but where the rest is no event or sp exceeds 1:
        // an entry's gradient is tot q - p, the rest's tot q - rem q / s
        const float tot = sp + rem;
        o.coef = have ? (tot * (rest.s * es_exp2((ref - mref) * a.c) * o.inv_total) - rem) / rest.s : 0.0f;
        o.inv_total *= tot;
    } else {
        o.live = top > -kExpInf;
        const float inv = 1.0f / v[0];
        L = v[1] * inv - v[2] * inv * a.inv_T * 0x1p10f - logf(v[0]) + lz * kLn2;
        o.coef = o.inv_total;
        p *= inv;
    }
    o.p = first ? p : -1.0f;
    if (k == 0) a.loss[r] = o.live ? w * L : 0.0f;
    return o;
}

// Leaves a row's statistics for the backward.
__device__ __forceinline__ void ds_save(const DistillArgs& a, int r, const DsRow& o) {
    const int k = threadIdx.x;
    if (k < a.K) a.entry_p[(size_t)r * a.K + k] = o.p;
    if (k == 0) {
        float* st = a.stats + (size_t)r * kDsRowStats;
        st[kDsRef] = o.ref;
        st[kDsCoef] = o.coef;
        st[kDsMax] = o.max;
        st[kDsInvTotal] = o.inv_total;
        st[kDsLive] = o.live ? 1.0f : 0.0f;
    }
}

// Loss of rows split over workgroups: each part's running maximum and sum in one read, entries kept out of
// the rest's sum by a bitmap; the part that arrives last joins them and takes the entries' logits.
// Bound: HBM: 512 x 151936 bf16 (156 MB) 30.8 us, 5.05 TB/s, a copy's rate; before a gradient it leaves what it reads
// to the caches (2048 x 128256 bf16, three rows in ten weightless, 353 MB fetched: 80 us, 4.4 TB/s).  4 x 32000
// fp32 6.6 us, 301 x 50257 17 (starts and ends of the launch, unaligned rows).
template <typename T, bool BUCKET>
__global__ __launch_bounds__(kDsThreads) void distill_forward_kernel(DistillArgs a) {
    extern __shared__ uint32_t bm[];
    __shared__ DsShared sh;
    __shared__ DsHash hash;
    __shared__ uint32_t last;
    constexpr int NW = kDsThreads / 64;
    const int S = a.S, r = blockIdx.x / S, p = blockIdx.x - r * S, tid = threadIdx.x;
    const float w = a.weight ? a.weight[r] : 1.0f;
    if (w == 0.0f) {  // the row does not count: not read
        if (p == 0 && tid == 0) {
            a.loss[r] = 0.0f;
            a.stats[(size_t)r * kDsRowStats + kDsLive] = 0.0f;
        }
        return;
    }
    const T* row = static_cast<const T*>(a.x) + (size_t)r * a.xstride;
    const int lo = p * a.part_len, len = min(a.V, lo + a.part_len) - lo;
    DsEntry e = ds_entry(a, r);
    ExpSum t = ds_stream<T, BUCKET>(row + lo, len, a.c, bm, [&] {
        hash.clear();
        if (BUCKET) {
            ds_clear_bits(bm, len);
            __syncthreads();
            if (e.id >= 0) ds_set_bit(bm, len, e.id - lo);
        }
        __syncthreads();
    });
    t.wave_merge(a.c);
    ds_put(sh, t);
    __syncthreads();
    t = ds_get<NW>(sh, a.c);
    if (exp_far(t.m, a.c)) {  // (every thread alike: a second read of the part, from the caches)
        const float mine = es_wave_sum(ds_far_sum<T, BUCKET>(row + lo, len, a.c, bm, t.m));
        __syncthreads();
        if ((tid & 63) == 0) sh.ws[tid >> 6] = mine;
        __syncthreads();
        t.s = 0.0f;
#pragma unroll
        for (int i = 0; i < NW; ++i) t.s += sh.ws[i];
    }
    if (S > 1) {
        // the part that arrives last joins them, in their order
        if (tid == 0) {
            ag_store64(&a.rec[(size_t)r * S + p], ((uint64_t)f2u(t.m) << 32) | f2u(t.s));
            stores_complete();
            last = ag_add32(&a.ctr[r], 1u) == (uint32_t)S - 1u ? 1u : 0u;
        }
        __syncthreads();
        if (!last) return;
        if (tid == 0) ag_store32(&a.ctr[r], 0u);
        t = ExpSum();
        const int part = tid & 63;
        if (part < S) {  // (S <= 64: a lane each, in every wave)
            const uint64_t v = ag_load64(&a.rec[(size_t)r * S + part]);
            t.m = u2f((uint32_t)(v >> 32));
            t.s = u2f((uint32_t)v);
        }
        t.wave_merge(a.c);
    }
    int slot = 0;
    if (e.id >= 0) {
        slot = hash.insert(e.id);
        e.x = Elem<T>::load1(row + e.id);
    }
    ds_put_entries<BUCKET>(a, e, sh);
    __syncthreads();
    const DsRow o = ds_finish<T, BUCKET>(a, r, t, w, e, slot, hash, sh);
    ds_save(a, r, o);
}

// The gradient of part p of row r.  Rows from the last to the first: those that the forward read last
// are still in the last-level cache.  Gradients are stored past the caches, which keeps the logits there
// (forward and backward of 2048 x 128256 bf16: 244 us, 287 with plain stores).
// Bound: HBM: of those rows 149 us, 353 MB fetched and 502 written, 5.7 TB/s; 301 x 50257 fp32 (121 MB) 22 us.
template <typename T>
__global__ __launch_bounds__(kDsThreads) void distill_backward_kernel(DistillArgs a) {
    constexpr int VEC = Elem<T>::kVec, U = 4;
    const int S = a.S, block = gridDim.x - 1 - blockIdx.x, r = block / S, p = block - r * S, tid = threadIdx.x;
    const T* row = static_cast<const T*>(a.x) + (size_t)r * a.xstride;
    T* out = static_cast<T*>(a.grad) + (size_t)r * a.gstride;
    const int lo = p * a.part_len, len = min(a.V, lo + a.part_len) - lo, nvec = len / VEC;
    const float* st = a.stats + (size_t)r * kDsRowStats;
    const float gs = (a.weight ? a.weight[r] : 1.0f) * (a.gout ? a.gout[r] : 1.0f) * a.inv_T;
    const int tail = nvec * VEC + tid;
    if (st[kDsLive] == 0.0f || gs == 0.0f) {
        const uint32_t zero[4] = {0u, 0u, 0u, 0u};
        for (int vi = tid; vi < nvec; vi += kDsThreads) ds_store<T>(out + lo, vi, zero);
        if (tail < len) out[lo + tail] = DsVec<T>::narrow(0.0f);
        return;
    }
    // this thread's teacher entry, where it lies in the part: read before anything is written
    // (the gradient may take the logits' place)
    int at = -1;
    float fix = 0.0f;
    if (tid < a.K) {
        const float P = a.entry_p[(size_t)r * a.K + tid];
        const int id = a.ids[(size_t)r * a.ids_stride + tid];
        if (!(P < 0.0f) && id >= lo && id < lo + len) {
            at = id;
            const float q = es_exp2((Elem<T>::load1(row + id) - st[kDsMax]) * a.c) * st[kDsInvTotal];
            fix = gs * (q - P);
        }
    }
    __syncthreads();
    const float m = st[kDsRef], ref = m * a.c, coef = st[kDsCoef] * gs;
    auto stream = [&](auto value) __attribute__((always_inline)) {
        for (int b = tid; b < nvec; b += U * kDsThreads) {
            uint32_t w[U][4];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int vi = b + u * kDsThreads;
                row_load<T>(row + lo, vi < nvec ? vi : b, w[u]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int vi = b + u * kDsThreads;
                float v[VEC];
                Elem<T>::from_words(w[u][0], w[u][1], w[u][2], w[u][3], v);
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] = value(v[j]);
                DsVec<T>::pack(v, w[u]);
                if (vi < nvec) ds_store<T>(out + lo, vi, w[u]);
            }
        }
        if (tail < len) out[lo + tail] = DsVec<T>::narrow(value(Elem<T>::load1(row + lo + tail)));
    };
    if (exp_far(m, a.c)) {
        stream([&](float v) __attribute__((always_inline)) { return es_exp2((v - m) * a.c) * coef; });
    } else {
        // (ref is off m c by its rounding, and so is every power)
        const float near = coef * es_exp2(-__builtin_fmaf(m, a.c, -ref));
        stream([&](float v) __attribute__((always_inline)) { return es_exp2(__builtin_fmaf(v, a.c, -ref)) * near; });
    }
    // the teacher's entries over what the stream wrote there, once that has arrived
    stores_complete();
    __syncthreads();
    if (at >= 0) out[at] = DsVec<T>::narrow(fix);
}

// Loss and gradient of rows that one workgroup holds in its registers (NV vectors a thread): every
// logit is read once and its gradient written once.  One workgroup for each compute unit, a row at a
// time; as a row's gradients are written, the next row's logits and entries are loaded into the
// registers they leave.  No barrier waits for memory: a vector that holds teacher entries (by the
// bitmap) takes their gradients from the hash, so nothing is written twice.
// Bound: HBM: 4096 x 128256 bf16 (1.05 GB read and as much written) 465 us, 4.5 TB/s of a copy's 5.07; forward and
// backward kernels take 593.  What is left is each row's two reductions, in which its workgroup moves nothing but
// the next row's loads.
template <typename T, bool BUCKET, int NV>
__global__ __launch_bounds__(kDsStepThreads) void distill_step_kernel(DistillArgs a) {
    constexpr int VEC = Elem<T>::kVec, U = 2, NW = kDsStepThreads / 64;
    extern __shared__ uint32_t bms[];  // two bitmaps: this row's and the next one's
    __shared__ DsShared sh;
    __shared__ DsHash hashes[2];
    const int tid = threadIdx.x, V = a.V, nvec = V / VEC, edge = nvec * VEC + tid, words = (V + 31) / 32;
    const T* x = static_cast<const T*>(a.x);
    T* grad = static_cast<T*>(a.grad);
    auto live = [&](int r) { return !a.weight || a.weight[r] != 0.0f; };
    uint32_t w[NV][4];
    float xe = 0.0f;  // the thread's logit past the last vector
    // What follows is for registers: the scheduler must not work on many vectors at once, nor the
    // compiler keep every vector's offsets, bounds or widened logits from one use to the next.
    auto fence = []() __attribute__((always_inline)) { __builtin_amdgcn_sched_barrier(0); };
    auto fresh = [](int v) __attribute__((always_inline)) {
        asm volatile("" : "+v"(v));
        return v;
    };
    // vectors past `end` repeat it: every load is unconditional
    auto fetch = [&](const T* row, int q, int end) __attribute__((always_inline)) {
        ds_load_once<T>(row, min(fresh(tid) + q * kDsStepThreads, end), w[q]);
    };
    int r = blockIdx.x;
    auto skip = [&]() {  // rows that do not count: zeros
        for (; r < a.N && !live(r); r += gridDim.x) {
            const uint32_t zero[4] = {0u, 0u, 0u, 0u};
            T* out = grad + (size_t)r * a.gstride;
            for (int vi = tid; vi < nvec; vi += kDsStepThreads) ds_store<T>(out, vi, zero);
            if (edge < V) out[edge] = DsVec<T>::narrow(0.0f);
            if (tid == 0) a.loss[r] = 0.0f;
        }
    };
    skip();
    if (r >= a.N) return;
    DsEntry e = ds_entry(a, r);
#pragma unroll
    for (int q = 0; q < NV; ++q) fetch(x + (size_t)r * a.xstride, q, nvec - 1);
    if (edge < V) xe = Elem<T>::load1(x + (size_t)r * a.xstride + edge);
    if (e.id >= 0) e.x = Elem<T>::load1(x + (size_t)r * a.xstride + e.id);
    hashes[0].clear();
    ds_clear_bits(bms, V);
    __syncthreads();
    // A row of 128256 bf16 takes a workgroup some 13 us of sums and then some 15 of reading and writing.
    // Started together the workgroups would keep time, and the memory idle while all sum: they start
    // up to most of a row's time apart.  Against a common start, us: bf16 1600 x 128256 231 -> 216, 4096 x
    // 487 -> 462, 3328 x 64000 219 -> 212; fp32 4000 x 32000 220 -> 213, but 2048 x
    // 64000 226 -> 231 (twice the sleep for rows of 64000 bf16 would lose: 224).  38 vectors, with a sleep of 5, 64, 133
    // units: bf16 1400 x 151936 232, 220, 219, 3000 x 442, 410, 404; f16 1500 x 140001 240, 246, 248, 2048 x 155000 329, 320, 312;
    // fp32 2048 x 70000 259, 256, 263, 1500 x 77000 221, 217, 225.
    constexpr int kApart = NV > 32 ? 64 : NV * 7 / 2;
    static_assert(kApart <= 127, "the instruction takes seven bits");
    for (int k = (int)((blockIdx.x >> 3) & 7u); k > 0; --k) __builtin_amdgcn_s_sleep(kApart);
    for (int parity = 0;; parity ^= 1) {
        const T* row = x + (size_t)r * a.xstride;
        T* out = grad + (size_t)r * a.gstride;
        const float wt = a.weight ? a.weight[r] : 1.0f;
        DsHash& hash = hashes[parity];
        uint32_t* bm = bms + parity * words;
        int slot = 0;
        if (e.id >= 0) {
            slot = hash.insert(e.id);
            ds_set_bit(bm, V, e.id);
        }
        __syncthreads();
        const bool edge_entry = edge < V && ((bm[edge >> 5] >> (edge & 31)) & 1u);
        // Once, or twice: a row whose largest logit m is far from zero is first moved by it, in its type (x - m is
        // exact where it counts, from m to 2 m or m / 2; what is rounded lies too far below).  Its entries, which may
        // be as far from a masked rest, stay.
        ExpSum rest;
        float moved = 0.0f;
        for (;;) {
            ExpRun t(a.c);
#pragma unroll
            for (int q0 = 0; q0 < NV; q0 += U) {
                uint32_t g[U][4];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int vi = fresh(tid) + (q0 + u) * kDsStepThreads;
                    if (BUCKET) ds_drop<T>(bm, min(vi, nvec - 1), w[q0 + u]);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        // (in place: what lies past the row is never written)
                        w[q0 + u][k] = vi < nvec ? w[q0 + u][k] : DsVec<T>::kNegInf;
                        asm volatile("" : "+v"(w[q0 + u][k]));
                        g[u][k] = w[q0 + u][k];
                    }
                }
                ds_add<T, U>(t, g, a.c);
                fence();
            }
            if (edge < V && !(BUCKET && edge_entry)) ds_add1(t, xe, a.c);
            ExpSum mine = t.close(a.c);
            mine.wave_merge(a.c);
            ds_put(sh, mine);
            ds_put_entries<BUCKET>(a, e, sh);
            __syncthreads();
            rest = ds_get<NW>(sh, a.c);
            if (!exp_far(rest.m, a.c)) break;
#pragma unroll
            for (int q = 0; q < NV; ++q) {
                float v[VEC];
#pragma unroll
                for (int k = 0; k < 4; ++k) asm volatile("" : "+v"(w[q][k]));
                Elem<T>::from_words(w[q][0], w[q][1], w[q][2], w[q][3], v);
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] -= rest.m;
                DsVec<T>::pack(v, w[q]);
#pragma unroll
                for (int k = 0; k < 4; ++k) asm volatile("" : "+v"(w[q][k]));
                fence();
            }
            xe -= rest.m;
            moved = rest.m;
            __syncthreads();  // every wave has the sums of this time
        }
        rest.m += moved;  // (moved: of 0)
        const DsRow o = ds_finish<T, BUCKET>(a, r, rest, wt, e, slot, hash, sh);
        const float gs = wt * (a.gout ? a.gout[r] : 1.0f) * a.inv_T;
        const bool on = o.live && gs != 0.0f;
        const float here = o.ref - moved, ref = here * a.c, coef = o.coef * gs * es_exp2(-__builtin_fmaf(here, a.c, -ref));
        if (!(o.p < 0.0f)) {  // (the first of its id)
            const float q = es_exp2((e.x - o.max) * a.c) * o.inv_total;
            hash.value[slot] = on ? gs * (q - o.p) : 0.0f;
        }
        r += gridDim.x;
        skip();
        const bool more = r < a.N;
        const T* after = more ? x + (size_t)r * a.xstride : row;
        const int end = more ? nvec - 1 : 0;
        e = more ? ds_entry(a, r) : DsEntry{-1, 0.0f, 0.0f};
        hashes[parity ^ 1].clear();
        ds_clear_bits(bms + (parity ^ 1) * words, V);
        __syncthreads();
        auto value = [&](float v) { return on ? es_exp2(__builtin_fmaf(v, a.c, -ref)) * coef : 0.0f; };
#pragma unroll
        for (int q = 0; q < NV; ++q) {
            const int vi = fresh(tid) + q * kDsStepThreads;
            float v[VEC];
#pragma unroll
            for (int k = 0; k < 4; ++k) asm volatile("" : "+v"(w[q][k]));
            Elem<T>::from_words(w[q][0], w[q][1], w[q][2], w[q][3], v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = value(v[j]);
            const uint32_t bits = ds_bits<T>(bm, min(vi, nvec - 1));
            if (bits) {
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if ((bits >> j) & 1u) v[j] = hash.of(min(vi, nvec - 1) * VEC + j);
            }
            uint32_t g[4];
            DsVec<T>::pack(v, g);
            if (vi < nvec) ds_store<T>(out + (size_t)q * kDsStepThreads * VEC, fresh(tid), g);
            fetch(after, q, end);
            fence();
        }
        if (edge < V) out[edge] = DsVec<T>::narrow(edge_entry ? hash.of(edge) : value(xe));
        if (more && edge < V) xe = Elem<T>::load1(after + edge);
        if (e.id >= 0) e.x = Elem<T>::load1(after + e.id);
        if (!more) return;
        __syncthreads();
    }
}

#define VWS_DISTILL_STEP(T, NV)                                                      \
    template __global__ void distill_step_kernel<T, false, NV>(DistillArgs);         \
    template __global__ void distill_step_kernel<T, true, NV>(DistillArgs);
#define VWS_DISTILL_INST(T)                                                   \
    VWS_DISTILL_STEP(T, 16)                                                   \
    VWS_DISTILL_STEP(T, 32)                                                   \
    VWS_DISTILL_STEP(T, 38)                                                   \
    template __global__ void distill_forward_kernel<T, false>(DistillArgs);   \
    template __global__ void distill_forward_kernel<T, true>(DistillArgs);    \
    template __global__ void distill_backward_kernel<T>(DistillArgs);
VWS_DISTILL_INST(float)
VWS_DISTILL_INST(uint16_t)
VWS_DISTILL_INST(_Float16)
#undef VWS_DISTILL_INST

}  // namespace vws
