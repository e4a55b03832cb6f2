// vws_distill.hip -- distillation from a teacher's top log-probabilities: loss, gradient, and
// both in one kernel.
//
// A row: student logits x [V], teacher entries (t_k, l_k), k < K, weight w, temperature T.
// With z = x / T, q = softmax(z):
//   renormalize: p = softmax_k(l / T);              L = w sum_k p_k (log p_k - log q_k)
//                                                   dL/dx_j = w / T (q_j - p_j)
//   bucket:      p = exp(l), r = 1 - sum p, s = sum of q outside the entries;
//                                                   L = w (sum_k ... + r log(r / s))
//                dL/dx_j = w / T (q_j - p_j) at the entries, w / T q_j (1 - r / s) elsewhere.
// Exponentials are powers of two of z2 = x * log2(e) / T relative to a maximum; one fma and one
// exp2 per logit.  s is the sum over the rest, never 1 - sum of the entries (which cancels when
// the student is sure), and the rest keeps its own maximum, so that log(s) and q_j / s stay finite
// however far the rest lies below the entries: q_j (1 - r / s) = e_j (s - r) / Z_rest with e_j and
// Z_rest relative to the rest's maximum.
#include "vws_device.h"
#include "vws_distill.h"
#include "vws_sampler.h"

namespace vws {

constexpr float kDsInf = __builtin_inff();
constexpr float kLn2 = 0x1.62e43p-1f;

__device__ __forceinline__ float ds_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// 16 bytes at any element's address: rows of an odd vocabulary start unaligned.
template <typename T> struct DsVec;
template <> struct DsVec<float> {
    typedef uint32_t U4 __attribute__((ext_vector_type(4), aligned(4)));
    static constexpr uint32_t kNegInf = 0xFF800000u;
    static __device__ __forceinline__ void set_neg_inf(uint32_t (&w)[4], int j) { w[j] = kNegInf; }
    static __device__ __forceinline__ void pack(const float* v, uint32_t (&w)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = f2u(v[i]);
    }
    static __device__ __forceinline__ float narrow(float v) { return v; }
};
template <> struct DsVec<uint16_t> {
    typedef uint32_t U4 __attribute__((ext_vector_type(4), aligned(2)));
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
    typedef uint32_t U4 __attribute__((ext_vector_type(4), aligned(2)));
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

// (vi: a 32-bit offset, at most 2 MB, on the row's pointer)
template <typename T>
__device__ __forceinline__ void ds_load(const T* row, int vi, uint32_t (&w)[4]) {
    const auto u = *reinterpret_cast<const typename DsVec<T>::U4*>(reinterpret_cast<const char*>(row) + 16u * (uint32_t)vi);
    w[0] = u[0]; w[1] = u[1]; w[2] = u[2]; w[3] = u[3];
}
template <typename T>
__device__ __forceinline__ void ds_store(T* row, int vi, const uint32_t (&w)[4]) {
    typename DsVec<T>::U4 u;
    u[0] = w[0]; u[1] = w[1]; u[2] = w[2]; u[3] = w[3];
    __builtin_nontemporal_store(u, reinterpret_cast<typename DsVec<T>::U4*>(reinterpret_cast<char*>(row) + 16u * (uint32_t)vi));
}

__device__ __forceinline__ float ds_lane_xor(float v, int s) { return u2f(lane_xor(f2u(v), s)); }
__device__ __forceinline__ float ds_wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = __builtin_fmaxf(v, ds_lane_xor(v, o));
    return v;
}
__device__ __forceinline__ float ds_wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += ds_lane_xor(v, o);
    return v;
}

// A running (maximum, sum of exp2(z2 - maximum)); the empty one is (-inf, 0).  NaN and +inf make
// the sum NaN, as log-softmax has it.
struct DsSum {
    float m = -kDsInf, s = 0.0f;
    __device__ __forceinline__ void merge(float om, float os) {
        const float n = __builtin_fmaxf(m, om), ref = n == -kDsInf ? 0.0f : n;
        s = s * ds_exp2(m - ref) + os * ds_exp2(om - ref);
        m = n;
    }
    __device__ __forceinline__ void wave_merge() {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) merge(ds_lane_xor(m, o), ds_lane_xor(s, o));
    }
};

// Adds U vectors (widened) to a thread's running sum: their maximum first, then one exponential
// each and one for the rescaling.
template <typename T, int U>
__device__ __forceinline__ void ds_add(DsSum& t, const uint32_t (&w)[U][4], float c) {
    constexpr int VEC = Elem<T>::kVec;
    float v[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) Elem<T>::from_words(w[u][0], w[u][1], w[u][2], w[u][3], v[u]);
    float g = v[0][0];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < VEC; ++j) g = __builtin_fmaxf(g, v[u][j]);
    const float n = __builtin_fmaxf(t.m, g * c), ref = n == -kDsInf ? 0.0f : n;
    float a[4] = {t.s * ds_exp2(t.m - ref), 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < VEC; ++j) a[j & 3] += ds_exp2(__builtin_fmaf(v[u][j], c, -ref));
    t.s = (a[0] + a[1]) + (a[2] + a[3]);
    t.m = n;
}

__device__ __forceinline__ void ds_add1(DsSum& t, float z) {
    t.merge(z, z == z && z < kDsInf ? (z == -kDsInf ? 0.0f : 1.0f) : __builtin_nanf(""));
}

// The bits of a part's elements that are teacher entries, from its first element on.
__device__ __forceinline__ void ds_bitmap(uint32_t* bm, int len, const int32_t* ids, int K, int lo, int threads) {
    for (int i = threadIdx.x; i < (len + 31) / 32; i += threads) bm[i] = 0u;
    __syncthreads();
    for (int k = threadIdx.x; k < K; k += threads) {
        const int d = ids[k] - lo;
        if (ids[k] >= 0 && d >= 0 && d < len) atomicOr(&bm[d >> 5], 1u << (d & 31));
    }
    __syncthreads();
}

// Sets the elements of vector vi whose bit is set to -inf.
template <typename T>
__device__ __forceinline__ void ds_drop(const uint32_t* bm, int vi, uint32_t (&w)[4]) {
    constexpr int VEC = Elem<T>::kVec;
    const uint32_t b = (bm[(vi * VEC) >> 5] >> ((vi * VEC) & 31)) & ((1u << VEC) - 1u);
    if (b) {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if ((b >> j) & 1u) DsVec<T>::set_neg_inf(w, j);
    }
}

// A part's running sum: elements [0, len) of `row`, without those whose bit is set (BUCKET).  The next
// four vectors' loads are issued before these are used; the first before `ready` (the bitmap).
template <typename T, bool BUCKET, typename F>
__device__ __forceinline__ DsSum ds_stream(const T* row, int len, float c, const uint32_t* bm, F ready) {
    constexpr int VEC = Elem<T>::kVec, U = 4;
    const int nvec = len / VEC, tid = threadIdx.x;
    uint32_t next[U][4];
    auto fetch = [&](int b) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u) ds_load<T>(row, min(b + u * kDsThreads, nvec - 1), next[u]);
    };
    if (nvec > 0) fetch(tid);
    ready();
    DsSum t;
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
    if (i < len && !(BUCKET && ((bm[i >> 5] >> (i & 31)) & 1u))) ds_add1(t, Elem<T>::load1(row + i) * c);
    return t;
}

// Sums and maxima over the first four waves of a workgroup (the teacher's entries), returned to
// every thread.  `red`: 16 floats of LDS.  All threads call.
struct DsBlock {
    float* red;
    template <typename F>
    __device__ __forceinline__ float reduce(float v, float none, F op) {
        const int wave = threadIdx.x >> 6;
        __syncthreads();
        if (wave < 4 && (threadIdx.x & 63) == 0) red[wave] = v;
        __syncthreads();
        float t = none;
#pragma unroll
        for (int i = 0; i < 4; ++i) t = op(t, red[i]);
        return t;
    }
    __device__ __forceinline__ float max(float v) {
        return reduce(ds_wave_max(v), -kDsInf, [](float a, float b) { return __builtin_fmaxf(a, b); });
    }
    __device__ __forceinline__ float sum(float v) {
        return reduce(ds_wave_sum(v), 0.0f, [](float a, float b) { return a + b; });
    }
};

struct DsRow {
    float ref, coef, max, inv_total;  // DistillStat
    bool live;
    float x, p;                       // this thread's entry: its logit, its P (-1: none)
};

// A row's loss and statistics from the running sum of its rest (BUCKET) or of all of it.  Called by
// every thread of a workgroup of at least 256; thread k < K has entry k.
struct DsShared {
    float red[16];
    float lpr[kDsMaxK];
    int32_t lid[kDsMaxK];
    // the entries' ids, hashed: an id, its first entry, its entries
    int32_t hid[2 * kDsMaxK];
    uint32_t hfirst[2 * kDsMaxK], hcount[2 * kDsMaxK];
};

template <typename T, bool BUCKET>
__device__ __forceinline__ DsRow ds_finish(const DistillArgs& a, int r, const T* row, DsSum rest, float w, DsShared& sh) {
    const int k = threadIdx.x, K = a.K;
    DsBlock blk{sh.red};
    for (int i = k; i < 2 * kDsMaxK; i += blockDim.x) {
        sh.hid[i] = -1;
        sh.hfirst[i] = ~0u;
        sh.hcount[i] = 0u;
    }
    int id = -1;
    float l = -kDsInf, x = 0.0f;
    if (k < K) {
        id = a.ids[(size_t)r * a.ids_stride + k];
        if (id < 0 || id >= a.V) id = -1;
        if (id >= 0) {
            l = a.lp[(size_t)r * a.lp_stride + k];
            x = Elem<T>::load1(row + id);
        }
        sh.lid[k] = id;
    }
    const bool valid = id >= 0;
    // the teacher's probabilities (the reductions' barriers order the table's clearing before its use)
    float p, logp;
    bool live;
    if (BUCKET) {
        logp = l;
        p = valid ? expf(l) : 0.0f;
        live = blk.max(valid ? 1.0f : 0.0f) > 0.0f;
    } else {
        logp = valid ? l * a.inv_T : -kDsInf;
        const float top = blk.max(valid && logp != logp ? kDsInf : logp);  // (a NaN makes the row NaN)
        live = top > -kDsInf;
        const float e = valid && live ? expf(logp - top) : 0.0f;
        const float tot = blk.sum(e);
        p = e / tot;
        logp = logp - top - logf(tot);
    }
    // entries that share an id: the first takes their probability together
    if (k < K) sh.lpr[k] = p;
    int slot = 0;
    if (valid) {  // (at most 256 of 512 places are taken)
        slot = (int)(((uint32_t)id * 2654435761u) >> 23);
        for (;;) {
            const int had = atomicCAS(&sh.hid[slot], -1, id);
            if (had == -1 || had == id) break;
            slot = (slot + 1) & (2 * kDsMaxK - 1);
        }
        atomicMin(&sh.hfirst[slot], (uint32_t)k);
        atomicAdd(&sh.hcount[slot], 1u);
    }
    __syncthreads();
    const bool first = valid && sh.hfirst[slot] == (uint32_t)k;
    float P = p;
    if (first && sh.hcount[slot] > 1u) {
        P = 0.0f;
        for (int j = 0; j < K; ++j)
            if (sh.lid[j] == id) P += sh.lpr[j];
    }
    // the student's total
    float M = rest.m, Z = rest.s;
    if (BUCKET) {
        M = __builtin_fmaxf(M, blk.max(first ? x * a.c : -kDsInf));
        const float mref = M == -kDsInf ? 0.0f : M;
        const float zk = blk.sum(first ? ds_exp2(__builtin_fmaf(x, a.c, -mref)) : 0.0f);
        Z = (rest.s != 0.0f ? rest.s * ds_exp2(rest.m - mref) : 0.0f) + zk;
    }
    const float mref = M == -kDsInf ? 0.0f : M;
    const float lz = log2f(Z);  // (-inf when no logit is finite: every log q is then -inf)
    const float logq = Z > 0.0f || Z != Z ? (__builtin_fmaf(x, a.c, -mref) - lz) * kLn2 : -kDsInf;
    float L = blk.sum(valid && !(p <= 0.0f) ? p * (logp - logq) : 0.0f);
    DsRow o;
    o.max = mref;
    o.inv_total = Z > 0.0f || Z != Z ? 1.0f / Z : 0.0f;
    o.ref = rest.m == -kDsInf ? 0.0f : rest.m;
    if (BUCKET) {
        const float sp = blk.sum(p);
        const float rr = 1.0f - sp;
        // a rest without a finite logit is no event
        const bool have = rest.s > 0.0f || rest.s != rest.s;
        const float rem = have && !(rr < 0.0f) ? rr : 0.0f;
        if (!(rem <= 0.0f)) L += rem * (logf(rem) - ((rest.m - mref) + log2f(rest.s) - lz) * kLn2);
        // the teacher's events add up to tot, 1 but where the rest is no event or sp exceeds 1:
        // an entry's gradient is tot q - p, the rest's tot q - rem q / s
        const float tot = sp + rem;
        o.coef = have ? (tot * (rest.s * ds_exp2(rest.m - mref) * o.inv_total) - rem) / rest.s : 0.0f;
        o.inv_total *= tot;
    } else {
        o.coef = o.inv_total;
    }
    o.live = live;
    o.x = x;
    o.p = first ? P : -1.0f;
    if (threadIdx.x == 0) a.loss[r] = live ? w * L : 0.0f;
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

template <typename T, bool BUCKET>
__global__ __launch_bounds__(kDsThreads) void distill_forward_kernel(DistillArgs a) {
    extern __shared__ uint32_t bm[];
    __shared__ DsShared sh;
    __shared__ float wm[kDsThreads / 64], ws[kDsThreads / 64];
    __shared__ uint32_t last;
    const int S = a.S, r = blockIdx.x / S, p = blockIdx.x - r * S, tid = threadIdx.x, wave = tid >> 6;
    const float w = a.weight ? a.weight[r] : 1.0f;
    if (w == 0.0f) {  // the row does not count: not read
        if (p == 0) {
            if (tid == 0) a.loss[r] = 0.0f;
            if (tid == 0) a.stats[(size_t)r * kDsRowStats + kDsLive] = 0.0f;
        }
        return;
    }
    const T* row = static_cast<const T*>(a.x) + (size_t)r * a.xstride;
    const int lo = p * a.part_len, len = min(a.V, lo + a.part_len) - lo;
    DsSum t = ds_stream<T, BUCKET>(row + lo, len, a.c, bm, [&] {
        if (BUCKET) ds_bitmap(bm, len, a.ids + (size_t)r * a.ids_stride, a.K, lo, kDsThreads);
    });
    t.wave_merge();
    if ((tid & 63) == 0) { wm[wave] = t.m; ws[wave] = t.s; }
    __syncthreads();
    t = DsSum();
#pragma unroll
    for (int i = 0; i < kDsThreads / 64; ++i) t.merge(wm[i], ws[i]);
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
        const int lane = tid & 63;
        t = DsSum();
        if (lane < S) {
            const uint64_t v = ag_load64(&a.rec[(size_t)r * S + lane]);
            t.m = u2f((uint32_t)(v >> 32));
            t.s = u2f((uint32_t)v);
        }
        t.wave_merge();
    }
    const DsRow o = ds_finish<T, BUCKET>(a, r, row, t, w, sh);
    ds_save(a, r, o);
}

// The gradient of part p of row r.  Rows from the last to the first: those that the forward read last
// are still in the last-level cache.
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
            const float q = ds_exp2(__builtin_fmaf(Elem<T>::load1(row + id), a.c, -st[kDsMax])) * st[kDsInvTotal];
            fix = gs * (q - P);
        }
    }
    __syncthreads();
    const float ref = st[kDsRef], coef = st[kDsCoef] * gs;
    for (int b = tid; b < nvec; b += U * kDsThreads) {
        uint32_t w[U][4];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int vi = b + u * kDsThreads;
            ds_load<T>(row + lo, vi < nvec ? vi : b, w[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int vi = b + u * kDsThreads;
            float v[VEC];
            Elem<T>::from_words(w[u][0], w[u][1], w[u][2], w[u][3], v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = ds_exp2(__builtin_fmaf(v[j], a.c, -ref)) * coef;
            DsVec<T>::pack(v, w[u]);
            if (vi < nvec) ds_store<T>(out + lo, vi, w[u]);
        }
    }
    if (tail < len) out[lo + tail] = DsVec<T>::narrow(ds_exp2(__builtin_fmaf(Elem<T>::load1(row + lo + tail), a.c, -ref)) * coef);
    // the teacher's entries over what the stream wrote there, once that has arrived
    stores_complete();
    __syncthreads();
    if (at >= 0) out[at] = DsVec<T>::narrow(fix);
}

// Loss and gradient of rows that one workgroup holds in its registers (NV vectors a thread): every
// logit is read once and its gradient written once.  One workgroup for each compute unit, a row at a
// time; as a row's gradients are written, the next row's logits are loaded into the registers they
// leave.
template <typename T, bool BUCKET, int NV>
__global__ __launch_bounds__(kDsStepThreads) void distill_step_kernel(DistillArgs a) {
    constexpr int VEC = Elem<T>::kVec, U = 2, W = kDsStepThreads / 64;
    extern __shared__ uint32_t bm[];
    __shared__ DsShared sh;
    __shared__ float wm[W], ws[W];
    const int tid = threadIdx.x, wave = tid >> 6, V = a.V, nvec = V / VEC, edge = nvec * VEC + tid;
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
        ds_load<T>(row, min(fresh(tid) + q * kDsStepThreads, end), w[q]);
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
#pragma unroll
    for (int q = 0; q < NV; ++q) fetch(x + (size_t)r * a.xstride, q, nvec - 1);
    if (edge < V) xe = Elem<T>::load1(x + (size_t)r * a.xstride + edge);
    for (;;) {
        const T* row = x + (size_t)r * a.xstride;
        T* out = grad + (size_t)r * a.gstride;
        const float wt = a.weight ? a.weight[r] : 1.0f;
        if (BUCKET) ds_bitmap(bm, V, a.ids + (size_t)r * a.ids_stride, a.K, 0, kDsStepThreads);
        DsSum t;
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
        const bool drop = BUCKET && edge < V && ((bm[edge >> 5] >> (edge & 31)) & 1u);
        if (edge < V && !drop) ds_add1(t, xe * a.c);
        t.wave_merge();
        if ((tid & 63) == 0) { wm[wave] = t.m; ws[wave] = t.s; }
        __syncthreads();
        t = DsSum();
#pragma unroll
        for (int i = 0; i < W; ++i) t.merge(wm[i], ws[i]);
        const DsRow o = ds_finish<T, BUCKET>(a, r, row, t, wt, sh);
        const float gs = wt * (a.gout ? a.gout[r] : 1.0f) * a.inv_T;
        const bool on = o.live && gs != 0.0f;
        const float ref = o.ref, coef = o.coef * gs;
        const int id = tid < a.K && !(o.p < 0.0f) ? sh.lid[tid] : -1;
        const float fix = gs * (ds_exp2(__builtin_fmaf(o.x, a.c, -o.max)) * o.inv_total - o.p);
        r += gridDim.x;
        skip();
        const bool more = r < a.N;
        const T* after = more ? x + (size_t)r * a.xstride : row;
        const int end = more ? nvec - 1 : 0;
#pragma unroll
        for (int q = 0; q < NV; ++q) {
            const int vi = fresh(tid) + q * kDsStepThreads;
            float v[VEC];
#pragma unroll
            for (int k = 0; k < 4; ++k) asm volatile("" : "+v"(w[q][k]));
            Elem<T>::from_words(w[q][0], w[q][1], w[q][2], w[q][3], v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = on ? ds_exp2(__builtin_fmaf(v[j], a.c, -ref)) * coef : 0.0f;
            uint32_t g[4];
            DsVec<T>::pack(v, g);
            if (vi < nvec) ds_store<T>(out + (size_t)q * kDsStepThreads * VEC, fresh(tid), g);
            fetch(after, q, end);
            fence();
        }
        if (edge < V) out[edge] = DsVec<T>::narrow(on ? ds_exp2(__builtin_fmaf(xe, a.c, -ref)) * coef : 0.0f);
        if (more && edge < V) xe = Elem<T>::load1(after + edge);
        // the teacher's entries over what was written there, once that has arrived
        stores_complete();
        __syncthreads();
        if (on && id >= 0) out[id] = DsVec<T>::narrow(fix);
        if (!more) return;
    }
}

#define VWS_DISTILL_STEP(T, NV)                                                      \
    template __global__ void distill_step_kernel<T, false, NV>(DistillArgs);         \
    template __global__ void distill_step_kernel<T, true, NV>(DistillArgs);
#define VWS_DISTILL_INST(T)                                                   \
    VWS_DISTILL_STEP(T, 16)                                                   \
    VWS_DISTILL_STEP(T, 32)                                                   \
    VWS_DISTILL_STEP(T, 40)                                                   \
    template __global__ void distill_forward_kernel<T, false>(DistillArgs);   \
    template __global__ void distill_forward_kernel<T, true>(DistillArgs);    \
    template __global__ void distill_backward_kernel<T>(DistillArgs);
VWS_DISTILL_INST(float)
VWS_DISTILL_INST(uint16_t)
VWS_DISTILL_INST(_Float16)
#undef VWS_DISTILL_INST

}  // namespace vws
