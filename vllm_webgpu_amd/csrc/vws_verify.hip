// vws_verify.hip -- verification of drafted tokens against the target's distribution.
//
// Request b has n drafts d_1 .. d_n and n + 1 rows of target logits.  Row i's distribution is the
// sampler's: y = x / T, m = max y, e = exp_det(y - m) over the set K_i that min-p, top-k and top-p
// keep (the sampler's rules and integer masses), p_i = e / S_i.  Draft i is accepted iff
// q_i(d_i) > 0 and u_i q_i(d_i) < p_i(d_i), q_i the distribution it was drawn from (1 at d_i without
// one); after the first refusal, at row a, a token is drawn from max(p_a - q_a, 0), after the last
// accepted draft from p_n, both by the sampler's exponential race.  The emitted tokens are then
// distributed as if the target had sampled them one by one.
//
// verify_rows_kernel reads every row once, split over workgroups, for its maximum and sum;
// verify_cut_kernel finds the kept set of the rows that their request cuts, of most from a short list;
// verify_mass_kernel (launches with a top-p) adds up the masses of the others, each split over
// workgroups; verify_token_kernel decides each request and races one of its rows.
#include "vws_device.h"
#include "vws_expsum.h"
#include "vws_sampler.h"
#include "vws_verify.h"

namespace vws {

template <typename T>
__device__ __forceinline__ void vf_load(const T* row, int vi, float (&v)[Elem<T>::kVec]) {
    uint32_t w[4];
    row_load<T>(row, vi, w);
    Elem<T>::from_words(w[0], w[1], w[2], w[3], v);
}

// N floats from element i of a row of any supported type.
template <int N>
__device__ __forceinline__ void vf_load_any(const void* row, int dtype, int i, float (&v)[N]) {
    if (dtype == VWS_DTYPE_F32) {
        const float* p = static_cast<const float*>(row) + i;
#pragma unroll
        for (int g = 0; g < N / 4; ++g) {
            const auto u = *reinterpret_cast<const RowVec<float>::U4*>(p + 4 * g);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[4 * g + j] = u2f(u[j]);
        }
    } else {
        typedef uint32_t U2 __attribute__((ext_vector_type(2), aligned(2)));
        const uint16_t* p = static_cast<const uint16_t*>(row) + i;
#pragma unroll
        for (int g = 0; g < N / 4; ++g) {
            const auto u = *reinterpret_cast<const U2*>(p + 4 * g);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint16_t h = (uint16_t)(u[j >> 1] >> (16 * (j & 1)));
                v[4 * g + j] = dtype == VWS_DTYPE_BF16 ? u2f((uint32_t)h << 16) : (float)__builtin_bit_cast(_Float16, h);
            }
        }
    }
}
__device__ __forceinline__ float vf_load_any1(const void* row, int dtype, int i) {
    if (dtype == VWS_DTYPE_F32) return static_cast<const float*>(row)[i];
    const uint16_t h = static_cast<const uint16_t*>(row)[i];
    return dtype == VWS_DTYPE_BF16 ? u2f((uint32_t)h << 16) : (float)__builtin_bit_cast(_Float16, h);
}
__device__ __forceinline__ size_t vf_esize(int dtype) { return dtype == VWS_DTYPE_F32 ? 4 : 2; }

// The request of row r: the last whose first row (cu[b] + b) lies at or before it.  64 bounds at a
// time, so two loads for up to 4096 requests; every lane of the calling wave returns it.  Bounds that
// decrease can name a row twice: this is the one request that it is taken for, VfRec::owner.
__device__ __forceinline__ int vf_request(const VerifyArgs& a, int r) {
    int lo = 0, n = a.B;
    while (n > 1) {
        const int step = (n + kWave - 1) / kWave, at = lane_id() * step;
        const int b = lo + min(at, n - 1);
        const uint64_t before = wave_ballot(at < n && a.cu[b] <= r - b);  // (r - b: any bound goes)
        const int skip = before ? (kWave - 1 - (int)__builtin_clzll(before)) * step : 0;
        lo += skip;
        n = min(step, n - skip);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

struct VfParams {
    float T, top_p, min_p;
    int k;
    bool greedy, cuts;
    bool sums;  // the row's sum of exponentials over all its tokens is used
};
__device__ __forceinline__ VfParams vf_params(const VerifyArgs& a, int b) {
    VfParams p;
    p.T = a.temperature ? a.temperature[b] : 0.0f;
    p.greedy = is_greedy(p.T);
    p.k = a.top_k ? a.top_k[b] : 0;
    if (p.k < 0 || p.k >= a.V) p.k = 0;
    p.top_p = a.top_p ? a.top_p[b] : 1.0f;
    p.min_p = a.min_p ? a.min_p[b] : 0.0f;
    p.cuts = !p.greedy && (p.k > 0 || 1.0f - p.top_p > 0.0f || p.min_p > 0.0f);
    p.sums = !p.greedy && p.k == 0 && !(p.min_p > 0.0f);
    return p;
}

// log2(e) / T of a row that is not greedy (T may be infinite: the least number above 0, by which -inf
// stays what it is).
__device__ __forceinline__ float vf_c(const VfParams& p) {
    return p.greedy ? 0.0f : __builtin_fmaxf(kExpLog2e / p.T, 0x1p-149f);
}

__device__ __forceinline__ uint64_t vf_pack(uint32_t key, int i) {
    return key ? ((uint64_t)key << 32) | (uint32_t)(0x7FFFFFFF - i) : 0ull;
}
__device__ __forceinline__ int vf_index(uint64_t top) { return top ? (int)(0x7FFFFFFFu - (uint32_t)top) : 0; }
__device__ __forceinline__ float vf_value(uint64_t top) {
    return top ? val_of((uint32_t)(top >> 32)) : __builtin_nanf("");
}

// Part p of row r: its largest logit, the lowest index that has it, and the sum of exponentials.
// NaN logits are never the largest and add nothing.  Of rows that are cut it leaves the maximum of
// every group (the kVfGroup vectors of a thread's iteration), with which verify_cut_kernel finds the
// few logits that matter without a second read of the row.
//
// Bound: HBM.  The next iteration's loads are issued before this one's are used, and the first
// before the request's parameters are known.  274 rows x 128256 fp32 (141 MB): 31.2 us, 4.5 TB/s of a copy's
// 5.07; 745 x 262144 bf16 (391 MB), most of them cut: 87 us, 4.5 TB/s, and 19 MB of groups' maxima written;
// small batches are one latency chain (6 x 128256 bf16 5.8 us, 4 x 32000 fp32 4.8).
template <typename T>
__global__ __launch_bounds__(kVfThreads) void verify_rows_kernel(VerifyArgs a) {
    constexpr int VEC = Elem<T>::kVec, U = kVfGroup;
    __shared__ uint64_t red_top[kVfThreads / 64];
    __shared__ float red_m[kVfThreads / 64], red_s[kVfThreads / 64];
    const int S = a.S, at = blockIdx.x / S, r = a.r0 + at, p = blockIdx.x - at * S, tid = threadIdx.x, wave = tid >> 6;
    const T* row = static_cast<const T*>(a.x) + (size_t)r * a.xstride;
    const int lo = p * a.part_len, len = min(a.V, lo + a.part_len) - lo, nvec = len / VEC;
    row += lo;
    uint32_t next[U][4];
    auto fetch = [&](int b) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int vi = b + u * kVfThreads;
            if (nvec > 0) row_load<T>(row, vi < nvec ? vi : nvec - 1, next[u]);
        }
    };
    fetch(tid);
    if (p == 0 && tid == 0) {
        if (r < a.B) a.ctr[r] = 0u;  // (R >= B)
        if (r == 0) *a.flat_n = 0u;
    }
    const int owner = vf_request(a, r);
    const VfParams prm = vf_params(a, owner);
    const float c = vf_c(prm);
    float* gmax = a.gmax + (size_t)r * a.groups + (size_t)p * (a.groups / S);
    ExpRun run(c);
    float best = __builtin_nanf("");  // the largest logit so far, and the first group that holds it
    int group = tid;
    for (int b = tid; b < nvec; b += U * kVfThreads) {
        float v[U][VEC];
#pragma unroll
        for (int u = 0; u < U; ++u) Elem<T>::from_words(next[u][0], next[u][1], next[u][2], next[u][3], v[u]);
        if (b + U * kVfThreads < nvec) fetch(b + U * kVfThreads);
        float g = v[0][0];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < VEC; ++j) g = b + u * kVfThreads < nvec ? __builtin_fmaxf(g, v[u][j]) : g;
        if (g == g && !(g <= best)) { best = g; group = b; }
        if (prm.cuts) gmax[(b / (U * kVfThreads)) * kVfThreads + tid] = g;
        if (prm.sums) {
            float acc[4] = {run.raise(g, c), 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool in = b + u * kVfThreads < nvec;
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float e = es_exp2(__builtin_fmaf(v[u][j], c, -run.ref));
                    acc[j & 3] += in && e == e ? e : 0.0f;
                }
            }
            run.s = (acc[0] + acc[1]) + (acc[2] + acc[3]);
        }
    }
    // the largest logit's first place in its group, where it is the wave's (every lane's group read
    // again was a third of the part)
    float most = best;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) most = __builtin_fmaxf(most, es_lane_xor(most, o));
    uint64_t top = 0ull;
    if (best == most) {  // (not of a thread without vectors: NaN)
        for (int u = U - 1; u >= 0; --u) {
            const int vi = group + u * kVfThreads;
            if (vi >= nvec) continue;
            float v[VEC];
            vf_load<T>(row, vi, v);
#pragma unroll
            for (int j = VEC - 1; j >= 0; --j)
                if (v[j] == best) top = vf_pack(key_of(v[j]), lo + vi * VEC + j);
        }
    }
    ExpSum t = run.close(c);
    const int i = nvec * VEC + tid;
    if (i < len) {
        const float x = Elem<T>::load1(row + i);
        top = vws_max64(top, vf_pack(key_of(x), lo + i));
        if (prm.sums && x == x) t.merge(x, x > -kExpInf ? 1.0f : 0.0f, c);
    }
    top = wave_max_u64(top);
    t.wave_merge(c);
    if ((tid & 63) == 0) { red_top[wave] = top; red_m[wave] = t.m; red_s[wave] = t.s; }
    __syncthreads();
    VfRec o{0ull, 0.0f, owner};
#pragma unroll
    for (int w = 0; w < kVfThreads / 64; ++w) o.top = vws_max64(o.top, red_top[w]);
    const float x_top = vf_value(o.top);
    if (prm.sums && exp_far(x_top, c)) {
        // far from zero: over y = fl(x / T), which the race and the masses take there (y spreads by its
        // rounding); a second read of the part, from the caches
        const float m = x_top / prm.T;
        float s = 0.0f;
        auto add = [&](float x) __attribute__((always_inline)) {
            const float e = es_exp2((x / prm.T - m) * kExpLog2e);
            s += e == e ? e : 0.0f;  // (NaN: x is, or x / T has no finite value)
        };
        for (int vi = tid; vi < nvec; vi += kVfThreads) {
            float v[VEC];
            vf_load<T>(row, vi, v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) add(v[j]);
        }
        if (i < len) add(Elem<T>::load1(row + i));
        s = es_wave_sum(s);
        if ((tid & 63) == 0) red_s[wave] = s;
        __syncthreads();
        if (tid == 0) {
#pragma unroll
            for (int w = 0; w < kVfThreads / 64; ++w) o.sum += red_s[w];
            a.rec[(size_t)r * S + p] = o;
        }
        return;
    }
    if (tid == 0) {
        ExpSum s;
#pragma unroll
        for (int w = 0; w < kVfThreads / 64; ++w) s.merge(red_m[w], red_s[w], c);
        o.sum = s.s;
        a.rec[(size_t)r * S + p] = o;
    }
}

// ---- rows that their request cuts ---------------------------------------------------------
//
// The kept set is that of vws_sample, decided on the integer masses w = floor(exp_det(y - m) 2^44):
// their sums do not depend on the order, so the set does not depend on how it is found.  Three ways,
// by what bounds the row's survivors:
//   * top-k or min-p: a bound on the logit below which nothing survives (the k-th largest of 256
//     maxima, joined from the groups' that the first pass left, or m + log(min_p)); the few logits
//     above it, read where a group's maximum reaches it, go into a list, which decides everything;
//   * top-p alone: the list of the logits above such a bound, if it holds the cut for any total
//     within the error of the first pass's sum (a peaked row);
//   * else the masses of all logits, summed in bins by the distance from the maximum;
//     the bin that holds the cut goes into a list (two reads of the row, one exp_det per logit).  16-bit
//     logits whose spacing is wider than a bin can overfill it with one value: 32 rows of 262144 bf16 with
//     mean 0 or 10, T 1.3, top-p 0.5, 116 us, with mean 20 (1/8 apart) 589.
//     verify_mass_kernel does that for the first kVfFlat such rows, all compute units at it
//     however few the rows, and verify_cut_kernel itself for further ones (rows of 128256 bf16 in
//     whole calls, with 64, 128, 256 rows taken: 80 such rows 128, 87, 87 us, 200 147, 154, 118, 320 217,
//     222, 190).
// A list that overflows (many equal logits) leaves the row to passes over its keys' bits.

constexpr int kVfCutWaves = kVfCutThreads / 64;
constexpr int kVfList = 2048;     // list entries (a row's candidates)
constexpr int kVfSmall = 512;     // entries that are compared with each other, all pairs
constexpr int kVfPairs = 128;     // (of one bin: more of them are mostly equal)
constexpr int kVfGroups = 1024;   // groups that are read for the list
constexpr int kVfPeaks = 256;     // maxima that bound the list
constexpr int kVfPeakMost = 232;  // of them, the last whose rank is used (the next are few and far between)

struct VfCutShared {
    uint64_t hist[kVfBins];
    uint64_t list[kVfList];       // key(y) << 32 | index
    uint32_t above[kVfSmall];     // of each listed element: the elements with larger keys
    uint32_t groups[kVfGroups];
    uint64_t red[kVfCutWaves];
    uint64_t out[4];
    float peaks[kVfPeaks];        // maxima, each of the groups of four threads
    uint32_t count, ngroups;
    uint32_t slot;                // the row's place in VerifyArgs::flat
    float bound;
};

__device__ __forceinline__ float vf_scaled(float x, float Tt) { return Tt == 1.0f ? x : x / Tt; }

// Calls fv(first index, logits) for every vector of a row and f(index, x) for the logits past them (each thread its
// vectors, then one element), or for its vectors [v0, v1) and, with `tail`, that element; the next four
// vectors are on their way while these are used.
template <typename T, typename FV, typename F>
__device__ __forceinline__ void vf_vectors(const T* row, int V, FV fv, F f, int v0 = 0, int v1 = 1 << 30, bool tail = true) {
    constexpr int VEC = Elem<T>::kVec, U = 4;
    const int tid = threadIdx.x, last = V / VEC, nvec = min(v1, last);
    if (nvec > v0) {
        uint32_t next[U][4];
        auto fetch = [&](int b) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < U; ++u) row_load<T>(row, min(b + u * kVfCutThreads, nvec - 1), next[u]);
        };
        fetch(v0 + tid);
        for (int b = v0 + tid; b < nvec; b += U * kVfCutThreads) {
            uint32_t w[U][4];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int k = 0; k < 4; ++k) w[u][k] = next[u][k];
            fetch(b + U * kVfCutThreads);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int vi = b + u * kVfCutThreads;
                if (vi >= nvec) break;
                float v[VEC];
                Elem<T>::from_words(w[u][0], w[u][1], w[u][2], w[u][3], v);
                fv(vi * VEC, v);
            }
        }
    }
    const int i = last * VEC + tid;
    if (tail && i < V) f(i, Elem<T>::load1(row + i));
}

// The same with f(index, x) for every logit.
template <typename T, typename F>
__device__ __forceinline__ void vf_each(const T* row, int V, F f, int v0 = 0, int v1 = 1 << 30, bool tail = true) {
    constexpr int VEC = Elem<T>::kVec;
    vf_vectors<T>(row, V, [&](int i, const float (&v)[VEC]) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) f(i + j, v[j]);
    }, f, v0, v1, tail);
}

// What the selection below runs over: a row's elements, or the list's.  each(f): f(index, key, y).
template <typename T> struct VfRowIter {
    const T* row;
    int V;
    float Tt;
    template <typename F> __device__ __forceinline__ void each(F f) const {
        const float t = Tt;
        vf_each<T>(row, V, [&](int i, float x) {
            const float y = vf_scaled(x, t);
            f(i, key_of(y), y);
        });
    }
};
struct VfListIter {
    const uint64_t* list;
    int n;
    template <typename F> __device__ __forceinline__ void each(F f) const {
        for (int j = threadIdx.x; j < n; j += kVfCutThreads) {
            const uint64_t v = list[j];
            f((int)(uint32_t)v, (uint32_t)(v >> 32), val_of((uint32_t)(v >> 32)));
        }
    }
};

__device__ __forceinline__ uint64_t vf_block_max(uint64_t v, VfCutShared& sh) {
    v = wave_max_u64(v);
    __syncthreads();
    if (lane_id() == 0) sh.red[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t t = 0;
#pragma unroll
    for (int i = 0; i < kVfCutWaves; ++i) t = vws_max64(t, sh.red[i]);
    return t;
}
__device__ __forceinline__ uint64_t vf_block_sum(uint64_t v, VfCutShared& sh) {
    v = wave_sum_u64(v);
    __syncthreads();
    if (lane_id() == 0) sh.red[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t t = 0;
#pragma unroll
    for (int i = 0; i < kVfCutWaves; ++i) t += sh.red[i];
    return t;
}

__device__ __forceinline__ void vf_clear(VfCutShared& sh) {
    __syncthreads();
    for (int i = threadIdx.x; i < kVfBins; i += kVfCutThreads) sh.hist[i] = 0ull;
    __syncthreads();
}
__device__ __forceinline__ void vf_count(VfCutShared& sh, int bin, uint64_t w) {
    atomicAdd(reinterpret_cast<unsigned long long*>(&sh.hist[bin]), (unsigned long long)w);
}

// Vectors of part p of a row.
template <typename T>
__device__ __forceinline__ int vf_part_vecs(const VerifyArgs& a, int p) {
    return (min(a.V, (p + 1) * a.part_len) - p * a.part_len) / Elem<T>::kVec;
}

// The bin of sh.hist (bins [0, n), n <= kVfBins, even) where the running sum from bin 0 up first
// exceeds `thr`, and the sum below it.  All threads call, two bins each; the total exceeds thr.
__device__ __forceinline__ void vf_find(VfCutShared& sh, int n, uint64_t thr, int* bin, uint64_t* below) {
    __syncthreads();
    const int lane = lane_id(), wave = threadIdx.x >> 6, at = 2 * (int)threadIdx.x;
    const uint64_t h0 = at < n ? sh.hist[at] : 0ull, h1 = at < n ? sh.hist[at + 1] : 0ull;
    uint64_t incl = h0 + h1;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const uint64_t t = __shfl_up(incl, o, kWave);
        if (lane >= o) incl += t;
    }
    if (lane == kWave - 1) sh.red[wave] = incl;
    __syncthreads();
    uint64_t c = incl - h0 - h1;
    for (int w = 0; w < wave; ++w) c += sh.red[w];
    if (c <= thr && thr < c + h0 + h1) {
        const bool second = c + h0 <= thr;
        sh.out[0] = (uint64_t)(at + (second ? 1 : 0));
        sh.out[1] = second ? c + h0 : c;
    }
    __syncthreads();
    *bin = (int)sh.out[0];
    *below = sh.out[1];
    __syncthreads();
}

// The key at which the running sum of weight(key, y) over ascending keys first exceeds thr, with the
// sum of all smaller keys: three passes, 11, 11 and 10 bits of the key.
template <typename I, typename W>
__device__ __forceinline__ uint32_t vf_select(const I& it, VfCutShared& sh, uint64_t thr, uint64_t* below, W weight) {
    uint32_t prefix = 0u;
    uint64_t under = 0ull;
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = pass == 2 ? 10 : 11;
        vf_clear(sh);
        it.each([&](int, uint32_t k, float y) {
            if (pass > 0 && (k >> (shift + bits)) != prefix) return;
            const uint64_t w = weight(k, y);
            if (w) vf_count(sh, (int)((k >> shift) & ((1u << bits) - 1u)), w);
        });
        int bin;
        uint64_t c;
        vf_find(sh, 1 << bits, thr - under, &bin, &c);
        under += c;
        prefix = (prefix << bits) | (uint32_t)bin;
    }
    *below = under;
    return prefix;
}

// The n-th (from 0) lowest index among the elements whose key is `key`: two passes.
template <typename I>
__device__ __forceinline__ int vf_nth_index(const I& it, VfCutShared& sh, uint32_t key, uint64_t n) {
    int hi = 0, lo = 0;
    uint64_t under;
    for (int pass = 0; pass < 2; ++pass) {
        vf_clear(sh);
        it.each([&](int i, uint32_t k, float) {
            if (k != key || (pass && (i >> 8) != hi)) return;
            vf_count(sh, pass ? (i & 255) : (i >> 8), 1ull);
        });
        vf_find(sh, pass ? 256 : kVfBins, n, pass ? &lo : &hi, &under);
        n -= under;
    }
    return hi * 256 + lo;
}

struct VfCut {
    uint64_t cut, kept;  // the smallest (key << 32 | index) kept, the kept masses' sum
};

// What a row keeps, and the rest of what the selection needs to know.
struct VfRule {
    float m, lp_min, q32;
    int k;
    __device__ __forceinline__ bool above(float y) const { return y - m >= lp_min; }
    __device__ __forceinline__ uint64_t mass(float y) const { return mass_of(exp_det(y - m)); }
};

// The kept set by passes over the elements, which hold everything that may survive (`n`: those that
// are not NaN).
template <typename I>
__device__ __forceinline__ VfCut vf_solve(const I& it, VfCutShared& sh, const VfRule& u, uint64_t n) {
    uint32_t kth = 1u;  // every key but a NaN's
    if (u.k > 0 && (uint64_t)u.k <= n) {
        uint64_t under;
        kth = vf_select(it, sh, n - (uint64_t)u.k, &under, [](uint32_t k, float) { return (uint64_t)(k ? 1u : 0u); });
    }
    uint64_t W = 0ull, kmin = ~0ull;
    it.each([&](int, uint32_t k, float y) {
        if (k >= kth && u.above(y)) {
            W += u.mass(y);
            kmin = vws_min64(kmin, k);
        }
    });
    VfCut o;
    W = vf_block_sum(W, sh);
    kmin = ~vf_block_max(~kmin, sh);
    o.cut = kmin << 32;
    o.kept = W;
    if (u.q32 > 0.0f && u.q32 < 1.0f) {
        const uint64_t thr = scale_floor(u.q32, W);
        uint64_t under;
        const uint32_t key = vf_select(it, sh, thr, &under, [&](uint32_t k, float y) -> uint64_t {
            return k >= kth && u.above(y) ? u.mass(y) : 0ull;
        });
        const uint64_t w = u.mass(val_of(key));
        const uint64_t gone = (thr - under) / w;  // of the elements with that key, the lowest indices
        o.cut = (uint64_t)key << 32;
        if (gone) o.cut |= (uint32_t)vf_nth_index(it, sh, key, gone);
        o.kept = W - under - gone * w;
    }
    return o;
}

// At most kVfSmall listed elements, thread j < n the j-th: its mass w, how many have a larger key, and
// the sum A of the masses above it in (key, index).  All pairs, spread over the workgroup.
struct VfRank {
    uint64_t mine, w, A;
    float y;
    int more;
};
__device__ __forceinline__ VfRank vf_rank(VfCutShared& sh, const VfRule& u, int n) {
    const int tid = threadIdx.x;
    VfRank o{0ull, 0ull, 0ull, 0.0f, 0};
    uint64_t* mass = sh.hist;
    uint64_t* A = sh.hist + kVfSmall;
    if (tid < n) {
        o.mine = sh.list[tid];
        o.y = val_of((uint32_t)(o.mine >> 32));
        o.w = u.mass(o.y);
        mass[tid] = o.w;
        A[tid] = 0ull;
        sh.above[tid] = 0u;
    }
    __syncthreads();
    int width = kWave;
    while (width < n) width *= 2;
    const int j = tid & (width - 1), parts = kVfCutThreads / width, len = (n + parts - 1) / parts;
    const int i0 = (tid / width) * len, i1 = min(n, i0 + len);
    if (j < n) {
        const uint64_t mine = sh.list[j];
        uint64_t sum = 0ull;
        uint32_t more = 0u;
#pragma unroll 4
        for (int i = i0; i < i1; ++i) {
            const uint64_t v = sh.list[i];
            sum += v > mine ? mass[i] : 0ull;
            more += (uint32_t)(v >> 32) > (uint32_t)(mine >> 32) ? 1u : 0u;
        }
        if (more) atomicAdd(&sh.above[j], more);
        if (sum) atomicAdd(reinterpret_cast<unsigned long long*>(&A[j]), (unsigned long long)sum);
    }
    __syncthreads();
    if (tid < n) {
        o.A = A[tid];
        o.more = (int)sh.above[tid];
    }
    return o;
}

// Sum of v over threads 0 .. kVfSmall - 1 (those past it pass 0), in every thread.
__device__ __forceinline__ uint64_t vf_small_sum(uint64_t v, VfCutShared& sh) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();
    if (wave < kVfSmall / kWave) {
        v = wave_sum_u64(v);
        if (lane_id() == 0) sh.red[wave] = v;
    }
    __syncthreads();
    uint64_t t = 0ull;
#pragma unroll
    for (int i = 0; i < kVfSmall / kWave; ++i) t += sh.red[i];
    return t;
}
// The kept elements' smallest (key, index) and the sum of their masses.
__device__ __forceinline__ VfCut vf_small_cut(bool on, const VfRank& e, VfCutShared& sh) {
    constexpr int W = kVfSmall / kWave;
    static_assert(2 * W <= kVfCutWaves, "two words a wave");
    const int wave = threadIdx.x >> 6;
    __syncthreads();
    if (wave < W) {
        const uint64_t s = wave_sum_u64(on ? e.w : 0ull), v = wave_max_u64(on ? ~e.mine : 0ull);
        if (lane_id() == 0) { sh.red[wave] = s; sh.red[W + wave] = v; }
    }
    __syncthreads();
    VfCut o{0ull, 0ull};
#pragma unroll
    for (int i = 0; i < W; ++i) {
        o.kept += sh.red[i];
        o.cut = vws_max64(o.cut, sh.red[W + i]);
    }
    o.cut = ~o.cut;
    return o;
}

// vf_solve for at most kVfSmall listed elements.  Those above a survivor survive too, so its A is
// the sum of survivors above it, and it is kept iff what lies up to it, W - A, exceeds floor(q W).
__device__ __forceinline__ VfCut vf_solve_small(VfCutShared& sh, const VfRule& u, int n) {
    const VfRank e = vf_rank(sh, u, n);
    bool on = (int)threadIdx.x < n && u.above(e.y) && (u.k <= 0 || e.more < u.k);
    if (u.q32 > 0.0f && u.q32 < 1.0f) {
        const uint64_t W = vf_small_sum(on ? e.w : 0ull, sh);
        on = on && W - e.A > scale_floor(u.q32, W);
    }
    return vf_small_cut(on, e, sh);
}

// The elements listed are the row's largest.  Whether top-p's cut lies among them, and is the same, for
// every total W in [lo, hi]: kept iff A < f(W) = W - floor(q W), which never falls.
__device__ __forceinline__ bool vf_solve_top(VfCutShared& sh, const VfRule& u, int n, double lo, double hi, VfCut* o) {
    const VfRank e = vf_rank(sh, u, n);
    const bool in = (int)threadIdx.x < n;
    const uint64_t Wl = (uint64_t)lo, Wh = (uint64_t)hi + 1ull;
    const uint64_t fl = Wl - scale_floor(u.q32, Wl), fh = Wh - scale_floor(u.q32, Wh);
    const bool sure = in && e.A < fl, open = in && e.A < fh && !sure;
    // (the sum of all masses listed is below 2^53: the count of open ones goes on top)
    const uint64_t total = vf_small_sum((in ? e.w : 0ull) + (open ? 1ull << 54 : 0ull), sh);
    // elements past the list have A >= total: refused for every W if total >= f(hi)
    if (total >= 1ull << 54 || total < fh) return false;
    *o = vf_small_cut(sure, e, sh);
    return true;
}

// The listed elements are those of one bin, with `under` below them: kept iff under and what lies
// up to it in the bin exceed thr.  `total`: the sum of all masses.
__device__ __forceinline__ VfCut vf_solve_bin(VfCutShared& sh, const VfRule& u, int n, uint64_t total, uint64_t under,
                                              uint64_t thr) {
    VfCut o;
    if (n <= kVfPairs) {
        const VfRank e = vf_rank(sh, u, n);
        const uint64_t in = vf_small_sum((int)threadIdx.x < n ? e.w : 0ull, sh);
        o = vf_small_cut((int)threadIdx.x < n && under + (in - e.A) > thr, e, sh);
        o.kept += total - under - in;
        return o;
    }
    // (in 16-bit logits a bin is mostly one value)
    const VfListIter it{sh.list, n};
    uint64_t hi = 0ull, lo = 0ull;
    it.each([&](int, uint32_t k, float) {
        hi = vws_max64(hi, k);
        lo = vws_max64(lo, (uint32_t)~k);
    });
    hi = vf_block_max(hi, sh);
    lo = vf_block_max(lo, sh);
    uint64_t c = 0ull;
    uint32_t key = (uint32_t)hi;
    if (key != ~(uint32_t)lo) key = vf_select(it, sh, thr - under, &c, [&](uint32_t, float y) { return u.mass(y); });
    const uint64_t q = u.mass(val_of(key));
    const uint64_t gone = (thr - under - c) / q;
    o.cut = (uint64_t)key << 32;
    if (gone) o.cut |= (uint32_t)vf_nth_index(it, sh, key, gone);
    o.kept = total - under - c - gone * q;
    return o;
}

// Lists the row's elements with lo <= x <= hi whose y passes `in`; false when those with lo <= x <= hi are
// more than the list holds.  One compute unit goes over the whole row, so a vector takes two compares
// an element and a branch; places are listed first, values looked up from there.
template <typename T, typename F>
__device__ __forceinline__ bool vf_collect(const T* row, int V, float Tt, VfCutShared& sh, float lo, float hi, F in) {
    constexpr int VEC = Elem<T>::kVec, kMine = kVfList / kVfCutThreads;
    __syncthreads();
    if (threadIdx.x == 0) sh.count = sh.ngroups = 0u;
    __syncthreads();
    auto add = [&](int i) {
        const uint32_t at = agg_reserve(&sh.ngroups);
        if (at < (uint32_t)kVfList) sh.list[at] = (uint32_t)i;
    };
    vf_vectors<T>(row, V, [&](int i, const float (&v)[VEC]) __attribute__((always_inline)) {
        uint32_t m = 0u;
#pragma unroll
        for (int j = 0; j < VEC; ++j) m |= v[j] >= lo && v[j] <= hi ? 1u << j : 0u;
        while (m) {
            add(i + (int)__builtin_ctz(m));
            m &= m - 1u;
        }
    }, [&](int i, float x) { if (x >= lo && x <= hi) add(i); });
    __syncthreads();
    const int n = (int)sh.ngroups;
    if (n > kVfList) return false;
    int at[kMine];
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
        const int e = (int)threadIdx.x + k * kVfCutThreads;
        at[k] = e < n ? (int)sh.list[e] : -1;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
        if (at[k] < 0) continue;
        const float y = vf_scaled(Elem<T>::load1(row + at[k]), Tt);
        if (in(y)) sh.list[agg_reserve(&sh.count)] = ((uint64_t)key_of(y) << 32) | (uint32_t)at[k];
    }
    __syncthreads();
    return true;
}

// Calls f(maximum, part, first vector) for the groups of a row that exist: kVfThreads of them to a
// quarter of the workgroup at a time, four loads in flight.
template <typename T, typename F>
__device__ __forceinline__ void vf_each_group(const VerifyArgs& a, const float* gmax, F f) {
    constexpr int U = 4, kStep = kVfCutThreads / kVfThreads;
    const int its = a.groups / a.S / kVfThreads, t = threadIdx.x & (kVfThreads - 1);
    int p = 0, it = __builtin_amdgcn_readfirstlane(threadIdx.x / kVfThreads);
    for (int g = threadIdx.x; g < a.groups; g += U * kVfCutThreads) {
        float m[U];
#pragma unroll
        for (int u = 0; u < U; ++u) m[u] = gmax[min(g + u * kVfCutThreads, a.groups - 1)];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            while (it >= its) { it -= its; ++p; }
            const int b = it * kVfGroup * kVfThreads + t;
            if (p < a.S && b < vf_part_vecs<T>(a, p)) f(m[u], p, b);
            it += kStep;
        }
    }
}

// Lists the row's elements with x >= t by the groups' maxima (and the few elements past the parts'
// last vectors); false when groups or elements are too many.
template <typename T>
__device__ __forceinline__ bool vf_gather(const VerifyArgs& a, const float* gmax, const T* row, float Tt, VfCutShared& sh,
                                          float t) {
    constexpr int VEC = Elem<T>::kVec, U = kVfGroup;
    const int tid = threadIdx.x;
    __syncthreads();
    if (tid == 0) sh.count = sh.ngroups = 0u;
    __syncthreads();
    vf_each_group<T>(a, gmax, [&](float m, int p, int b) {
        if (m >= t) {
            const uint32_t at = agg_reserve(&sh.ngroups);
            // (parts are whole vectors but for the last: a part's place in vectors of the row)
            if (at < (uint32_t)kVfGroups) sh.groups[at] = (uint32_t)(p * (a.part_len / VEC) + b);
        }
    });
    __syncthreads();
    const int n = (int)sh.ngroups;
    if (n > kVfGroups) return false;
    auto add = [&](float x, int i) {
        if (x >= t) {
            const uint32_t at = agg_reserve(&sh.count);
            if (at < (uint32_t)kVfList) sh.list[at] = ((uint64_t)key_of(vf_scaled(x, Tt)) << 32) | (uint32_t)i;
        }
    };
    for (int k = tid; k < n * U; k += kVfCutThreads) {
        const int b = (int)sh.groups[k / U], p = b / (a.part_len / VEC), vi = b + (k % U) * kVfThreads;
        if (vi >= p * (a.part_len / VEC) + vf_part_vecs<T>(a, p)) continue;
        float v[VEC];
        vf_load<T>(row, vi, v);
#pragma unroll
        for (int j = 0; j < VEC; ++j) add(v[j], vi * VEC + j);
    }
    const int i = a.V / VEC * VEC + tid;
    if (i < a.V) add(Elem<T>::load1(row + i), i);
    __syncthreads();
    return sh.count <= (uint32_t)kVfList;
}

// The maxima of a row's groups, joined into kVfPeaks.
template <typename T>
__device__ __forceinline__ void vf_join_peaks(const VerifyArgs& a, const float* gmax, VfCutShared& sh) {
    float m = -kExpInf;
    vf_each_group<T>(a, gmax, [&](float g, int, int) { m = __builtin_fmaxf(m, g); });
    m = __builtin_fmaxf(m, es_lane_xor(m, 1));
    m = __builtin_fmaxf(m, es_lane_xor(m, 2));
    static_assert(kVfCutThreads / kVfPeaks == 4, "a maximum for every four threads");
    if ((threadIdx.x & 3) == 0) sh.peaks[threadIdx.x / 4] = m;
    __syncthreads();
}

// The n-th largest (from 1) of the row's peaks, with its low 16 bits cleared (a bound below it): found
// bit by bit by one wave.  -inf when fewer are finite.
__device__ __forceinline__ float vf_peak(VfCutShared& sh, int n) {
    if (threadIdx.x < kWave) {
        uint32_t k[kVfPeaks / kWave];
#pragma unroll
        for (int i = 0; i < kVfPeaks / kWave; ++i) k[i] = key_of(sh.peaks[i * kWave + lane_id()]);
        uint32_t ans = 0u;
#pragma unroll
        for (int b = 31; b >= 16; --b) {
            const uint32_t cand = ans | (1u << b);
            int c = 0;
#pragma unroll
            for (int i = 0; i < kVfPeaks / kWave; ++i) c += __popcll(wave_ballot(k[i] >= cand));
            if (c >= n) ans = cand;
        }
        if (threadIdx.x == 0) sh.bound = ans >= 0x00800000u ? val_of(ans) : -kExpInf;  // (below: -inf or none)
    }
    __syncthreads();
    return sh.bound;
}

struct VfRow {
    uint64_t top, cut;
    float m, sum;
    int owner;  // VfRec::owner
    bool sure;  // greedy, or the maximum is not finite: the row's distribution is its argmax
    bool far;   // exp_far of the maximum
};

// Row r's statistics from its parts, in every lane of the calling wave.
__device__ __forceinline__ VfRow vf_join(const VerifyArgs& a, const VfParams& prm, int r) {
    VfRec v{0ull, 0.0f, 0};
    if (lane_id() < a.S) v = a.rec[(size_t)r * a.S + lane_id()];
    VfRow o;
    o.owner = (int)__builtin_amdgcn_readfirstlane((uint32_t)v.owner);
    o.top = wave_max_u64(v.top);
    o.cut = 0ull;
    const float x = vf_value(o.top), part = vf_value(v.top), c = vf_c(prm);
    o.m = prm.greedy ? x : x / prm.T;
    o.sure = prm.greedy || !(__builtin_fabsf(o.m) < kExpInf);
    o.far = exp_far(x, c);
    const float e = es_exp2(o.far ? (part / prm.T - o.m) * kExpLog2e : (part - x) * c);
    o.sum = es_wave_sum(v.sum > 0.0f ? v.sum * e : 0.0f);
    return o;
}

// Bins of a row's masses, by distance from the maximum: what lies further than `far` holds less than
// q W (W is at least the maximum's own mass), so the cut does not lie there.
struct VfFar {
    float far, scale;
    __device__ __forceinline__ VfFar(const VfRule& u, int V) {
        far = __builtin_fminf(logf((float)V / u.q32) + 0.01f, 31.0f);
        scale = (float)(kVfBins - 1) / far;
    }
    __device__ __forceinline__ int bin(float d) const { return (int)(d * scale); }
};

// Adds the masses of a row's vectors [v0, v1) to the bins; returns those further away (this thread's).
//
// Bound: VALU, so the arithmetic is cut to what a mass needs, to the same bits: y = fl(x / T) from the
// reciprocal by two exact remainders (correctly rounded: the first makes the quotient faithful;
// for temperatures whose reciprocal is far from subnormal), exp_det without the cases that
// d <= 0 excludes, its scaling and the mass's in one ldexp.
template <typename T>
__device__ __forceinline__ uint64_t vf_masses(const T* row, int V, float Tt, VfCutShared& sh, const VfRule& u, int v0, int v1,
                                              bool tail) {
    const VfFar fr(u, V);
    const float inv = 1.0f / Tt;
    const bool quick = Tt < 0x1p60f;
    uint64_t rest = 0ull;
    vf_each<T>(row, V, [&](int, float x) {
        float y;
        if (quick) {
            y = x * inv;
            y = __builtin_fmaf(__builtin_fmaf(-y, Tt, x), inv, y);
            y = __builtin_fmaf(__builtin_fmaf(-y, Tt, x), inv, y);
        } else {
            y = x / Tt;
        }
        const float d = y - u.m;  // (NaN where y overflows: no mass, as its exp_det is 0)
        float n;
        const float p = exp_mantissa(d, &n);
        // 2^44 exp(d), 0 from where a mass is 0 (d < -31: below 2^-44)
        const float f = d >= -31.0f ? __builtin_ldexpf(p, (int)n + 44) : 0.0f;
        const float hf = __builtin_truncf(f * 0x1p-32f);
        const uint64_t q = ((uint64_t)(uint32_t)hf << 32) | (uint32_t)__builtin_fmaf(-hf, 0x1p32f, f);
        if (-d < fr.far) vf_count(sh, fr.bin(-d), q);
        else rest += q;
    }, v0, v1, tail);
    return rest;
}

// The kept set of a row from its bins in sh.hist and the masses beyond; false when the cut's bin does
// not fit the list.
template <typename T>
__device__ __forceinline__ bool vf_flat(const T* row, int V, float Tt, VfCutShared& sh, const VfRule& u, uint64_t rest, VfCut* o) {
    const VfFar fr(u, V);
    uint64_t in = 0ull;
    __syncthreads();
    for (int i = threadIdx.x; i < kVfBins; i += kVfCutThreads) in += sh.hist[i];
    in = vf_block_sum(in, sh);
    const uint64_t total = in + rest, thr = scale_floor(u.q32, total);
    if (total - thr > in) return false;
    // from the maximum down: the cut lies where the running sum reaches total - thr
    int bin;
    uint64_t over;
    vf_find(sh, kVfBins, total - thr - 1ull, &bin, &over);
    const uint64_t under = total - over - sh.hist[bin];
    const float yhi = u.m - (float)bin / fr.scale, ylo = u.m - (float)(bin + 1) / fr.scale;
    const float slack = (__builtin_fabsf(u.m) + 32.0f) * 0x1p-20f;
    if (!vf_collect<T>(row, V, Tt, sh, Tt * (ylo - slack), Tt * (yhi + slack), [&](float y) {
            const float d = u.m - y;
            return d < fr.far && fr.bin(d) == bin;
        }))
        return false;
    *o = vf_solve_bin(sh, u, (int)sh.count, total, under, thr);
    return true;
}

__device__ __forceinline__ VfRule vf_rule(const VfParams& prm, const VfRow& w) {
    VfRule u;
    u.m = w.m;
    u.q32 = 1.0f - prm.top_p;
    u.k = prm.k;
    u.lp_min = prm.min_p > 0.0f ? log_det(prm.min_p < 1.0f ? prm.min_p : 1.0f) : -kExpInf;
    return u;
}

// The kept set by passes over the whole row.
template <typename T>
__device__ __forceinline__ VfCut vf_solve_row(const T* row, int V, float Tt, VfCutShared& sh, const VfRule& u) {
    uint64_t n = 0ull;
    vf_each<T>(row, V, [&](int, float x) {
        const float y = vf_scaled(x, Tt);  // (NaN at T = inf where x is not finite)
        n += y == y ? 1u : 0u;
    });
    n = vf_block_sum(n, sh);
    return vf_solve(VfRowIter<T>{row, V, Tt}, sh, u, n);
}

// Thread 0: row r's own statistics in place of its parts' (which every wave has read).
__device__ __forceinline__ void vf_write(const VerifyArgs& a, int r, const VfRow& w, const VfCut& o) {
    VfRec c;
    c.top = w.top;
    c.owner = w.owner;
    c.sum = (float)o.kept * 0x1p-44f;
    a.rec[(size_t)r * a.S] = c;
    a.cut[r] = o.cut;
}

// One workgroup per row: the kept set of a row that its request cuts, as the smallest
// (key(y) << 32 | index) kept, and the sum of its exponentials.  The n-th largest of 256 peaks (maxima
// of groups, each from its own logits) is a lower bound of the n-th largest logit, so the logits above it
// are a list of n or a few more, read by way of the groups' maxima alone (a number for 16 or 32 logits).
// Top-k is decided in the list if k <= kVfPeakMost; top-p if the list's masses reach p of the row's sum even at the
// edge of that sum's error.
//
// Bound: latency, a chain of about ten barriers for one row (6 rows x 128256 17 us, 150 x 151936
// with a top-k 13.5), then rows a compute unit: 745 x 262144 42 us, of which 31 MB fetched.  Reading
// the row again in its place took 120 us of one request's 155, and of the 745 rows 1.1 ms.
template <typename T>
__global__ __launch_bounds__(kVfCutThreads) void verify_cut_kernel(VerifyArgs a) {
    __shared__ VfCutShared sh;
    const int r = a.r0 + (int)blockIdx.x;
    const VfParams prm = vf_params(a, a.rec[(size_t)r * a.S].owner);
    if (!prm.cuts) return;
    const T* row = static_cast<const T*>(a.x) + (size_t)r * a.xstride;
    const float Tt = prm.T;
    const int V = a.V;
    const VfRow w = vf_join(a, prm, r);
    const VfRule u = vf_rule(prm, w);
    VfCut o{0ull, 0ull};
    if (!w.sure) {
        const float* gmax = a.gmax + (size_t)r * a.groups;
        vf_join_peaks<T>(a, gmax, sh);
        // y = fl(x / T) and y - m round, and a maximum's group may hold the k-th largest itself:
        // a margin of some ulps below the bound keeps every element that could survive
        // (T 2^-120: where y is subnormal)
        const float tiny = Tt * 0x1p-120f;
        auto below = [tiny](float x) { return x - __builtin_fabsf(x) * 0x1p-20f - tiny; };
        bool done = false;
        bool listed = false;  // the list holds everything kept
        if (u.q32 >= 1.0f) {
            // only the last of (key, index)
            const uint32_t mk = key_of(u.m);
            uint64_t last = 0ull;
            vf_each<T>(row, V, [&](int i, float x) {
                if (key_of(vf_scaled(x, Tt)) == mk) last = vws_max64(last, ((uint64_t)mk << 32) | (uint32_t)i);
            });
            o.cut = vf_block_max(last, sh);
            o.kept = 1ull << 44;
            done = true;
        } else if (u.k > 0 || u.lp_min > -kExpInf) {
            float t = -kExpInf;
            if (u.k > 0 && u.k <= kVfPeakMost) t = below(vf_peak(sh, u.k));
            if (u.lp_min > -kExpInf) {
                const float y = u.m + u.lp_min;
                t = __builtin_fmaxf(t, Tt * (y - (__builtin_fabsf(u.m) - u.lp_min) * 0x1p-20f) - tiny);
            }
            const bool k_listed = u.k == 0 || t > -kExpInf;
            if (k_listed && vf_gather<T>(a, gmax, row, Tt, sh, t)) {
                const int n = (int)sh.count;
                o = n <= kVfSmall ? vf_solve_small(sh, u, n) : vf_solve(VfListIter{sh.list, n}, sh, u, (uint64_t)n);
                done = listed = true;
            }
        } else {
            // top-p alone.  The first pass's sum is off by at most 2^-22 (2 |m| + 64) of itself: y and
            // y - m round to 2^-24 of |m| + 31 (beyond which a mass is 0), the exponent's fma and
            // its constant likewise, the exponential and the sums by a few 2^-24.  A far row's is
            // over the masses' own y.
            const double W = (double)w.sum * 0x1p44, am = w.far ? 0.0 : (double)__builtin_fabsf(u.m);
            const double eps = 0x1p-22 * (2.0 * am + 64.0);
            // the 100 or so logits above the 84th of 256 maxima
            const float t = below(vf_peak(sh, 84));
            if (t > -kExpInf && vf_gather<T>(a, gmax, row, Tt, sh, t) && sh.count <= (uint32_t)kVfSmall)
                done = listed = vf_solve_top(sh, u, (int)sh.count, W * (1.0 - eps), W * (1.0 + eps), &o);
            if (!done) {
                // for verify_mass_kernel, or (the launch has many such rows) here
                // (a word of its own: others may still be reading the count on which vf_gather gave up)
                if (threadIdx.x == 0) sh.slot = ag_add32(a.flat_n, 1u);
                __syncthreads();
                const uint32_t at = sh.slot;
                if (at < (uint32_t)min(a.R, kVfFlat)) {
                    VfFlat& f = a.flat[at];
                    for (int i = threadIdx.x; i < kVfBins; i += kVfCutThreads) f.hist[i] = 0ull;
                    if (threadIdx.x == 0) {
                        f.row = r;
                        f.ctr = 0u;
                        f.rest = 0ull;
                    }
                    return;
                }
                vf_clear(sh);
                const uint64_t rest = vf_block_sum(vf_masses<T>(row, V, Tt, sh, u, 0, V, true), sh);
                done = vf_flat<T>(row, V, Tt, sh, u, rest, &o);
            }
        }
        if (!done) o = vf_solve_row<T>(row, V, Tt, sh, u);
        // the kept tokens for the race, where the list holds them and they are few
        int32_t* kept = a.kept + (size_t)r * (1 + kVfKept);
        const int n = listed ? (int)sh.count : 0;
        __syncthreads();
        if (threadIdx.x == 0) sh.ngroups = 0u;
        __syncthreads();
        for (int j = threadIdx.x; j < n; j += kVfCutThreads)
            if (sh.list[j] >= o.cut) {
                const uint32_t at = agg_reserve(&sh.ngroups);
                if (at < (uint32_t)kVfKept) kept[1 + at] = (int32_t)(uint32_t)sh.list[j];
            }
        __syncthreads();
        if (threadIdx.x == 0) kept[0] = listed && sh.ngroups <= (uint32_t)kVfKept ? (int32_t)sh.ngroups : -1;
    }
    __syncthreads();  // every wave has read the row's parts
    if (threadIdx.x == 0) vf_write(a, r, w, o);
}

// The rows that verify_cut_kernel has left, each split over as many workgroups as there are for it; the
// part that arrives last finishes the row.  Exact masses fall into bins by distance from the maximum
// (integers: no order of the atomics changes them); the bin where the sum passes p is then read
// and decided.
//
// Bound: the last part's chain (for a row of 262144 about 18 us of masses and 5 of waiting in its own sum, 16
// of the deciding bin's read by one compute unit, 8 of its order; 27 in all for one row of 128256).  70 such
// rows of 745: 54 us, against 165 by verify_cut_kernel alone, where they held up the launch; with no such row 1
// to 4 us, the price of a launch with a top-p.
template <typename T>
__global__ __launch_bounds__(kVfCutThreads) void verify_mass_kernel(VerifyArgs a) {
    __shared__ VfCutShared sh;
    const int rows = min((int)min(*a.flat_n, (uint32_t)kVfFlat), a.R);
    if (rows == 0) return;
    const int parts = min((int)gridDim.x / rows, 64), at = blockIdx.x / parts, p = blockIdx.x - at * parts;
    if (at >= rows) return;
    VfFlat& f = a.flat[at];
    const int r = f.row;
    const VfParams prm = vf_params(a, a.rec[(size_t)r * a.S].owner);
    const T* row = static_cast<const T*>(a.x) + (size_t)r * a.xstride;
    const VfRow w = vf_join(a, prm, r);
    const VfRule u = vf_rule(prm, w);
    const int V = a.V, nvec = V / Elem<T>::kVec, len = (nvec + parts - 1) / parts;
    vf_clear(sh);
    // (a part past the row's end only arrives; the last takes the elements past the vectors)
    const uint64_t mine = vf_masses<T>(row, V, prm.T, sh, u, min(p * len, nvec), min((p + 1) * len, nvec), p == parts - 1);
    uint64_t rest = vf_block_sum(mine, sh);
    for (int i = threadIdx.x; i < kVfBins; i += kVfCutThreads)
        if (const uint64_t h = sh.hist[i]) ag_add64(&f.hist[i], h);
    if (threadIdx.x == 0 && rest) ag_add64(&f.rest, rest);
    stores_complete();
    __syncthreads();
    if (threadIdx.x == 0) sh.count = ag_add32(&f.ctr, 1u);
    __syncthreads();
    if (sh.count != (uint32_t)parts - 1u) return;
    for (int i = threadIdx.x; i < kVfBins; i += kVfCutThreads) sh.hist[i] = ag_load64(&f.hist[i]);
    rest = ag_load64(&f.rest);
    VfCut o;
    if (!vf_flat<T>(row, V, prm.T, sh, u, rest, &o)) o = vf_solve_row<T>(row, V, prm.T, sh, u);
    if (threadIdx.x == 0) {
        vf_write(a, r, w, o);
        a.kept[(size_t)r * (1 + kVfKept)] = -1;
    }
}

// ---- decision and race ----------------------------------------------------------------------

// Row r's statistics for the decision, in every lane of the calling wave.
__device__ __forceinline__ VfRow vf_row(const VerifyArgs& a, const VfParams& prm, int r) {
    if (!prm.cuts) return vf_join(a, prm, r);
    const VfRec v = a.rec[(size_t)r * a.S];
    VfRow o;
    o.top = v.top;
    o.cut = a.cut[r];
    o.m = vf_value(v.top) / prm.T;
    o.sum = v.sum;
    o.owner = v.owner;
    o.sure = !(__builtin_fabsf(o.m) < kExpInf);
    return o;
}

__device__ __forceinline__ bool vf_kept(const VfRow& w, float y, int i) {
    const uint32_t k = key_of(y);
    return k != 0u && (((uint64_t)k << 32) | (uint32_t)i) >= w.cut;
}

// Part p of request b's race; every part decides the request for itself.
//
// A draw is argmax w / E, E = -ln u; as E >= 1 - u, a token whose w / (1 - u) is below the best so far needs
// no logarithm.  Rows whose kept tokens are listed race those alone.
// Bound: for uncut rows the reads (64 x 128256 fp32 logits, draft's probabilities and uniforms, 82 MB fetched:
// 24 us, 4.1 TB/s of the 98 they hold); for listed ones the latency of decision and race (48 requests, top-k 50: 9 us, 22.6 reading
// the row; one request 5.8); 256 mixed requests of 262144 bf16 44 us, Philox for the tokens near the best.
template <typename T>
__global__ __launch_bounds__(kVfThreads) void verify_token_kernel(VerifyArgs a) {
    constexpr int VEC = Elem<T>::kVec;
    __shared__ VfRow rows[kVfMaxDrafts + 1];
    __shared__ uint64_t red[kVfThreads / 64];
    __shared__ uint32_t last, shared_bound;
    const int S2 = a.S2, at = blockIdx.x / S2, b = a.r0 + at, p = blockIdx.x - at * S2, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const VfParams prm = vf_params(a, b);
    const int first = a.cu[b], end = a.cu[b + 1], n = (int)((uint32_t)end - (uint32_t)first), K1 = a.K + 1;
    auto misfit = [&] {  // bounds that do not fit: no token
        if (p > 0) return;
        for (int i = tid; i < K1; i += kVfThreads) {
            a.tokens[(size_t)b * K1 + i] = -1;
            a.logprobs[(size_t)b * K1 + i] = 0.0f;
        }
        if (tid == 0) a.accepted[b] = -1;
    };
    if (first < 0 || end < first || n > a.K || end > a.D) return misfit();
    for (int i = wave; i <= n; i += kVfThreads / 64) {
        const VfRow w = vf_row(a, prm, first + b + i);
        if (lane == 0) rows[i] = w;
    }
    __syncthreads();
    const T* x0 = static_cast<const T*>(a.x) + (size_t)(first + b) * a.xstride;
    const char* q0 = static_cast<const char*>(a.q) + (a.q ? (size_t)first * a.qstride * vf_esize(a.qdtype) : 0);
    const size_t qbytes = (size_t)a.qstride * vf_esize(a.qdtype);
    const uint64_t seed = a.rng_seed ? a.rng_seed[b] : a.rng_key;
    const uint64_t offset = a.rng_seed ? (a.rng_offset ? a.rng_offset[b] : 0ull) : (uint64_t)(uint32_t)b;
    // lane i decides draft i (every wave the same)
    bool ok = false;
    int d = -1;
    float lp = 0.0f;
    if (lane < n) {
        d = a.drafts[first + lane];
        const VfRow w = rows[lane];
        if (d >= 0 && d < a.V) {
            if (w.sure) {
                ok = d == vf_index(w.top);
            } else {
                const float x = Elem<T>::load1(x0 + (size_t)lane * a.xstride + d), y = x / prm.T;
                const float e = vf_kept(w, y, d) ? exp_det(y - w.m) : 0.0f;
                const float qd = a.q ? vf_load_any1(q0 + (size_t)lane * qbytes, a.qdtype, d) : 1.0f;
                const float u = a.u ? a.au[first + lane] : philox_uniform(seed, offset, kVfAcceptBase + (uint32_t)lane);
                ok = qd > 0.0f && u * qd < e / w.sum;
                lp = (y - w.m) - logf(w.sum);
            }
        }
    }
    // Rows that decreasing bounds make another request's have its statistics, and its cut or none: what
    // this request would read of them from here on need not have been written.  (n <= 64; every wave alike)
    if (wave_ballot(rows[min(lane, n)].owner != b || rows[n].owner != b)) return misfit();
    const uint64_t refused = wave_ballot(!ok && lane < n);
    const int acc = refused ? (int)__builtin_ctzll(refused) : n;
    const VfRow w = rows[acc];
    const T* row = x0 + (size_t)acc * a.xstride;
    uint64_t best = 0ull;
    if (!w.sure) {
        const int drop = !a.q && acc < n ? a.drafts[first + acc] : -1;  // the residual without q: without the draft
        const char* q = a.q && acc < n ? q0 + (size_t)acc * qbytes : nullptr;
        const float inv = 1.0f / w.sum;
        const float* u = a.u ? a.u + (size_t)b * a.ustride : nullptr;
        // The largest key so far, of the workgroup, is a bound: a key is w / E with E = -ln u >= 1 - u
        // >= 2^-24, so an element whose w (from the hardware's exp2, with its error on top) stays
        // below bound (1 - u) cannot win, and a logit below tl cannot whatever its uniform.
        // (Far from zero fl(x_top c) says nothing of that: an infinite scale, nothing is left out.)
        const float c = vf_c(prm), x_top = vf_value(w.top), m2 = x_top * c;
        const float eps = 1.0f + 0x1p-22f * (2.0f * __builtin_fabsf(w.m) + 64.0f);
        const float scale = exp_far(x_top, c) ? kExpInf : (q ? inv : 1.0f) * eps;
        const float y_cut = w.cut ? val_of((uint32_t)(w.cut >> 32)) : -kExpInf;
        const float x_cut = w.cut ? prm.T * (y_cut - __builtin_fabsf(y_cut) * 0x1p-20f) - prm.T * 0x1p-120f : -kExpInf;
        float bound = 0.0f;
        auto add = [&](int i, float x, float qi, float ui) {
            const float y = x / prm.T;
            if (!vf_kept(w, y, i) || i == drop) return;
            const float e = exp_det(y - w.m);
            const float wt = q ? __builtin_fmaxf(e * inv - qi, 0.0f) : e;
            if (!(wt > 0.0f)) return;
            const float key = wt / (0.0f - log_det(ui));
            if (key >= 0.0f) {
                best = vws_max64(best, vf_pack(f2u(key) + 1u, i));
                if (key < kExpInf) bound = __builtin_fmaxf(bound, key * 0.9999f);
            }
        };
        auto can_win = [&](float x, float qi, float ui) {
            const float e = es_exp2(__builtin_fmaf(x, c, -m2)) * scale;
            return !((q ? e - qi : e) < bound * (1.0f - ui)) || !(ui < 1.0f);  // (true for NaN)
        };
        // a cut row whose kept tokens are listed: they alone, by the first part
        const int32_t* kept = a.kept + (size_t)(first + b + acc) * (1 + kVfKept);
        const int nkept = prm.cuts ? kept[0] : -1;
        if (nkept >= 0 && p > 0) return;
        for (int k = tid; k < nkept; k += kVfThreads) {
            const int i = kept[1 + k];
            add(i, Elem<T>::load1(row + i), q ? vf_load_any1(q, a.qdtype, i) : 0.0f,
                u ? u[i] : philox_uniform(seed, offset, (uint32_t)i));
        }
        const int lo = p * a.part2_len, len = nkept >= 0 ? 0 : min(a.V, lo + a.part2_len) - lo, nvec = len / VEC;
        // the most probable token's key first (each thread for itself): a good bound
        if (nkept < 0) {
            const int i = vf_index(w.top);
            add(i, x_top, q ? vf_load_any1(q, a.qdtype, i) : 0.0f, u ? u[i] : philox_uniform(seed, offset, (uint32_t)i));
        }
        if (tid == 0) shared_bound = f2u(bound);
        __syncthreads();
        const bool dense = w.cut == 0ull && (u || q);  // read q and u with the logits
        constexpr int U = 2;
        for (int b0 = tid; b0 < nvec; b0 += U * kVfThreads) {
            float v[U][VEC], qv[U][VEC], uv[U][VEC];
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const int vi = min(b0 + k * kVfThreads, nvec - 1), i0 = lo + vi * VEC;
                vf_load<T>(row + lo, vi, v[k]);
                if (dense && q) vf_load_any<VEC>(q, a.qdtype, i0, qv[k]);
                if (dense && u) vf_load_any<VEC>(u, VWS_DTYPE_F32, i0, uv[k]);
            }
            bound = __builtin_fmaxf(bound, u2f(__hip_atomic_load(&shared_bound, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP)));
            const float had = bound;
            // (1 / c = T ln 2; the slack covers the roundings)
            const float lg = m2 + __builtin_amdgcn_logf(bound / scale) - 24.01f;
            const float tl = __builtin_fmaxf(x_cut, (lg - __builtin_fabsf(lg) * 0x1p-20f - __builtin_fabsf(m2) * 0x1p-20f) * (prm.T * 0x1.62e43p-1f));
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const int vi = b0 + k * kVfThreads, i0 = lo + vi * VEC;
#pragma unroll
                for (int g = 0; g < VEC; g += 4) {
                    const float top4 = __builtin_fmaxf(__builtin_fmaxf(v[k][g], v[k][g + 1]), __builtin_fmaxf(v[k][g + 2], v[k][g + 3]));
                    if (!(vi < nvec && top4 >= tl)) continue;
                    float q4[4] = {}, u4[4];
                    if (dense && q) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) q4[j] = qv[k][g + j];
                    } else if (q) {
                        vf_load_any<4>(q, a.qdtype, i0 + g, q4);
                    }
                    if (dense && u) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) u4[j] = uv[k][g + j];
                    } else if (u) {
                        vf_load_any<4>(u, VWS_DTYPE_F32, i0 + g, u4);
                    } else {
                        philox_uniforms_aligned<4>(seed, offset, (uint32_t)(i0 + g), u4);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (can_win(v[k][g + j], q4[j], u4[j])) add(i0 + g + j, v[k][g + j], q4[j], u4[j]);
                }
            }
            if (bound > had) atomicMax(&shared_bound, f2u(bound));  // (positive floats order as their bits)
        }
        const int i = lo + nvec * VEC + tid;
        if (i < lo + len)
            add(i, Elem<T>::load1(row + i), q ? vf_load_any1(q, a.qdtype, i) : 0.0f,
                u ? u[i] : philox_uniform(seed, offset, (uint32_t)i));
        // the part that arrives last has the winner
        best = wave_max_u64(best);
        if (lane == 0) red[wave] = best;
        __syncthreads();
        best = 0ull;
#pragma unroll
        for (int k = 0; k < kVfThreads / 64; ++k) best = vws_max64(best, red[k]);
        if (S2 > 1 && nkept < 0) {
            if (tid == 0) {
                ag_store64(&a.best[(size_t)b * S2 + p], best);
                stores_complete();
                last = ag_add32(&a.ctr[b], 1u) == (uint32_t)S2 - 1u ? 1u : 0u;
            }
            __syncthreads();
            if (!last) return;
            best = wave_max_u64(lane < S2 ? ag_load64(&a.best[(size_t)b * S2 + lane]) : 0ull);
        }
    } else if (p > 0) {
        return;
    }
    if (wave != 0) return;
    // no valid key (an empty residual): the most probable token
    const int token = vf_index(w.sure || !best ? w.top : best);
    float tlp = 0.0f;
    if (!w.sure) {
        const float y = Elem<T>::load1(row + token) / prm.T;
        tlp = (y - w.m) - logf(w.sum);
    }
    for (int i = lane; i < K1; i += kWave) {
        a.tokens[(size_t)b * K1 + i] = i < acc ? d : (i == acc ? token : -1);
        a.logprobs[(size_t)b * K1 + i] = i < acc ? lp : (i == acc ? tlp : 0.0f);
    }
    if (lane == 0) a.accepted[b] = acc;
}

#define VWS_VERIFY_INST(T)                                       \
    template __global__ void verify_rows_kernel<T>(VerifyArgs);  \
    template __global__ void verify_cut_kernel<T>(VerifyArgs);   \
    template __global__ void verify_mass_kernel<T>(VerifyArgs);  \
    template __global__ void verify_token_kernel<T>(VerifyArgs);
VWS_VERIFY_INST(float)
VWS_VERIFY_INST(uint16_t)
VWS_VERIFY_INST(_Float16)
#undef VWS_VERIFY_INST

}  // namespace vws
