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
// Three kernels: verify_rows_kernel reads every row once, split over workgroups, for its maximum and
// sum; verify_cut_kernel finds the kept set of the rows that their request cuts; verify_token_kernel
// decides each request and races one of its rows, split over workgroups.
#include "vws_device.h"
#include "vws_sampler.h"
#include "vws_verify.h"

namespace vws {

constexpr float kVfInf = __builtin_inff();

__device__ __forceinline__ float vf_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// 16 bytes at any element's address: rows of an odd vocabulary start unaligned.
template <typename T> struct VfVec { typedef uint32_t U4 __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct VfVec<float> { typedef uint32_t U4 __attribute__((ext_vector_type(4), aligned(4))); };

template <typename T>
__device__ __forceinline__ void vf_load(const T* row, int vi, float (&v)[Elem<T>::kVec]) {
    const auto u = *reinterpret_cast<const typename VfVec<T>::U4*>(row + (size_t)vi * Elem<T>::kVec);
    Elem<T>::from_words(u[0], u[1], u[2], u[3], v);
}

// N floats from element i of a row of any supported type.
template <int N>
__device__ __forceinline__ void vf_load_any(const void* row, int dtype, int i, float (&v)[N]) {
    if (dtype == VWS_DTYPE_F32) {
        const float* p = static_cast<const float*>(row) + i;
#pragma unroll
        for (int g = 0; g < N / 4; ++g) {
            const auto u = *reinterpret_cast<const VfVec<float>::U4*>(p + 4 * g);
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

// The request of row r: the number of requests whose first row lies at or before it, less one.
// Every lane of the calling wave returns it.
__device__ __forceinline__ int vf_request(const VerifyArgs& a, int r) {
    int n = 0;
    for (int b0 = 0; b0 < a.B; b0 += kWave) {
        const int b = b0 + lane_id();
        n += __popcll(wave_ballot(b < a.B && a.cu[min(b, a.B)] + b <= r));
    }
    return n > 0 ? n - 1 : 0;
}

struct VfParams {
    float T, top_p, min_p;
    int k;
    bool greedy, cuts;
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
    return p;
}

__device__ __forceinline__ float vf_lane_xor(float v, int s) { return u2f(lane_xor(f2u(v), s)); }

// A running (maximum, sum of exp2(x c - maximum)).
struct VfSum {
    float m = -kVfInf, s = 0.0f;
    __device__ __forceinline__ void merge(float om, float os) {
        const float n = __builtin_fmaxf(m, om), ref = n == -kVfInf ? 0.0f : n;
        s = s * vf_exp2(m - ref) + os * vf_exp2(om - ref);
        m = n;
    }
    __device__ __forceinline__ void wave_merge() {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) merge(vf_lane_xor(m, o), vf_lane_xor(s, o));
    }
};

__device__ __forceinline__ uint64_t vf_pack(uint32_t key, int i) {
    return key ? ((uint64_t)key << 32) | (uint32_t)(0x7FFFFFFF - i) : 0ull;
}
__device__ __forceinline__ int vf_index(uint64_t top) { return top ? (int)(0x7FFFFFFFu - (uint32_t)top) : 0; }
__device__ __forceinline__ float vf_value(uint64_t top) {
    return top ? val_of((uint32_t)(top >> 32)) : __builtin_nanf("");
}

// Part p of row r: its largest logit, the lowest index that has it, and the sum of exponentials.
// NaN logits are never the largest and add nothing.
template <typename T>
__global__ __launch_bounds__(kVfThreads) void verify_rows_kernel(VerifyArgs a) {
    constexpr int VEC = Elem<T>::kVec, U = 4;
    __shared__ uint64_t red_top[kVfThreads / 64];
    __shared__ float red_m[kVfThreads / 64], red_s[kVfThreads / 64];
    const int S = a.S, r = blockIdx.x / S, p = blockIdx.x - r * S, tid = threadIdx.x, wave = tid >> 6;
    if (p == 0 && tid == 0 && r < a.B) a.ctr[r] = 0u;  // (R >= B)
    const VfParams prm = vf_params(a, vf_request(a, r));
    if (prm.cuts) return;
    const float c = prm.greedy ? 0.0f : 0x1.715476p+0f / prm.T;
    const T* row = static_cast<const T*>(a.x) + (size_t)r * a.xstride;
    const int lo = p * a.part_len, len = min(a.V, lo + a.part_len) - lo, nvec = len / VEC;
    row += lo;
    VfSum t;
    float best = __builtin_nanf("");  // the largest logit so far, and the first group of U vectors that holds it
    int group = tid;
    for (int b = tid; b < nvec; b += U * kVfThreads) {
        float v[U][VEC];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int vi = b + u * kVfThreads;
            vf_load<T>(row, vi < nvec ? vi : b, v[u]);
        }
        float g = v[0][0];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < VEC; ++j) g = __builtin_fmaxf(g, v[u][j]);
        if (g == g && !(g <= best)) { best = g; group = b; }
        if (!prm.greedy) {
            const float n = __builtin_fmaxf(t.m, g * c), ref = n == -kVfInf ? 0.0f : n;
            float acc[4] = {t.s * vf_exp2(t.m - ref), 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool in = b + u * kVfThreads < nvec;
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float e = vf_exp2(__builtin_fmaf(v[u][j], c, -ref));
                    acc[j & 3] += in && e == e ? e : 0.0f;
                }
            }
            t.s = (acc[0] + acc[1]) + (acc[2] + acc[3]);
            t.m = n;
        }
    }
    // the largest logit's first place in its group
    uint64_t top = 0ull;
    if (tid < nvec) {
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
    const int i = nvec * VEC + tid;
    if (i < len) {
        const float x = Elem<T>::load1(row + i);
        top = vws_max64(top, vf_pack(key_of(x), lo + i));
        if (!prm.greedy && x == x) t.merge(x * c, x > -kVfInf ? 1.0f : 0.0f);
    }
    top = wave_max_u64(top);
    t.wave_merge();
    if ((tid & 63) == 0) { red_top[wave] = top; red_m[wave] = t.m; red_s[wave] = t.s; }
    __syncthreads();
    if (tid == 0) {
        VfRec o;
        VfSum s;
        o.top = 0ull;
#pragma unroll
        for (int w = 0; w < kVfThreads / 64; ++w) {
            o.top = vws_max64(o.top, red_top[w]);
            s.merge(red_m[w], red_s[w]);
        }
        o.m2 = s.m;
        o.sum = s.s;
        a.rec[(size_t)r * S + p] = o;
    }
}

// ---- rows that their request cuts ---------------------------------------------------------

constexpr int kVfBins = 2048;
constexpr int kVfCutWaves = kVfCutThreads / 64;

struct VfCutShared {
    uint64_t hist[kVfBins];
    uint64_t red[kVfCutWaves];
    uint64_t out[4];
};

// Calls f(index, y) for every element of a row (each thread its vectors, then one tail element).
template <typename T, typename F>
__device__ __forceinline__ void vf_each(const T* row, int V, float Tt, F f) {
    constexpr int VEC = Elem<T>::kVec;
    const int nvec = V / VEC;
    for (int vi = threadIdx.x; vi < nvec; vi += kVfCutThreads) {
        float v[VEC];
        vf_load<T>(row, vi, v);
#pragma unroll
        for (int j = 0; j < VEC; ++j) f(vi * VEC + j, Tt == 1.0f ? v[j] : v[j] / Tt);
    }
    const int i = nvec * VEC + threadIdx.x;
    if (i < V) {
        const float x = Elem<T>::load1(row + i);
        f(i, Tt == 1.0f ? x : x / Tt);
    }
}

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

// The bin of sh.hist (bins [0, n), n a multiple of 64, up to kVfBins) where the running sum from
// bin 0 up first exceeds `thr`, and the sum below it.  All threads call; the total exceeds thr.
__device__ __forceinline__ void vf_find(VfCutShared& sh, int n, uint64_t thr, int* bin, uint64_t* below) {
    __syncthreads();
    if (threadIdx.x < kWave) {
        const int per = n / kWave, lane = lane_id();
        uint64_t s = 0;
        for (int i = 0; i < per; ++i) s += sh.hist[lane * per + i];
        uint64_t incl = s;
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) {
            const uint64_t t = __shfl_up(incl, o, kWave);
            if (lane >= o) incl += t;
        }
        uint64_t c = incl - s;
        if (c <= thr && thr < incl) {
            int i = 0;
            while (c + sh.hist[lane * per + i] <= thr) { c += sh.hist[lane * per + i]; ++i; }
            sh.out[0] = (uint64_t)(lane * per + i);
            sh.out[1] = c;
        }
    }
    __syncthreads();
    *bin = (int)sh.out[0];
    *below = sh.out[1];
    __syncthreads();
}

// The key at which the running sum of weight(key, y) over ascending keys first exceeds thr, with the
// sum of all smaller keys: three passes over the row, 11, 11 and 10 bits of the key.
template <typename T, typename W>
__device__ __forceinline__ uint32_t vf_select(const T* row, int V, float Tt, VfCutShared& sh, uint64_t thr,
                                              uint64_t* below, W weight) {
    uint32_t prefix = 0u;
    uint64_t under = 0ull;
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = pass == 2 ? 10 : 11;
        for (int i = threadIdx.x; i < kVfBins; i += kVfCutThreads) sh.hist[i] = 0ull;
        __syncthreads();
        vf_each<T>(row, V, Tt, [&](int, float y) {
            const uint32_t k = key_of(y);
            if (pass > 0 && (k >> (shift + bits)) != prefix) return;
            const uint64_t w = weight(k, y);
            if (w) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.hist[(k >> shift) & ((1u << bits) - 1u)]),
                             (unsigned long long)w);
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

// The n-th (from 0) lowest index among the row's elements whose key is `key`: two passes over the row.
template <typename T>
__device__ __forceinline__ int vf_nth_index(const T* row, int V, float Tt, VfCutShared& sh, uint32_t key, uint64_t n) {
    int hi = 0, lo = 0;
    uint64_t under;
    for (int pass = 0; pass < 2; ++pass) {
        for (int i = threadIdx.x; i < kVfBins; i += kVfCutThreads) sh.hist[i] = 0ull;
        __syncthreads();
        vf_each<T>(row, V, Tt, [&](int i, float y) {
            if (key_of(y) != key || (pass && (i >> 8) != hi)) return;
            atomicAdd(reinterpret_cast<unsigned long long*>(&sh.hist[pass ? (i & 255) : (i >> 8)]), 1ull);
        });
        vf_find(sh, pass ? 256 : kVfBins, n, pass ? &lo : &hi, &under);
        n -= under;
    }
    return hi * 256 + lo;
}

// One workgroup per row: the kept set of a row that its request cuts, as the smallest
// (key(y) << 32 | index) kept, and the sum of its exponentials.
template <typename T>
__global__ __launch_bounds__(kVfCutThreads) void verify_cut_kernel(VerifyArgs a) {
    __shared__ VfCutShared sh;
    const int r = blockIdx.x;
    const VfParams prm = vf_params(a, vf_request(a, r));
    if (!prm.cuts) return;
    const T* row = static_cast<const T*>(a.x) + (size_t)r * a.xstride;
    const float Tt = prm.T;
    const int V = a.V;
    uint64_t top = 0ull, nvalid = 0ull;
    vf_each<T>(row, V, 1.0f, [&](int i, float x) {
        const uint32_t k = key_of(x);
        top = vws_max64(top, vf_pack(k, i));
        nvalid += k ? 1u : 0u;
    });
    top = vf_block_max(top, sh);
    nvalid = vf_block_sum(nvalid, sh);
    const float m = vf_value(top) / Tt;
    VfRec o;
    o.top = top;
    o.m2 = m;
    o.sum = 0.0f;
    uint64_t cut = 0ull;
    if (__builtin_fabsf(m) < kVfInf) {
        const float lp_min = prm.min_p > 0.0f ? log_det(prm.min_p < 1.0f ? prm.min_p : 1.0f) : -kVfInf;
        uint32_t kth = 1u;  // every key but a NaN's
        if (prm.k > 0 && (uint64_t)prm.k <= nvalid) {
            uint64_t under;
            kth = vf_select<T>(row, V, Tt, sh, nvalid - (uint64_t)prm.k, &under,
                               [](uint32_t k, float) { return (uint64_t)(k ? 1u : 0u); });
        }
        auto weight = [=](uint32_t k, float y) -> uint64_t {
            const float d = y - m;
            return k >= kth && d >= lp_min ? mass_of(exp_det(d)) : 0ull;
        };
        // (the kept set without top-p, as one bound on the key)
        uint64_t W = 0ull, kmin = ~0ull;
        vf_each<T>(row, V, Tt, [&](int, float y) {
            const uint32_t k = key_of(y);
            if (k >= kth && y - m >= lp_min) {
                W += mass_of(exp_det(y - m));
                kmin = vws_min64(kmin, k);
            }
        });
        W = vf_block_sum(W, sh);
        kmin = ~vf_block_max(~kmin, sh);
        cut = kmin << 32;
        uint64_t kept = W;
        const float q32 = 1.0f - prm.top_p;
        if (q32 >= 1.0f) {
            // only the last of (key, index)
            uint64_t lastk = 0ull;
            const uint32_t mk = key_of(m);
            vf_each<T>(row, V, Tt, [&](int i, float y) {
                if (key_of(y) == mk) lastk = vws_max64(lastk, ((uint64_t)mk << 32) | (uint32_t)i);
            });
            cut = vf_block_max(lastk, sh);
            kept = 1ull << 44;
        } else if (q32 > 0.0f) {
            const uint64_t thr = scale_floor(q32, W);
            uint64_t under;
            const uint32_t key = vf_select<T>(row, V, Tt, sh, thr, &under, weight);
            const uint64_t w = mass_of(exp_det(val_of(key) - m));
            const uint64_t gone = (thr - under) / w;  // of the elements with that key, the lowest indices
            cut = (uint64_t)key << 32;
            if (gone) cut |= (uint32_t)vf_nth_index<T>(row, V, Tt, sh, key, gone);
            kept = W - under - gone * w;
        }
        o.sum = (float)kept * 0x1p-44f;
    }
    if (threadIdx.x == 0) {
        a.rec[(size_t)r * a.S] = o;
        a.cut[r] = cut;
    }
}

// ---- decision and race ----------------------------------------------------------------------

struct VfRow {
    uint64_t top, cut;
    float m, sum;
    bool sure;  // greedy, or the maximum is not finite: the row's distribution is its argmax
};

// Row r's statistics from its parts, in every lane of the calling wave.
__device__ __forceinline__ VfRow vf_row(const VerifyArgs& a, const VfParams& prm, int r) {
    VfRow o;
    VfRec v{0ull, -kVfInf, 0.0f};
    const int lane = lane_id();
    if (prm.cuts) {
        v = a.rec[(size_t)r * a.S];
        o.top = v.top;
        o.cut = a.cut[r];
        o.m = v.m2;
        o.sum = v.sum;
        o.sure = !(__builtin_fabsf(v.m2) < kVfInf);
        return o;
    }
    if (lane < a.S) v = a.rec[(size_t)r * a.S + lane];
    VfSum t;
    t.m = v.m2;
    t.s = v.sum;
    o.top = wave_max_u64(v.top);
    o.cut = 0ull;
    const float x = vf_value(o.top);
    o.m = prm.greedy ? x : x / prm.T;
    o.sure = prm.greedy || !(__builtin_fabsf(o.m) < kVfInf);
    t.wave_merge();
    // relative to x c - maximum, whose rounding leaves the largest element's own term off 1
    o.sum = t.s * vf_exp2(-__builtin_fmaf(x, prm.greedy ? 0.0f : 0x1.715476p+0f / prm.T, -t.m));
    return o;
}

__device__ __forceinline__ bool vf_kept(const VfRow& w, float y, int i) {
    const uint32_t k = key_of(y);
    return k != 0u && (((uint64_t)k << 32) | (uint32_t)i) >= w.cut;
}

// Part p of request b's race; every part decides the request for itself.
template <typename T>
__global__ __launch_bounds__(kVfThreads) void verify_token_kernel(VerifyArgs a) {
    constexpr int VEC = Elem<T>::kVec;
    __shared__ VfRow rows[kVfMaxDrafts + 1];
    __shared__ uint64_t red[kVfThreads / 64];
    __shared__ uint32_t last;
    const int S2 = a.S2, b = blockIdx.x / S2, p = blockIdx.x - b * S2, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const VfParams prm = vf_params(a, b);
    const int first = a.cu[b], n = a.cu[b + 1] - first, K1 = a.K + 1;
    if (first < 0 || n < 0 || n > a.K || first > a.D - n) {  // bounds that do not fit: no token
        if (p == 0) {
            for (int i = tid; i < K1; i += kVfThreads) {
                a.tokens[(size_t)b * K1 + i] = -1;
                a.logprobs[(size_t)b * K1 + i] = 0.0f;
            }
            if (tid == 0) a.accepted[b] = -1;
        }
        return;
    }
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
        auto add = [&](int i, float x, float qi, float ui) {
            const float y = x / prm.T;
            if (!vf_kept(w, y, i) || i == drop) return;
            const float e = exp_det(y - w.m);
            const float wt = q ? __builtin_fmaxf(e * inv - qi, 0.0f) : e;
            if (!(wt > 0.0f)) return;
            const float key = wt / (0.0f - log_det(ui));
            if (key >= 0.0f) best = vws_max64(best, vf_pack(f2u(key) + 1u, i));
        };
        const int lo = p * a.part2_len, len = min(a.V, lo + a.part2_len) - lo, nvec = len / VEC;
        for (int vi = tid; vi < nvec; vi += kVfThreads) {
            float v[VEC], qv[VEC] = {}, uv[VEC];
            const int i0 = lo + vi * VEC;
            vf_load<T>(row + lo, vi, v);
            if (q) vf_load_any<VEC>(q, a.qdtype, i0, qv);
            if (u) vf_load_any<VEC>(u, VWS_DTYPE_F32, i0, uv);
            else philox_uniforms_aligned<VEC>(seed, offset, (uint32_t)i0, uv);
#pragma unroll
            for (int j = 0; j < VEC; ++j) add(i0 + j, v[j], qv[j], uv[j]);
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
        if (S2 > 1) {
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
    template __global__ void verify_token_kernel<T>(VerifyArgs);
VWS_VERIFY_INST(float)
VWS_VERIFY_INST(uint16_t)
VWS_VERIFY_INST(_Float16)
#undef VWS_VERIFY_INST

}  // namespace vws
