// vws_cache.hip -- a paged cache's writes: keys and values appended with the position rotation applied on the
// way, and the accepted nodes of a drafted tree moved up behind their context.
//
// The pair (a, b) of a head at position t turns by theta = t f: (a cos - b sin, b cos + a sin).  A fp32 product
// t f is off by up to half an ulp of itself, at t = 2^20 by 2^-4 radians; so the angle is taken in 64 bits, as
// a fraction of a turn, whose sine and cosine are then those of a small fp32 angle.
#include "vws_cache.h"
#include "vws_device.h"
#include "vws_sampler.h"

namespace vws {

typedef uint32_t CacheU4 __attribute__((ext_vector_type(4), aligned(2)));  // 16 bytes at any element's address
struct CacheVec { uint32_t w[4]; };

__device__ __forceinline__ CacheVec cache_load(const uint16_t* p) {
    const CacheU4 u = *reinterpret_cast<const CacheU4*>(p);
    return {{u[0], u[1], u[2], u[3]}};
}
__device__ __forceinline__ void cache_store(uint16_t* p, const CacheVec& v) {
    CacheU4 u;
    u[0] = v.w[0]; u[1] = v.w[1]; u[2] = v.w[2]; u[3] = v.w[3];
    *reinterpret_cast<CacheU4*>(p) = u;
}

template <typename T>
__device__ __forceinline__ uint32_t cache_pack(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t cache_pack<uint16_t>(float lo, float hi) {
    return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)lo) | ((uint32_t)__builtin_bit_cast(uint16_t, (__bf16)hi) << 16);
}
template <>
__device__ __forceinline__ uint32_t cache_pack<_Float16>(float lo, float hi) {
    return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)lo) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)hi) << 16);
}
template <typename T>
__device__ __forceinline__ CacheVec cache_pack8(const float (&v)[8]) {
    return {{cache_pack<T>(v[0], v[1]), cache_pack<T>(v[2], v[3]), cache_pack<T>(v[4], v[5]), cache_pack<T>(v[6], v[7])}};
}

// A slot's page and place in it; false outside the cache.
__device__ __forceinline__ bool cache_slot(const CacheView& c, int slot, int* page, int* off) {
    *page = slot >> c.pshift;
    *off = slot & ((1 << c.pshift) - 1);
    return slot >= 0 && *page < c.pages;
}

// What bounds both writes is HBM: 16384 tokens of 32 + 4 heads take 74 us, 4.5 TB/s read and written (a copy's 4.9), 4096 17
// us; 701 tokens of trees 8.2 us, of which the chain slot, load, store is most, and the call 12.

// Queries and keys of `group` tokens.  A head is `units` of 16 bytes or 32: pairs of vectors that turn together (or
// vectors of four pairs), then vectors that do not turn; a thread has one unit of several heads, and loads four of them
// before it turns any, the first four before the cosines and sines are there (one at a time: 16384 tokens 100 us, 74).
template <typename T>
__device__ __forceinline__ void append_rotate(const AppendArgs& a, float* cs) {
    constexpr int U = 4;
    const int t0 = blockIdx.x * a.group, n = min(a.group, a.T - t0), half = a.R >> 1, tid = threadIdx.x;
    const CacheView& c = a.c;
    const int turned = a.interleaved ? a.R >> 3 : half >> 3, units = turned + ((c.D - a.R) >> 3), heads = a.Hq + c.heads;
    const int first = tid / units, u = tid - first * units, step = kApThreads / units;
    const bool turns = u < turned, wide = turns && !a.interleaved;
    const int d = turns ? u * 8 : a.R + (u - turned) * 8;  // the unit's first element
    // this thread's (token, head), which advances by `step` heads
    int t = 0, h = first;
    auto wrap = [&]() __attribute__((always_inline)) {
        while (h >= heads && t < n) {
            h -= heads;
            ++t;
        }
    };
    wrap();
    bool live = first < step && t < n;  // (the last few threads may have no unit)
    CacheVec x[U], z[U];
    uint16_t* to[U];
    int at[U];  // token, or -1
    auto load = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            at[i] = -1;
            if (live) {
                const uint16_t* from;
                bool store = true;
                if (h < a.Hq) {
                    from = a.q + (int64_t)(t0 + t) * a.qts + (int64_t)h * a.qhs + d;
                    to[i] = a.qo + (int64_t)(t0 + t) * a.qots + (int64_t)h * a.qohs + d;
                } else {
                    int page = 0, off = 0;
                    store = cache_slot(c, a.slots[t0 + t], &page, &off);
                    from = a.k + (int64_t)(t0 + t) * a.kts + (int64_t)(h - a.Hq) * a.khs + d;
                    to[i] = c.k + (int64_t)page * c.kps + ((int64_t)((h - a.Hq) << c.pshift) + off) * c.D + d;
                }
                if (store) {
                    at[i] = t;
                    x[i] = cache_load(from);
                    if (wide) z[i] = cache_load(from + half);
                }
                h += step;
                wrap();
                live = t < n;
            }
        }
    };
    load();
    for (int i = tid; i < n * half; i += kApThreads) {
        const int k = i / half, f = i - k * half;
        double turn = (double)a.positions[t0 + k] * (double)a.inv_freq[f] * 0.15915494309189533577;
        turn -= __builtin_rint(turn);
        float s, co;
        sincospif(2.0f * (float)turn, &s, &co);
        cs[2 * i] = co * a.scale;
        cs[2 * i + 1] = s * a.scale;
    }
    if (half) __syncthreads();
    for (;;) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (at[i] < 0) continue;
            if (!turns) {
                cache_store(to[i], x[i]);
                continue;
            }
            float v[8], y[8];
            Elem<T>::from_words(x[i].w[0], x[i].w[1], x[i].w[2], x[i].w[3], v);
            if (!wide) {
                const float* p = cs + 2 * (at[i] * half + u * 4);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    y[2 * j] = v[2 * j] * p[2 * j] - v[2 * j + 1] * p[2 * j + 1];
                    y[2 * j + 1] = v[2 * j + 1] * p[2 * j] + v[2 * j] * p[2 * j + 1];
                }
                cache_store(to[i], cache_pack8<T>(y));
            } else {
                const float* p = cs + 2 * (at[i] * half + u * 8);
                float w[8], r[8];
                Elem<T>::from_words(z[i].w[0], z[i].w[1], z[i].w[2], z[i].w[3], w);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    y[j] = v[j] * p[2 * j] - w[j] * p[2 * j + 1];
                    r[j] = w[j] * p[2 * j] + v[j] * p[2 * j + 1];
                }
                cache_store(to[i], cache_pack8<T>(y));
                cache_store(to[i] + half, cache_pack8<T>(r));
            }
        }
        if (!live) break;
        load();
    }
}

// Values of one head: a page keeps a dimension's tokens together, so a tile of tokens is turned in LDS.  Eight
// tokens whose slots fill an aligned eight of a page (a run's inside) leave as one 16-byte store for each
// dimension, the eights of one dimension side by side; other tokens element by element.  A token is looked up where its
// eight would begin, which another tile may hold.
struct AppendValues {
    int32_t slot[kApValueTokens + 14];  // from 7 tokens before the tile to 7 behind it; -1: none
    int32_t eight[kApValueTokens], one[kApValueTokens];  // tokens that begin an eight, tokens of none
    uint32_t eights, ones;
};
__device__ __forceinline__ void append_values(const AppendArgs& a, AppendValues& sh, uint16_t* x) {
    const CacheView& c = a.c;
    const int b = blockIdx.x - a.wgs, tile = b / c.heads, h = b - tile * c.heads, t0 = tile * kApValueTokens, tid = threadIdx.x;
    const int n = min(kApValueTokens, a.T - t0), have = min(kApValueTokens + 7, a.T - t0), D = c.D, pitch = D + 2, vecs = D >> 3;
    const int most = c.pages << c.pshift;  // (at most 2^31 - 1: the launcher's check)
    if (tid < 2) (tid ? sh.ones : sh.eights) = 0u;
    for (int i = tid; i < kApValueTokens + 14; i += kApThreads) {
        const int t = t0 - 7 + i;
        const int s = t >= 0 && t < a.T ? a.slots[t] : -1;
        sh.slot[i] = s >= 0 && s < most ? s : -1;
    }
    for (int i = tid; i < have * vecs; i += kApThreads) {
        const int t = i / vecs, d = (i - t * vecs) * 8;
        const CacheVec w = cache_load(a.v + (int64_t)(t0 + t) * a.vts + (int64_t)h * a.vhs + d);
        uint32_t* to = reinterpret_cast<uint32_t*>(x + t * pitch + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) to[j] = w.w[j];
    }
    __syncthreads();
    if (tid < n && sh.slot[tid + 7] >= 0) {
        // whether the eight slots from where this token's eight begins (7 tokens before the tile at the earliest) follow
        // each other
        const int begin = tid + 7 - (sh.slot[tid + 7] & 7), s0 = sh.slot[tid + 7] & ~7;
        bool whole = true;
#pragma unroll
        for (int j = 0; j < 8; ++j) whole &= sh.slot[begin + j] == s0 + j;
        if (!whole) sh.one[atomicAdd(&sh.ones, 1u)] = tid;
    }
    __syncthreads();
    // (in order, so that neighbours are stored together)
    if (tid < 64) {
        const int s = tid < n ? sh.slot[tid + 7] : -1;
        bool begins = s >= 0 && (s & 7) == 0;
        if (begins) {
#pragma unroll
            for (int j = 1; j < 8; ++j) begins &= sh.slot[tid + 7 + j] == s + j;
        }
        const uint64_t all = wave_ballot(begins);
        if (begins) sh.eight[lane_prefix(all)] = tid;
        if (tid == 0) sh.eights = (uint32_t)__builtin_popcountll(all);
    }
    __syncthreads();
    auto at = [&](int s, int d) {
        return c.v + (int64_t)(s >> c.pshift) * c.vps + ((int64_t)(h * D + d) << c.pshift) + (s & ((1 << c.pshift) - 1));
    };
    const int eights = (int)sh.eights, ones = (int)sh.ones;
    constexpr int kSide = kApValueTokens / 8;
    for (int i = tid; i < kSide * D; i += kApThreads) {
        const int e = i % kSide, d = i / kSide;
        if (e >= eights) continue;
        const int t = sh.eight[e];
        CacheVec v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v.w[j] = (uint32_t)x[(t + 2 * j) * pitch + d] | ((uint32_t)x[(t + 2 * j + 1) * pitch + d] << 16);
        cache_store(at(sh.slot[t + 7], d), v);
    }
    const int wave = tid >> 6, lane = tid & 63;
    for (int i = wave; i < ones; i += kApThreads / 64) {
        const int t = sh.one[i];
        for (int d = lane; d < D; d += 64) *at(sh.slot[t + 7], d) = x[t * pitch + d];
    }
}

// Keys rotated, queries rotated, values turned: one launch, the rotating workgroups first.
template <typename T>
__global__ __launch_bounds__(kApThreads) void append_kernel(AppendArgs a) {
    extern __shared__ __align__(16) char append_lds[];
    __shared__ AppendValues sh;
    if ((int)blockIdx.x < a.wgs) append_rotate<T>(a, reinterpret_cast<float*>(append_lds));
    else append_values(a, sh, reinterpret_cast<uint16_t*>(append_lds));
}

// A request's position; false where it lies in no page (what it leaves then is no place).
__device__ __forceinline__ bool cache_position(const CompactArgs& a, int b, int pos, int* page, int* off) {
    const int i = pos >> a.c.pshift;
    if (pos < 0 || i >= a.max_pages) return false;
    *page = a.table[(int64_t)b * a.table_stride + i];
    *off = pos & ((1 << a.c.pshift) - 1);
    return *page >= 0 && *page < a.c.pages;
}

// One head of one request: a chain of table, load and store, 4.9 us for one request and 7.8 for 200 of 4 heads (700 moves of
// 2 KB; the call's host work is as long).  Entry j's node never lies before position j, so entries are taken in order, some at
// a time: all read before any is written.
constexpr int kCpEntries = 16;
__global__ __launch_bounds__(kApThreads) void compact_kernel(CompactArgs a) {
    __shared__ int32_t src[kCpEntries], dst[kCpEntries], spage[kCpEntries], dpage[kCpEntries];
    const CacheView& c = a.c;
    const int b = blockIdx.x / c.heads, h = blockIdx.x - b * c.heads, tid = threadIdx.x, D = c.D;
    const int context = a.context[b], vecs = D >> 3;
    const int32_t* path = a.path + (int64_t)b * a.path_stride;
    for (int j0 = 1; j0 < a.width; j0 += kCpEntries) {
        const int n = min(kCpEntries, a.width - j0);
        bool any = false;
        if (tid < n) {
            const int node = path[j0 + tid];
            // (a node before its entry, or past a tree's end, is no accepted path's)
            int sp = 0, so = 0, dp = 0, d = 0;
            const bool moves = context >= 0 && context <= kCacheMaxPosition && node > j0 + tid && node < VWS_MAX_TREE_NODES && cache_position(a, b, context + node, &sp, &so) &&
                               cache_position(a, b, context + j0 + tid, &dp, &d);
            src[tid] = moves ? so : -1;
            spage[tid] = sp;
            dst[tid] = d;
            dpage[tid] = dp;
            any = node >= 0;
        }
        if (!__syncthreads_or(any)) return;
        CacheVec key[kCpEntries * 256 / 8 / kApThreads];
        uint16_t val[kCpEntries];
#pragma unroll
        for (int u = 0; u < kCpEntries * 256 / 8 / kApThreads; ++u) {
            const int i = tid + u * kApThreads, e = i / vecs, d = (i - e * vecs) * 8;
            if (e < n && src[e] >= 0) key[u] = cache_load(c.k + (int64_t)spage[e] * c.kps + ((int64_t)(h << c.pshift) + src[e]) * D + d);
        }
        if (tid < D)
#pragma unroll
            for (int e = 0; e < kCpEntries; ++e)
                if (e < n && src[e] >= 0) val[e] = c.v[(int64_t)spage[e] * c.vps + ((int64_t)(h * D + tid) << c.pshift) + src[e]];
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kCpEntries * 256 / 8 / kApThreads; ++u) {
            const int i = tid + u * kApThreads, e = i / vecs, d = (i - e * vecs) * 8;
            if (e < n && src[e] >= 0) cache_store(c.k + (int64_t)dpage[e] * c.kps + ((int64_t)(h << c.pshift) + dst[e]) * D + d, key[u]);
        }
        if (tid < D)
#pragma unroll
            for (int e = 0; e < kCpEntries; ++e)
                if (e < n && src[e] >= 0) c.v[(int64_t)dpage[e] * c.vps + ((int64_t)(h * D + tid) << c.pshift) + dst[e]] = val[e];
        // (what this pass has written the next one's loads must see)
        stores_complete();
        __syncthreads();
    }
}

template __global__ void append_kernel<uint16_t>(AppendArgs);
template __global__ void append_kernel<_Float16>(AppendArgs);

}  // namespace vws
