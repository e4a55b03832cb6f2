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

// Queries and keys of `group` tokens: cosines and sines once for a token, then 16 bytes of each half of a pair (or
// of four pairs) at a time.
template <typename T>
__device__ __forceinline__ void append_rotate(const AppendArgs& a, float* cs) {
    const int t0 = blockIdx.x * a.group, n = min(a.group, a.T - t0), half = a.R >> 1, tid = threadIdx.x;
    const CacheView& c = a.c;
    for (int i = tid; i < n * half; i += kApThreads) {
        const int t = i / half, f = i - t * half;
        double turns = (double)a.positions[t0 + t] * (double)a.inv_freq[f] * 0.15915494309189533577;
        turns -= __builtin_rint(turns);
        float s, co;
        sincospif(2.0f * (float)turns, &s, &co);
        cs[2 * i] = co * a.scale;
        cs[2 * i + 1] = s * a.scale;
    }
    if (half) __syncthreads();
    // a head's units: pairs of vectors (or vectors) that turn, then vectors that do not
    const int turned = a.interleaved ? a.R >> 3 : half >> 3, units = turned + ((c.D - a.R) >> 3), heads = a.Hq + c.heads;
    const int total = n * heads * units;
    for (int i = tid; i < total; i += kApThreads) {
        const int hu = i / units, u = i - hu * units, t = hu / heads, h = hu - t * heads;
        const uint16_t* from;
        uint16_t* to;
        if (h < a.Hq) {
            from = a.q + (int64_t)(t0 + t) * a.qts + (int64_t)h * a.qhs;
            to = a.qo + (int64_t)(t0 + t) * a.qots + (int64_t)h * a.qohs;
        } else {
            int page, off;
            if (!cache_slot(c, a.slots[t0 + t], &page, &off)) continue;
            from = a.k + (int64_t)(t0 + t) * a.kts + (int64_t)(h - a.Hq) * a.khs;
            to = c.k + (int64_t)page * c.kps + ((int64_t)((h - a.Hq) << c.pshift) + off) * c.D;
        }
        if (u >= turned) {
            const int d = a.R + (u - turned) * 8;
            cache_store(to + d, cache_load(from + d));
            continue;
        }
        float x[8], y[8];
        if (a.interleaved) {
            const float* p = cs + 2 * (t * half + u * 4);
            const CacheVec w = cache_load(from + u * 8);
            Elem<T>::from_words(w.w[0], w.w[1], w.w[2], w.w[3], x);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                y[2 * j] = x[2 * j] * p[2 * j] - x[2 * j + 1] * p[2 * j + 1];
                y[2 * j + 1] = x[2 * j + 1] * p[2 * j] + x[2 * j] * p[2 * j + 1];
            }
            cache_store(to + u * 8, cache_pack8<T>(y));
        } else {
            const float* p = cs + 2 * (t * half + u * 8);
            const CacheVec w0 = cache_load(from + u * 8), w1 = cache_load(from + half + u * 8);
            float z[8], r[8];
            Elem<T>::from_words(w0.w[0], w0.w[1], w0.w[2], w0.w[3], x);
            Elem<T>::from_words(w1.w[0], w1.w[1], w1.w[2], w1.w[3], z);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                y[j] = x[j] * p[2 * j] - z[j] * p[2 * j + 1];
                r[j] = z[j] * p[2 * j] + x[j] * p[2 * j + 1];
            }
            cache_store(to + u * 8, cache_pack8<T>(y));
            cache_store(to + half + u * 8, cache_pack8<T>(r));
        }
    }
}

// Values of one head: a page keeps a dimension's tokens together, so a tile of tokens is turned in LDS.  Eight
// tokens whose slots fill an aligned eighth of a page (a run's inside) leave as one 16-byte store for
// each dimension; a token is looked up where its eight would begin, which another tile may hold.
struct AppendValues {
    int32_t slot[kApValueTokens + 14];  // from 7 tokens before the tile to 7 behind it; -1: none
    uint16_t x[(kApValueTokens + 7) * (256 + 2)];
};
__device__ __forceinline__ void append_values(const AppendArgs& a, AppendValues& sh) {
    const CacheView& c = a.c;
    const int b = blockIdx.x - a.wgs, tile = b / c.heads, h = b - tile * c.heads, t0 = tile * kApValueTokens, tid = threadIdx.x;
    const int n = min(kApValueTokens, a.T - t0), have = min(kApValueTokens + 7, a.T - t0), D = c.D, pitch = D + 2, vecs = D >> 3;
    const int most = c.pages << c.pshift;  // (at most 2^31 - 1: the launcher's check)
    for (int i = tid; i < kApValueTokens + 14; i += kApThreads) {
        const int t = t0 - 7 + i;
        const int s = t >= 0 && t < a.T ? a.slots[t] : -1;
        sh.slot[i] = s >= 0 && s < most ? s : -1;
    }
    for (int i = tid; i < have * vecs; i += kApThreads) {
        const int t = i / vecs, d = (i - t * vecs) * 8;
        const CacheVec w = cache_load(a.v + (int64_t)(t0 + t) * a.vts + (int64_t)h * a.vhs + d);
        uint32_t* to = reinterpret_cast<uint32_t*>(sh.x + t * pitch + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) to[j] = w.w[j];
    }
    __syncthreads();
    // whether eight slots in a row begin at the tile's token i (from -7 on)
    auto eight = [&](int i) {
        if (i < -7 || i + 7 >= kApValueTokens + 7) return false;
        const int s = sh.slot[i + 7];
        if (s < 0 || (s & 7)) return false;
#pragma unroll
        for (int j = 1; j < 8; ++j)
            if (sh.slot[i + 7 + j] != s + j) return false;
        return true;
    };
    auto at = [&](int s, int d) {
        return c.v + (int64_t)(s >> c.pshift) * c.vps + ((int64_t)(h * D + d) << c.pshift) + (s & ((1 << c.pshift) - 1));
    };
    const int wave = tid >> 6, lane = tid & 63;
    for (int i = wave; i < n; i += kApThreads / 64) {
        const int s = sh.slot[i + 7];
        if (s < 0) continue;
        const int first = i - (s & 7);
        if (eight(first)) {
            if (first != i) continue;  // (its eight's first token stores it)
            for (int d = lane; d < D; d += 64) {
                CacheVec v;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    v.w[j] = (uint32_t)sh.x[(i + 2 * j) * pitch + d] | ((uint32_t)sh.x[(i + 2 * j + 1) * pitch + d] << 16);
                cache_store(at(s, d), v);
            }
        } else {
            for (int d = lane; d < D; d += 64) *at(s, d) = sh.x[i * pitch + d];
        }
    }
}

// Keys rotated, queries rotated, values turned: one launch, the rotating workgroups first.
template <typename T>
__global__ __launch_bounds__(kApThreads) void append_kernel(AppendArgs a) {
    __shared__ union {
        float cs[kApThreads * 8];
        AppendValues v;
    } sh;
    if ((int)blockIdx.x < a.wgs) append_rotate<T>(a, sh.cs);
    else append_values(a, sh.v);
}

// A request's position; false where it lies in no page (what it leaves then is no place).
__device__ __forceinline__ bool cache_position(const CompactArgs& a, int b, int pos, int* page, int* off) {
    const int i = pos >> a.c.pshift;
    if (pos < 0 || i >= a.max_pages) return false;
    *page = a.table[(int64_t)b * a.table_stride + i];
    *off = pos & ((1 << a.c.pshift) - 1);
    return *page >= 0 && *page < a.c.pages;
}

// One head of one request.  Entry j's node never lies before position j, so entries are taken in order, some at
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
