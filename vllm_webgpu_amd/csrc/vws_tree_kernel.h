// vws_tree_kernel.h -- attention of drafted trees over a paged cache, instantiated by vws_tree_bf16.hip and
// vws_tree_f16.hip.
//
// A request's rows are its (node, query head of a key head) pairs: all of them read the same keys.
// For 32 keys at a time a wave takes S^T = K Q^T and O^T += V^T P^T by 16x16x32 matrix instructions.  A
// lane holds one row's column of S^T throughout, so softmax statistics need no exchange but between the four
// lanes of a row, and the exponentials of its keys are at once the second product's operand: the keys
// of the first product's two tiles are dealt out so that lane group g gets keys 8g .. 8g + 7.  Keys and values
// come from the cache in their operand layout (16 bytes a lane; the cache keeps values by dimension for that), so
// neither passes through LDS.
// The running reference of a row is raised only when some score exceeds it by 2^8 (P in 16 bits keeps its
// relative precision there, and sums are in 32): nearly every step then neither exchanges nor rescales.
#pragma once

#include "vws_device.h"
#include "vws_tree.h"

namespace vws {

typedef float TrF4 __attribute__((ext_vector_type(4)));
typedef uint32_t TrU4 __attribute__((ext_vector_type(4)));
typedef TrU4 TrU4a2 __attribute__((aligned(2)));

constexpr float kTrInf = __builtin_inff();
constexpr float kTrRaise = 8.0f;

__device__ __forceinline__ float tr_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float tr_xor(float v, int s) { return u2f(lane_xor(f2u(v), s)); }

template <typename T> struct TrElem;
template <> struct TrElem<uint16_t> {
    typedef __bf16 V8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ TrF4 mma(const TrU4& a, const TrU4& b, const TrF4& c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)lo) | ((uint32_t)__builtin_bit_cast(uint16_t, (__bf16)hi) << 16);
    }
    static constexpr uint32_t kExp = 0x7F80u;  // the exponent's bits: all set where a value is not finite
};
template <> struct TrElem<_Float16> {
    typedef _Float16 V8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ TrF4 mma(const TrU4& a, const TrU4& b, const TrF4& c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)lo) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)hi) << 16);
    }
    static constexpr uint32_t kExp = 0x7C00u;
};

__device__ __forceinline__ uint32_t tr_ones(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }

// A request's bounds, the same in every kernel: false where they do not fit.
struct TrBounds { int t0, n, context, len; };
__device__ __forceinline__ bool tr_bounds(const TreeArgs& a, int b, TrBounds* o) {
    o->t0 = a.cu[b];
    const int end = a.cu[b + 1];
    o->n = end - o->t0;
    if (o->t0 < 0 || end > a.T || end <= o->t0 || o->n > a.max_nodes) return false;
    const int most = (int)min((int64_t)a.max_pages << a.c.pshift, (int64_t)kCacheMaxPosition);
    o->context = min(max(a.context[b], 0), most);
    o->len = o->n < most - o->context ? o->context + o->n : most;
    return true;
}

// The keys [kb, kb + 32) that a row of node `node` sees, of those before `len`.
__device__ __forceinline__ uint32_t tr_seen(const TreeArgs& a, const TrBounds& o, int node, int kb) {
    const int rel = kb - o.context;
    uint32_t w;
    if (rel <= -32) {
        w = ~0u;
    } else if (!a.visible) {
        w = tr_ones(node - rel + 1);
    } else {
        const uint32_t* row = a.visible + (int64_t)(o.t0 + node) * a.visible_stride;
        auto word = [&](int i) { return i >= 0 && i < a.words ? row[i] : 0u; };
        if (rel < 0) {
            w = tr_ones(-rel) | (word(0) << -rel);
        } else {
            const int i = rel >> 5, s = rel & 31;
            w = s ? (word(i) >> s) | (word(i + 1) << (32 - s)) : word(i);
        }
    }
    return w & tr_ones(o.len - kb);
}

// A workgroup's rows: MT tiles of 16 for each of WM waves; the other 4 / WM waves of each take the keys in turn.
template <typename T, int D, int MT, int WM>
__global__ __launch_bounds__(kTrThreads) void tree_kernel(TreeArgs a) {
    constexpr int WK = 4 / WM, KS = D / 32, DT = D / 16, kAcc = MT * DT * 4 + MT * 2;
    constexpr int kSlots = WK / 2 * WM;  // waves that hand over at once
    __shared__ float merge[kSlots > 0 ? kSlots * kAcc * 64 : 1];
    typedef TrElem<T> E;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave % WM, wk = wave / WM;
    const int i16 = lane & 15, g = lane >> 4;
    // workgroups of the same keys lie eight apart, on one chiplet
    const int per = 8 * a.blocks, item = (blockIdx.x / per) * 8 + (blockIdx.x & 7), mb = (blockIdx.x % per) >> 3;
    const int bs = item / a.c.heads, h = item - bs * a.c.heads, b = bs / a.splits, split = bs - b * a.splits;
    if (b >= a.B) return;
    TrBounds o;
    if (!tr_bounds(a, b, &o)) return;
    const int rows = o.n * a.group, m0 = (mb * WM + wm) * MT * 16;
    const int k0 = split * a.chunk, k1 = min(o.len, k0 + a.chunk);
    if (mb * WM * MT * 16 >= rows || (k0 >= o.len && split > 0)) return;
    const int pm = (1 << a.c.pshift) - 1;
    const uint16_t* const kh = a.c.k + (((int64_t)h << a.c.pshift) * D);
    const uint16_t* const vh = a.c.v + (((int64_t)h << a.c.pshift) * D);
    const int32_t* const table = a.table + (int64_t)b * a.table_stride;

    TrU4 q[MT][KS];
    int node[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int m = m0 + mt * 16 + i16;
        node[mt] = m / a.group;
        const uint16_t* p = a.q + (int64_t)(o.t0 + node[mt]) * a.qts + (int64_t)(h * a.group + m - node[mt] * a.group) * a.qhs + 8 * g;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            TrU4 z = {0u, 0u, 0u, 0u};
            q[mt][s] = m < rows ? *reinterpret_cast<const TrU4a2*>(p + 32 * s) : z;
        }
    }
    TrF4 acc[MT][DT];
    float ref[MT], sum[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        ref[mt] = -kTrInf;
        sum[mt] = 0.0f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[mt][dt] = TrF4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    TrU4 kf[2][KS], vf[DT];
    const int oct = i16 >> 2;  // the eight keys that this lane's row of K lies in
    // pages of the lane's keys and values at kb: entries past the request's last are not read
    auto page_at = [&](int pos) __attribute__((always_inline)) { return table[min(pos, o.len - 1) >> a.c.pshift]; };
    auto good = [&](int p) __attribute__((always_inline)) { return (uint32_t)p < (uint32_t)a.c.pages; };
    auto load_k = [&](int kb, int page) __attribute__((always_inline)) {
        const uint16_t* p = kh + (int64_t)(good(page) ? page : 0) * a.c.kps + (((kb + 8 * oct) & pm) + (i16 & 3)) * D + 8 * g;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            kf[0][s] = *reinterpret_cast<const TrU4*>(p + 32 * s);
            kf[1][s] = *reinterpret_cast<const TrU4*>(p + 4 * D + 32 * s);
        }
    };
    auto load_v = [&](int kb, int page) __attribute__((always_inline)) {
        const uint16_t* p = vh + (int64_t)(good(page) ? page : 0) * a.c.vps + ((i16 << a.c.pshift) + ((kb + 8 * g) & pm));
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) vf[dt] = *reinterpret_cast<const TrU4*>(p + ((16 * dt) << a.c.pshift));
    };

    // one step; edge: some of its keys may be hidden from some rows
    auto step = [&](bool edge, int kb, int pk, int pv, int next, int pk_next, int pv_next) __attribute__((always_inline)) {
        TrF4 s[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                s[mt][t] = TrF4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < KS; ++k) s[mt][t] = E::mma(kf[t][k], q[mt][k], s[mt][t]);
            }
        if (next < k1) load_k(next, pk_next);
        uint32_t seen[MT];
        if (edge) {
            // (lanes 0, 4, 8 and 12 hold the four eights' pages)
            const uint64_t ok = wave_ballot(good(pk));
            uint32_t live = 0u;
#pragma unroll
            for (int e = 0; e < 4; ++e) live |= (ok >> (4 * e)) & 1u ? 0xFFu << (8 * e) : 0u;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                seen[mt] = (m0 + mt * 16 + i16 < rows ? tr_seen(a, o, node[mt], kb) : 0u) & live;
                const uint32_t mine = seen[mt] >> (8 * g);
#pragma unroll
                for (int j = 0; j < 8; ++j) s[mt][j >> 2][j & 3] = (mine >> j) & 1u ? s[mt][j >> 2][j & 3] : -kTrInf;
            }
        }
        bool raise = false;
        float top[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            float m = __builtin_fmaxf(s[mt][0][0], s[mt][1][0]);
#pragma unroll
            for (int j = 1; j < 4; ++j) m = __builtin_fmaxf(m, __builtin_fmaxf(s[mt][0][j], s[mt][1][j]));
            top[mt] = m * a.c2;
            raise |= top[mt] > ref[mt] + kTrRaise;
        }
        if (wave_ballot(raise)) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                float m = __builtin_fmaxf(top[mt], tr_xor(top[mt], 16));
                m = __builtin_fmaxf(ref[mt], __builtin_fmaxf(m, tr_xor(m, 32)));
                const float f = m == -kTrInf ? 1.0f : tr_exp2(ref[mt] - m);
                ref[mt] = m;
                sum[mt] *= f;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) acc[mt][dt] *= f;
            }
        }
        TrU4 p[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const float r = ref[mt] == -kTrInf ? 0.0f : ref[mt];
            float e[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) e[j] = tr_exp2(__builtin_fmaf(s[mt][j >> 2][j & 3], a.c2, -r));
            sum[mt] += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
#pragma unroll
            for (int j = 0; j < 4; ++j) p[mt][j] = E::pack(e[2 * j], e[2 * j + 1]);
        }
        bool odd = false;
        if (edge) {
            // values of keys that no row sees are nothing's; others that are not finite stay out of the common
            // product (0 times them is not 0)
            const int have = good(pv) ? min(max(o.len - kb - 8 * g, 0), 8) : 0;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t sh = 16 * (j & 1);
                    const bool bad = ((vf[dt][j >> 1] >> sh) & E::kExp) == E::kExp;
                    odd |= bad && j < have;
                    if (bad || j >= have) vf[dt][j >> 1] &= ~(0xFFFFu << sh);
                }
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) acc[mt][dt] = E::mma(vf[dt], p[mt], acc[mt][dt]);
        if (wave_ballot(odd)) {
            // a product for each key that has such values, added for the rows that see it
            load_v(kb, pv);
#pragma unroll 1
            for (int e = 0; e < 32 && kb + e < o.len; ++e) {
                const uint32_t sh = 16 * (e & 1);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    TrU4 one = {0u, 0u, 0u, 0u};
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const bool mine = g == (e >> 3) && w == ((e & 7) >> 1) && good(pv) && ((vf[dt][w] >> sh) & E::kExp) == E::kExp;
                        one[w] = mine ? vf[dt][w] & (0xFFFFu << sh) : 0u;
                    }
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        const TrF4 more = E::mma(one, p[mt], TrF4{0.0f, 0.0f, 0.0f, 0.0f});
                        if ((seen[mt] >> e) & 1u) acc[mt][dt] += more;
                    }
                }
            }
        }
        if (next < k1) load_v(next, pv_next);
    };

    int kb = k0 + wk * kTrKeys;
    constexpr int kStep = WK * kTrKeys;
    if (kb < k1) {
        int pk = page_at(kb + 8 * oct), pv = page_at(kb + 8 * g);
        load_k(kb, pk);
        load_v(kb, pv);
        int pk1 = page_at(kb + kStep + 8 * oct), pv1 = page_at(kb + kStep + 8 * g);
        for (; kb < k1; kb += kStep) {
            const int pk2 = page_at(kb + 2 * kStep + 8 * oct), pv2 = page_at(kb + 2 * kStep + 8 * g);
            step(kb + kTrKeys > o.context || wave_ballot(!good(pk)), kb, pk, pv, kb + kStep, pk1, pv1);
            pk = pk1; pv = pv1;
            pk1 = pk2; pv1 = pv2;
        }
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        sum[mt] += tr_xor(sum[mt], 16);
        sum[mt] += tr_xor(sum[mt], 32);
    }

    // the waves of the same rows, joined by halves
    for (int half = WK / 2; half > 0; half >>= 1) {
        if (half != WK / 2) __syncthreads();
        if (wk >= half && wk < 2 * half) {
            float* to = merge + ((wk - half) * WM + wm) * kAcc * 64 + lane;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                to[(2 * mt) * 64] = ref[mt];
                to[(2 * mt + 1) * 64] = sum[mt];
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) to[(2 * MT + (mt * DT + dt) * 4 + r) * 64] = acc[mt][dt][r];
            }
        }
        __syncthreads();
        if (wk < half) {
            const float* from = merge + (wk * WM + wm) * kAcc * 64 + lane;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const float other = from[(2 * mt) * 64], m = __builtin_fmaxf(ref[mt], other), z = m == -kTrInf ? 0.0f : m;
                const float f = tr_exp2(ref[mt] - z), f1 = tr_exp2(other - z);
                ref[mt] = m;
                sum[mt] = sum[mt] * f + from[(2 * mt + 1) * 64] * f1;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        acc[mt][dt][r] = acc[mt][dt][r] * f + from[(2 * MT + (mt * DT + dt) * 4 + r) * 64] * f1;
            }
        }
    }
    if (wk > 0) return;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int m = m0 + mt * 16 + i16;
        if (m >= rows) continue;
        if (a.splits == 1) {
            const float inv = sum[mt] == 0.0f ? 0.0f : 1.0f / sum[mt];
            uint16_t* p = a.out + (int64_t)(o.t0 + node[mt]) * a.ots + (int64_t)(h * a.group + m - node[mt] * a.group) * a.ohs + 4 * g;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                typedef uint32_t U2 __attribute__((ext_vector_type(2), aligned(2)));
                U2 w;
                w[0] = E::pack(acc[mt][dt][0] * inv, acc[mt][dt][1] * inv);
                w[1] = E::pack(acc[mt][dt][2] * inv, acc[mt][dt][3] * inv);
                *reinterpret_cast<U2*>(p + 16 * dt) = w;
            }
        } else {
            const int64_t rec = ((int64_t)(b * a.splits + split) * a.c.heads + h) * a.rows + m;
            float* p = a.part + rec * D + 4 * g;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<TrF4*>(p + 16 * dt) = acc[mt][dt];
            if (g == 0) {
                a.stat[2 * rec] = ref[mt];
                a.stat[2 * rec + 1] = sum[mt];
            }
        }
    }
}

// Joins the parts of a request's rows, a wave each.
template <typename T, int D>
__global__ __launch_bounds__(kTrThreads) void tree_join_kernel(TreeArgs a) {
    typedef TrElem<T> E;
    constexpr int N = (D + 63) / 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, quads = (a.rows + 3) / 4;
    const int bh = blockIdx.x / quads, m = (blockIdx.x - bh * quads) * 4 + wave, b = bh / a.c.heads, h = bh - b * a.c.heads;
    TrBounds o;
    if (!tr_bounds(a, b, &o) || m >= o.n * a.group) return;
    const int parts = max(1, (o.len + a.chunk - 1) / a.chunk);
    const int64_t first = ((int64_t)b * a.splits * a.c.heads + h) * a.rows + m, pitch = (int64_t)a.c.heads * a.rows;
    float top = -kTrInf;
    for (int i = lane; i < parts; i += 64) top = __builtin_fmaxf(top, a.stat[2 * (first + i * pitch)]);
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) top = __builtin_fmaxf(top, tr_xor(top, s));
    const float z = top == -kTrInf ? 0.0f : top;
    float total = 0.0f, v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = 0.0f;
    for (int i = 0; i < parts; ++i) {
        const int64_t rec = first + i * pitch;
        const float f = tr_exp2(a.stat[2 * rec] - z);
        total += a.stat[2 * rec + 1] * f;
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (lane + 64 * j < D) v[j] += a.part[rec * D + lane + 64 * j] * f;
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    const int node = m / a.group;
    uint16_t* p = a.out + (int64_t)(o.t0 + node) * a.ots + (int64_t)(h * a.group + m - node * a.group) * a.ohs;
#pragma unroll
    for (int j = 0; j < N; ++j)
        if (lane + 64 * j < D) p[lane + 64 * j] = (uint16_t)E::pack(v[j] * inv, 0.0f);
}

#define VWS_TREE(T, D, MT)                                      \
    template __global__ void tree_kernel<T, D, 1, 1>(TreeArgs);  \
    template __global__ void tree_kernel<T, D, MT, 2>(TreeArgs); \
    template __global__ void tree_kernel<T, D, MT, 4>(TreeArgs); \
    template __global__ void tree_join_kernel<T, D>(TreeArgs);
#define VWS_TREES(T)                                                          \
    VWS_TREE(T, 64, 2) VWS_TREE(T, 96, 2) VWS_TREE(T, 128, 2)                 \
    template __global__ void tree_kernel<T, 64, 2, 1>(TreeArgs);              \
    template __global__ void tree_kernel<T, 96, 2, 1>(TreeArgs);              \
    template __global__ void tree_kernel<T, 128, 2, 1>(TreeArgs);             \
    VWS_TREE(T, 192, 1) VWS_TREE(T, 256, 1)

}  // namespace vws
