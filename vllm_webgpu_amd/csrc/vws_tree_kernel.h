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

// All ones in the halves of a word that are not finite (E's exponents; without compares, whose masks would take
// scalar registers).
template <typename E>
__device__ __forceinline__ uint32_t tr_odd(uint32_t w) {
    const uint32_t top = ((w & (E::kExp * 0x10001u)) + (0x8000u - E::kExp) * 0x10001u) & 0x80008000u;
    return (top << 1) - (top >> 15);
}
// 0 or all ones, by bit i.
__device__ __forceinline__ uint32_t tr_bit(uint32_t w, int i) { return 0u - ((w >> i) & 1u); }

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

// Floats that a lane hands over.
constexpr int tr_acc(int D, int MT) { return MT * (D / 4 + 2); }
// Bytes of a step's keys, and of its values, that a wave keeps in LDS.
constexpr int tr_tile(int D) { return 2 * kTrKeys * D; }
constexpr int tr_lds(int D, int MT) {
    const int ring = kTrThreads / 64 * 2 * tr_tile(D), merge = kTrThreads / 128 * 64 * 4 * tr_acc(D, MT);
    return ring > merge ? ring : merge;
}

// 64 times 16 bytes into LDS, lane by lane from `to` on.
__device__ __forceinline__ void tr_fetch(char* to, const uint16_t* from) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}
// Until at most N of a wave's latest loads are on their way.
template <int N>
__device__ __forceinline__ void tr_arrived() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Until what a wave has read from LDS is in its registers, and may be overwritten there.
__device__ __forceinline__ void tr_read() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// Where a tile keeps 16-byte chunk c of key row i (0 .. 15), and chunk c of dimension row i of its values: lanes
// that read together lie in different banks.
template <int D>
__device__ __forceinline__ int tr_key_place(int c, int i) { return c ^ (i & (D % 128 == 0 ? 15 : D % 64 == 0 ? 7 : 3)); }
__device__ __forceinline__ int tr_value_place(int c, int i) { return c ^ ((i >> 1 & 2) | ((i >> 1 ^ i >> 3) & 1)); }

// MT tiles of 16 rows, from m0 on; the workgroup's four waves take the keys in turn, 32 at a time, each through LDS
// of its own (no wave waits for another), and join what they have in LDS.
template <typename T, int D, int MT>
__device__ __forceinline__ void tree_rows(const TreeArgs& a, const TrBounds& o, int b, int h, int split, int m0, char* lds) {
    constexpr int WK = kTrThreads / 64, KS = D / 32, DT = D / 16, kAcc = tr_acc(D, MT), kStep = WK * kTrKeys;
    constexpr int kTile = tr_tile(D), kLoads = D / 16;  // loads of a tile
    typedef TrElem<T> E;
    const int lane = threadIdx.x & 63, wk = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i16 = lane & 15, g = lane >> 4, rows = o.n * a.group;
    const int k0 = split * a.chunk, k1 = min(o.len, k0 + a.chunk), first = k0 + wk * kTrKeys;
    const int pm = (1 << a.c.pshift) - 1;
    const uint16_t* const kh = a.c.k + (((int64_t)h << a.c.pshift) * D);
    const uint16_t* const vh = a.c.v + (((int64_t)h << a.c.pshift) * D);
    // (the table is read as constants: its entries are the same for every lane)
    typedef const __attribute__((address_space(4))) int32_t* Entry;
    const Entry table = (Entry)(a.table + (int64_t)b * a.table_stride);

    TrU4 q[MT][KS];
    TrF4 acc[MT][DT];
    float ref[MT], sum[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        ref[mt] = -kTrInf;
        sum[mt] = 0.0f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[mt][dt] = TrF4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    char* const ring = lds + wk * 2 * kTile;
    // the pages of a step's four eights of keys (entries past the request's last are not read), 0 for those that do not exist, and
    // the keys that lie in pages that do
    struct Pages { int p[4]; uint32_t live; };
    auto pages_at = [&](int kb) __attribute__((always_inline)) {
        Pages s;
        s.live = 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int p = table[min(kb + 8 * e, o.len - 1) >> a.c.pshift];
            const bool good = (uint32_t)p < (uint32_t)a.c.pages;
            s.p[e] = good ? p : 0;
            s.live |= good ? 0xFFu << (8 * e) : 0u;
        }
        return s;
    };
    auto fetch_k = [&](const Pages& s, int kb) __attribute__((always_inline)) {
        const uint16_t* at[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) at[e] = kh + (int64_t)s.p[e] * a.c.kps + ((kb + 8 * e) & pm) * D;
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const int n = 64 * j + lane, key = n / (D / 8), c = n - key * (D / 8), i = (key >> 3) * 4 + (key & 3);
            const uint16_t* base = at[(64 * j) / D];
            // (of 96 dimensions a load may span two eights)
            if ((64 * j) / D != (64 * j + 63) / D) base = key >= 8 * ((64 * j) / D + 1) ? at[(64 * j + 63) / D] : base;
            tr_fetch(ring + 1024 * j, base + (key & 7) * D + 8 * tr_key_place<D>(c, i));
        }
    };
    auto fetch_v = [&](const Pages& s, int kb) __attribute__((always_inline)) {
        const int r = lane >> 2, e = tr_value_place(lane & 3, r);  // this lane's dimension and eight
        const int p01 = e & 1 ? s.p[1] : s.p[0], p23 = e & 1 ? s.p[3] : s.p[2];
        const uint16_t* p = vh + (int64_t)(e & 2 ? p23 : p01) * a.c.vps + ((r << a.c.pshift) + ((kb + 8 * e) & pm));
#pragma unroll
        for (int j = 0; j < kLoads; ++j) tr_fetch(ring + kTile + 1024 * j, p + ((16 * j) << a.c.pshift));
    };
    auto key_of_tile = [&](int t, int s) __attribute__((always_inline)) {
        const int key = 8 * (i16 >> 2) + 4 * t + (i16 & 3);
        return *reinterpret_cast<const TrU4*>(ring + key * (2 * D) + 16 * tr_key_place<D>(4 * s + g, i16));
    };
    auto value_of_tile = [&](int dt) __attribute__((always_inline)) {
        return *reinterpret_cast<const TrU4*>(ring + kTile + (16 * dt + i16) * 64 + 16 * tr_value_place(g, i16));
    };

    // one step, of keys kb and on; the tiles take the next one's as soon as the products have read them
    auto step = [&](int kb, uint32_t live, const Pages& next_pages) __attribute__((always_inline)) {
        const int next = kb + kStep;
        const bool more = next < k1, edge = kb + kTrKeys > o.context || live != ~0u;
        tr_arrived<kLoads>();  // (but for the values)
        TrF4 s[MT][2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const TrU4 f = key_of_tile(t, k);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) s[mt][t] = E::mma(f, q[mt][k], k ? s[mt][t] : TrF4{0.0f, 0.0f, 0.0f, 0.0f});
            }
        }
        uint32_t seen[MT];
        if (edge) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const int m = m0 + mt * 16 + i16;
                seen[mt] = (m < rows ? tr_seen(a, o, m / a.group, kb) : 0u) & live;
                const uint32_t mine = seen[mt] >> (8 * g);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t keep = tr_bit(mine, j);
                    s[mt][j >> 2][j & 3] = u2f((f2u(s[mt][j >> 2][j & 3]) & keep) | (0xFF800000u & ~keep));
                }
            }
        }
        tr_read();
        if (more) fetch_k(next_pages, next);
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
                const float w = m == -kTrInf ? 1.0f : tr_exp2(ref[mt] - m);
                ref[mt] = m;
                sum[mt] *= w;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) acc[mt][dt] *= w;
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
        if (more) tr_arrived<kLoads>();  // (but for the next keys)
        else tr_arrived<0>();
        if (!edge) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const TrU4 f = value_of_tile(dt);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) acc[mt][dt] = E::mma(f, p[mt], acc[mt][dt]);
            }
        } else {
            // values of keys that no row sees are nothing's; others that are not finite stay out of the common product
            // (0 times them is not 0)
            const uint32_t have = (tr_ones(o.len - kb) & live) >> (8 * g);
            uint32_t keep[4], odd = 0u;
#pragma unroll
            for (int w = 0; w < 4; ++w) keep[w] = (tr_bit(have, 2 * w) & 0xFFFFu) | (tr_bit(have, 2 * w + 1) << 16);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                TrU4 f = value_of_tile(dt);
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint32_t x = f[w] & keep[w], bad = tr_odd<E>(x);
                    odd |= bad;
                    f[w] = x & ~bad;
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) acc[mt][dt] = E::mma(f, p[mt], acc[mt][dt]);
            }
            if (wave_ballot(odd != 0u)) {
                // a product for each key that has such values, added for the rows that see it
#pragma unroll 1
                for (int e = 0; e < 32 && kb + e < o.len; ++e) {
                    const uint32_t mine = g == (e >> 3) && ((live >> e) & 1u) ? 0xFFFFu << (16 * (e & 1)) : 0u;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) {
                        TrU4 f = value_of_tile(dt);
#pragma unroll
                        for (int w = 0; w < 4; ++w) f[w] &= w == ((e & 7) >> 1) ? mine & tr_odd<E>(f[w]) : 0u;
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            const TrF4 add = E::mma(f, p[mt], TrF4{0.0f, 0.0f, 0.0f, 0.0f});
                            const uint32_t on = tr_bit(seen[mt], e);
#pragma unroll
                            for (int r = 0; r < 4; ++r) acc[mt][dt][r] += u2f(f2u(add[r]) & on);
                        }
                    }
                }
            }
        }
        tr_read();
        if (more) fetch_v(next_pages, next);
    };

    int kb = first;
    if (kb < k1) {
        const Pages now = pages_at(kb);
        fetch_k(now, kb);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const int m = m0 + mt * 16 + i16, node = m / a.group;
            const uint16_t* p = a.q + (int64_t)(o.t0 + node) * a.qts + (int64_t)(h * a.group + m - node * a.group) * a.qhs + 8 * g;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                TrU4 z = {0u, 0u, 0u, 0u};
                q[mt][s] = m < rows ? *reinterpret_cast<const TrU4a2*>(p + 32 * s) : z;
            }
        }
        fetch_v(now, kb);
        // (queries are waited for here, not by way of everything in flight in every step)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(q[mt][s]));
        uint32_t live = now.live;
        for (; kb < k1; kb += kStep) {
            const Pages next = pages_at(kb + kStep);
            step(kb, live, next);
            live = next.live;
        }
    }
    tr_arrived<0>();  // (what lands in LDS lands before it is used for something else)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        sum[mt] += tr_xor(sum[mt], 16);
        sum[mt] += tr_xor(sum[mt], 32);
    }

    // the waves, joined by halves, where their tiles were
    float* const merge = reinterpret_cast<float*>(lds);
    auto give = [&](int half) __attribute__((always_inline)) {
        __syncthreads();
        if (wk >= half && wk < 2 * half) {
            float* to = merge + (wk - half) * kAcc * 64 + lane;
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
            const float* from = merge + wk * kAcc * 64 + lane;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const float other = from[(2 * mt) * 64], m = __builtin_fmaxf(ref[mt], other), z = m == -kTrInf ? 0.0f : m;
                const float w = tr_exp2(ref[mt] - z), w1 = tr_exp2(other - z);
                ref[mt] = m;
                sum[mt] = sum[mt] * w + from[(2 * mt + 1) * 64] * w1;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        acc[mt][dt][r] = acc[mt][dt][r] * w + from[(2 * MT + (mt * DT + dt) * 4 + r) * 64] * w1;
            }
        }
    };
    static_assert(WK == 4, "two halvings");
    give(2);
    give(1);
    if (wk > 0) return;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int m = m0 + mt * 16 + i16;
        if (m >= rows) continue;
        if (a.splits == 1) {
            const float inv = sum[mt] == 0.0f ? 0.0f : 1.0f / sum[mt];
            const int node = m / a.group;
            uint16_t* p = a.out + (int64_t)(o.t0 + node) * a.ots + (int64_t)(h * a.group + m - node * a.group) * a.ohs + 4 * g;
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

// A workgroup's rows: up to MT tiles, as many as its request has there.
template <typename T, int D, int MT>
__global__ __launch_bounds__(kTrThreads, 2) void tree_kernel(TreeArgs a) {
    __shared__ __align__(1024) char lds[tr_lds(D, MT)];
    // workgroups of the same keys lie eight apart, on one chiplet
    const int per = 8 * a.blocks, item = (blockIdx.x / per) * 8 + (blockIdx.x & 7), mb = (blockIdx.x % per) >> 3;
    const int bs = item / a.c.heads, h = item - bs * a.c.heads, b = bs / a.splits, split = bs - b * a.splits;
    if (b >= a.B) return;
    TrBounds o;
    if (!tr_bounds(a, b, &o)) return;
    const int rows = o.n * a.group, m0 = mb * MT * 16;
    if (m0 >= rows || (split * a.chunk >= o.len && split > 0)) return;
    if (MT == 1 || rows - m0 <= 16) tree_rows<T, D, 1>(a, o, b, h, split, m0, lds);
    else tree_rows<T, D, MT>(a, o, b, h, split, m0, lds);
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

#define VWS_TREE(T, D)                                       \
    template __global__ void tree_kernel<T, D, 1>(TreeArgs);  \
    template __global__ void tree_join_kernel<T, D>(TreeArgs);
// (past 128 dimensions two tiles do not fit the registers)
#define VWS_TREES(T)                                          \
    VWS_TREE(T, 64) VWS_TREE(T, 96) VWS_TREE(T, 128)          \
    VWS_TREE(T, 192) VWS_TREE(T, 256)                         \
    template __global__ void tree_kernel<T, 64, 2>(TreeArgs); \
    template __global__ void tree_kernel<T, 96, 2>(TreeArgs); \
    template __global__ void tree_kernel<T, 128, 2>(TreeArgs);

}  // namespace vws
