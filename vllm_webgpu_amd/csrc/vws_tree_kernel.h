// vws_tree_kernel.h -- attention of drafted trees over a paged cache, instantiated by vws_tree_bf16.hip and
// vws_tree_f16.hip.
//
// A request's rows are its (node, query head of a key head) pairs: all of them read the same keys.
// For 32 keys at a time a wave takes S^T = K Q^T and O^T += V^T P^T by 16x16x32 matrix instructions.  A
// lane holds one row's column of S^T throughout, so softmax statistics need no exchange but between the four
// lanes of a row, and the exponentials of its keys are at once the second product's operand: the keys
// of the first product's two tiles are dealt out so that lane group g gets keys 8g .. 8g + 7.  The cache keeps
// values by dimension, so that both products' operands are 16 bytes of a row.
// Keys and values pass through LDS, by loads that go there directly: whole lines of a page, each lane's 16 bytes
// at a place where the products' reads find them in different banks (64 trees of up to 32 nodes over 8192 tokens took
// 1001 us from memory straight to the operands' lanes, whose loads touch sixteen rows each; 398 by way of LDS).
// The running reference of a row is raised only when some score exceeds it by more than 2^kRaise: nearly every step then
// neither exchanges nor rescales.  Sums are in 32 bits, of the unrounded exponentials; P is rounded to the cache's type,
// which is what the matrix instructions take, by at most 2^-8 (bf16) or 2^-11 of itself.  f16 has steps of 2^-24 below
// 2^-14: there the reference lies 2^kLift below the largest score, so that weights down to 2^-25 of the largest are rounded as
// any others, and 2^20 smaller ones lose less than 2^-16 in all (a first token of value 0, 17.5 nats above 131071 others in one
// part: the result is off by 0.03 %, with the reference at the largest score by 50; the time is the same).
//
// What bounds it is the cache's one read: 64 requests over 8192 tokens, 128 dimensions, take 241 us with one node each (5.2
// TB/s), 243 with 8 and 259 with up to 32 (4.9); three over 131000 293 (5.5 TB/s, reads alone).  From 64
// nodes of four heads on it is the arithmetic: 256 rows, 64 requests over 4096 tokens, 448 us, 0.6 PFLOP/s, with an
// exponential, two fmas and a rounding for every 512 of the products' operations.  One small request (12 nodes over 1900) takes
// 12 us and 4 for the join, of which 8.7 are a step's own latency (one key): launch, bounds, table, tile, products, joins.
#pragma once

#include <type_traits>

#include "vws_device.h"
#include "vws_tree.h"

namespace vws {

typedef float TrF4 __attribute__((ext_vector_type(4)));
typedef uint32_t TrU4 __attribute__((ext_vector_type(4)));
typedef TrU4 TrU4a2 __attribute__((aligned(2)));

constexpr float kTrInf = __builtin_inff();
// Scores (times log2 e) past this are far from zero: a 32-bit number's step is then no longer small beside 1, and a score less
// its rounded reference may be any power of two.  The reference of a row that holds one lies in LDS, two such steps lower, so that the
// largest weight is no less than kLift says, and its scores are taken less that reference in every step and end at
// kMost: keys whose scores differ by less than their rounding may weigh the same there.  It is part of raising a
// reference, without a branch (0.2 to 0.6 % of 64 requests' time, 2 % of a single tree's; with a branch around it 0.5 to 1 and 5).
constexpr float kTrFar = 0x1p22f;
__device__ __forceinline__ bool tr_far(float x) { return __builtin_fabsf(x) > kTrFar && __builtin_fabsf(x) < kTrInf; }

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
    // powers of two: that a score may exceed its reference, that the largest exceeds it at least, and at most far from zero
    static constexpr float kRaise = 8.0f, kLift = 0.0f, kMost = 64.0f;
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
    static constexpr float kRaise = 15.0f, kLift = 11.0f, kMost = 15.0f;  // (2^16 is infinite)
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
    o->n = (int)((uint32_t)end - (uint32_t)o->t0);
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
// Steps that a workgroup keeps in LDS (128 KB of 128 or 256 dimensions), and of those each lane.
constexpr int tr_steps(int D, int waves) { return D > 128 ? 4 : waves; }
constexpr int tr_deep(int D, int waves, int WM) { return tr_steps(D, waves) * WM / waves; }
// Waves of a SIMD: two, of one workgroup or two; of four waves past 128 dimensions the LDS holds one workgroup.
constexpr int tr_waves(int D, int waves) { return D > 128 && waves == 4 ? 1 : 2; }
constexpr int tr_lds(int D, int MT, int waves) {
    const int ring = tr_steps(D, waves) * 2 * tr_tile(D), merge = waves / 2 * 64 * 4 * tr_acc(D, MT);
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

// The workgroup's waves meet; what each has in flight stays so.
__device__ __forceinline__ void tr_meet() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Of 256 dimensions, operands are read four at a time: read ahead without a bound they do not fit the registers (79
// spilled of eight waves; a tree of 16 nodes, 64 requests, 493 us and 444).
template <int D>
__device__ __forceinline__ void tr_narrow(int i) {
    if (D > 192 && i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
}

// Where a tile keeps 16-byte chunk c of key row i (0 .. 15), and chunk c of dimension row i of its values: lanes
// that read together lie in different banks.
template <int D>
__device__ __forceinline__ int tr_key_place(int c, int i) { return c ^ (i & (D % 128 == 0 ? 15 : D % 64 == 0 ? 7 : 3)); }
__device__ __forceinline__ int tr_value_place(int c, int i) { return c ^ ((i >> 1 & 2) | ((i >> 1 ^ i >> 3) & 1)); }

// (Two tiles of rows a wave read each operand once for both; four spill.)
// MT tiles of 16 rows for each of WM waves, from m0 on.  The workgroup's waves make WAVES / WM lanes, which take the
// keys in turn, 32 at a time, each through LDS of its own, and join what they have there.  A lane of one wave waits for
// no other; the waves of a wider one share its tiles, and meet once a step.  `far`: the references of rows far from zero, 16 MT
// of each wave.
template <typename T, int D, int MT, int WAVES, int WM>
__device__ __forceinline__ void tree_rows(const TreeArgs& a, const TrBounds& o, int b, int h, int split, int m0, char* lds, float* far) {
    constexpr int WK = WAVES / WM, KS = D / 32, DT = D / 16, kAcc = tr_acc(D, MT), kStep = WK * kTrKeys;
    constexpr int kTile = tr_tile(D), kLoads = D / 16;  // loads of a tile
    constexpr int kMine = 2 * kLoads / WM;              // ... of a step's two that a wave makes
    constexpr int kDeep = tr_deep(D, WAVES, WM);        // steps of a lane's LDS
    static_assert(2 * kLoads % WM == 0, "every wave makes as many");
    typedef TrElem<T> E;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wk = wave / WM, wm = wave % WM;
    const int i16 = lane & 15, g = lane >> 4, rows = o.n * a.group;
    m0 += wm * MT * 16;
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

    char* const ring = lds + wk * kDeep * 2 * kTile;
    auto far_ref = [&](int mt) __attribute__((always_inline)) -> float& {
        int i = i16;
        asm volatile("" : "+v"(i));  // (the address is rarely needed: not kept in a register)
        return far[(wave * MT + mt) * 16 + i];
    };
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) far_ref(mt) = -kTrInf;
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
    // A wave's share (part of WM: every WM-th load) of a step's keys (what & 1) and of its values (what & 2), to the tiles
    // at `to`
    auto fetch = [&](const Pages& s, int kb, char* to, int part, auto what) __attribute__((always_inline)) {
        constexpr int kWhat = decltype(what)::value;
        if (kWhat & 1) {
            const uint16_t* at[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) at[e] = kh + (int64_t)s.p[e] * a.c.kps + ((kb + 8 * e) & pm) * D;
#pragma unroll
            for (int i = 0; i < (kLoads + WM - 1) / WM; ++i) {
                // (a load's first and last eight differ for 96 dimensions only)
                const int j = i * WM + part, e0 = (64 * j) / D, e1 = (64 * j + 63) / D;
                if (kLoads % WM && j >= kLoads) continue;
                const int n = 64 * j + lane, key = n / (D / 8), c = n - key * (D / 8), row = (key >> 3) * 4 + (key & 3);
                const uint16_t* base = e0 & 2 ? (e0 & 1 ? at[3] : at[2]) : (e0 & 1 ? at[1] : at[0]);
                if (D % 64) {
                    const uint16_t* last = e1 & 2 ? (e1 & 1 ? at[3] : at[2]) : (e1 & 1 ? at[1] : at[0]);
                    base = key >= 8 * (e0 + 1) ? last : base;
                }
                tr_fetch(to + 1024 * j, base + (key & 7) * D + 8 * tr_key_place<D>(c, row));
            }
        }
        if (kWhat & 2) {
            const int r = lane >> 2, e = tr_value_place(lane & 3, r);  // this lane's dimension and eight
            const int p01 = e & 1 ? s.p[1] : s.p[0], p23 = e & 1 ? s.p[3] : s.p[2];
            const uint16_t* const p = vh + (int64_t)(e & 2 ? p23 : p01) * a.c.vps + ((r << a.c.pshift) + ((kb + 8 * e) & pm));
#pragma unroll
            for (int i = 0; i < (kLoads + WM - 1) / WM; ++i) {
                // (of 96 dimensions half of four waves make one load of keys more, the others one of values)
                const int j = i * WM + (kLoads % WM ? (part + WM / 2) % WM : part);
                if (kLoads % WM && j >= kLoads) continue;
                tr_fetch(to + kTile + 1024 * j, p + ((16 * j) << a.c.pshift));
            }
        }
    };
    typedef std::integral_constant<int, 1> Keys;
    typedef std::integral_constant<int, 2> Values;
    typedef std::integral_constant<int, 3> Both;
    auto key_of_tile = [&](const char* tile, int t, int s) __attribute__((always_inline)) {
        const int key = 8 * (i16 >> 2) + 4 * t + (i16 & 3);
        return *reinterpret_cast<const TrU4*>(tile + key * (2 * D) + 16 * tr_key_place<D>(4 * s + g, i16));
    };
    auto value_of_tile = [&](const char* tile, int dt) __attribute__((always_inline)) {
        return *reinterpret_cast<const TrU4*>(tile + kTile + (16 * dt + i16) * 64 + 16 * tr_value_place(g, i16));
    };

    // one step, of keys kb and on, whose tiles lie at `tile`: keys_read once the first product has read the keys,
    // values_here before the second one reads the values
    auto step = [&](int kb, uint32_t live, const char* tile, auto keys_read, auto values_here) __attribute__((always_inline)) {
        const bool edge = kb + kTrKeys > o.context || live != ~0u;
        TrF4 s[MT][2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const TrU4 f = key_of_tile(tile, t, k);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) s[mt][t] = E::mma(f, q[mt][k], k ? s[mt][t] : TrF4{0.0f, 0.0f, 0.0f, 0.0f});
                tr_narrow<D>(k);
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
        keys_read();
        bool raise = false;
        float top[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            float m = __builtin_fmaxf(s[mt][0][0], s[mt][1][0]);
#pragma unroll
            for (int j = 1; j < 4; ++j) m = __builtin_fmaxf(m, __builtin_fmaxf(s[mt][0][j], s[mt][1][j]));
            top[mt] = m * a.c2;
            raise |= top[mt] > ref[mt] + E::kRaise;
        }
        if (wave_ballot(raise)) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                float m = __builtin_fmaxf(top[mt], tr_xor(top[mt], 16));
                m = __builtin_fmaxf(m, tr_xor(m, 32));
                const float was = ref[mt] == -kTrInf ? far_ref(mt) : ref[mt];
                m = __builtin_fmaxf(was, tr_far(m) ? m - E::kLift - __builtin_fabsf(m) * 0x1p-22f : m - E::kLift);
                const float w = m == -kTrInf ? 1.0f : tr_exp2(was - m);
                // (without a reference in its register a row comes here in every step)
                const bool off = tr_far(m);
                ref[mt] = off ? -kTrInf : m;
                far_ref(mt) = off ? m : -kTrInf;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float x = s[mt][j >> 2][j & 3], y = __builtin_fmaf(x, a.c2, -m);
                    s[mt][j >> 2][j & 3] = off ? (y > E::kMost ? E::kMost : y) * a.back : x;
                }
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
        values_here();
        if (!edge) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const TrU4 f = value_of_tile(tile, dt);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) acc[mt][dt] = E::mma(f, p[mt], acc[mt][dt]);
                tr_narrow<D>(dt);
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
                TrU4 f = value_of_tile(tile, dt);
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint32_t x = f[w] & keep[w], bad = tr_odd<E>(x);
                    odd |= bad;
                    f[w] = x & ~bad;
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) acc[mt][dt] = E::mma(f, p[mt], acc[mt][dt]);
                tr_narrow<D>(dt);
            }
            if (wave_ballot(odd != 0u)) {
                // a product for each key that has such values, added for the rows that see it
#pragma unroll 1
                for (int e = 0; e < 32 && kb + e < o.len; ++e) {
                    const uint32_t mine = g == (e >> 3) && ((live >> e) & 1u) ? 0xFFFFu << (16 * (e & 1)) : 0u;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) {
                        TrU4 f = value_of_tile(tile, dt);
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
    };

    auto load_q = [&]() __attribute__((always_inline)) {
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
    };
    // (queries are waited for once, not by way of everything in flight in every step)
    auto q_here = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(q[mt][s]));
    };
    if constexpr (WM == 1) {
        // a step's tiles take the next one's keys and values as soon as the products have read them
        if (first < k1) {
            const Pages now = pages_at(first);
            fetch(now, first, ring, 0, Keys());
            load_q();
            fetch(now, first, ring, 0, Values());
            q_here();
            uint32_t live = now.live;
            for (int kb = first; kb < k1; kb += kStep) {
                const Pages next = pages_at(kb + kStep);
                const bool more = kb + kStep < k1;
                tr_arrived<kLoads>();  // (but for the values)
                step(kb, live, ring,
                     [&]() __attribute__((always_inline)) {
                         tr_read();
                         if (more) fetch(next, kb + kStep, ring, 0, Keys());
                     },
                     [&]() __attribute__((always_inline)) {
                         if (more) tr_arrived<kLoads>();  // (but for the next keys)
                         else tr_arrived<0>();
                     });
                if (more) fetch(next, kb + kStep, ring, 0, Values());
                live = next.live;
            }
        }
    } else {
        // the tiles of kDeep - 1 steps are on their way; past the last key they are the last page's, not used
        constexpr int kAhead = kDeep - 1;
        static_assert(kAhead > 0, "");
        const int steps = (k1 - k0 + kStep - 1) / kStep;
        const bool idle = m0 >= rows;
        uint32_t live[kAhead];
        load_q();
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const Pages s = pages_at(first + i * kStep);
            fetch(s, first + i * kStep, ring + i * 2 * kTile, wm, Both());
            live[i] = s.live;
        }
        q_here();
        char *tile = ring, *free = ring + kAhead * 2 * kTile;
        for (int i = 0, kb = first; i < steps; ++i, kb += kStep) {
            tr_arrived<(kAhead - 1) * kMine>();
            tr_meet();  // (this step's tiles are whole, and the last one's have been read)
            const Pages s = pages_at(kb + kAhead * kStep);
            fetch(s, kb + kAhead * kStep, free, wm, Both());
            if (kb < k1 && !idle) step(kb, live[0], tile, []() {}, []() {});
#pragma unroll
            for (int j = 0; j + 1 < kAhead; ++j) live[j] = live[j + 1];
            live[kAhead - 1] = s.live;
            free = tile;
            tile = tile == ring + kAhead * 2 * kTile ? ring : tile + 2 * kTile;
        }
    }
    tr_arrived<0>();  // (what lands in LDS lands before it is used for something else)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        sum[mt] += tr_xor(sum[mt], 16);
        sum[mt] += tr_xor(sum[mt], 32);
        if (ref[mt] == -kTrInf) ref[mt] = far_ref(mt);
    }

    // the waves, joined by halves, where their tiles were
    float* const merge = reinterpret_cast<float*>(lds);
    auto give = [&](int half) __attribute__((always_inline)) {
        __syncthreads();
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
    if (WK > 4) give(4);
    if (WK > 2) give(2);
    if (WK > 1) give(1);
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
                a.stat[2 * rec] = sum[mt] == sum[mt] ? ref[mt] : sum[mt];  // (a NaN without a reference counts in the join)
                a.stat[2 * rec + 1] = sum[mt];
            }
        }
    }
}

// A workgroup's rows: up to 16 MT for each of WIDE groups of its waves, which share them as its request has them.
template <typename T, int D, int MT, int WAVES, int WIDE>
__global__ __launch_bounds__(64 * WAVES, tr_waves(D, WAVES)) void tree_kernel(TreeArgs a) {
    constexpr int kThreads = 64 * WAVES, kRows = 16 * MT * WIDE;
    __shared__ __align__(1024) char lds[tr_lds(D, MT, WAVES)];
    __shared__ float far[16 * MT * WAVES];
    // workgroups of the same keys lie eight apart, on one chiplet
    const int per = 8 * a.blocks, item = (blockIdx.x / per) * 8 + (blockIdx.x & 7), mb = (blockIdx.x % per) >> 3;
    const int bs = item / a.c.heads, h = item - bs * a.c.heads, split = bs % a.splits;
    int b = bs / a.splits;
    if (b >= a.B) return;
    TrBounds o;
    if (a.longest_first) {
        // the workgroups that start last would leave most of the chip idle if theirs were the longest requests
        int* const lens = reinterpret_cast<int*>(lds);
        const int t = threadIdx.x;
        int mine = -1;
        if (t < a.B) mine = tr_bounds(a, t, &o) ? o.len : 0;
        lens[t] = mine;
        __syncthreads();
        int before = 0;
        for (int i = 0; i < a.B; ++i) before += lens[i] > mine || (lens[i] == mine && i < t) ? 1 : 0;
        if (t < a.B && before == b) lens[kThreads] = t;
        __syncthreads();
        b = __builtin_amdgcn_readfirstlane(lens[kThreads]);
        __syncthreads();
    }
    if (!tr_bounds(a, b, &o)) return;
    const int m0 = mb * kRows, rows = o.n * a.group - m0;
    if (rows <= 0 || (split * a.chunk >= o.len && split > 0)) return;
    if constexpr (WIDE == 8) {
        if (rows > 4 * 16 * MT) tree_rows<T, D, MT, WAVES, 8>(a, o, b, h, split, m0, lds, far);
        else tree_rows<T, D, MT, WAVES, 4>(a, o, b, h, split, m0, lds, far);
    } else if constexpr (WIDE == 4) {
        if (rows > 2 * 16 * MT) tree_rows<T, D, MT, WAVES, 4>(a, o, b, h, split, m0, lds, far);
        else if (rows > 16 * MT) tree_rows<T, D, MT, WAVES, 2>(a, o, b, h, split, m0, lds, far);
        else tree_rows<T, D, MT, WAVES, 1>(a, o, b, h, split, m0, lds, far);
    } else {
        if (MT == 1 || rows <= 16) tree_rows<T, D, 1, WAVES, 1>(a, o, b, h, split, m0, lds, far);
        else tree_rows<T, D, MT, WAVES, 1>(a, o, b, h, split, m0, lds, far);
    }
}

// Joins the parts of a request's rows, 16 bytes of a part's row a lane: D / 4 lanes a row, as many rows of a
// request's key head as a workgroup has room for.  Latency: 4.0 us for 5 parts of 48 rows, 5.8 for 10 of 64.  A launch of its own: the
// parts of 128 rows are too much for the workgroup that would come last; those of 32 and fewer, where it is a quarter of the
// time, would not be, and take it too.
template <typename T, int D>
__global__ __launch_bounds__(kTrThreads) void tree_join_kernel(TreeArgs a) {
    typedef TrElem<T> E;
    constexpr int kLanes = D / 4, kRows = kTrThreads / kLanes;
    const int tid = threadIdx.x, groups = (a.max_nodes * a.group + kRows - 1) / kRows;
    const int bh = blockIdx.x / groups, b = bh / a.c.heads, h = bh - b * a.c.heads;
    const int m = (blockIdx.x - bh * groups) * kRows + tid / kLanes, d = 4 * (tid % kLanes);
    TrBounds o;
    if (tid >= kRows * kLanes || !tr_bounds(a, b, &o) || m >= o.n * a.group) return;
    const int parts = max(1, (o.len + a.chunk - 1) / a.chunk);
    const int64_t pitch = (int64_t)a.c.heads * a.rows, first = (int64_t)b * a.splits * pitch + (int64_t)h * a.rows + m;
    // a running reference, eight parts' loads in flight
    constexpr int U = 8;
    float top = -kTrInf, total = 0.0f;
    TrF4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i0 = 0; i0 < parts; i0 += U) {
        TrF4 x[U];
        float r[U], s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t rec = first + min(i0 + u, parts - 1) * pitch;
            r[u] = a.stat[2 * rec];
            s[u] = a.stat[2 * rec + 1];
            x[u] = *reinterpret_cast<const TrF4*>(a.part + rec * D + d);
        }
        float m1 = top;
#pragma unroll
        for (int u = 0; u < U; ++u) m1 = __builtin_fmaxf(m1, i0 + u < parts ? r[u] : -kTrInf);
        const float z = m1 == -kTrInf ? 0.0f : m1, f = tr_exp2(top - z);
        top = m1;
        total *= f;
        v *= f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            // (of weight 0 too: a value that is no number counts whatever its weight)
            const bool in = i0 + u < parts;
            const float w = in ? tr_exp2(r[u] - z) : 0.0f;
            total += (in ? s[u] : 0.0f) * w;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += (in ? x[u][j] : 0.0f) * w;
        }
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    const int node = m / a.group;
    typedef uint32_t U2 __attribute__((ext_vector_type(2), aligned(2)));
    U2 w;
    w[0] = E::pack(v[0] * inv, v[1] * inv);
    w[1] = E::pack(v[2] * inv, v[3] * inv);
    *reinterpret_cast<U2*>(a.out + (int64_t)(o.t0 + node) * a.ots + (int64_t)(h * a.group + m - node * a.group) * a.ohs + d) = w;
}

#define VWS_TREE(T, D)                                            \
    template __global__ void tree_kernel<T, D, 1, 4, 1>(TreeArgs); \
    template __global__ void tree_join_kernel<T, D>(TreeArgs);
#define VWS_TREE_128(T, D)                                           \
    VWS_TREE(T, D)                                                    \
    template __global__ void tree_kernel<T, D, 2, 4, 1>(TreeArgs);    \
    template __global__ void tree_kernel<T, D, 2, 8, 4>(TreeArgs);
// (past 128 dimensions two tiles do not fit the registers, nor eight steps the LDS)
#define VWS_TREE_256(T, D)                                           \
    VWS_TREE(T, D)                                                    \
    template __global__ void tree_kernel<T, D, 1, 8, 8>(TreeArgs);
#define VWS_TREES(T)                                                     \
    VWS_TREE_128(T, 64) VWS_TREE_128(T, 96) VWS_TREE_128(T, 128)          \
    VWS_TREE_256(T, 192) VWS_TREE_256(T, 256)

}  // namespace vws
