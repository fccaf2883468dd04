// The attention of one new token over the paged cache: the kernel, instantiated per type by wt_kv_attend_*.hip.
#pragma once
#include "wt_kv.h"

namespace wt {

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float fl2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr float KV_LOWEST = -3.402823466e38f;   // the running maximum's start: finite, so x - m is never inf - inf
constexpr float KV_LOG2E = 1.44269504088896340736f;

// CT: what the pages hold; T: queries and results.
// Matrix instructions take 16-bit operands as they are; 8-bit codes become bf16 (exactly), and then the queries are split
// into bf16 parts whose sum they are: bf16 1, f16 2, f32 3.  f32 pages use the f32 instruction.
template <typename CT, typename T, int HD>
struct KvKind {
    static constexpr bool F32 = sizeof(CT) == 4, E4M3 = sizeof(CT) == 1;
    static constexpr bool F16 = !F32 && !E4M3 && __is_same(CT, f16_t);
    static constexpr int KB = F32 ? 16 : 32;                // keys a wave takes at a time
    static constexpr int NT = KB / 16;                      // ... in tiles of 16
    static constexpr int GK = KB / 4;                       // keys a lane group holds the weights and values of
    static constexpr int QP = !E4M3 ? 1 : __is_same(T, bf16_t) ? 1 : __is_same(T, f16_t) ? 2 : 3;
    // The second product is one of bf16 operands for every page type but f32: a weight is the sum of WP bf16 numbers (as many bits as results
    // hold, and 5 more at least), an f16 value of two, exactly; a bf16 value and an 8-bit code are one
    static constexpr int WP = sizeof(T) == 4 ? 3 : 2, VP = F16 ? 2 : 1;
    static constexpr float SLACK = 8.f;   // by what the running maximum may be outgrown before it moves
};

// d index of the first of the 8 (f32: 4) elements that lane group g takes of contraction step s; K and Q use the same one.
// 8-bit pages: two steps of a full 64 share one 16-byte load.
template <typename CT, int HD>
__device__ __forceinline__ constexpr int kv_d(int s, int g) {
    if (sizeof(CT) == 4) return s * 16 + g * 4;
    if (sizeof(CT) == 1 && (s / 2 + 1) * 64 <= HD) return s / 2 * 64 + g * 16 + (s & 1) * 8;
    return s * 32 + g * 8;
}

template <typename CT, typename T, int HD>
struct KvFrag {
    using K = KvKind<CT, T, HD>;
    static constexpr int STEPS = HD / (K::F32 ? 16 : 32), EV = HD / 16;
    static constexpr int KD = K::E4M3 ? 2 : 4;                                       // dwords a step and tile
    static constexpr int VD = (EV * (int)sizeof(CT) + 3) / 4;                        // dwords of a key's values
    uint32_t k[K::NT][STEPS][KD];
    uint32_t v[K::GK][VD];
    uint2 ke, ve;   // 8-bit pages: exponents of the lane group's 8 keys (keys by themselves, PG 1: in .x that of key lane % 32)
};

// N bytes from a place aligned to as many of them as a power of two allows (16 at most).  Non-temporal: keys and values are
// read once; with it long calls stream at 6.57 instead of 5.67 TB/s (bf16, 128 values), 7.41 instead of 6.32 (f16, 64).
template <int N>
__device__ __forceinline__ void kv_fetch(uint32_t *dst, const char *src) {
    if constexpr (N == 2) dst[0] = *reinterpret_cast<const uint16_t *>(src);
    else if constexpr (N == 6) {
        const uint16_t *s = reinterpret_cast<const uint16_t *>(src);
        dst[0] = s[0] | (uint32_t)s[1] << 16, dst[1] = s[2];
    } else if constexpr (N <= 16 || N == 24) {
        constexpr int D = N / 4;
        typedef uint32_t V __attribute__((ext_vector_type(D < 2 ? 2 : D)));
        if constexpr (D == 4 || D == 2) {
            const V p = __builtin_nontemporal_load(reinterpret_cast<const V *>(src));
#pragma unroll
            for (int i = 0; i < D; ++i) dst[i] = p[i];
        } else {
            using P = Pack<uint32_t, D>;
            const P p = *reinterpret_cast<const P *>(src);
#pragma unroll
            for (int i = 0; i < D; ++i) dst[i] = p.v[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N / 16; ++i) kv_fetch<16>(dst + 4 * i, src + 16 * i);
    }
}

// Where a block's rows are, for this lane: byte offsets from the tensors' starts.
//   PG 32: a page size that the block divides: the block is in one page, the offsets the wave's
//   PG  8: one that a lane group's GK keys (8, f32 4) divide: each group is in one page
//   PG  1: any other: each key by itself
template <int PG, int NT, int GK>
struct KvSpot {
    int64_t k[PG == 1 ? NT : 1], v[PG == 1 ? GK : 1];
    int64_t e[1];
};

// A wave's share of one (sequence, key head, tile of 16 * QT queries)
template <typename CT, typename T, int HD, int PG, int NW, int QT>
struct KvWave {
    using K = KvKind<CT, T, HD>;
    using Frag = KvFrag<CT, T, HD>;
    using Spot = KvSpot<PG, K::NT, K::GK>;
    static constexpr int STEPS = Frag::STEPS, EV = Frag::EV, ITEM = sizeof(CT);

    const KvAttend &a;
    const int lane, g, n;
    const int32_t *row;   // the sequence's row of the table
    int len, h;
    bool bad = false;
    uint32_t koff, voff;  // PG 32: this lane's byte offsets inside a page
    // queries
    u4 q[QT][K::F32 ? 1 : K::QP][K::F32 ? 1 : STEPS];
    f4 qf[QT][K::F32 ? STEPS : 1];
    // state
    f4 o[QT][EV];
    float m[QT], l[QT];

    __device__ __forceinline__ KvWave(const KvAttend &args) : a(args), lane(threadIdx.x & 63), g((threadIdx.x & 63) >> 4), n(threadIdx.x & 15) {}

    // table entries of the block at p0 (the wave's, or this lane's for its K and V rows)
    struct Ids {
        int k, v;
    };
    __device__ __forceinline__ int kkey(int t) const { return (n >> 2) * K::GK + t * 4 + (n & 3); }
    __device__ __forceinline__ Ids ids(int p0) const { return ids(p0, len); }
    __device__ __forceinline__ Ids ids(int p0, int len) const {
        Ids id;
        if constexpr (PG == 32) {
            id.k = id.v = row[__builtin_amdgcn_readfirstlane((int)page_of(a.c.div, (uint32_t)min(p0, len - 1)))];
        } else if constexpr (PG == 8) {
            id.k = row[page_of(a.c.div, (uint32_t)min(p0 + (n >> 2) * K::GK, len - 1))];
            id.v = row[page_of(a.c.div, (uint32_t)min(p0 + g * K::GK, len - 1))];
        } else {
            id.k = id.v = row[page_of(a.c.div, (uint32_t)min(p0 + (lane & (K::KB - 1)), len - 1))];
        }
        return id;
    }
    __device__ __forceinline__ int checked(int page, bool *wrong) const {
        const bool w = (uint32_t)page >= (uint32_t)a.c.n_pages;
        *wrong |= w;
        return w ? 0 : page;
    }
    __device__ __forceinline__ void place(int p0, const Ids &id, Spot &s) {
        if constexpr (PG == 32) {
            const int page = checked(__builtin_amdgcn_readfirstlane(id.k), &bad);
            const int slot = p0 - (int)(page_of(a.c.div, (uint32_t)p0) * a.c.div.d);
            s.k[0] = (page * a.k.page + h * a.k.head + slot * a.k.slot) * ITEM;
            s.v[0] = (page * a.v.page + h * a.v.head + slot * a.v.slot) * ITEM;
            s.e[0] = ((int64_t)page * a.c.n_heads + h) * a.c.page_size + slot;
        } else if constexpr (PG == 8) {
            const int last = (len - 1) & -K::GK;
            const int pk = min(p0 + (n >> 2) * K::GK, last), pv = min(p0 + g * K::GK, last);
            const int page_k = checked(id.k, &bad), page_v = checked(id.v, &bad);
            const int slot_k = pk - (int)(page_of(a.c.div, (uint32_t)pk) * a.c.div.d) + (n & 3);
            const int slot_v = pv - (int)(page_of(a.c.div, (uint32_t)pv) * a.c.div.d);
            s.k[0] = (page_k * a.k.page + h * a.k.head + slot_k * a.k.slot + kv_d<CT, HD>(0, g)) * ITEM;
            s.v[0] = (page_v * a.v.page + h * a.v.head + slot_v * a.v.slot + n * EV) * ITEM;
            s.e[0] = ((int64_t)page_v * a.c.n_heads + h) * a.c.page_size + slot_v;
        } else {
            const int p = min(p0 + (lane & (K::KB - 1)), len - 1);
            const int page = checked(id.k, &bad);
            const int slot = p - (int)(page_of(a.c.div, (uint32_t)p) * a.c.div.d);
            const int64_t kk = (page * a.k.page + h * a.k.head + slot * a.k.slot) * ITEM, vv = (page * a.v.page + h * a.v.head + slot * a.v.slot) * ITEM;
            s.e[0] = ((int64_t)page * a.c.n_heads + h) * a.c.page_size + slot;
#pragma unroll
            for (int t = 0; t < K::NT; ++t) s.k[t] = shfl64(kk, kkey(t)) + kv_d<CT, HD>(0, g) * ITEM;
#pragma unroll
            for (int j = 0; j < K::GK; ++j) s.v[j] = shfl64(vv, g * K::GK + j) + n * EV * ITEM;
        }
    }
    static __device__ __forceinline__ int64_t shfl64(int64_t v, int src) {
        const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)v, src, 64), hi = (uint32_t)__shfl((int)(uint32_t)(v >> 32), src, 64);
        return (int64_t)((uint64_t)hi << 32 | lo);
    }

    __device__ __forceinline__ void fetch(Frag &f, const Spot &s) const {
        const char *kp = static_cast<const char *>(a.k.p), *vp = static_cast<const char *>(a.v.p);
#pragma unroll
        for (int t = 0; t < K::NT; ++t) {
            const char *r;
            if constexpr (PG == 32) r = kp + s.k[0] + (uint32_t)(koff + t * 4 * (uint32_t)a.k.slot * ITEM);
            else if constexpr (PG == 8) r = kp + s.k[0] + t * 4 * a.k.slot * ITEM;
            else r = kp + s.k[t];
#pragma unroll
            for (int st = 0; st < STEPS; ++st) {
                const char *p = r + (kv_d<CT, HD>(st, 0) - kv_d<CT, HD>(0, 0)) * ITEM;
                constexpr int PAIRED = HD / 64 * 2;   // 8-bit pages: steps that share a load
                if constexpr (!K::E4M3) kv_fetch<16>(f.k[t][st], p);
                else if (st < PAIRED) {
                    if (st & 1) continue;
                    uint32_t w[4];
                    kv_fetch<16>(w, p);
                    f.k[t][st][0] = w[0], f.k[t][st][1] = w[1], f.k[t][st + 1][0] = w[2], f.k[t][st + 1][1] = w[3];
                } else   // (behind the last full 64 the lane groups are 8 apart instead of 16)
                    kv_fetch<8>(f.k[t][st], p + (kv_d<CT, HD>(st, g) - kv_d<CT, HD>(st, 0) - kv_d<CT, HD>(0, g)) * ITEM);
            }
        }
#pragma unroll
        for (int j = 0; j < K::GK; ++j) {
            const char *r;
            if constexpr (PG == 32) r = vp + s.v[0] + (uint32_t)(voff + j * (uint32_t)a.v.slot * ITEM);
            else if constexpr (PG == 8) r = vp + s.v[0] + j * a.v.slot * ITEM;
            else r = vp + s.v[j];
            kv_fetch<EV * ITEM>(f.v[j], r);
        }
        if constexpr (K::E4M3) {
            if constexpr (PG == 1) {
                f.ke.x = a.k.e[s.e[0]], f.ve.x = a.v.e[s.e[0]];
            } else {
                const int64_t e = s.e[0] + (PG == 32 ? g * 8 : 0);
                f.ke = *reinterpret_cast<const uint2 *>(a.k.e + e), f.ve = *reinterpret_cast<const uint2 *>(a.v.e + e);
            }
        }
    }

    static __device__ __forceinline__ f4 mma_bf16(u4 x, u4 y, f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, x), __builtin_bit_cast(bf8, y), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f4 mma(u4 x, u4 y, f4 c) {   // of operands as pages and queries hold them
        if constexpr (K::F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, x), __builtin_bit_cast(h8, y), c, 0, 0, 0);
        else return mma_bf16(x, y, c);
    }
    static __device__ __forceinline__ uint32_t codes(uint32_t w, bool high) {   // two 8-bit codes as bf16
        return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.f, true))
                    : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.f, false));
    }
    // the next bf16 part of two numbers, which become what is left of them
    static __device__ __forceinline__ uint32_t part(float &x, float &y) {
        const fl2 v = {x, y};
        const uint32_t w = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf2));
        x -= __uint_as_float(w << 16), y -= __uint_as_float(w & 0xffff0000u);
        return w;
    }

    // One block of KB keys.  Scores as (keys x queries) tiles: A rows are keys, chosen so that lane group g gets keys g * GK
    // ... + GK - 1 of its query (column n) in order; they are, without leaving the lane, the B operand of (values^T x
    // weights), whose contraction slots are numbered alike.
    __device__ __forceinline__ void block(Frag &f, int p0) {
        constexpr int GK = K::GK;
        float x[QT][GK];
#pragma unroll
        for (int t = 0; t < K::NT; ++t) {
            f4 s[QT];
#pragma unroll
            for (int y = 0; y < QT; ++y) s[y] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < STEPS; ++st) {
                if constexpr (K::F32) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int y = 0; y < QT; ++y) s[y] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(f.k[t][st][i]), qf[y][st][i], s[y], 0, 0, 0);
                } else {
                    u4 w;
                    if constexpr (K::E4M3)
                        w = u4{codes(f.k[t][st][0], false), codes(f.k[t][st][0], true), codes(f.k[t][st][1], false), codes(f.k[t][st][1], true)};
                    else w = u4{f.k[t][st][0], f.k[t][st][1], f.k[t][st][2], f.k[t][st][3]};
#pragma unroll
                    for (int p = K::QP - 1; p >= 0; --p)
#pragma unroll
                        for (int y = 0; y < QT; ++y) s[y] = mma(w, q[y][p][st], s[y]);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int y = 0; y < QT; ++y) x[y][t * 4 + r] = s[y][r];
        }
        // PG 1: exponents of key and value, each from the lane that has them (16 sequences of 4000 ... 12000 positions, 8 heads of 128, pages
        // of 100: 56 us; 75 with a load of a byte for every key of the lane group)
        uint32_t both[PG == 1 && K::E4M3 ? 8 : 1];
        if constexpr (K::E4M3) {
            if constexpr (PG == 1) {
#pragma unroll
                for (int j = 0; j < 8; ++j) both[j] = (uint32_t)__shfl((int)(f.ke.x | f.ve.x << 8), g * 8 + j, 64);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float e = exp_of((PG == 1 ? both[PG == 1 ? j : 0] : (j < 4 ? f.ke.x : f.ke.y) >> (j % 4 * 8)) & 255u);
#pragma unroll
                for (int y = 0; y < QT; ++y) x[y][j] *= e;
            }
        }
#pragma unroll
        for (int y = 0; y < QT; ++y)
#pragma unroll
            for (int j = 0; j < GK; ++j) x[y][j] *= a.scale;
        uint32_t off = 0;   // keys of this lane group behind the end
        if (p0 + K::KB > len) {
#pragma unroll
            for (int j = 0; j < GK; ++j)
                if (p0 + g * GK + j >= len) {
                    off |= 1u << j;
#pragma unroll
                    for (int y = 0; y < QT; ++y) x[y][j] = -__builtin_inff();
#pragma unroll
                    for (int i = 0; i < Frag::VD; ++i) f.v[j][i] = 0;
                }
        }
        float p[QT][GK];
#pragma unroll
        for (int y = 0; y < QT; ++y) {
            float top = x[y][0];
#pragma unroll
            for (int j = 1; j < GK; ++j) top = fmaxf(top, x[y][j]);
            if (__any(top > m[y] + K::SLACK)) {   // rare once the maximum is found: the reference moves, all sums with it
                top = fmaxf(top, __shfl_xor(top, 16, 64));
                top = fmaxf(top, __shfl_xor(top, 32, 64));
                const float mn = fmaxf(m[y], top), c = __builtin_amdgcn_exp2f((m[y] - mn) * KV_LOG2E);
                m[y] = mn;
                l[y] *= c;
#pragma unroll
                for (int i = 0; i < EV; ++i) o[y][i] *= c;
            }
#pragma unroll
            for (int j = 0; j < GK; ++j) p[y][j] = __builtin_amdgcn_exp2f((x[y][j] - m[y]) * KV_LOG2E);
#pragma unroll
            for (int j = 0; j < GK; ++j) l[y] += p[y][j];
        }
        if constexpr (K::E4M3) {   // the value's power of two goes into its weight
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float e = exp_of((PG == 1 ? both[PG == 1 ? j : 0] >> 8 : (j < 4 ? f.ve.x : f.ve.y) >> (j % 4 * 8)) & 255u);
#pragma unroll
                for (int y = 0; y < QT; ++y) p[y][j] *= off >> j & 1 ? 0.f : e;
            }
        }
        if constexpr (K::F32) {
#pragma unroll
            for (int j = 0; j < GK; ++j)
#pragma unroll
                for (int i = 0; i < EV; ++i)
#pragma unroll
                    for (int y = 0; y < QT; ++y) o[y][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(f.v[j][i]), p[y][j], o[y][i], 0, 0, 0);
        } else {
            // With one bf16 number for a weight a result is off by up to 2^-8 where few keys share the weight, with two by 2^-17, which 16-bit
            // results do not show; f32 results (over 8-bit pages) take three, all 24 bits.  f16 weights would spare the splitting of f16 values (32
            // sequences of 1500, 20 heads of 64: 46.4 instead of 48.2 us; 447 keys of 8 heads: 6.0 instead of 6.9; 4000 keys of 32 values: 35
            // instead of 42), but they lose bits from e^-12 of the largest weight on: a key's weight of e^-20 was off by 6 %.
            // Values arrive as rows (key j: EV neighbouring columns a lane) and are needed as columns: 16-bit pairs of rows are
            // interleaved by byte permutes, f16 ones as they are split.
            u4 weight[QT][K::WP];
#pragma unroll
            for (int y = 0; y < QT; ++y)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float w0 = p[y][2 * i], w1 = p[y][2 * i + 1];
#pragma unroll
                    for (int n = 0; n < K::WP; ++n) weight[y][n][i] = part(w0, w1);
                }
            uint32_t w[8][EV / 2];
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int i = 0; i < EV / 2; ++i) {
                    if constexpr (K::E4M3) w[j][i] = codes(f.v[j][i / 2], i & 1);
                    else w[j][i] = f.v[j][i];
                }
#pragma unroll
            for (int i = 0; i < EV; ++i) {
                // (columns in turn: registers for one more wave a SIMD; 128 short tables of 8 bits, f32: 12.8 -> 12.3 us)
                if constexpr (K::F16 || K::WP > 2) __builtin_amdgcn_sched_barrier(0);
                u4 vt[K::VP];
#pragma unroll
                for (int jj = 0; jj < 4; ++jj) {
                    const uint32_t w0 = w[2 * jj][i / 2], w1 = w[2 * jj + 1][i / 2];
                    if constexpr (K::F16) {
                        float v0 = (float)__builtin_bit_cast(h2, w0)[i & 1], v1 = (float)__builtin_bit_cast(h2, w1)[i & 1];
#pragma unroll
                        for (int n = 0; n < K::VP; ++n) vt[n][jj] = part(v0, v1);
                    } else
                        vt[0][jj] = __builtin_amdgcn_perm(w1, w0, i & 1 ? 0x07060302u : 0x05040100u);
                }
#pragma unroll
                for (int n = K::WP + K::VP - 2; n >= 0; --n)   // the small products first; that of both last parts is 2^-18 of the largest
#pragma unroll
                    for (int h = 0; h < K::VP; ++h)
                        if (n - h >= 0 && n - h < K::WP && !(h > 0 && n - h == K::WP - 1))
#pragma unroll
                            for (int y = 0; y < QT; ++y) o[y][i] = mma_bf16(vt[h], weight[y][n - h], o[y][i]);
            }
        }
    }

    // the queries in two steps, so that the first block's loads are on their way before the conversion waits
    static constexpr int QE = K::F32 ? 4 : 8;
    struct Raw {
        Pack<T, QE> p[QT][STEPS];
    };
    __device__ __forceinline__ void queries_load(Raw &raw, int s, int hq0, int rows) const {
#pragma unroll
        for (int y = 0; y < QT; ++y) {
            const T *src = static_cast<const T *>(a.q) + s * a.q_row + (hq0 + min(y * 16 + n, rows - 1)) * a.q_head;
#pragma unroll
            for (int st = 0; st < STEPS; ++st) {
                const int d = kv_d<CT, HD>(st, g);
                if (a.q_aligned) raw.p[y][st] = *reinterpret_cast<const Pack<T, QE> *>(src + d);
                else {
#pragma unroll
                    for (int i = 0; i < QE; ++i) raw.p[y][st].v[i] = src[d + i];
                }
            }
        }
    }
    __device__ __forceinline__ void queries_take(const Raw &raw, int rows) {   // columns without a query are zeros
#pragma unroll
        for (int y = 0; y < QT; ++y) {
            const bool in = y * 16 + n < rows;
#pragma unroll
            for (int st = 0; st < STEPS; ++st) {
                if constexpr (K::F32) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) qf[y][st][i] = in ? raw.p[y][st].v[i] : 0.f;
                } else if constexpr (K::QP == 1) {
                    const u4 w = __builtin_bit_cast(u4, raw.p[y][st]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) q[y][0][st][i] = in ? w[i] : 0u;
                } else {
                    float v[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = in ? to_f(raw.p[y][st].v[i]) : 0.f;
#pragma unroll
                    for (int p = 0; p < K::QP; ++p)
#pragma unroll
                        for (int i = 0; i < 4; ++i) q[y][p][st][i] = part(v[2 * i], v[2 * i + 1]);
                }
            }
        }
    }

    // blocks b, b + NW, ... < end of this sequence and head; two sets of registers, the next block's loads always in
    // flight.  `first`: table entries of block b, loaded before the length was known (and not clamped to it).
    __device__ __forceinline__ void run(int b, int end, Ids first, const Raw &raw, int rows) {
#pragma unroll
        for (int y = 0; y < QT; ++y) {
            m[y] = KV_LOWEST, l[y] = 0.f;
#pragma unroll
            for (int i = 0; i < EV; ++i) o[y][i] = f4{0.f, 0.f, 0.f, 0.f};
        }
        if (b >= end) return;
        if constexpr (PG == 32) {
            koff = (uint32_t)(kkey(0) * (uint32_t)a.k.slot + kv_d<CT, HD>(0, g)) * ITEM;
            voff = (uint32_t)(g * K::GK * (uint32_t)a.v.slot + n * EV) * ITEM;
        }
        // (a block behind the last one is the last one again: its loads hit the cache and its numbers are not used)
        const auto next = [&](int x) { return x + NW < end ? x + NW : x; };
        if (PG != 32 && (b + 1) * K::KB > len) first = ids(b * K::KB);
        Frag f[2];
        Spot sp;
        place(b * K::KB, first, sp);
        int nb = next(b);
        Ids id = ids(nb * K::KB);
        fetch(f[0], sp);
        queries_take(raw, rows);
        while (true) {
            place(nb * K::KB, id, sp);
            int n2 = next(nb);
            id = ids(n2 * K::KB);
            fetch(f[1], sp);
            block(f[0], b * K::KB);
            if (nb == b) break;
            b = nb, nb = n2;
            place(nb * K::KB, id, sp);
            n2 = next(nb);
            id = ids(n2 * K::KB);
            fetch(f[0], sp);
            block(f[1], b * K::KB);
            if (nb == b) break;
            b = nb, nb = n2;
        }
    }
};

__device__ __forceinline__ int64_t kv_capacity(const KvAttend &a) { return (int64_t)a.t.width * a.c.page_size; }
__device__ __forceinline__ int kv_length(const KvAttend &a, int raw, bool *wrong) {   // a length outside of the table counts as zero, its results as NaN
    *wrong = raw < 0 || raw > kv_capacity(a);
    return *wrong ? 0 : raw;
}
__device__ __forceinline__ uint32_t kv_div(uint64_t x, uint64_t y) {   // where the quotient fits 32 bits (a share that does not is hours of work); the wave's operands
    return ((x | y) >> 32) == 0 ? (uint32_t)x / (uint32_t)y : (uint32_t)(x / y);
}

// Partial results travel between workgroups, which may run on different XCDs with an L2 each: stored through to memory and
// loaded from there (the agent's scope in the instruction itself).  Fences of that scope around plain stores write back and
// invalidate whole L2s: with them, 131071 positions took 246 us instead of 171.
constexpr int KV_AGENT = 16;
template <int HD, int QT>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t kv_partials(const KvAttend &a) {
    return __builtin_amdgcn_make_buffer_rsrc(a.partials, 0, a.n_wg * 2 * kv_slot(HD, QT) * 4, 0x00020000);
}
__device__ __forceinline__ void kv_put(__amdgpu_buffer_rsrc_t p, int at, float v) { __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), p, at * 4, 0, KV_AGENT); }
__device__ __forceinline__ void kv_put(__amdgpu_buffer_rsrc_t p, int at, f4 v) { __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, v), p, at * 4, 0, KV_AGENT); }
__device__ __forceinline__ float kv_get(__amdgpu_buffer_rsrc_t p, int at) { return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(p, at * 4, 0, KV_AGENT)); }
__device__ __forceinline__ f4 kv_get4(__amdgpu_buffer_rsrc_t p, int at) { return __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(p, at * 4, 0, KV_AGENT)); }

template <typename T>
__device__ __forceinline__ void kv_result(const KvAttend &a, int s, int head, int d, f4 v) {
    T *dst = static_cast<T *>(a.out) + s * a.o_row + head * a.o_head + d;
    Pack<T, 4> out;
#pragma unroll
    for (int x = 0; x < 4; ++x) out.v[x] = from_f<T>(v[x]);
    if (a.o_aligned) *reinterpret_cast<Pack<T, 4> *>(dst) = out;
    else {
#pragma unroll
        for (int x = 0; x < 4; ++x) dst[x] = out.v[x];
    }
}

// One workgroup's part of one (sequence, key head, query tile): blocks [b0, b1).  What the waves found is joined in LDS and
// goes out as the result, or as a partial one (slot >= 0).  LATE: the length is not known yet (all blocks are meant then):
// queries and first table entries are loaded beside it.
template <bool LATE, typename CT, typename T, int HD, int PG, int NW, int QT>
__device__ __forceinline__ void kv_segment(KvWave<CT, T, HD, PG, NW, QT> &w, const KvAttend &a, float *lds, int s, int pair, int len, bool bad_len,
                                           int b0, int b1, int slot) {
    constexpr int EV = HD / 16, KB = KvKind<CT, T, HD>::KB, R = 16 * QT;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = pair / a.q_tiles, qt = pair % a.q_tiles;
    const int hq0 = h * a.group + qt * R, rows = min(R, a.group - qt * R);
    w.row = a.t.t + s * a.t.stride;
    w.h = h;
    typename KvWave<CT, T, HD, PG, NW, QT>::Raw raw;
    const int late_len = LATE ? a.lengths[s] : 0;
    const auto first = w.ids((b0 + wave) * KB, LATE ? (int)kv_capacity(a) : max(len, 1));
    w.queries_load(raw, s, hq0, rows);
    if constexpr (LATE) {
        len = __builtin_amdgcn_readfirstlane(kv_length(a, late_len, &bad_len));
        b1 = (len + KB - 1) / KB;
    }
    w.len = len;
    w.bad = bad_len;
    w.run(b0 + wave, b1, first, raw, rows);
    if (__any(w.bad) && w.lane == 0) kv_report(a.c.error, bad_len ? WT_KV_BAD_POSITION : WT_KV_BAD_PAGE);
    const bool bad = __any(w.bad);
    float *lm = lds, *ll = lds + NW * R, *lo = lds + NW * 2 * R;
#pragma unroll
    for (int y = 0; y < QT; ++y) {
        float l = bad ? __builtin_nanf("") : w.l[y];
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        const int r = y * 16 + w.n;
        if (w.lane < 16) lm[wave * R + r] = w.m[y], ll[wave * R + r] = l;
        if (r < rows) {
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int i = 0; i < EV; ++i) lo[(wave * rows + r) * HD + (4 * w.g + x) * EV + i] = w.o[y][i][x];
        }
    }
    __syncthreads();
    const __amdgpu_buffer_rsrc_t part = kv_partials<HD, QT>(a);
    const int at = slot * kv_slot(HD, QT);
    for (int e = threadIdx.x; e < rows * (HD / 4); e += NW * 64) {
        const int r = e / (HD / 4), d = e % (HD / 4) * 4;
        float mm = lm[r];
#pragma unroll
        for (int i = 1; i < NW; ++i) mm = fmaxf(mm, lm[i * R + r]);
        f4 acc = {0.f, 0.f, 0.f, 0.f};
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            const float c = __builtin_amdgcn_exp2f((lm[i * R + r] - mm) * KV_LOG2E);
            const f4 x = *reinterpret_cast<const f4 *>(&lo[(i * rows + r) * HD + d]);
#pragma unroll
            for (int y = 0; y < 4; ++y) acc[y] = fmaf(x[y], c, acc[y]);
            sum = fmaf(ll[i * R + r], c, sum);
        }
        if (slot >= 0) {
            kv_put(part, at + 4 * R + e * 4, acc);
            if (d == 0) kv_put(part, at + r, mm), kv_put(part, at + R + r, sum);
        } else {
            const bool empty = len == 0 && !bad_len;
#pragma unroll
            for (int y = 0; y < 4; ++y) acc[y] = empty ? 0.f : acc[y] / sum;
            kv_result<T>(a, s, hq0 + r, d, acc);
            if (a.lse && d == 0) a.lse[(int64_t)s * a.n_q_heads + hq0 + r] = empty ? -__builtin_inff() : mm + logf(sum);
        }
    }
}

// The last workgroup of a pair to arrive joins its partial results.  A thread takes four columns of a row, and where there
// are more threads than that and more than KV_JOIN parts, every LANES-th part; KV_JOIN parts are loaded at a time, in an order
// that never changes.  One workgroup reads partial results at some 48 GB/s, so with more than two KV_GROUPs of parts the last of
// each group joins the group, and the last of those the groups, and so on (90 parts of 8 queries of 256 values: 30 us by one
// workgroup alone; 24 queries of 128 values over 24000 and 48000 positions of 8 heads, groups of 16 / 8: 36.3 / 33.6, 54.2 / 51.4 us).
template <int QT>
constexpr int KV_GROUP = QT == 2 ? 8 : 16;

// parts first, first + step, ... (count of them; number i stands in slot_of(i), its maxima and sums `stats` floats into it) ->
// the result, or one part, in the slot of `first`, its maxima and sums in the second place for them
template <typename T, int HD, int NW, int QT, typename SlotOf>
__device__ __forceinline__ void kv_reduce(const KvAttend &a, float *lds, int s, int hq0, int rows, SlotOf slot_of, int first, int step, int count,
                                          int stats, bool result) {
    constexpr int NTH = NW * 64, R = 16 * QT, SLOT = kv_slot(HD, QT);
    const __amdgpu_buffer_rsrc_t parts = kv_partials<HD, QT>(a);
    const int quads = rows * (HD / 4);
    const int lanes = kv_join_lanes(NTH, quads, count);
    for (int e0 = 0; e0 < quads; e0 += NTH / lanes) {
        const int e = e0 + threadIdx.x / lanes, mine = threadIdx.x % lanes;
        const bool in = e < quads && kv_join_grouped(threadIdx.x, lanes, NTH);
        const int r = in ? e / (HD / 4) : 0, d = in ? e % (HD / 4) * 4 : 0;
        float mm = KV_LOWEST, sum = 0.f;
        f4 acc = {0.f, 0.f, 0.f, 0.f};
        for (int i0 = mine; i0 < count; i0 += lanes * KV_JOIN) {
            float m[KV_JOIN], l[KV_JOIN];
            f4 o[KV_JOIN];
#pragma unroll
            for (int i = 0; i < KV_JOIN; ++i) {
                const bool there = i0 + i * lanes < count;
                const int p = slot_of(first + (there ? i0 + i * lanes : i0) * step) * SLOT;
                m[i] = kv_get(parts, p + stats + r), l[i] = kv_get(parts, p + stats + R + r);
                o[i] = kv_get4(parts, p + 4 * R + r * HD + d);
            }
            __builtin_amdgcn_sched_barrier(0);   // (else maxima are waited for before the last loads are on their way: 37.7 instead of 27.1 us
                                                 // for 131072 positions of one head with 16 queries)
            float mn = mm;
#pragma unroll
            for (int i = 0; i < KV_JOIN; ++i) mn = fmaxf(mn, m[i]);   // (one that stands in for a missing part changes nothing, then weighs nothing)
            const float c = __builtin_amdgcn_exp2f((mm - mn) * KV_LOG2E);
            sum *= c, acc *= c, mm = mn;
#pragma unroll
            for (int i = 0; i < KV_JOIN; ++i) {
                const bool there = i0 + i * lanes < count;
                const float w = there ? __builtin_amdgcn_exp2f((m[i] - mm) * KV_LOG2E) : 0.f;
                sum = fmaf(l[i], w, sum);
#pragma unroll
                for (int x = 0; x < 4; ++x) acc[x] = fmaf(o[i][x], w, acc[x]);
            }
        }
        if (lanes > 1) {
            float *mine_lds = lds + 6 * threadIdx.x;
            mine_lds[0] = mm, mine_lds[1] = sum;
#pragma unroll
            for (int x = 0; x < 4; ++x) mine_lds[2 + x] = acc[x];
            __syncthreads();
            if (in && mine == 0)
                for (int i = 1; i < lanes; ++i) {
                    const float *p = mine_lds + 6 * i;
                    const float mn = fmaxf(mm, p[0]);
                    const float c0 = __builtin_amdgcn_exp2f((mm - mn) * KV_LOG2E), c1 = __builtin_amdgcn_exp2f((p[0] - mn) * KV_LOG2E);
                    sum = sum * c0 + p[1] * c1;
#pragma unroll
                    for (int x = 0; x < 4; ++x) acc[x] = acc[x] * c0 + p[2 + x] * c1;
                    mm = mn;
                }
            __syncthreads();
        }
        if (in && mine == 0) {
            if (result) {
#pragma unroll
                for (int x = 0; x < 4; ++x) acc[x] /= sum;
                kv_result<T>(a, s, hq0 + r, d, acc);
                if (a.lse && d == 0) a.lse[(int64_t)s * a.n_q_heads + hq0 + r] = mm + logf(sum);
            } else {   // (only this thread reads these columns of the slot; its maxima others may still read)
                const int p = slot_of(first) * SLOT;
                kv_put(parts, p + 4 * R + r * HD + d, acc);
                if (d == 0) kv_put(parts, p + 2 * R - stats + r, mm), kv_put(parts, p + 3 * R - stats + r, sum);
            }
        }
    }
}

// Counts this workgroup's arrival, its stores being out; true in the last of `of`, which leaves the counter at zero.
__device__ __forceinline__ bool kv_last(int32_t *counter, int of, float *lds) {
    wait_vmcnt0();     // every wave's stores are where the others read them before the count
    __syncthreads();   // (and lds is free)
    int *last = reinterpret_cast<int *>(lds);
    if (threadIdx.x == 0) {
        const int before = atomicAdd(counter, 1);
        *last = before == of - 1;
        if (before == of - 1) *counter = 0;
    }
    __syncthreads();
    const bool is = *last;
    __syncthreads();   // (lds is free again)
    return is;
}

template <typename T, int HD, int NW, int QT>
__device__ __forceinline__ void kv_join(const KvAttend &a, float *lds, int s, int pair, int first_wg, int n_parts) {
    const int h = pair / a.q_tiles, qt = pair % a.q_tiles;
    constexpr int R = 16 * QT;
    const int hq0 = h * a.group + qt * R, rows = min(R, a.group - qt * R);
    // the first part stands in the slot of a segment that goes on, the others in that of one that came from before
    const auto slot_of = [&](int i) { return 2 * (first_wg + i) + (i == 0 ? 1 : 0); };
    constexpr int G = KV_GROUP<QT>;
    static_assert(2 * G * G * G >= WT_KV_WORKSPACE_ZEROED / 16, "parts of one pair: a workgroup each");
    const int i = blockIdx.x - first_wg;
    for (int level = 0, step = 1;; ++level, step *= G) {
        const int left = (n_parts + step - 1) / step;   // parts 0, step, 2 * step ... are still to be joined
        const bool result = left <= 2 * G;
        const int first = result ? 0 : i / (step * G) * G, count = result ? left : min(G, left - first);
        // counters of this pair's own: level 0 in the first half, the others in the second (those of level 1 at multiples of G * G);
        // level 2 is the last
        int32_t *counter = a.counters + (level == 0 ? 0 : 2 * a.n_wg) + slot_of(level < 2 ? first * step : 1);
        if (!kv_last(counter, count, lds)) return;
        kv_reduce<T, HD, NW, QT>(a, lds, s, hq0, rows, slot_of, first * step, step, count, level & 1 ? 2 * R : 0, result);
        if (result) return;
    }
}

// Short tables: one workgroup per (sequence, key head, query tile).  One head is bound by what a compute unit streams and by the
// chain length -> table -> keys -> joining waves (447 keys of 8 heads, f16, 64 values: 7.1 us), many by memory (32 sequences of 1500, 20
// heads: 47 us, 5.2 TB/s).
template <typename CT, typename T, int HD, int PG, int NW, int QT>
__global__ __launch_bounds__(NW * 64, HD * QT <= 128 ? 2 : 1) void kv_attend_direct_kernel(const KvAttend a) {
    extern __shared__ __attribute__((aligned(16))) float kv_lds[];
    const unsigned pairs = a.c.n_heads * a.q_tiles;
    KvWave<CT, T, HD, PG, NW, QT> w(a);
    kv_segment<true, CT, T, HD, PG, NW, QT>(w, a, kv_lds, blockIdx.x / pairs, blockIdx.x % pairs, 0, false, 0, 0, -1);
}

// Longer ones: one workgroup a compute unit, equal shares.  Bound by memory; 131071 positions of 8 heads, bf16, 128 values: 88 us (6.1
// TB/s), 16 sequences of 17 ... 32768: 61 us (5.6), 4 of 50001 ... 65537 in 8 bits: 80 us (5.9).  Two workgroups a compute unit
// progress unevenly: their ends lay between 55 and 106 us where one's lay between 76 and 99.
template <typename CT, typename T, int HD, int PG, int NW, int QT>
__global__ __launch_bounds__(NW * 64, HD * QT <= 128 ? 2 : 1) void kv_attend_kernel(const KvAttend a) {
    extern __shared__ __attribute__((aligned(16))) float kv_lds[];
    constexpr int KB = KvKind<CT, T, HD>::KB, UNIT = KB * NW;
    const int lane = threadIdx.x & 63;
    const int pairs = a.c.n_heads * a.q_tiles;   // of one sequence
    KvWave<CT, T, HD, PG, NW, QT> w(a);
    // All pairs stand in a row, sequence by sequence, each with seg_cost units for what a segment costs by itself (queries,
    // joining the waves) and then one for every NW blocks of keys; workgroup i takes the i-th share of the row.
    const int n_seqs = a.t.n_seqs, head = a.seg_cost;
    int raw = 0, base = 0;   // lengths of 64 sequences from `base` on, one a lane
    const auto load = [&](int s0) {
        base = s0;
        raw = a.lengths[min(s0 + lane, n_seqs - 1)];
    };
    const auto units = [&](int r) {
        bool wrong;
        return (kv_length(a, r, &wrong) + UNIT - 1) / UNIT;
    };
    uint64_t total = 0;
    for (int s0 = 0; s0 < n_seqs; s0 += 64) {
        load(s0);
        total += s0 + lane < n_seqs ? units(raw) + head : 0;
    }
    for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o, 64);
    total *= pairs;
    total = (uint64_t)__builtin_amdgcn_readfirstlane((int)(total >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)total);
    const uint32_t share = max((uint32_t)a.min_share, kv_div(total + a.n_wg - 1, a.n_wg));
    uint64_t u = (uint64_t)blockIdx.x * share;
    const uint64_t u_end = min(u + share, total);
    if (u >= u_end) return;
    // the sequence u falls into: prefix sums, 64 sequences at a time
    int s = 0;
    uint64_t before = 0;   // units in front of sequence s
    for (int s0 = 0; s0 < n_seqs; s0 += 64) {
        if (base != s0) load(s0);
        const uint64_t mine = s0 + lane < n_seqs ? (uint64_t)(units(raw) + head) * pairs : 0;
        uint64_t incl = mine;
        for (int o = 1; o < min(64, n_seqs); o <<= 1) {
            const uint64_t x = __shfl_up(incl, o, 64);
            incl += lane >= o ? x : 0;
        }
        const uint64_t above = __ballot(before + incl > u);
        const int first = above ? __ffsll((unsigned long long)above) - 1 : 63;
        const uint64_t add = __shfl(above ? incl - mine : incl, first, 64);
        before += (uint64_t)__builtin_amdgcn_readfirstlane((int)(add >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)add);
        if (above) {
            s = s0 + first;
            break;
        }
    }
    while (u < u_end) {
        if (s >= base + 64) load(base + 64);
        bool wrong;
        const int len = kv_length(a, __builtin_amdgcn_readlane(raw, s - base), &wrong);
        const int n = (len + UNIT - 1) / UNIT, cost = n + head;
        const int pair = (int)kv_div(u - before, cost);
        const uint64_t p0 = before + (uint64_t)pair * cost;   // the pair's first unit, and that of its keys
        const uint64_t k0 = p0 + head;
        const uint64_t stop = min(p0 + cost, u_end);
        const int from = u > k0 ? (int)(u - k0) : 0, to = stop > k0 ? (int)(stop - k0) : 0;
        if (n == 0 ? u == p0 : to > from) {   // (an empty sequence belongs to the workgroup that holds its first unit)
            const bool whole = from == 0 && to == n;
            const int slot = whole ? -1 : 2 * (int)blockIdx.x + (from == 0 ? 1 : 0);
            kv_segment<false, CT, T, HD, PG, NW, QT>(w, a, kv_lds, s, pair, len, wrong, from * NW, min(to * NW, (len + KB - 1) / KB), slot);
            if (!whole) {
                const int first_wg = (int)kv_div(k0, share), last_wg = (int)kv_div(k0 + n - 1, share);
                kv_join<T, HD, NW, QT>(a, kv_lds, s, pair, first_wg, last_wg - first_wg + 1);
            }
            __syncthreads();   // lds is free
        }
        u = stop;
        if (u >= before + (uint64_t)cost * pairs) before += (uint64_t)cost * pairs, ++s;
    }
}

template <typename CT, typename T, int HD, int PG>
static int kv_attend_go(const KvAttend &a, unsigned grid, hipStream_t st) {
    const int tile = 16 * a.q_wide, rows = a.group < tile ? a.group : tile;
    void (*kernel)(KvAttend) = !a.direct     ? kv_attend_kernel<CT, T, HD, PG, KV_WAVES, 1>
                               : a.waves == 2 ? kv_attend_direct_kernel<CT, T, HD, PG, 2, 1>
                                              : kv_attend_direct_kernel<CT, T, HD, PG, KV_WAVES, 1>;
    if constexpr (HD <= KV_WIDE_HD)
        if (a.q_wide == 2) kernel = a.direct ? kv_attend_direct_kernel<CT, T, HD, PG, KV_WAVES, 2> : kv_attend_kernel<CT, T, HD, PG, KV_WAVES, 2>;
    size_t lds = sizeof(float) * a.waves * (2 * tile + (size_t)rows * HD);
    if (!a.direct && lds < sizeof(float) * KV_WAVES * 64 * 6) lds = sizeof(float) * KV_WAVES * 64 * 6;   // what the join of partial results takes
    if (lds > 64 * 1024)   // (16 queries of 256 values, 32 of 128)
        WT_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(64 * a.waves), lds, st, a);
    WT_HIP(hipGetLastError());
    return WT_OK;
}

// page sizes: see KvSpot
template <typename CT, typename T, int HD>
static int kv_attend_pages(const KvAttend &a, unsigned grid, hipStream_t st) {
    using K = KvKind<CT, T, HD>;
    if (a.c.page_size % K::KB == 0) return kv_attend_go<CT, T, HD, 32>(a, grid, st);
    if (a.c.page_size % K::GK == 0) return kv_attend_go<CT, T, HD, 8>(a, grid, st);
    return kv_attend_go<CT, T, HD, 1>(a, grid, st);
}

template <typename CT, typename T>
static int kv_attend_widths(const KvAttend &a, unsigned grid, hipStream_t st) {
    switch (a.c.head_dim) {
        case 32: return kv_attend_pages<CT, T, 32>(a, grid, st);
        case 64: return kv_attend_pages<CT, T, 64>(a, grid, st);
        case 96: return kv_attend_pages<CT, T, 96>(a, grid, st);
        case 128: return kv_attend_pages<CT, T, 128>(a, grid, st);
        default: return kv_attend_pages<CT, T, 256>(a, grid, st);
    }
}

}  // namespace wt
