// What the paged cache's kernels share: places of positions, types, argument checks.  Layout: include/wtalign.h, wt_kv_*.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "wt_common.h"
#include "wt_kv_plan.h"

namespace wt {

// position -> (page index, slot) for any page size: q = (p * m) >> s with m = ceil(2^s / d), s = 31 + ceil(log2 d), is exact
// for 0 <= p < 2^31 and m < 2^32
struct PageDiv {
    uint32_t d, m, s;
};
inline PageDiv page_div(int d) {
    PageDiv r = {(uint32_t)d, 0, 31};
    while ((1ull << (r.s - 31)) < (uint64_t)d) ++r.s;
    r.m = (uint32_t)(((1ull << r.s) + d - 1) / d);   // d = 1: 2^31
    return r;
}
__device__ __forceinline__ uint32_t page_of(PageDiv v, uint32_t p) { return (uint32_t)(((uint64_t)p * v.m) >> v.s); }

struct KvRows {   // one of the two tensors of a cache
    void *p;
    uint8_t *e;
    int64_t page, head, slot;   // strides in elements
};
struct KvDims {
    int n_pages, n_heads, page_size, head_dim;
    PageDiv div;
    int32_t *error;
};
struct KvTable {
    const int32_t *t;
    int64_t stride;
    int n_seqs, width;
};

__device__ __forceinline__ void kv_report(int32_t *error, int bits) {
    if (error) atomicOr(error, bits);
}

// Page and slot of position `pos` of sequence `seq`; false (and the error word) where one of them is out of range.
__device__ __forceinline__ bool kv_place(const KvDims &c, const KvTable &t, int seq, int pos, int *page, int *slot) {
    if ((uint32_t)seq >= (uint32_t)t.n_seqs) {
        kv_report(c.error, WT_KV_BAD_SEQUENCE);
        return false;
    }
    const uint32_t pi = page_of(c.div, (uint32_t)pos);
    if (pi >= (uint32_t)t.width) {
        kv_report(c.error, WT_KV_BAD_POSITION);
        return false;
    }
    *page = t.t[(int64_t)seq * t.stride + pi];
    *slot = pos - (int)(pi * c.div.d);
    if ((uint32_t)*page >= (uint32_t)c.n_pages) {
        kv_report(c.error, WT_KV_BAD_PAGE);
        return false;
    }
    return true;
}

// ---- types ----------------------------------------------------------------------------------------------------------
typedef float f4 __attribute__((ext_vector_type(4)));
struct fp8_t {
    uint8_t b;
};
struct bf16_t {
    uint16_t b;
};
struct f16_t {
    uint16_t b;
};
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(f16_t v) { return __half2float(__ushort_as_half(v.b)); }
__device__ __forceinline__ float to_f(bf16_t v) { return __uint_as_float((uint32_t)v.b << 16); }
__device__ __forceinline__ float to_f(fp8_t v) { return __builtin_amdgcn_cvt_f32_fp8((int)v.b, 0); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ f16_t from_f<f16_t>(float v) { return {__half_as_ushort(__float2half(v))}; }
template <>
__device__ __forceinline__ bf16_t from_f<bf16_t>(float v) {   // round to nearest even, NaN stays NaN
    const uint32_t u = __float_as_uint(v);
    return {(uint16_t)((u & 0x7fffffffu) > 0x7f800000u ? (u >> 16) | 0x40u : (u + 0x7fffu + ((u >> 16) & 1u)) >> 16)};
}
// the power of two that a stored exponent byte stands for (0, which no row of a written cache has, stands for 0)
__device__ __forceinline__ float exp_of(uint32_t e) { return __uint_as_float(e << 23); }

template <typename T, int N>
struct alignas((sizeof(T) * N & -(sizeof(T) * N)) > 16 ? 16 : sizeof(T) * N & -(sizeof(T) * N)) Pack {   // N elements that travel together
    T v[N];
};
static_assert(sizeof(Pack<float, 6>) == 24 && sizeof(Pack<uint16_t, 6>) == 12 && sizeof(Pack<uint16_t, 8>) == 16, "no padding");


// arguments of one attention call, as its kernels take them (wt_kv_attend.h)
struct KvAttend {
    KvRows k, v;
    KvDims c;
    KvTable t;
    const void *q;
    int64_t q_row, q_head;
    int n_q_heads, group;            // query heads, those of a key head
    int q_wide, q_tiles;             // ... are taken 16 * q_wide at a time, in q_tiles tiles
    float scale;
    const int32_t *lengths;
    void *out;
    int64_t o_row, o_head;
    float *lse;
    bool q_aligned, o_aligned;       // every row of q starts on 16 bytes; of out, on four elements
    // schedule
    int direct;                      // one workgroup per (sequence, key head, tile), no workspace
    int waves;                       // of a workgroup: KV_WAVES, or 2
    int n_wg, min_share, seg_cost;
    int32_t *counters;               // 4 * n_wg, zero between calls
    float *partials;                 // 2 * n_wg slots: a tile's maxima and sums, the same of a joined group, sums of values
};

}  // namespace wt
