// A paged key-value cache: writing it (plain, or in 8 bits with one power of two per row), reading it back, and the
// attention of one new token per sequence over it.  Layout and formulas: include/wtalign.h, wt_kv_*.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "wt_common.h"

namespace wt {

// position -> (page index, slot) for any page size: q = (p * m) >> s with m = ceil(2^s / d), s = 31 + ceil(log2 d), is exact
// for 0 <= p < 2^31 and m < 2^32
struct PageDiv {
    uint32_t d, m, s;
};
static PageDiv page_div(int d) {
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

// ---- writing rows ---------------------------------------------------------------------------------------------------
// A row (one head of one token) is HD values; LPR lanes take EPL = HD / LPR of them each, so that a lane moves 16 bytes of
// the source (24 for 96 values).  A workgroup takes RT consecutive rows of the call, slots innermost: the rows of a
// prompt that share a line of the cache (64-value rows of 8 bits: two a line) are written by one workgroup, and a lane
// group reads and writes whole 64 ... 256 byte runs on both sides.
template <typename ST, int HD>
struct RowSplit {
    static constexpr int EPL = HD == 96 ? 6 : 16 / (int)sizeof(ST);
    static constexpr int LPR = HD / EPL;
};
constexpr int KV_RT = 16;

template <typename ST, typename CT, int HD>
__device__ __forceinline__ void kv_store_row(const KvRows &x, const KvDims &c, const ST *src, int64_t off, int64_t eoff, int lane) {
    constexpr int EPL = RowSplit<ST, HD>::EPL, LPR = RowSplit<ST, HD>::LPR;
    const Pack<ST, EPL> in = *reinterpret_cast<const Pack<ST, EPL> *>(src + lane * EPL);
    if constexpr (sizeof(CT) != 1) {
        *reinterpret_cast<Pack<ST, EPL> *>(static_cast<ST *>(x.p) + off + lane * EPL) = in;
    } else {
        float f[EPL];
        float a = 0.f;
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
            f[i] = to_f(in.v[i]);
            const float m = fabsf(f[i]);
            a = m < __builtin_inff() ? fmaxf(a, m) : a;   // infinities and NaN do not choose the power
        }
#pragma unroll
        for (int o = 1; o < LPR; o <<= 1) a = fmaxf(a, __shfl_xor(a, o, 64));
        // least E with a <= 448 * 2^(E - 127); 448 = 1.75 * 2^8, so E = exponent - 8, one more where the fraction is over .75
        const int e = min(max((int)((__float_as_uint(a) + 0x1fffffu) >> 23) - 8, 1), 254);
        const float inv = __uint_as_float((uint32_t)(254 - e) << 23);   // a power of two: the product is exact
        Pack<uint8_t, EPL> out;
#pragma unroll
        for (int i = 0; i < EPL; i += 2) {
            const float u = f[i] * inv, v = f[i + 1] * inv;
            const uint32_t w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(u, v, 0, false);
            out.v[i] = fabsf(f[i]) < __builtin_inff() ? (uint8_t)w : 0x7f;
            out.v[i + 1] = fabsf(f[i + 1]) < __builtin_inff() ? (uint8_t)(w >> 8) : 0x7f;
        }
        uint8_t *dst = static_cast<uint8_t *>(x.p) + off + lane * EPL;
        if constexpr (EPL == 8) *reinterpret_cast<uint2 *>(dst) = *reinterpret_cast<const uint2 *>(out.v);
        else if constexpr (EPL == 4) *reinterpret_cast<uint32_t *>(dst) = *reinterpret_cast<const uint32_t *>(out.v);
        else {
#pragma unroll
            for (int i = 0; i < EPL; i += 2) *reinterpret_cast<uint16_t *>(dst + i) = *reinterpret_cast<const uint16_t *>(out.v + i);
        }
        if (lane == 0) x.e[eoff] = (uint8_t)e;
    }
}

template <typename ST, typename CT, int HD>
__global__ __launch_bounds__(256) void kv_append_kernel(KvRows k, KvRows v, KvDims c, KvTable t, const ST *__restrict__ ks,
                                                        const ST *__restrict__ vs, int64_t k_row, int64_t k_head, int64_t v_row,
                                                        int64_t v_head, int n_rows, const int32_t *__restrict__ sequences,
                                                        const int32_t *__restrict__ positions) {
    constexpr int LPR = RowSplit<ST, HD>::LPR, HPW = 256 / LPR / KV_RT < 1 ? 1 : 256 / LPR / KV_RT, RPW = 256 / LPR / HPW;
    const int g = threadIdx.x / LPR, lane = threadIdx.x % LPR;
    const int h = blockIdx.y * HPW + g / RPW;
    const int r = blockIdx.x * RPW + g % RPW;
    if (r >= n_rows || h >= c.n_heads) return;   // whole lane groups
    const int pos = positions[r];
    if (pos < 0) return;
    int page, slot;
    if (!kv_place(c, t, sequences ? sequences[r] : r, pos, &page, &slot)) return;
    const int64_t eoff = ((int64_t)page * c.n_heads + h) * c.page_size + slot;
    kv_store_row<ST, CT, HD>(k, c, ks + r * k_row + h * k_head, page * k.page + h * k.head + slot * k.slot, eoff, lane);
    kv_store_row<ST, CT, HD>(v, c, vs + r * v_row + h * v_head, page * v.page + h * v.head + slot * v.slot, eoff, lane);
}

// ---- reading rows back ----------------------------------------------------------------------------------------------
template <typename DT, typename CT, int HD>
__device__ __forceinline__ void kv_load_row(const KvRows &x, DT *dst, int64_t off, int64_t eoff, bool ok, float fill, int lane) {
    constexpr int EPL = RowSplit<DT, HD>::EPL;
    Pack<DT, EPL> out;
    if (!ok) {
#pragma unroll
        for (int i = 0; i < EPL; ++i) out.v[i] = from_f<DT>(fill);
    } else if constexpr (sizeof(CT) != 1) {
        out = *reinterpret_cast<const Pack<DT, EPL> *>(static_cast<const DT *>(x.p) + off + lane * EPL);
    } else {
        const float f = exp_of(x.e[eoff]);
        const uint8_t *src = static_cast<const uint8_t *>(x.p) + off + lane * EPL;
        uint32_t w[(EPL + 3) / 4];
        if constexpr (EPL == 8) {
            const uint2 u = *reinterpret_cast<const uint2 *>(src);
            w[0] = u.x, w[1] = u.y;
        } else if constexpr (EPL == 4) w[0] = *reinterpret_cast<const uint32_t *>(src);
        else {
            const uint16_t *s = reinterpret_cast<const uint16_t *>(src);
            w[0] = s[0] | (uint32_t)s[1] << 16, w[1] = s[2];
        }
#pragma unroll
        for (int i = 0; i < EPL; ++i) out.v[i] = from_f<DT>(to_f(fp8_t{(uint8_t)(w[i / 4] >> (i % 4 * 8))}) * f);
    }
    *reinterpret_cast<Pack<DT, EPL> *>(dst + lane * EPL) = out;
}

template <typename DT, typename CT, int HD>
__global__ __launch_bounds__(256) void kv_gather_kernel(KvRows k, KvRows v, KvDims c, KvTable t, DT *__restrict__ kd,
                                                        DT *__restrict__ vd, int n_rows, const int32_t *__restrict__ sequences,
                                                        const int32_t *__restrict__ positions) {
    constexpr int LPR = RowSplit<DT, HD>::LPR, HPW = 256 / LPR / KV_RT < 1 ? 1 : 256 / LPR / KV_RT, RPW = 256 / LPR / HPW;
    const int g = threadIdx.x / LPR, lane = threadIdx.x % LPR;
    const int h = blockIdx.y * HPW + g / RPW;
    const int r = blockIdx.x * RPW + g % RPW;
    if (r >= n_rows || h >= c.n_heads) return;
    const int pos = positions[r];
    int page = 0, slot = 0;
    const bool ok = pos >= 0 && kv_place(c, t, sequences ? sequences[r] : r, pos, &page, &slot);
    const float fill = pos < 0 ? 0.f : __builtin_nanf("");
    const int64_t eoff = ((int64_t)page * c.n_heads + h) * c.page_size + slot;
    const int64_t to = ((int64_t)r * c.n_heads + h) * HD;
    kv_load_row<DT, CT, HD>(k, kd + to, page * k.page + h * k.head + slot * k.slot, eoff, ok, fill, lane);
    kv_load_row<DT, CT, HD>(v, vd + to, page * v.page + h * v.head + slot * v.slot, eoff, ok, fill, lane);
}

// ---- attention of one new token ---------------------------------------------------------------------------------------
// One workgroup per (sequence, query head); a wave takes every fourth run of 64 positions, a lane one key of the run: its
// score, the run's maximum and sum by wave reductions, then all lanes over the run's values, HD / 64 columns each.
constexpr int KV_NEG_WAVES = 4;
template <typename T, typename CT>
__global__ __launch_bounds__(256) void kv_attend_kernel(KvRows k, KvRows v, KvDims c, KvTable t, const T *__restrict__ q, int64_t q_row,
                                                        int64_t q_head, int n_q_heads, float scale,
                                                        const int32_t *__restrict__ lengths, T *__restrict__ out, int64_t o_row,
                                                        int64_t o_head, float *__restrict__ lse) {
    __shared__ float qs[256], part[KV_NEG_WAVES][256], pm[KV_NEG_WAVES], pl[KV_NEG_WAVES];
    const int s = blockIdx.x / n_q_heads, hq = blockIdx.x % n_q_heads, h = hq / (n_q_heads / c.n_heads);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hd = c.head_dim;
    if ((int)threadIdx.x < hd) qs[threadIdx.x] = to_f(q[s * q_row + hq * q_head + threadIdx.x]);
    int len = lengths[s];
    bool bad = false;
    if (len < 0 || len > (int64_t)t.width * c.page_size) {
        if (threadIdx.x == 0) kv_report(c.error, WT_KV_BAD_POSITION);
        bad = true;
        len = 0;
    }
    __syncthreads();
    const float LOWEST = -3.402823466e38f;
    float m = LOWEST, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int p0 = wave * 64; p0 < len; p0 += KV_NEG_WAVES * 64) {
        const int pos = p0 + lane;
        const bool in = pos < len;
        int page = 0, slot = 0;
        const bool ok = in && kv_place(c, t, s, pos, &page, &slot);
        bad |= in && !ok;
        float x = -__builtin_inff(), ve = 0.f;
        if (ok) {
            const CT *row = static_cast<const CT *>(k.p) + page * k.page + h * k.head + slot * k.slot;
            float a = 0.f;
            for (int d = 0; d < hd; ++d) a = fmaf(qs[d], to_f(row[d]), a);
            if constexpr (sizeof(CT) == 1) {
                const int64_t eo = ((int64_t)page * c.n_heads + h) * c.page_size + slot;
                a *= exp_of(k.e[eo]);
                ve = exp_of(v.e[eo]);
            } else
                ve = 1.f;
            x = a * scale;
        }
        const float mn = fmaxf(m, wave_max(x)), f = expf(m - mn), p = ok ? expf(x - mn) : 0.f;
        l = l * f + wave_sum(p);
        m = mn;
        for (int i = 0; i < 4; ++i) o[i] *= f;
        const int n = min(64, len - p0);
        for (int j = 0; j < n; ++j) {
            if (!__shfl((int)ok, j, 64)) continue;
            const float pj = __shfl(p, j, 64) * __shfl(ve, j, 64);
            const CT *row = static_cast<const CT *>(v.p) + __shfl(page, j, 64) * v.page + h * v.head + __shfl(slot, j, 64) * v.slot;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (lane + i * 64 < hd) o[i] = fmaf(pj, to_f(row[lane + i * 64]), o[i]);
        }
    }
    if (__any(bad)) l = __builtin_nanf("");
    for (int i = 0; i < 4; ++i)
        if (lane + i * 64 < hd) part[wave][lane + i * 64] = o[i];
    if (lane == 0) pm[wave] = m, pl[wave] = l;
    __syncthreads();
    float mm = LOWEST, ll = 0.f;
    for (int w = 0; w < KV_NEG_WAVES; ++w) mm = fmaxf(mm, pm[w]);
    for (int w = 0; w < KV_NEG_WAVES; ++w) ll += pl[w] * expf(pm[w] - mm);
    if ((int)threadIdx.x < hd) {
        float a = 0.f;
        for (int w = 0; w < KV_NEG_WAVES; ++w) a += part[w][threadIdx.x] * expf(pm[w] - mm);
        out[s * o_row + hq * o_head + threadIdx.x] = from_f<T>(len == 0 && ll == 0.f ? 0.f : a / ll);
    }
    if (lse && threadIdx.x == 0) lse[(int64_t)s * n_q_heads + hq] = mm + logf(ll);
}

// ---- host -----------------------------------------------------------------------------------------------------------
static int kv_check(const char *what, const wt_kv_cache *c, int dtype, const int32_t *table, int64_t table_stride, int n_seqs,
                    int table_width) {
    if (!c || !c->k || !c->v || c->n_pages <= 0 || c->n_heads <= 0 || c->page_size <= 0 || c->reserved != 0) {
        set_error("%s: null cache or pages, or a size below one", what);
        return WT_E_BADARG;
    }
    if (c->dtype < WT_DTYPE_F32 || c->dtype > WT_DTYPE_E4M3 || dtype < WT_DTYPE_F32 || dtype > WT_DTYPE_BF16 ||
        (c->dtype != WT_DTYPE_E4M3 && c->dtype != dtype)) {
        set_error("%s: dtype %d against a cache of dtype %d", what, dtype, c->dtype);
        return WT_E_BADARG;
    }
    if ((c->dtype == WT_DTYPE_E4M3) != (c->k_exp != nullptr) || (c->dtype == WT_DTYPE_E4M3) != (c->v_exp != nullptr)) {
        set_error("%s: an 8 bit cache has exponents, another has none", what);
        return WT_E_BADARG;
    }
    const int d = c->head_dim;
    if (d != 32 && d != 64 && d != 96 && d != 128 && d != 256) {
        set_error("%s: head_dim %d (32, 64, 96, 128 and 256 are supported)", what, d);
        return WT_E_UNSUPPORTED;
    }
    const int64_t per16 = c->dtype == WT_DTYPE_F32 ? 4 : c->dtype == WT_DTYPE_E4M3 ? 16 : 8;
    const int64_t st[6] = {c->k_page_stride, c->k_head_stride, c->k_slot_stride, c->v_page_stride, c->v_head_stride, c->v_slot_stride};
    for (int i = 0; i < 6; ++i)
        if (st[i] < 0 || st[i] % per16 != 0) {
            set_error("%s: cache stride %lld is not a multiple of 16 bytes", what, (long long)st[i]);
            return WT_E_BADARG;
        }
    if (((uintptr_t)c->k | (uintptr_t)c->v) & 15) {
        set_error("%s: the cache's pages are not 16-byte aligned", what);
        return WT_E_BADARG;
    }
    if (!table || n_seqs < 0 || table_width <= 0 || (n_seqs > 1 && table_stride < table_width) ||
        (int64_t)table_width * c->page_size > 0x7fffffffll) {
        set_error("%s: bad table (%d sequences of %d pages, %lld apart)", what, n_seqs, table_width, (long long)table_stride);
        return WT_E_BADARG;
    }
    return WT_OK;
}

static KvRows kv_k(const wt_kv_cache *c) { return {c->k, c->k_exp, c->k_page_stride, c->k_head_stride, c->k_slot_stride}; }
static KvRows kv_v(const wt_kv_cache *c) { return {c->v, c->v_exp, c->v_page_stride, c->v_head_stride, c->v_slot_stride}; }
static KvDims kv_dims(const wt_kv_cache *c) {
    return {c->n_pages, c->n_heads, c->page_size, c->head_dim, page_div(c->page_size), c->error};
}

static int kv_check_rows(const char *what, const void *k, const void *v, int n_rows, int n_seqs, const int32_t *sequences,
                         const int32_t *positions) {
    if (!k || !v || !positions || n_rows < 0 || (!sequences && n_rows > n_seqs)) {
        set_error("%s: null pointer, or %d rows for %d sequences", what, n_rows, n_seqs);
        return WT_E_BADARG;
    }
    if (((uintptr_t)k | (uintptr_t)v) & 15) {
        set_error("%s: the rows are not 16-byte aligned", what);
        return WT_E_BADARG;
    }
    return WT_OK;
}

// F(T, HD) over the supported head widths; T, CT over the types
#define WT_KV_WIDTHS(F, A, B)       \
    switch (c->head_dim) {          \
        case 32: F(A, B, 32); break;   \
        case 64: F(A, B, 64); break;   \
        case 96: F(A, B, 96); break;   \
        case 128: F(A, B, 128); break; \
        default: F(A, B, 256); break;  \
    }
#define WT_KV_TYPES(M, F)                                      \
    if (c->dtype == WT_DTYPE_E4M3) {                           \
        if (dtype == WT_DTYPE_F32) M(F, float, fp8_t)          \
        else if (dtype == WT_DTYPE_F16) M(F, f16_t, fp8_t)     \
        else M(F, bf16_t, fp8_t)                               \
    } else if (dtype == WT_DTYPE_F32) M(F, float, float)       \
    else if (dtype == WT_DTYPE_F16) M(F, f16_t, f16_t)         \
    else M(F, bf16_t, bf16_t)

template <typename ST, int HD>
static dim3 kv_row_grid(int n_rows, int n_heads) {
    constexpr int LPR = RowSplit<ST, HD>::LPR, HPW = 256 / LPR / KV_RT < 1 ? 1 : 256 / LPR / KV_RT, RPW = 256 / LPR / HPW;
    return dim3((unsigned)((n_rows + RPW - 1) / RPW), (unsigned)((n_heads + HPW - 1) / HPW));
}

int kv_append(const wt_kv_cache *c, const void *k, const void *v, int dtype, int64_t k_row, int64_t k_head, int64_t v_row, int64_t v_head,
              int n_rows, const int32_t *table, int64_t table_stride, int n_seqs, int table_width, const int32_t *sequences,
              const int32_t *positions, hipStream_t st) {
    int rc = kv_check("wt_kv_append", c, dtype, table, table_stride, n_seqs, table_width);
    if (!rc) rc = kv_check_rows("wt_kv_append", k, v, n_rows, n_seqs, sequences, positions);
    if (rc) return rc;
    const int64_t per16 = dtype == WT_DTYPE_F32 ? 4 : 8;
    if (((k_row | k_head | v_row | v_head) & (per16 - 1)) != 0) {
        set_error("wt_kv_append: a stride of the rows is not a multiple of 16 bytes");
        return WT_E_BADARG;
    }
    if (n_rows == 0) return WT_OK;
#define WT_KV_GO(ST, CT, HD)                                                                                                     \
    hipLaunchKernelGGL((kv_append_kernel<ST, CT, HD>), (kv_row_grid<ST, HD>(n_rows, c->n_heads)), dim3(256), 0, st, kv_k(c), kv_v(c), \
                       kv_dims(c), (KvTable{table, table_stride, n_seqs, table_width}), (const ST *)k, (const ST *)v, k_row, k_head,   \
                       v_row, v_head, n_rows, sequences, positions)
#define WT_KV_M(F, A, B) WT_KV_WIDTHS(F, A, B)
    WT_KV_TYPES(WT_KV_M, WT_KV_GO)
#undef WT_KV_GO
    WT_HIP(hipGetLastError());
    return WT_OK;
}

int kv_gather(const wt_kv_cache *c, void *k, void *v, int dtype, int n_rows, const int32_t *table, int64_t table_stride, int n_seqs,
              int table_width, const int32_t *sequences, const int32_t *positions, hipStream_t st) {
    int rc = kv_check("wt_kv_gather", c, dtype, table, table_stride, n_seqs, table_width);
    if (!rc) rc = kv_check_rows("wt_kv_gather", k, v, n_rows, n_seqs, sequences, positions);
    if (rc) return rc;
    if (n_rows == 0) return WT_OK;
#define WT_KV_GO(DT, CT, HD)                                                                                                     \
    hipLaunchKernelGGL((kv_gather_kernel<DT, CT, HD>), (kv_row_grid<DT, HD>(n_rows, c->n_heads)), dim3(256), 0, st, kv_k(c), kv_v(c), \
                       kv_dims(c), (KvTable{table, table_stride, n_seqs, table_width}), (DT *)k, (DT *)v, n_rows, sequences, positions)
    WT_KV_TYPES(WT_KV_M, WT_KV_GO)
#undef WT_KV_GO
    WT_HIP(hipGetLastError());
    return WT_OK;
}

int64_t kv_attend_workspace(const wt_kv_cache *c, int n_seqs, int n_q_heads, int table_width) { return 0; }

int kv_attend(const wt_kv_cache *c, const void *q, int dtype, int64_t q_row, int64_t q_head, int n_seqs, int n_q_heads, float scale,
              const int32_t *table, int64_t table_stride, int table_width, const int32_t *lengths, void *out, int64_t o_row,
              int64_t o_head, float *lse, void *workspace, int64_t workspace_bytes, hipStream_t st) {
    const int rc = kv_check("wt_kv_attend", c, dtype, table, table_stride, n_seqs, table_width);
    if (rc) return rc;
    if (!q || !out || !lengths || n_q_heads <= 0 || n_q_heads % c->n_heads != 0 || (int64_t)n_seqs * n_q_heads > 0x7fffffffll) {
        set_error("wt_kv_attend: null pointer, or %d query heads over %d key heads", n_q_heads, c->n_heads);
        return WT_E_BADARG;
    }
    if (n_seqs == 0) return WT_OK;
#define WT_KV_GO(T, CT)                                                                                                              \
    hipLaunchKernelGGL((kv_attend_kernel<T, CT>), dim3((unsigned)(n_seqs * n_q_heads)), dim3(256), 0, st, kv_k(c), kv_v(c), kv_dims(c), \
                       (KvTable{table, table_stride, n_seqs, table_width}), (const T *)q, q_row, q_head, n_q_heads, scale, lengths, (T *)out, \
                       o_row, o_head, lse)
#define WT_KV_ONE(F, A, B) { F(A, B); }
    WT_KV_TYPES(WT_KV_ONE, WT_KV_GO)
#undef WT_KV_GO
    WT_HIP(hipGetLastError());
    return WT_OK;
}

}  // namespace wt
