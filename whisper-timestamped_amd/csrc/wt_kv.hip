// A paged key-value cache: writing it (plain, or in 8 bits with one power of two per row), reading it back, and the
// attention of one new token per sequence over it.  Layout and formulas: include/wtalign.h, wt_kv_*.
#include "wt_kv.h"
#include <type_traits>

namespace wt {

// ---- writing rows and reading them back -----------------------------------------------------------------------------
// A row (one head of one token) is HD values; LPR lanes take EPL = HD / LPR of them each, so that a lane moves 16 bytes
// outside of the cache (24 or 12 where a row is 96 values).  A workgroup takes up to 16 consecutive rows of the call, slots
// innermost: rows of a prompt that share a line of the cache (64 values of 8 bits: two a line) are written by one
// workgroup, and every lane group moves whole runs of 64 ... 256 bytes on both sides.  Both directions are bound by memory:
// a lane finds its row's place once and has KV_HU heads' keys and values in flight, past the caches (one head, plain loads: 35 / 168 /
// 97 us instead of 31 / 124 / 64 for the following).  20000 rows of 8 heads, bf16, 128 values: 31 us (5.3 TB/s read and written); 40000 rows
// of 20 heads, f16, 64 values, into 8 bits 61 us and back 62; 111000 rows of 8 heads of 128 from 8 bits to bf16 64 us (5.4).
template <typename T, int HD>
struct RowSplit {
    static constexpr int EPL = HD == 96 ? 6 : 16 / (int)sizeof(T);
    static constexpr int LPR = HD / EPL;
    static constexpr int GROUPS = 256 / LPR;                 // lane groups of a workgroup: RPW rows x HPW heads
    static constexpr int RPW = GROUPS < 16 ? GROUPS : 16;
    static constexpr int HPW = GROUPS / RPW;
};
constexpr int KV_HU = 4;
constexpr int KV_MAX_ROWS = 1 << 25;   // rows of one launch (4 a workgroup at least, a grid has less than 2^32 threads)

template <int N>   // N bytes as the widest loads and stores their alignment allows
struct Bytes {
    static constexpr int W = N % 16 == 0 ? 16 : N % 8 == 0 ? 8 : N % 4 == 0 ? 4 : 2;
    typedef uint32_t v4 __attribute__((ext_vector_type(4)));
    typedef uint32_t v2 __attribute__((ext_vector_type(2)));
    using Word = std::conditional_t<W == 16, v4, std::conditional_t<W == 8, v2, std::conditional_t<W == 4, uint32_t, uint16_t>>>;
    Word w[N / W];
    __device__ __forceinline__ void load(const void *p) {
#pragma unroll
        for (int i = 0; i < N / W; ++i) w[i] = __builtin_nontemporal_load(static_cast<const Word *>(p) + i);
    }
    __device__ __forceinline__ void store(void *p) const {
#pragma unroll
        for (int i = 0; i < N / W; ++i) __builtin_nontemporal_store(w[i], static_cast<Word *>(p) + i);
    }
};

template <typename ST, int EPL, int LPR>
__device__ __forceinline__ void kv_quantise(const Bytes<EPL * sizeof(ST)> &src, Bytes<EPL> &dst, int *exponent) {
    ST in[EPL];
    __builtin_memcpy(in, &src, sizeof(in));
    float f[EPL];
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
        f[i] = to_f(in[i]);
        const float m = fabsf(f[i]);
        a = m < __builtin_inff() ? fmaxf(a, m) : a;   // infinities and NaN do not choose the power
    }
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1) a = fmaxf(a, __shfl_xor(a, o, 64));
    // least E with a <= 448 * 2^(E - 127); 448 = 1.75 * 2^8, so E = exponent - 8, one more where the fraction is over .75
    const int e = min(max((int)((__float_as_uint(a) + 0x1fffffu) >> 23) - 8, 1), 254);
    const float inv = __uint_as_float((uint32_t)(254 - e) << 23);   // a power of two: the product is exact
    uint8_t out[EPL];
#pragma unroll
    for (int i = 0; i < EPL; i += 2) {
        const uint32_t w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[i] * inv, f[i + 1] * inv, 0, false);
        out[i] = fabsf(f[i]) < __builtin_inff() ? (uint8_t)w : 0x7f;
        out[i + 1] = fabsf(f[i + 1]) < __builtin_inff() ? (uint8_t)(w >> 8) : 0x7f;
    }
    __builtin_memcpy(&dst, out, EPL);
    *exponent = e;
}

template <typename ST, typename CT, int HD>
__global__ __launch_bounds__(256) void kv_append_kernel(KvRows k, KvRows v, KvDims c, KvTable t, const ST *__restrict__ ks,
                                                        const ST *__restrict__ vs, int64_t k_row, int64_t k_head, int64_t v_row,
                                                        int64_t v_head, int row0, int n_rows, const int32_t *__restrict__ sequences,
                                                        const int32_t *__restrict__ positions) {
    using R = RowSplit<ST, HD>;
    constexpr int EPL = R::EPL;
    const int g = threadIdx.x / R::LPR, lane = threadIdx.x % R::LPR;
    const int r = row0 + blockIdx.x * R::RPW + g % R::RPW, h0 = blockIdx.y * R::HPW * KV_HU + g / R::RPW;
    if (g >= R::GROUPS || r >= n_rows) return;   // whole lane groups
    const int pos = positions[r];
    Bytes<EPL * sizeof(ST)> kr[KV_HU], vr[KV_HU];
#pragma unroll
    for (int i = 0; i < KV_HU; ++i) {   // (beside the look-up of the place)
        const int h = min(h0 + i * R::HPW, c.n_heads - 1);
        kr[i].load(ks + r * k_row + h * k_head + lane * EPL);
        vr[i].load(vs + r * v_row + h * v_head + lane * EPL);
    }
    int page, slot;
    if (pos < 0 || !kv_place(c, t, sequences ? sequences[r] : r, pos, &page, &slot)) return;
#pragma unroll
    for (int i = 0; i < KV_HU; ++i) {
        const int h = h0 + i * R::HPW;
        if (h >= c.n_heads) break;
        CT *kd = static_cast<CT *>(k.p) + (page * k.page + h * k.head + slot * k.slot + lane * EPL);
        CT *vd = static_cast<CT *>(v.p) + (page * v.page + h * v.head + slot * v.slot + lane * EPL);
        if constexpr (sizeof(CT) != 1) {
            kr[i].store(kd), vr[i].store(vd);
        } else {
            Bytes<EPL> out;
            int ke, ve;
            kv_quantise<ST, EPL, R::LPR>(kr[i], out, &ke);
            out.store(kd);
            kv_quantise<ST, EPL, R::LPR>(vr[i], out, &ve);
            out.store(vd);
            const int64_t eoff = ((int64_t)page * c.n_heads + h) * c.page_size + slot;
            if (lane == 0) k.e[eoff] = (uint8_t)ke, v.e[eoff] = (uint8_t)ve;
        }
    }
}

template <typename DT, typename CT, int EPL>
__device__ __forceinline__ void kv_emit(const Bytes<EPL * sizeof(CT)> &src, uint32_t e, bool ok, float fill, DT *dst) {
    Bytes<EPL * sizeof(DT)> out;
    if constexpr (sizeof(CT) != 1) out = src;
    if (sizeof(CT) == 1 || !ok) {
        DT val[EPL];
        if constexpr (sizeof(CT) == 1) {
            uint8_t b[EPL];
            __builtin_memcpy(b, &src, EPL);
            const float f = exp_of(e);
#pragma unroll
            for (int i = 0; i < EPL; ++i) val[i] = from_f<DT>(to_f(fp8_t{b[i]}) * f);
        }
        if (!ok)
#pragma unroll
            for (int i = 0; i < EPL; ++i) val[i] = from_f<DT>(fill);
        __builtin_memcpy(&out, val, sizeof(out));
    }
    out.store(dst);
}

template <typename DT, typename CT, int HD>
__global__ __launch_bounds__(256) void kv_gather_kernel(KvRows k, KvRows v, KvDims c, KvTable t, DT *__restrict__ kd,
                                                        DT *__restrict__ vd, int row0, int n_rows, const int32_t *__restrict__ sequences,
                                                        const int32_t *__restrict__ positions) {
    using R = RowSplit<DT, HD>;
    constexpr int EPL = R::EPL;
    const int g = threadIdx.x / R::LPR, lane = threadIdx.x % R::LPR;
    const int r = row0 + blockIdx.x * R::RPW + g % R::RPW, h0 = blockIdx.y * R::HPW * KV_HU + g / R::RPW;
    if (g >= R::GROUPS || r >= n_rows) return;
    const int pos = positions[r];
    int page = 0, slot = 0;
    const bool ok = pos >= 0 && kv_place(c, t, sequences ? sequences[r] : r, pos, &page, &slot);
    if (!ok) page = 0, slot = 0;   // (a row of the cache all the same: read, not used)
    const float fill = pos < 0 ? 0.f : __builtin_nanf("");
    Bytes<EPL * sizeof(CT)> kr[KV_HU], vr[KV_HU];
    uint32_t ke[KV_HU], ve[KV_HU];
#pragma unroll
    for (int i = 0; i < KV_HU; ++i) {
        const int h = min(h0 + i * R::HPW, c.n_heads - 1);
        kr[i].load(static_cast<const CT *>(k.p) + (page * k.page + h * k.head + slot * k.slot + lane * EPL));
        vr[i].load(static_cast<const CT *>(v.p) + (page * v.page + h * v.head + slot * v.slot + lane * EPL));
        if constexpr (sizeof(CT) == 1) {
            const int64_t eoff = ((int64_t)page * c.n_heads + h) * c.page_size + slot;
            ke[i] = k.e[eoff], ve[i] = v.e[eoff];
        } else
            ke[i] = ve[i] = 0;
    }
#pragma unroll
    for (int i = 0; i < KV_HU; ++i) {
        const int h = h0 + i * R::HPW;
        if (h >= c.n_heads) break;
        const int64_t to = ((int64_t)r * c.n_heads + h) * HD + lane * EPL;
        kv_emit<DT, CT, EPL>(kr[i], ke[i], ok, fill, kd + to);
        kv_emit<DT, CT, EPL>(vr[i], ve[i], ok, fill, vd + to);
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------
static int kv_check(const char *what, const wt_kv_cache *c, int dtype, const int32_t *table, int64_t table_stride, int n_seqs,
                    int table_width) {
    if (!c || !c->k || !c->v || c->n_pages <= 0 || c->n_heads <= 0 || c->n_heads > 65535 || c->page_size <= 0 || c->reserved != 0) {
        set_error("%s: null cache or pages, a size below one, or more than 65535 heads", what);
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
    if (((uintptr_t)c->k_exp | (uintptr_t)c->v_exp) & 15) {
        set_error("%s: the exponents are not 16-byte aligned", what);
        return WT_E_BADARG;
    }
    if (!table || n_seqs < 0 || table_width <= 0 || (n_seqs > 1 && table_stride < table_width) ||
        (int64_t)table_width * c->page_size > WT_KV_MAX_POSITIONS) {
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
    if (!k || !v || !positions || n_rows < 0 || n_rows > (1 << 30) || (!sequences && n_rows > n_seqs)) {
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

template <typename T, int HD>
static dim3 kv_row_grid(int n_rows, int n_heads) {
    using R = RowSplit<T, HD>;
    return dim3((unsigned)((n_rows + R::RPW - 1) / R::RPW), (unsigned)((n_heads + R::HPW * KV_HU - 1) / (R::HPW * KV_HU)));
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
#define WT_KV_GO(ST, CT, HD)                                                                                                   \
    hipLaunchKernelGGL((kv_append_kernel<ST, CT, HD>), (kv_row_grid<ST, HD>(end - r0, c->n_heads)), dim3(256), 0, st, kv_k(c), kv_v(c), \
                       kv_dims(c), (KvTable{table, table_stride, n_seqs, table_width}), (const ST *)k, (const ST *)v, k_row, k_head, v_row, \
                       v_head, r0, end, sequences, positions)
#define WT_KV_M(F, A, B) WT_KV_WIDTHS(F, A, B)
    for (int64_t r = 0; r < n_rows; r += KV_MAX_ROWS) {
        const int r0 = (int)r, end = (int)(r + KV_MAX_ROWS < n_rows ? r + KV_MAX_ROWS : n_rows);
        WT_KV_TYPES(WT_KV_M, WT_KV_GO)
        WT_HIP(hipGetLastError());
    }
#undef WT_KV_GO
    return WT_OK;
}

int kv_gather(const wt_kv_cache *c, void *k, void *v, int dtype, int n_rows, const int32_t *table, int64_t table_stride, int n_seqs,
              int table_width, const int32_t *sequences, const int32_t *positions, hipStream_t st) {
    int rc = kv_check("wt_kv_gather", c, dtype, table, table_stride, n_seqs, table_width);
    if (!rc) rc = kv_check_rows("wt_kv_gather", k, v, n_rows, n_seqs, sequences, positions);
    if (rc) return rc;
    if (n_rows == 0) return WT_OK;
#define WT_KV_GO(DT, CT, HD)                                                                                                   \
    hipLaunchKernelGGL((kv_gather_kernel<DT, CT, HD>), (kv_row_grid<DT, HD>(end - r0, c->n_heads)), dim3(256), 0, st, kv_k(c), kv_v(c), \
                       kv_dims(c), (KvTable{table, table_stride, n_seqs, table_width}), (DT *)k, (DT *)v, r0, end, sequences, positions)
    for (int64_t r = 0; r < n_rows; r += KV_MAX_ROWS) {
        const int r0 = (int)r, end = (int)(r + KV_MAX_ROWS < n_rows ? r + KV_MAX_ROWS : n_rows);
        WT_KV_TYPES(WT_KV_M, WT_KV_GO)
        WT_HIP(hipGetLastError());
    }
#undef WT_KV_GO
    return WT_OK;
}

// ---- attention of one new token: schedule ------------------------------------------------------------------------------
int scratch_kv(hipStream_t st, size_t bytes, void **out);
int kv_attend_f32(const KvAttend &, unsigned, hipStream_t);
int kv_attend_f16(const KvAttend &, unsigned, hipStream_t);
int kv_attend_bf16(const KvAttend &, unsigned, hipStream_t);
int kv_attend_e4m3_f32(const KvAttend &, unsigned, hipStream_t);
int kv_attend_e4m3_f16(const KvAttend &, unsigned, hipStream_t);
int kv_attend_e4m3_bf16(const KvAttend &, unsigned, hipStream_t);

__global__ void kv_zero_kernel(int32_t *p) { p[blockIdx.x * 256 + threadIdx.x] = 0; }
int kv_clear(void *workspace, hipStream_t st) {
    hipLaunchKernelGGL(kv_zero_kernel, dim3(WT_KV_WORKSPACE_ZEROED / 1024), dim3(256), 0, st, (int32_t *)workspace);
    WT_HIP(hipGetLastError());
    return WT_OK;
}
static int64_t kv_most_workspace(int n_wg) {   // of any call
    const int64_t narrow = kv_workspace(n_wg, 256, 1), wide = kv_workspace(n_wg, KV_WIDE_HD, 2);
    return narrow > wide ? narrow : wide;
}

static int kv_plan(const wt_kv_cache *c, int n_seqs, int n_q_heads, int table_width, KvPlan *p) {
    static int cus[16] = {0};   // per device; two threads that fill it write the same
    int dev = 0;
    WT_HIP(hipGetDevice(&dev));
    int n = dev < 16 ? cus[dev] : 0;
    if (n == 0) {
        WT_HIP(hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev));
        if (dev < 16) cus[dev] = n;
    }
    *p = kv_plan(n, *c, n_seqs, n_q_heads, table_width);
    return WT_OK;
}

static int kv_check_heads(const wt_kv_cache *c, int n_seqs, int n_q_heads) {
    if (n_q_heads <= 0 || n_q_heads % c->n_heads != 0 || (int64_t)n_seqs * n_q_heads > 0x7fffffffll) {
        set_error("wt_kv_attend: %d query heads over %d key heads, %d sequences", n_q_heads, c->n_heads, n_seqs);
        return WT_E_BADARG;
    }
    return WT_OK;
}

int64_t kv_attend_workspace(const wt_kv_cache *c, int n_seqs, int n_q_heads, int table_width) {
    static const int32_t none = 0;
    int rc = kv_check("wt_kv_attend_workspace", c, c && c->dtype != WT_DTYPE_E4M3 ? c->dtype : 0, &none, table_width, n_seqs, table_width);
    if (!rc) rc = kv_check_heads(c, n_seqs, n_q_heads);
    KvPlan p, one;   // (fewer sequences may be split where these are not)
    if (!rc) rc = kv_plan(c, n_seqs, n_q_heads, table_width, &p);
    if (!rc) rc = kv_plan(c, 1, n_q_heads, table_width, &one);
    return rc ? rc : p.bytes > one.bytes ? p.bytes : one.bytes;
}

int kv_attend(const wt_kv_cache *c, const void *q, int dtype, int64_t q_row, int64_t q_head, int n_seqs, int n_q_heads, float scale,
              const int32_t *table, int64_t table_stride, int table_width, const int32_t *lengths, void *out, int64_t o_row,
              int64_t o_head, float *lse, void *workspace, int64_t workspace_bytes, hipStream_t st) {
    int rc = kv_check("wt_kv_attend", c, dtype, table, table_stride, n_seqs, table_width);
    if (rc) return rc;
    if (!q || !out || !lengths) {
        set_error("wt_kv_attend: null pointer");
        return WT_E_BADARG;
    }
    if ((rc = kv_check_heads(c, n_seqs, n_q_heads))) return rc;
    const int64_t item = dtype == WT_DTYPE_F32 ? 4 : 2, held = c->dtype == WT_DTYPE_E4M3 ? 1 : item;
    if (((uintptr_t)q | (uintptr_t)out) & (item - 1)) {
        set_error("wt_kv_attend: q or out is not aligned to its elements");
        return WT_E_BADARG;
    }
    if ((c->k_slot_stride > c->v_slot_stride ? c->k_slot_stride : c->v_slot_stride) * held * 32 > 0x7fffffffll) {
        set_error("wt_kv_attend: slots of a page are too far apart");
        return WT_E_UNSUPPORTED;
    }
    if (n_seqs == 0) return WT_OK;
    KvPlan p;
    if ((rc = kv_plan(c, n_seqs, n_q_heads, table_width, &p))) return rc;
    if (p.bytes > 0) {
        if (workspace) {
            if (workspace_bytes < p.bytes || ((uintptr_t)workspace & 15)) {
                set_error("wt_kv_attend: workspace of %lld bytes, %lld needed, 16-byte aligned", (long long)workspace_bytes, (long long)p.bytes);
                return WT_E_BADARG;
            }
        } else {
            hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
            WT_HIP(hipStreamIsCapturing(st, &cap));
            if (cap != hipStreamCaptureStatusNone) {
                set_error("wt_kv_attend: a captured call needs a workspace of its own (%lld bytes)", (long long)p.bytes);
                return WT_E_CAPTURE;
            }
            if ((rc = scratch_kv(st, (size_t)kv_most_workspace(p.n_wg), &workspace))) return rc;
        }
    }
    KvAttend a;
    a.k = kv_k(c), a.v = kv_v(c), a.c = kv_dims(c), a.t = KvTable{table, table_stride, n_seqs, table_width};
    a.q = q, a.q_row = q_row, a.q_head = q_head;
    a.n_q_heads = n_q_heads, a.group = n_q_heads / c->n_heads, a.q_wide = p.q_wide, a.q_tiles = p.q_tiles;
    a.scale = scale, a.lengths = lengths, a.out = out, a.o_row = o_row, a.o_head = o_head, a.lse = lse;
    a.q_aligned = (((uintptr_t)q | (uint64_t)(q_row * item) | (uint64_t)(q_head * item)) & 15) == 0;
    a.o_aligned = (((uintptr_t)out | (uint64_t)(o_row * item) | (uint64_t)(o_head * item)) & (4 * item - 1)) == 0;
    a.direct = p.direct, a.waves = p.waves, a.n_wg = p.n_wg, a.min_share = p.min_share, a.seg_cost = p.seg_cost;
    a.counters = (int32_t *)workspace;
    a.partials = workspace ? (float *)((char *)workspace + WT_KV_WORKSPACE_ZEROED) : nullptr;
    if (c->dtype == WT_DTYPE_E4M3)
        return dtype == WT_DTYPE_F32 ? kv_attend_e4m3_f32(a, p.grid, st) : dtype == WT_DTYPE_F16 ? kv_attend_e4m3_f16(a, p.grid, st) : kv_attend_e4m3_bf16(a, p.grid, st);
    return dtype == WT_DTYPE_F32 ? kv_attend_f32(a, p.grid, st) : dtype == WT_DTYPE_F16 ? kv_attend_f16(a, p.grid, st) : kv_attend_bf16(a, p.grid, st);
}

}  // namespace wt
