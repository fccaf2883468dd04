// Decisions of the paged cache's attention that the host can be asked about without a GPU: plain arithmetic, shared with its kernels.
#pragma once
#include <hip/hip_runtime.h>

#include "wtalign.h"

namespace wt {

// The join of partial results: threads that share four columns, each taking every lanes-th of `count` parts, KV_JOIN at a time.
constexpr int KV_JOIN = 8;
__host__ __device__ inline int kv_join_lanes(int threads, int quads, int count) {
    const int most = threads / quads > 1 ? threads / quads : 1, useful = (count + KV_JOIN - 1) / KV_JOIN;
    return most < useful ? most : useful;
}
// Whether `thread` belongs to a whole group of lanes: where lanes do not divide the workgroup, its last threads belong to none, and a
// sum over the group would run past the workgroup's LDS.
__host__ __device__ inline bool kv_join_grouped(int thread, int lanes, int threads) { return thread / lanes < threads / lanes; }

// ---- who does what in a call of the attention -------------------------------------------------------------------------
constexpr int KV_WAVES = 4;   // waves of a workgroup of the attention kernel
constexpr int KV_WIDE_HD = 128;   // widest heads whose queries may be taken 32 at a time (beyond, registers run out)
constexpr int kv_slot(int head_dim, int q_wide) { return q_wide * (64 + 16 * head_dim); }   // floats of a partial result
inline int64_t kv_workspace(int n_wg, int head_dim, int q_wide) { return WT_KV_WORKSPACE_ZEROED + (int64_t)n_wg * 2 * kv_slot(head_dim, q_wide) * 4; }
constexpr int64_t KV_MAX_GRID = 1 << 23;   // workgroups of one launch: a grid has less than 2^32 threads

struct KvPlan {
    int q_wide, q_tiles, direct, waves, n_wg, min_share, seg_cost;
    unsigned grid;
    int64_t bytes;
};

inline KvPlan kv_plan(int cus, const wt_kv_cache &c, int n_seqs, int n_q_heads, int table_width) {   // on a card of that many compute units
    const int n = cus;
    KvPlan p;
    const int group = n_q_heads / c.n_heads;
    const int64_t heads = (int64_t)n_seqs * c.n_heads, narrow = heads * ((group + 15) / 16);
    const int64_t key_bytes = 2ll * c.head_dim * (c.dtype == WT_DTYPE_F32 ? 4 : c.dtype == WT_DTYPE_E4M3 ? 1 : 2);   // and its value's
    p.n_wg = n < WT_KV_WORKSPACE_ZEROED / 16 ? n : WT_KV_WORKSPACE_ZEROED / 16;   // (four counters each)
    const int64_t unit = key_bytes * KV_WAVES * (c.dtype == WT_DTYPE_F32 ? 16 : 32);   // a block of each of KV_WAVES waves: 8 to 128 KB
    // The least share of a workgroup, 1 / 2 / 4 units, us, 2 heads of 768 KB and one of 2 MB, 8 queries each: units of 16 KB, 8 bits, 64 values 10.8 / 10.8 / 10.9
    // and 11.0 / 11.7 / 13.1, f16, 32 values 10.4 / 9.9 / 9.9 and 10.3 / 11.0 / 12.1; of 32 KB, f16, 64 values 10.3 / 9.8 / 10.6 and 11.1 / 11.1 / 12.1,
    // 8 bits, 128 values 10.9 / 11.1 / 12.2 and 12.6 / 12.9 / 13.8; of 64 KB, bf16, 128 values 11.1 / 11.8 / 14.5 and 12.5 / 12.4 / 15.5; of 128 KB, bf16,
    // 256 values 16.9 / 20.8 / 28.3 and 17.1 / 19.7 / 28.2.
    p.min_share = unit < 32 * 1024 ? 2 : 1;
    // A segment of its own costs about two units (16 sequences up to 32768, without / 2 / 4 / 8: 107 / 64 / 65 / 68 us).
    p.seg_cost = 2;
    // One workgroup streams keys and values at some 48 GB/s whatever its waves (four 8.8 us, eight 9.7, sixteen 11.5 over 250 KB), and
    // splitting them costs 3 to 5 us.  Direct / shares, us: 8 and 32 heads of 192, 256 and 384 KB: f16, 64 values (units of 32 KB) 7.7 / 8.0,
    // 9.0 / 8.0, 11.6 / 8.9 and 8.2 / 9.0, 9.8 / 9.8, 13.4 / 9.9; bf16, 128 values (64 KB) 7.7 / 9.4, 8.9 / 9.4, 11.0 / 10.1 and 8.9 / 10.7, 10.7 /
    // 10.8, 14.1 / 11.0; 128 heads of 256, 384 and 512 KB: 11.2 / 13.0, 15.1 / 15.5, 18.9 / 18.1 and 12.4 / 15.6, 16.3 / 18.0, 20.1 / 20.4; 256
    // heads of 512 KB 23.1 / 24.6 and 24.6 / 26.3.
    const int64_t capacity = (int64_t)table_width * c.page_size * key_bytes;
    const auto is_direct = [&](int64_t pairs) {
        const int64_t kb = unit <= 32 * 1024 ? (pairs <= n / 4 ? 208 : pairs <= n / 2 ? 384 : 512) : pairs <= n / 4 ? 320 : 512;
        return capacity <= kb * 1024 && pairs <= KV_MAX_GRID;
    };
    // More than 16 query heads a key head: 32 at a time read keys and values half as often, but leave one wave a SIMD where a key is more than
    // 64 values of 16 bits, and their partial results are twice as long.  16 / 32 at a time, us, 24 query heads a key head.  Whole tables of
    // 448 keys, 128, 256 and 384 tiles of 16: bf16, 128 values 12.5 / 14.1, 14.5 / 14.8, 23.2 / 15.5, f32, 64 values 11.7 / 13.7, 13.1 /
    // 14.0, 21.0 / 14.4.  5120 tiles of 32, 128, 224, 448 keys: bf16, 128 values 41 / 59, 86 / 85, 117 / 102, 188 / 137, 96 values 30 / 53, 49 /
    // 65, 73 / 81, 125 / 106, 8 bits, 128 values 34 / 60, 50 / 71, 65 / 82, 104 / 102; f16, 64 values 21 / 21, 49 / 34, 70 / 45, 118 / 69, f32, 64
    // values 39 / 27 ... 179 / 106, 128 values 81 / 76 ... 402 / 238.  Shares, tables of 50, 100 and 300 (8 bits) or 600 MB in all: bf16, 128 values
    // 24.0 / 26.3, 41.5 / 33.6, 193 / 109, f16, 64 values 23.9 / 21.9, 39.8 / 31.1, 192 / 110, 8 bits, 128 values 28.0 / 28.5, 42.6 / 40.5, 106 / 73.
    const bool widen = is_direct(narrow) ? narrow > n && (c.head_dim <= 64 || c.dtype == WT_DTYPE_F32 || capacity >= 128 * 1024)
                                         : (double)heads * (double)capacity >= 64. * 1024 * 1024;
    p.q_wide = group > 16 && c.head_dim <= KV_WIDE_HD && widen ? 2 : 1;
    p.q_tiles = (group + 16 * p.q_wide - 1) / (16 * p.q_wide);
    const int64_t pairs = heads * p.q_tiles;
    p.direct = is_direct(pairs);
    // Where the pairs fill the card by themselves, workgroups of two waves let more of them run at once.  Four / two waves, us:
    // f16, 64 values, 256 pairs of 1..448 keys 7.0 / 8.4, 512 8.9 / 9.5 and of 448 each 13.5 / 12.6, 1536 of 1..448 16.2 / 14.9, 5120 39.4 / 36.3; bf16, 128
    // values, 512 of 1..448 15.5 / 14.1, 768 of 448 35.3 / 31.9; f32, 768 of 10..1000 34.8 / 38.6, 1536 of 1..448 27.5 / 24.1; 8 bits, 1536 of 10..1000
    // 18.2 / 21.3, 5120 of 1..448 26.0 / 23.0.
    p.waves = p.direct && p.q_wide == 1 && pairs >= n * (c.dtype == WT_DTYPE_F32 ? 6 : c.dtype == WT_DTYPE_E4M3 ? 12 : 2) ? 2 : KV_WAVES;
    p.grid = p.direct ? (unsigned)pairs : (unsigned)p.n_wg;
    p.bytes = p.direct ? 0 : kv_workspace(p.n_wg, c.head_dim, p.q_wide);
    return p;
}

}  // namespace wt
