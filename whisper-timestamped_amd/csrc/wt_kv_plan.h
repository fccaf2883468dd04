// Decisions of the paged cache's attention that the host can be asked about without a GPU: plain arithmetic, shared with its kernels.
#pragma once
#include <hip/hip_runtime.h>

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

}  // namespace wt
