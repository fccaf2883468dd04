// What the library's per-stream memory is kept by.
#pragma once
#include <hip/hip_runtime.h>

#include <atomic>
#include <cstdint>
#include <utility>

namespace wt {

// hipStreamPerThread is one handle for another stream in every thread: it is kept apart by the calling thread (numbered from 1, a number
// is never given twice).  Any other handle is one stream, whoever uses it.
using StreamKey = std::pair<hipStream_t, uint64_t>;
inline StreamKey stream_key(hipStream_t st) {
    static std::atomic<uint64_t> threads{0};
    thread_local uint64_t me = 0;
    if (st != hipStreamPerThread) return {st, 0};
    if (me == 0) me = ++threads;
    return {st, me};
}

}  // namespace wt
