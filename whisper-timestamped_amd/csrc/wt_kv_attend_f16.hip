// wt_kv_attend over pages of f16_t, queries and results of f16_t (the kernel: wt_kv_attend.h)
#include "wt_kv_attend.h"

namespace wt {
int kv_attend_f16(const KvAttend &a, unsigned grid, hipStream_t st) { return kv_attend_widths<f16_t, f16_t>(a, grid, st); }
}  // namespace wt
