// wt_kv_attend over pages of float, queries and results of float (the kernel: wt_kv_attend.h)
#include "wt_kv_attend.h"

namespace wt {
int kv_attend_f32(const KvAttend &a, unsigned grid, hipStream_t st) { return kv_attend_widths<float, float>(a, grid, st); }
}  // namespace wt
