// wt_kv_attend over pages of fp8_t, queries and results of float (the kernel: wt_kv_attend.h)
#include "wt_kv_attend.h"

namespace wt {
int kv_attend_e4m3_f32(const KvAttend &a, unsigned grid, hipStream_t st) { return kv_attend_widths<fp8_t, float>(a, grid, st); }
}  // namespace wt
