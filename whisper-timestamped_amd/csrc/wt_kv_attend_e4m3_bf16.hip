// wt_kv_attend over pages of fp8_t, queries and results of bf16_t (the kernel: wt_kv_attend.h)
#include "wt_kv_attend.h"

namespace wt {
int kv_attend_e4m3_bf16(const KvAttend &a, unsigned grid, hipStream_t st) { return kv_attend_widths<fp8_t, bf16_t>(a, grid, st); }
}  // namespace wt
