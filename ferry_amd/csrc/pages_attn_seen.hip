// pages_attn_seen.hip -- the kernels of pages_attn.hpp for rows that see a part of
// what is before them (a window with sinks, a tree of drafts): a file of its own, as each
// set takes a minute to compile.
#include "pages_attn.hpp"

void ferry_amd::launch_attend_seen(const PageView& v, int layer, int dtype, const AttendArgs& a, const Scratch& ws,
                                   int forms, int grid, hipStream_t s) {
  if (dtype == FERRY_F32) launch_forms<FERRY_F32, kSeen>(v, layer, a, ws, forms, grid, s);
  else if (dtype == FERRY_F16) launch_forms<FERRY_F16, kSeen>(v, layer, a, ws, forms, grid, s);
  else if (dtype == FERRY_BF16) launch_forms<FERRY_BF16, kSeen>(v, layer, a, ws, forms, grid, s);
  else launch_forms<FERRY_FP8_E4M3, kSeen>(v, layer, a, ws, forms, grid, s);
}
