// pages_attn_seen.hip -- the kernels of pages_attn.hpp for rows that see a part of
// what is before them (a window with sinks, a tree of drafts): a file of its own, as each
// set takes half a minute to compile.
#include "pages_attn.hpp"

namespace {

template <int DT>
void launch(const PageView& v, int layer, const AttendArgs& a, const Scratch& ws, int forms, bool wide, int grid, hipStream_t s) {
  if constexpr (DT != FERRY_F32) {
    if (wide) {
      k_attend<DT, 3, kSeenWide><<<grid, threads_of(kSeenWide), 0, s>>>(v, layer, a, ws);
      return;
    }
  }
  launch_forms<DT, kSeen>(v, layer, a, ws, forms, grid, s);
}

}  // namespace

void ferry_amd::launch_attend_seen(const PageView& v, int layer, int dtype, const AttendArgs& a, const Scratch& ws,
                                   int forms, bool wide, int grid, hipStream_t s) {
  if (dtype == FERRY_F32) launch<FERRY_F32>(v, layer, a, ws, forms, wide, grid, s);
  else if (dtype == FERRY_F16) launch<FERRY_F16>(v, layer, a, ws, forms, wide, grid, s);
  else if (dtype == FERRY_BF16) launch<FERRY_BF16>(v, layer, a, ws, forms, wide, grid, s);
  else launch<FERRY_FP8_E4M3>(v, layer, a, ws, forms, wide, grid, s);
}
