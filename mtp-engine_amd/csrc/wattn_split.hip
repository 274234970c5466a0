// Instantiations of the split windowed attention kernel (wattn_split.hpp).
#include "wattn_split.hpp"

namespace mtp {

namespace {
template <int CT, int D, bool MERGE>
WinKernel form(int rt, bool paged) {
  if constexpr (MERGE) {
    if (rt == 1) return paged ? win_merge_kernel<CT, D, 1, true> : win_merge_kernel<CT, D, 1, false>;
    return paged ? win_merge_kernel<CT, D, 2, true> : win_merge_kernel<CT, D, 2, false>;
  } else {
    if (rt == 1) return paged ? win_split_kernel<CT, D, 1, true> : win_split_kernel<CT, D, 1, false>;
    return paged ? win_split_kernel<CT, D, 2, true> : win_split_kernel<CT, D, 2, false>;
  }
}
template <int CT, bool MERGE>
WinKernel dims(int d, int rt, bool paged) {
  if (rt != 1 && rt != 2) return nullptr;
  if (d == 64) return form<CT, 64, MERGE>(rt, paged);
  if (d == 128) return form<CT, 128, MERGE>(rt, paged);
  return nullptr;
}
template <bool MERGE>
WinKernel types(int ct, int d, int rt, bool paged) {
  switch (ct) {
    case MTP_F32: return dims<MTP_F32, MERGE>(d, rt, paged);
    case MTP_BF16: return dims<MTP_BF16, MERGE>(d, rt, paged);
    case MTP_F16: return dims<MTP_F16, MERGE>(d, rt, paged);
  }
  return nullptr;
}
}  // namespace

WinKernel win_split_pick(int ct, int d, int rt, bool paged) {
  return types<false>(ct, d, rt, paged);
}
WinKernel win_merge_pick(int ct, int d, int rt, bool paged) {
  return types<true>(ct, d, rt, paged);
}

}  // namespace mtp
