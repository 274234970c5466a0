// Instantiations of the split windowed attention kernel (wattn_split.hpp).
#include "wattn_split.hpp"

namespace mtp {

namespace {
template <int CT, int D, int RT>
WinKernel split(bool paged, int nw) {
  if (paged) return nw == 4 ? win_split_kernel<CT, D, RT, true, 4> : win_split_kernel<CT, D, RT, true, 8>;
  return nw == 4 ? win_split_kernel<CT, D, RT, false, 4> : win_split_kernel<CT, D, RT, false, 8>;
}
template <int CT, int D>
WinKernel join(bool paged, int waves) {
  if (paged) return waves == 1 ? win_join_kernel<CT, D, true, 1> : win_join_kernel<CT, D, true, 4>;
  return waves == 1 ? win_join_kernel<CT, D, false, 1> : win_join_kernel<CT, D, false, 4>;
}
template <int CT>
WinKernel split_of(int d, int rt, bool paged, int nw) {
  if (d == 64) return rt == 1 ? split<CT, 64, 1>(paged, nw) : split<CT, 64, 2>(paged, nw);
  if (d == 128) return rt == 1 ? split<CT, 128, 1>(paged, nw) : split<CT, 128, 2>(paged, nw);
  return nullptr;
}
template <int CT>
WinKernel join_of(int d, bool paged, int waves) {
  return d == 64 ? join<CT, 64>(paged, waves) : d == 128 ? join<CT, 128>(paged, waves) : nullptr;
}
}  // namespace

WinKernel win_split_pick(int ct, int d, int rt, bool paged, int nw) {
  switch (ct) {
    case MTP_F32: return split_of<MTP_F32>(d, rt, paged, nw);
    case MTP_BF16: return split_of<MTP_BF16>(d, rt, paged, nw);
    case MTP_F16: return split_of<MTP_F16>(d, rt, paged, nw);
  }
  return nullptr;
}
WinKernel win_join_pick(int ct, int d, bool paged, int waves) {
  switch (ct) {
    case MTP_F32: return join_of<MTP_F32>(d, paged, waves);
    case MTP_BF16: return join_of<MTP_BF16>(d, paged, waves);
    case MTP_F16: return join_of<MTP_F16>(d, paged, waves);
  }
  return nullptr;
}

}  // namespace mtp
