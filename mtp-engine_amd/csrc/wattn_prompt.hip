// Instantiations of the windowed attention kernel for prompts (wattn_prompt.hpp).
#include "wattn_prompt.hpp"

namespace mtp {

namespace {
template <int CT, int D>
WinKernel waves(int nw) {
  return nw == 8 ? win_prompt_kernel<CT, D, 8> : nw == 4 ? win_prompt_kernel<CT, D, 4> : nullptr;
}
template <int CT>
WinKernel dims(int d, int nw) {
  return d == 64 ? waves<CT, 64>(nw) : d == 128 ? waves<CT, 128>(nw) : nullptr;
}
}  // namespace

WinKernel win_prompt_pick(int ct, int d, int nw) {
  return ct == MTP_BF16 ? dims<MTP_BF16>(d, nw) : ct == MTP_F16 ? dims<MTP_F16>(d, nw) : nullptr;
}

}  // namespace mtp
