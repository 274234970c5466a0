// Instantiations of the windowed attention kernel for prompts (wattn_prompt.hpp).
#include "wattn_prompt.hpp"

namespace mtp {

namespace {
template <int CT>
WinKernel dims(int d) {
  constexpr int NW = kWinPromptRows / 32;
  return d == 64 ? win_prompt_kernel<CT, 64, NW> : d == 128 ? win_prompt_kernel<CT, 128, NW> : nullptr;
}
}  // namespace

WinKernel win_prompt_pick(int ct, int d) {
  return ct == MTP_BF16 ? dims<MTP_BF16>(d) : ct == MTP_F16 ? dims<MTP_F16>(d) : nullptr;
}

}  // namespace mtp
