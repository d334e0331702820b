// The MoE block of a few tokens (few.hpp) for FP8 experts.
#include "few.hpp"

namespace xtu {
namespace few {

hipError_t run_fp8(const FewArgs& f, const Plan& p, hipStream_t stream) {
  return launch_few<kFP8>(f, p, stream);
}

}  // namespace few
}  // namespace xtu
