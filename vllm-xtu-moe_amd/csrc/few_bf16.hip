// The MoE block of a few tokens (few.hpp) for BF16 experts.
#include "few.hpp"

namespace xtu {
namespace few {

hipError_t run_bf16(const FewArgs& f, const Plan& p, hipStream_t stream) {
  return launch_few<kBF16>(f, p, stream);
}

}  // namespace few
}  // namespace xtu
