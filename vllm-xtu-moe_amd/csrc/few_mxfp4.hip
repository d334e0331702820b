// The MoE block of a few tokens (few.hpp) for MXFP4 experts.
#include "few.hpp"

namespace xtu {
namespace few {

hipError_t run_mxfp4(const FewArgs& f, const Plan& p, hipStream_t stream) {
  return launch_few<kMXFP4>(f, p, stream);
}

}  // namespace few
}  // namespace xtu
