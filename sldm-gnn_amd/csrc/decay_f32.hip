// fp32 instances of the decay attention kernel.
#include "decay.hpp"

namespace sldm_decay {
void run_f32(const Args& a, int roles, bool out, hipStream_t stream) {
  out ? dispatch<float, true>(a, roles, stream) : dispatch<float, false>(a, roles, stream);
}
}  // namespace sldm_decay
