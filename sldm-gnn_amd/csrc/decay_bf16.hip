// bf16 instances of the decay attention kernel.
#include "decay.hpp"

namespace sldm_decay {
void run_bf16(const Args& a, int roles, bool out, hipStream_t stream) {
  out ? dispatch<uint16_t, true>(a, roles, stream) : dispatch<uint16_t, false>(a, roles, stream);
}
}  // namespace sldm_decay
