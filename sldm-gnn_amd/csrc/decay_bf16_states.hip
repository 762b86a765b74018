// bf16 instances of the decay attention kernel that walk to the state alone.
#include "decay_bf16.hpp"

namespace sldm_decay {

void run_bf16_states(const Args& a, hipStream_t st) {
  if (!all_fast(a, false, 8)) launch<4, 4, false, false>(a, st);
  else by_rows<false>(a, st);
}

}  // namespace sldm_decay
