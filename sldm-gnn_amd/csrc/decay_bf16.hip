// bf16 instances of the decay attention kernel that write outputs, and the choice.
#include "decay_bf16.hpp"

namespace sldm_decay {

void run_bf16_states(const Args& a, hipStream_t st);

void run_bf16(const Args& a, bool out, hipStream_t st) {
  if (!out) run_bf16_states(a, st);
  else if (!all_fast(a, out, 8)) launch<4, 4, true, false>(a, st);
  else by_rows<true>(a, st);
}

}  // namespace sldm_decay
