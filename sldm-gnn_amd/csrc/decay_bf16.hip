// bf16 instances of the decay attention kernel: outputs in plain rounding, and states
// alone.
#include "decay_bf16.hpp"

namespace sldm_decay {

void run_bf16_exact(const Args& a, hipStream_t st);

void run_bf16(const Args& a, bool out, hipStream_t st) {
  bool exact = a.T <= kShort;
  for (int i = 0; i < a.roles; ++i) exact = exact || a.role[i].s1;
  if (!all_fast(a, out, 8)) {
    if (out) launch<4, 4, true, true, false>(a, st);
    else launch<4, 4, false, true, false>(a, st);
  } else if (!out) {
    by_rows<false, true>(a, st);
  } else if (exact) {
    run_bf16_exact(a, st);
  } else {
    by_rows<true, false>(a, st);
  }
}

}  // namespace sldm_decay
