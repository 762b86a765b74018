// bf16 instances of the decay attention kernel: short sequences, and walks whose
// state is an output.
#include "decay_bf16.hpp"

namespace sldm_decay {
void run_bf16_exact(const Args& a, hipStream_t st) { by_rows<true, true>(a, st); }
}  // namespace sldm_decay
