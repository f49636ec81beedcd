// Heads of 65 to 96 units (attention.hip).
#include "attention_fwd.h"

namespace cpmk {

int attn_launch_96(const Attention& a, unsigned grid, hipStream_t st) { return attn_launch<3>(a, grid, st); }

}  // namespace cpmk
