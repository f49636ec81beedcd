// Heads of 129 to 256 units (attention.hip).
#include "attention_fwd.h"

namespace cpmk {

int attn_launch_256(const Attention& a, unsigned grid, hipStream_t st) { return attn_launch<8>(a, grid, st); }

}  // namespace cpmk
