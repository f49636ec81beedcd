// Heads of up to 64 units (attention.hip).
#include "attention_fwd.h"

namespace cpmk {

int attn_launch_64(const Attention& a, unsigned grid, hipStream_t st) { return attn_launch<2>(a, grid, st); }

}  // namespace cpmk
