// Heads of 97 to 128 units (attention.hip).
#include "attention_fwd.h"

namespace cpmk {

int attn_launch_128(const Attention& a, unsigned grid, hipStream_t st) { return attn_launch<4>(a, grid, st); }

}  // namespace cpmk
