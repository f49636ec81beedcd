// Heads of 129 to 256 units (attention_bwd.hip).
#include "attention_grad.h"

namespace cpmk {

int attn_grad_launch_256(const AttentionGrad& a, unsigned dq_grid, unsigned dkv_grid, hipStream_t st) { return grad_launch<8>(a, dq_grid, dkv_grid, st); }

}  // namespace cpmk
