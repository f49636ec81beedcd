// Heads of up to 64 units (attention_bwd.hip).
#include "attention_grad.h"

namespace cpmk {

int attn_grad_launch_64(const AttentionGrad& a, unsigned dq_grid, unsigned dkv_grid, hipStream_t st) { return grad_launch<2>(a, dq_grid, dkv_grid, st); }

}  // namespace cpmk
