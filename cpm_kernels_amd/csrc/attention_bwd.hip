// Gradients of the attention over fp16 keys and values (attention.hip), the probabilities computed again from the scores and the forward pass's log of their sums:
//
//     p_ij = exp(s_ij - lse_i),  dv_j = sum_i p_ij do_i,  dp_ij = do_i v_j,  D_i = do_i o_i,  ds_ij = p_ij (dp_ij - D_i),
//     dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dbias[h, bucket] = sum of ds_ij over the pairs of that bucket
//
// Two kernels, so that every sum has one owner and no atomics decide its order: k_attn_dq has queries and goes over their keys, k_attn_dkv has keys and goes over the queries of all heads
// that share them.  Both form scores and dp, seven products of queries and keys in all where a kernel that shared them would need five and a sum in memory that grows in any order.
//
// ds and p are rounded to fp16 for the last products.  p is taken times 2^15 (exact, in the exponent).  |dp_ij - D_i| is at most 2 |do_i| max |v_j|: ds is taken times the power of two that
// brings this bound to 2^15 (a row's own in k_attn_dq, the largest row's in k_attn_dkv), so that it neither overflows beside a loss scale nor vanishes without one.
// The forward pass has left the values' largest magnitude, k_attn_dq, which comes first, leaves D and the gradients'.
#include <algorithm>
#include "attention_grad.h"

using namespace cpmk;

extern "C" {

// Workspace, in floats: D, norms, sums by distance
static int64_t attn_workspace(int64_t batch, int64_t heads, int64_t tokens, int64_t entries, int64_t (&at)[3]) {
    const int64_t row_tiles = ceil_div(tokens, kGradRows);
    at[0] = batch * heads * tokens;
    at[1] = at[0] + batch * heads * row_tiles;
    at[2] = at[1] + batch * heads * row_tiles * entries;
    return at[2];
}

int64_t cpmk_attention_backward_workspace(int32_t batch, int32_t heads, int32_t kv_heads, int32_t tokens, int32_t length, int32_t max_distance, int bidirectional) {
    if (batch <= 0 || heads <= 0 || kv_heads <= 0 || tokens < 0 || length < 0 || heads % kv_heads || tokens > kAttnLong || length > kAttnLong) return 0;
    if (!grid_fits((int64_t)batch * heads) || max_distance < 0 || (int64_t)max_distance * (bidirectional ? 2 : 1) > 1024) return 0;
    int64_t at[3];
    const int64_t entries = max_distance ? max_distance + (bidirectional ? std::max(max_distance - 1, 1) : 0) + 2 * kBiasPad : 0;
    return attn_workspace(batch, heads, tokens, entries, at) * (int64_t)sizeof(float);
}

int cpmk_attention_backward(int32_t batch, int32_t heads, int32_t kv_heads, int32_t tokens, int32_t dim, int32_t length, const void* q, int64_t q_batch, int64_t q_head, int64_t q_token,
                            int64_t q_unit, const void* k, int64_t k_batch, int64_t k_head, int64_t k_token, int64_t k_unit, const void* v, int64_t v_batch, int64_t v_head, int64_t v_token,
                            int64_t v_unit, const void* lens_each, int32_t len, const void* pos_each, int32_t pos, int causal, float scale, const void* bias, const void* mapping,
                            int32_t num_buckets, int32_t max_distance, int bidirectional, const void* mask, int64_t mask_batch, int64_t mask_token, const void* out, int64_t out_batch,
                            int64_t out_head, int64_t out_token, int64_t out_unit, const void* lse, const void* rest, const void* dout, int64_t dout_batch, int64_t dout_head, int64_t dout_token,
                            int64_t dout_unit, void* dq, int64_t dq_batch, int64_t dq_head, int64_t dq_token, int64_t dq_unit, void* dk, int64_t dk_batch, int64_t dk_head, int64_t dk_token,
                            int64_t dk_unit, void* dv, int64_t dv_batch, int64_t dv_head, int64_t dv_token, int64_t dv_unit, void* dbias, void* workspace, void* stream) {
    clear_stale_error();
    AttentionGrad a;
    a.q = {(half_t*)q, q_batch, q_head, q_token, q_unit}, a.k = {(half_t*)k, k_batch, k_head, k_token, k_unit}, a.v = {(half_t*)v, v_batch, v_head, v_token, v_unit};
    a.out = {(half_t*)out, out_batch, out_head, out_token, out_unit}, a.dout = {(half_t*)dout, dout_batch, dout_head, dout_token, dout_unit};
    a.dq = {(half_t*)dq, dq_batch, dq_head, dq_token, dq_unit}, a.dk = {(half_t*)dk, dk_batch, dk_head, dk_token, dk_unit}, a.dv = {(half_t*)dv, dv_batch, dv_head, dv_token, dv_unit};
    a.lens_each = (const int32_t*)lens_each, a.pos_each = (const int32_t*)pos_each, a.len = len, a.pos = pos;
    a.table = (const half_t*)bias, a.mapping = (const int32_t*)mapping, a.buckets = num_buckets, a.distances = max_distance, a.dtable = (half_t*)dbias;
    a.mask = (const uint8_t*)mask, a.mask_batch = mask_batch, a.mask_token = mask_token;
    a.lse = (float*)lse, a.rest = (half_t*)rest, a.scale = scale * kLog2e, a.natural_scale = scale, a.causal = causal != 0;
    a.tokens = tokens, a.dim = dim, a.length = length, a.parts = nullptr;
    bool empty;
    if (int e = attn_check(a, batch, heads, kv_heads, bidirectional, empty)) return e;
    if (empty) return 0;
    if (tokens == 0) a.mask = nullptr;          // (it has no rows to read)
    if ((tokens > 0 && any_null(lse, rest, dout, dq)) || (length > 0 && any_null(dk, dv)) || !workspace || (dbias && !bias)) return CPMK_EBADARG;
    a.row_tiles = (int32_t)ceil_div(tokens, kGradRows), a.query_tiles = (int32_t)ceil_div(tokens, kAttnTile);
    a.splits = tokens > 0 ? attn_plan(batch, heads, kv_heads, tokens, dim, length, false, true).splits : 0;        // (the forward pass's: where it has left the values' magnitudes)
    const int64_t dkv_blocks = (int64_t)batch * kv_heads * ceil_div(length, kGradRows);
    if (!grid_fits((int64_t)batch * heads * a.row_tiles) || !grid_fits(dkv_blocks + heads)) return CPMK_ETOOBIG;
    int64_t at[3];
    attn_workspace(batch, heads, tokens, dbias ? a.distances - a.first_distance + 2 * kBiasPad : 0, at);
    a.delta = (float*)workspace, a.dout_top = a.delta + at[0], a.table_parts = dbias ? a.delta + at[1] : nullptr;
    a.batch = batch, a.rows_in_all = (int64_t)batch * heads * tokens;
    hipStream_t st = (hipStream_t)stream;
    const unsigned dq_grid = (unsigned)((int64_t)batch * heads * a.row_tiles), dkv_grid = (unsigned)dkv_blocks;
    if (int e = dim <= 64   ? attn_grad_launch_64(a, dq_grid, dkv_grid, st)
                : dim <= 96 ? attn_grad_launch_96(a, dq_grid, dkv_grid, st)
                : dim <= 128 ? attn_grad_launch_128(a, dq_grid, dkv_grid, st)
                             : attn_grad_launch_256(a, dq_grid, dkv_grid, st))
        return e;
    return launch_status();
}

}  // extern "C"
