// Attention over fp16 keys and values, forward:
//
//     out[i] = sum_j p_ij v_j,   p_ij = exp(s_ij - m_i) / sum_j exp(s_ij - m_i),   s_ij = scale q_i k_j + bias[bucket(at_i - j)]
//
// over the keys j that length, causality and mask leave, in one pass over the keys: the running maximum m_i and the sum are kept beside the weighted values, which are scaled when the
// maximum grows.  Nothing of the size of the scores is in memory.
//
// A workgroup has 128 queries of a head, 32 a wave, and goes over its keys in tiles of 64 that all its waves read from LDS.  Scores are formed transposed (keys as rows), so a lane holds
// keys of one query, and its probabilities, rounded to fp16, are the second product's operand as they are.  fp16 keeps their bits: they are at most 2^15 and their maximum is 2^7 at least
// (the running maximum follows the true one at a distance of up to 2^8), so what falls below fp16's normal range is less than 2^-21 of the row's largest.  Sums are fp32, of the
// unrounded probabilities.  For training (TRAIN) what their rounding leaves is multiplied by the values as well, and what the result's rounding leaves is kept: the
// backward pass subtracts two nearly equal numbers where a query looks at one key, do_i v_j and do_i out_i, and the second has to be as exact as the first.  Where there are few rows the
// keys are cut into parts, which k_attn_join adds up.
//
// Bound by products and exponentials together: a score costs an exponential and about five vector operations beside 4 dim operations of products, so heads of 128 units come nearer to what
// the matrix cores give than those of 64.  128 queries, so that a tile is read from memory once for all of them; tiles of 64 keys, so that two workgroups fit a compute unit and one's
// products run beside the other's exponentials.  Measured: 2000 queries of 32 heads, 8 of keys, dim 128, 8011 keys, causal: 275 us, 0.84 PFLOP/s; 8 x 64 heads of 64, 512 tokens, biases and a
// mask of keys: 100 us, 0.34; 64 keys more for 8 x 32 heads of 512 queries, dim 128: 4.5 us, 0.96.
#include <algorithm>
#include "attention_fwd.h"

namespace cpmk {

// Parts joined under the largest of their maxima: a wave a row, its lanes along the units.  `rows` of them lie together: queries of a head, or (few) rows of a head of keys.
__global__ __launch_bounds__(256) void k_attn_join(Attention a, AttnPlan plan, uint32_t total_rows) {
    const int lane = threadIdx.x & 63, rows = plan.rows;
    const uint32_t id = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= total_rows) return;
    const int32_t group = plan.few ? a.group : 1, heads = plan.few ? a.held : a.heads, of_head = a.tokens * group;
    const int32_t in_head = id % (uint32_t)of_head;
    const uint32_t bh = id / (uint32_t)of_head;
    const int64_t b = bh / (uint32_t)heads;
    const int32_t rt = in_head / rows, r = in_head - rt * rows, query = in_head / group, h = (bh - (uint32_t)b * heads) * group + in_head - query * group;
    const AttnRange range = attn_range(a, b);
    const AttnParts p = attn_parts(a, range, min(rt * rows + rows - 1, of_head - 1) / group, plan.least, plan.tile);
    const int64_t size = (int64_t)rows * (a.dim + 2);
    const float* const part = a.parts + ((int64_t)bh * a.row_tiles + rt) * a.splits * size;
    const float* const tops = part + rows * a.dim + r;
    float m = -__builtin_inff();
    for (int i = lane; i < p.parts; i += 64) m = fmaxf(m, tops[i * size]);
    m = wave_max(m);
    const float base = m == -__builtin_inff() ? 0.0f : m;
    float total = 0.0f, value[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int first = 0; first < p.parts; first += 64) {
        // a lane a part: its weight; then eight parts' sums at a time, all on their way together
        const bool real = first + lane < p.parts;
        const float* const mine = tops + (first + (real ? lane : 0)) * size;
        const float weight = real ? __builtin_amdgcn_exp2f(mine[0] - base) : 0.0f;
        total = __builtin_fmaf(real ? mine[rows] : 0.0f, weight, total);
        const int n = min(64, p.parts - first);
        for (int i = 0; i < n; i += 8) {
            float x[8][4];
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (c * 64 < a.dim) x[k][c] = part[(first + min(i + k, n - 1)) * size + r * a.dim + min(c * 64 + lane, a.dim - 1)];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float f = i + k < n ? __shfl(weight, i + k) : 0.0f;
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (c * 64 < a.dim) value[c] = __builtin_fmaf(x[k][c], f, value[c]);
            }
        }
    }
    total = wave_sum(total);
    half_t* const out = a.out.at(b, h) + query * a.out.token;
#pragma unroll
    for (int c = 0; c < 4; ++c)
        if (c * 64 + lane < a.dim) {
            const int64_t at = (int64_t)(c * 64 + lane) * a.out.unit;
            const float x = total == 0.0f ? 0.0f : value[c] / total;
            const half_t r = round_f16(x);
            out[at] = r;
            if (a.lse) a.rest[out - a.out.p + at] = (half_t)((x - (float)r) * kRest);
        }
    if (a.lse && lane == 0) a.lse[(b * a.heads + h) * a.tokens + query] = total == 0.0f ? __builtin_inff() : base - kLift + __builtin_amdgcn_logf(total);
}

// Which kernel a call takes, and how it is divided.  k_attn_few, where units are neighbours, up to 32 rows of a head of keys (8 x 32 heads on 8 of 128, 4096 keys, 4 to 32 rows: 29 to 33 us
// and k_attn 53 to 55; 32 x 16 heads of 64, 1024 keys, one head a head of keys: 23 to 26 and 23 to 24), and where four heads or more share one, up to 192 rows of up to 32 queries: k_attn goes
// over the keys once for each head, with 128 rows for a handful (8 x 32 heads on 8 of 64, 4096 keys, 36, 64, 128 rows: 25, 26, 30 us and 45, 45, 49; 2 x 32 on 4 of 128, 16384 keys, 192 and
// 256 rows: 43, 55 and 55, 56; two heads that share: 48 and 64 rows 18, 19 and 18, 19; of 256 units 64 rows 31 and 25).  Elsewhere keys are cut into as many parts as let the device's
// compute units each have two workgroups, of four tiles at least.
AttnPlan attn_plan(int64_t batch, int64_t heads, int64_t held, int64_t tokens, int32_t dim, int64_t length, bool rows_of_keys, bool train) {
    const int64_t of_head = tokens * (heads / held);
    const bool shared = heads >= 4 * held && tokens <= 32 && of_head <= 192 && dim <= 128;
    if (rows_of_keys && !train && (of_head <= 32 || shared) && dim % 8 == 0 && length > 0) {
        AttnPlan p = attn_few_plan(batch, held, of_head, dim, length);
        p.few = true;
        return p;
    }
    AttnPlan p;
    p.few = false, p.rows = kAttnRows, p.waves = 4, p.tile = kAttnTile, p.least = kAttnLeast;
    p.row_tiles = (int)ceil_div(tokens, kAttnRows);
    const int64_t base = batch * heads * p.row_tiles, tiles = ceil_div(length, kAttnTile), units = compute_units();
    p.splits = (int)std::max<int64_t>(1, std::min(2 * units / base, tiles / kAttnLeast));
    return p;
}

}  // namespace cpmk

using namespace cpmk;

extern "C" {

// (enough for either kernel: which one a call takes depends on its strides too)
int64_t cpmk_attention_forward_workspace(int32_t batch, int32_t heads, int32_t kv_heads, int32_t tokens, int32_t dim, int32_t length) {
    if (batch <= 0 || heads <= 0 || kv_heads <= 0 || tokens <= 0 || dim <= 0 || length <= 0 || heads % kv_heads) return 0;
    if (dim > 256 || tokens > kAttnLong || length > kAttnLong || !grid_fits((int64_t)batch * heads)) return 0;
    int64_t most = 0;
    for (int few = 0; few < 2; ++few) {
        const AttnPlan p = attn_plan(batch, heads, kv_heads, tokens, dim, length, few, false);
        if (p.splits > 1) most = std::max(most, (int64_t)batch * (p.few ? kv_heads : heads) * p.row_tiles * p.splits * p.rows * (dim + 2) * (int64_t)sizeof(float));
    }
    return most;
}

int cpmk_attention_forward(int32_t batch, int32_t heads, int32_t kv_heads, int32_t tokens, int32_t dim, int32_t length, const void* q, int64_t q_batch, int64_t q_head, int64_t q_token,
                           int64_t q_unit, const void* k, int64_t k_batch, int64_t k_head, int64_t k_token, int64_t k_unit, const void* v, int64_t v_batch, int64_t v_head, int64_t v_token,
                           int64_t v_unit, const void* lens_each, int32_t len, const void* pos_each, int32_t pos, int causal, float scale, const void* bias, const void* mapping,
                           int32_t num_buckets, int32_t max_distance, int bidirectional, const void* mask, int64_t mask_batch, int64_t mask_token, void* out, int64_t out_batch,
                           int64_t out_head, int64_t out_token, int64_t out_unit, void* lse, void* rest, void* workspace, void* stream) {
    clear_stale_error();
    Attention a;
    a.q = {(half_t*)q, q_batch, q_head, q_token, q_unit}, a.k = {(half_t*)k, k_batch, k_head, k_token, k_unit}, a.v = {(half_t*)v, v_batch, v_head, v_token, v_unit};
    a.out = {(half_t*)out, out_batch, out_head, out_token, out_unit};
    a.lens_each = (const int32_t*)lens_each, a.pos_each = (const int32_t*)pos_each, a.len = len, a.pos = pos;
    a.table = (const half_t*)bias, a.mapping = (const int32_t*)mapping, a.buckets = num_buckets, a.distances = max_distance;
    a.mask = (const uint8_t*)mask, a.mask_batch = mask_batch, a.mask_token = mask_token;
    a.lse = (float*)lse, a.rest = (half_t*)rest, a.scale = scale * kLog2e, a.causal = causal != 0;
    a.tokens = tokens, a.dim = dim, a.length = length;
    bool empty;
    if (int e = attn_check(a, batch, heads, kv_heads, bidirectional, empty)) return e;
    if (empty || tokens == 0) return 0;
    if (lse && !rest) return CPMK_EBADARG;
    const AttnPlan plan = attn_plan(batch, heads, kv_heads, tokens, dim, length, k_unit == 1 && v_unit == 1 && !(mask && length < 4), lse != nullptr);          // (of masks k_attn_few reads four bytes at a time)
    a.row_tiles = plan.row_tiles, a.splits = plan.splits, a.parts = (float*)workspace;
    if (a.splits > 1 && !workspace) return CPMK_EBADARG;
    const int64_t grid = (int64_t)batch * heads * a.row_tiles * a.splits, rows = (int64_t)batch * heads * tokens;
    if (!grid_fits(grid) || !grid_fits(rows)) return CPMK_ETOOBIG;
    a.rows_in_all = rows;
    hipStream_t st = (hipStream_t)stream;
    const unsigned g = (unsigned)grid;
    const int e = plan.few    ? attn_few_launch(a, plan, batch, st)
                  : dim <= 64 ? attn_launch_64(a, g, st)
                  : dim <= 96 ? attn_launch_96(a, g, st)
                  : dim <= 128 ? attn_launch_128(a, g, st)
                               : attn_launch_256(a, g, st);
    if (e) return e;
    if (a.splits > 1) hipLaunchKernelGGL(k_attn_join, dim3((unsigned)ceil_div(rows, 4)), dim3(256), 0, st, a, plan, (uint32_t)rows);
    return launch_status();
}

}  // extern "C"
