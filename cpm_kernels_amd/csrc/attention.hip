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
// backward pass subtracts two nearly equal numbers where a query looks at one key, do_i v_j and do_i out_i, and the second has to be as exact as the first.  Where there are few rows the keys are cut into parts, which k_attn_join adds up.
#include <algorithm>
#include "attention.h"

namespace cpmk {

constexpr int kAttnRows = 128, kAttnLeast = 4;       // queries of a workgroup; tiles of a part, at least
constexpr int kLazy = 8;            // log2 of how far the running maximum may lie below the true one
constexpr float kLift = 7.0f;       // log2 of the largest probability's size right behind a change of the maximum

template <int NT, bool BIAS, int LAY, bool TRAIN>
__global__ __launch_bounds__(256, NT <= 4 ? 2 : 1) void k_attn(Attention a) {
    constexpr int D = NT <= 2 ? 64 : NT <= 4 ? 128 : 256, KS = NT * 2, kTileBytes = kAttnTile * D * 2;
    extern __shared__ __attribute__((aligned(128))) int8_t lds[];        // two buffers of keys, two of values, biases
    __shared__ uint32_t bad[3][2];              // tokens of a tile whose values are no finite numbers; those of tile t in t % 3
    __shared__ uint32_t mask_bits[2][kAttnRows][2];
    __shared__ __attribute__((aligned(16))) float mask_caps[2][kAttnTile];
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    float* const biases = reinterpret_cast<float*>(lds + 4 * kTileBytes);
    const uint32_t inner = (uint32_t)a.group * a.row_tiles * a.splits;
    uint32_t unit, w;
    attn_deal(blockIdx.x, gridDim.x / inner, inner, unit, w);
    const int64_t b = unit / (uint32_t)a.held;
    const int32_t kvh = unit - (uint32_t)b * a.held;
    const int32_t split = w % (uint32_t)a.splits;
    w /= (uint32_t)a.splits;
    // (of a causal chunk the last queries see most keys: their workgroups come first)
    const int32_t qt = a.row_tiles - 1 - (int32_t)(w % (uint32_t)a.row_tiles);
    const int32_t h = kvh * a.group + w / (uint32_t)a.row_tiles;
    const AttnRange range = attn_range(a, b);
    const AttnParts parts = attn_parts(a, range, min(qt * kAttnRows + kAttnRows - 1, a.tokens - 1), kAttnLeast, kAttnTile);
    const bool looks = TRAIN && qt == a.row_tiles - 1 && h == kvh * a.group;         // for the largest magnitude of the values: the workgroup whose queries see most keys of a head
    if (split >= parts.parts) {
        if (looks && tid == 0) a.lse[a.rows_in_all + (b * a.held + kvh) * a.splits + split] = 0.0f;
        return;
    }

    const int32_t q_first = qt * kAttnRows + wave * 32;
    const int32_t query = min(q_first + col, a.tokens - 1);         // (queries past the end repeat the last one)
    const int32_t where = range.pos + query, limit = a.causal ? min(range.len, where + 1) : range.len;
    // what all and what any of the wave's queries see, and what all of the workgroup's do
    const int32_t last = min(q_first + 31, a.tokens - 1);
    const int32_t all_see = a.causal ? min(range.len, range.pos + min(q_first, a.tokens - 1) + 1) : range.len;
    const int32_t any_sees = q_first >= a.tokens ? 0 : a.causal ? min(range.len, range.pos + last + 1) : range.len;
    const int32_t every_sees = a.causal ? min(range.len, range.pos + qt * kAttnRows + 1) : range.len;
    const float scale = a.scale == 0.0f ? 1.0f : fabsf(a.scale);         // (of queries times its sign: the largest score is the largest product)
    const bool masked = a.mask != nullptr;
    const half_t *const keys = a.k.at(b, kvh), *const values = a.v.at(b, kvh);
    const bool each = masked && a.mask_token != 0;          // a row of the mask for each query, or one for all
    const uint8_t* const mask = masked ? a.mask + b * a.mask_batch + min(qt * kAttnRows + (tid >> 1), a.tokens - 1) * a.mask_token : nullptr;

    // Keys, and the mask's bits, come a tile before the values: scores of the next tile are formed beside this one's sums.
    const int32_t t_begin = split * parts.per_part, t_end = min(t_begin + parts.per_part, parts.tiles);
    AttnTiles<D, LAY> ks, vs;
    ks.init(keys, a.k, a.dim, tid, wave, lane);
    vs.init(values, a.v, a.dim, tid, wave, lane);
    AttnMaskShare ms;
    ushort8_t largest = {0, 0, 0, 0, 0, 0, 0, 0};
    const auto guarded = [&](int32_t t) { return masked || (t + 1) * kAttnTile > every_sees; };       // (a value that is no finite number must not reach the queries that do not see it)
    auto fetch = [&](int32_t t) __attribute__((always_inline)) {
        if (t + 1 < t_end) {
            ks.fetch(lds + ((t + 1) & 1) * kTileBytes, a.dim, (t + 1) * kAttnTile, range.len, tid, wave, lane);
            if (each) ms.load(mask, (t + 1) * kAttnTile + (tid & 1) * 32, a.length);
            else if (masked && tid < kAttnTile) ms.byte = mask[min((t + 1) * kAttnTile + tid, a.length - 1)];
        }
        if (t >= t_begin && t < t_end) vs.fetch(lds + (2 + (t & 1)) * kTileBytes, a.dim, t * kAttnTile, range.len, tid, wave, lane);
    };
    if (tid < 6) bad[tid >> 1][tid & 1] = 0;
    if (LAY == kDirect && a.dim < D) {
        attn_clear(lds, 4 * kTileBytes, tid, 256);
        __syncthreads();
    }
    if (LAY != kDirect) fetch(t_begin - 1);
    half8_t q[KS];
    if (LAY == kColumns && a.q.token == 1) {
        attn_bring_columns<D>(a.q, a.q.at(b, h), qt * kAttnRows, a.tokens, a.dim, tid, lds + 2 * kTileBytes);
        __syncthreads();
        attn_keep_columns<D, KS>(q, lds + 2 * kTileBytes, wave, lane);
    } else
        attn_keep<KS>(q, a.q, a.q.at(b, h) + query * a.q.token, a.dim, half);
    if (!(a.scale > 0.0f))
#pragma unroll
        for (int s = 0; s < KS; ++s) q[s] *= (half_t)(a.scale < 0.0f ? -1.0f : 0.0f);
    if (BIAS) attn_biases(a, h, scale, biases, tid, 256);
    __syncthreads();
    if (LAY == kDirect) fetch(t_begin - 1);

    const uint32_t at_rows = attn_rows_at<D>(lane), at_units = attn_units_at<D>(lane);
    float16_tv acc[NT], s[2];
    half8_t p[4], left[TRAIN ? 4 : 1];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n] = kZero16;
    float top = -__builtin_inff(), sum = 0.0f;
    auto scores_of = [&](int32_t t) {
        const int8_t* const tile = lds + (t & 1) * kTileBytes;
        if (BIAS) {
            const float* const first = attn_window(a, biases, where - t * kAttnTile, half);
            attn_begin(s[0], 0, first);
            attn_begin(s[1], 1, first);
        } else
            s[0] = s[1] = kZero16;
#pragma unroll
        for (int u = 0; u < KS; ++u)
#pragma unroll
            for (int blk = 0; blk < 2; ++blk) s[blk] = __builtin_amdgcn_mfma_f32_32x32x16_f16(attn_rows<D>(tile, at_rows, blk, u), q[u], s[blk], 0, 0, 0);
    };
    auto sums_of = [&](int32_t t) {
        const int8_t* const tile = lds + (2 + (t & 1)) * kTileBytes;
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const half8_t v = attn_units<D>(tile, at_units, n, e >> 1, e & 1);
                acc[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[e], acc[n], 0, 0, 0);
                if (TRAIN) acc[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, left[e], acc[n], 0, 0, 0);
            }
    };
    for (int32_t t = t_begin - 1; t < t_end; ++t) {
        const int32_t k0 = t * kAttnTile;
        const bool active = t >= t_begin && k0 < any_sees;
        if (active) {
            if (k0 + kAttnTile > all_see) {
                const int32_t seen = limit - k0 - half * 4;
#pragma unroll
                for (int blk = 0; blk < 2; ++blk)
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[blk][i] = blk * 32 + (i >> 2) * 8 + (i & 3) < seen ? s[blk][i] : -__builtin_inff();
            }
            if (masked) {
#pragma unroll
                for (int blk = 0; blk < 2; ++blk) {
                    if (each) attn_cap_each(s[blk], mask_bits[t & 1][wave * 32 + col][blk] >> (half * 4));
                    else attn_cap(s[blk], blk, half, mask_caps[t & 1]);
                }
            }
            float m = s[0][0];
#pragma unroll
            for (int blk = 0; blk < 2; ++blk)
#pragma unroll
                for (int j = 0; j < 16; ++j) m = fmaxf(m, s[blk][j]);
            m *= scale;
            {
                const auto both = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, m), __builtin_bit_cast(uint32_t, m), false, false);
                const uint32_t low = both[0], high = both[1];       // (a bit cast of a vector's element itself takes the first one's)
                m = fmaxf(__builtin_bit_cast(float, low), __builtin_bit_cast(float, high));
            }
            if (__builtin_amdgcn_ballot_w64(m > top + kLazy)) {
                const float now = fmaxf(m, top), f = now == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(top - now);
                top = now;
                sum *= f;
#pragma unroll
                for (int n = 0; n < NT; ++n) acc[n] *= f;
            }
            const float shift = kLift - (top == -__builtin_inff() ? 0.0f : top);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float part = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e >> 1][(e & 1) * 8 + j], scale, shift));
                    part += x;
                    p[e][j] = (half_t)x;
                    if (TRAIN) left[e][j] = (half_t)(x - (float)p[e][j]);
                }
                sum += part;
            }
        }
        if (LAY == kDirect) wait_vmcnt<0>();
        if (t + 1 < t_end) {
            ks.place(lds + ((t + 1) & 1) * kTileBytes, a.dim, (t + 1) * kAttnTile, range.len, tid, wave, lane, nullptr);
            if (each) mask_bits[(t + 1) & 1][tid >> 1][tid & 1] = ms.bits(mask, (t + 1) * kAttnTile + (tid & 1) * 32, a.length);
            else if (masked && tid < kAttnTile) mask_caps[(t + 1) & 1][tid] = ms.byte ? __builtin_inff() : -__builtin_inff();
        }
        if (t >= t_begin) {
            int8_t* const tile = lds + (2 + (t & 1)) * kTileBytes;
            if (looks) largest = vs.largest(largest, tile, wave, lane);
            vs.place(tile, a.dim, k0, range.len, tid, wave, lane, guarded(t) ? bad[(uint32_t)t % 3] : nullptr);
        }
        if (tid < 2) bad[(uint32_t)(t + 1) % 3][tid] = 0;          // (last looked at two tiles ago)
        if (LAY != kDirect) fetch(t + 1);
        __syncthreads();
        if (LAY == kDirect) fetch(t + 1);
        if (active) {           // (behind the last tile: scores that nobody looks at)
            const uint32_t spoilt[2] = {bad[(uint32_t)t % 3][0], bad[(uint32_t)t % 3][1]};
            if (spoilt[0] | spoilt[1]) {        // a query that sees such a key has no number for a result
                bool sees = false;
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int j = 0; j < 8; ++j) sees |= (spoilt[e >> 1] >> (half * 4 + (e & 1) * 16 + (j >> 2) * 8 + (j & 3)) & 1) && !(p[e][j] == (half_t)0);
                if (sees) sum = __builtin_nanf("");
            }
            sums_of(t);
            scores_of(t + 1);
            attn_pace<4 * NT * (TRAIN ? 2 : 1), 8 * NT, 2 * KS, BIAS ? 16 : 0>();
        } else if ((t + 1) * kAttnTile < any_sees && t + 1 < t_end) {
            scores_of(t + 1);
            attn_pace<0, 0, 2 * KS, BIAS ? 16 : 0>();
        }
    }
    sum += __shfl_xor(sum, 32);
    __syncthreads();            // (the tiles are done with)
    if (looks) {
        // (numbers that are none or infinite count as the largest one: the keys past the end among them are zeros or copies)
        const uint32_t m = wave_max_u32(min(absbits_max_of(largest), 0x7bffu));
        if (lane == 0) bad[0][0] = 0;
        __syncthreads();
        if (lane == 0) atomicMax(&bad[0][0], m);
        __syncthreads();
        if (tid == 0) a.lse[a.rows_in_all + (b * a.held + kvh) * a.splits + split] = (float)__builtin_bit_cast(half_t, (uint16_t)bad[0][0]);
    }
    const bool real = q_first + col < a.tokens;
    const int64_t row = (b * a.heads + h) * a.tokens + query;
    if (a.splits > 1) {
        if (!real) return;
        struct __attribute__((packed, aligned(4))) Float4Any { float x, y, z, w; };         // (a workspace is aligned to 4 bytes)
        float* const part = a.parts + (((b * a.heads + h) * a.row_tiles + qt) * a.splits + split) * kAttnRows * (a.dim + 2);
        const int r = wave * 32 + col;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int u = n * 32 + c * 8 + half * 4;
                if (u + 4 <= a.dim) *reinterpret_cast<Float4Any*>(part + r * a.dim + u) = Float4Any{acc[n][c * 4], acc[n][c * 4 + 1], acc[n][c * 4 + 2], acc[n][c * 4 + 3]};
                else
                    for (int e = 0; e < 4; ++e)
                        if (u + e < a.dim) part[r * a.dim + u + e] = acc[n][c * 4 + e];
            }
        if (half == 0) {
            part[kAttnRows * a.dim + r] = top;
            part[kAttnRows * a.dim + kAttnRows + r] = sum;
        }
        return;
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    int8_t* const own = lds + wave * D * 80;
    attn_write<NT>(a.out, a.out.at(b, h), acc, inv, q_first, a.tokens, a.dim, lane, own);
    if (!TRAIN) return;
    attn_write<NT, true>(a.out, a.rest + (a.out.at(b, h) - a.out.p), acc, inv, q_first, a.tokens, a.dim, lane, own);
    if (real && half == 0) a.lse[row] = sum == 0.0f ? __builtin_inff() : top - kLift + __builtin_amdgcn_logf(sum);
}

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

// Which kernel a call takes, and how it is divided.  Keys are cut into as many parts as let the device's compute units each have a workgroup, of four tiles at least.
AttnPlan attn_plan(int64_t batch, int64_t heads, int64_t held, int64_t tokens, int32_t dim, int64_t length, bool rows_of_keys, bool train) {
    const int64_t of_head = tokens * (heads / held);
    if (rows_of_keys && !train && of_head <= 32 && dim % 8 == 0 && length > 0) {
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

template <int NT, bool BIAS, int LAY, bool TRAIN>
static int attn_launch(const Attention& a, unsigned grid, hipStream_t st) {
    constexpr int D = NT <= 2 ? 64 : NT <= 4 ? 128 : 256;
    const int lds = 4 * kAttnTile * D * 2 + (a.table ? (a.distances - a.first_distance + 2 * kBiasPad) * 4 : 0);
    static std::atomic<bool> done[64];
    if (int e = enable_dynamic_lds((const void*)k_attn<NT, BIAS, LAY, TRAIN>, 150 * 1024, done)) return e;
    hipLaunchKernelGGL((k_attn<NT, BIAS, LAY, TRAIN>), dim3(grid), dim3(256), lds, st, a);
    return 0;
}
template <int NT, bool BIAS, int LAY>
static int attn_launch(const Attention& a, unsigned grid, hipStream_t st) {
    return a.lse ? attn_launch<NT, BIAS, LAY, true>(a, grid, st) : attn_launch<NT, BIAS, LAY, false>(a, grid, st);
}
template <int NT, bool BIAS>
static int attn_launch(const Attention& a, unsigned grid, hipStream_t st) {
    const int lay = attn_layout(a.k, a.v, a.dim);
    return lay == kDirect ? attn_launch<NT, BIAS, kDirect>(a, grid, st) : lay == kColumns ? attn_launch<NT, BIAS, kColumns>(a, grid, st) : attn_launch<NT, BIAS, kAnyLayout>(a, grid, st);
}
template <int NT>
static int attn_launch(const Attention& a, unsigned grid, hipStream_t st) {
    return a.table ? attn_launch<NT, true>(a, grid, st) : attn_launch<NT, false>(a, grid, st);
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
    const AttnPlan plan = attn_plan(batch, heads, kv_heads, tokens, dim, length, k_unit == 1 && v_unit == 1, lse != nullptr);
    a.row_tiles = plan.row_tiles, a.splits = plan.splits, a.parts = (float*)workspace;
    if (a.splits > 1 && !workspace) return CPMK_EBADARG;
    const int64_t grid = (int64_t)batch * heads * a.row_tiles * a.splits, rows = (int64_t)batch * heads * tokens;
    if (!grid_fits(grid) || !grid_fits(rows)) return CPMK_ETOOBIG;
    a.rows_in_all = rows;
    hipStream_t st = (hipStream_t)stream;
    const unsigned g = (unsigned)grid;
    const int e = plan.few    ? attn_few_launch(a, plan, batch, st)
                  : dim <= 64 ? attn_launch<2>(a, g, st)
                  : dim <= 96 ? attn_launch<3>(a, g, st)
                  : dim <= 128 ? attn_launch<4>(a, g, st)
                               : attn_launch<8>(a, g, st);
    if (e) return e;
    if (a.splits > 1) hipLaunchKernelGGL(k_attn_join, dim3((unsigned)ceil_div(rows, 4)), dim3(256), 0, st, a, plan, (uint32_t)rows);
    return launch_status();
}

}  // extern "C"
