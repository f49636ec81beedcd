// k_attn_dq and k_attn_dkv of attention_bwd.hip (the mathematics: there), compiled for each size of heads by itself.
//
// Both bound by products beside vector operations.  Measured, 1 x 32 heads on 8, 8192 tokens, dim 128, causal: k_attn_dq 850 us (0.97 PFLOP/s of its three products), k_attn_dkv 1680 (0.65 of
// its four: one wave a SIMD, its products 32 % of the cycles); 8 x 64 heads of 64, 512 tokens, causal, biases with their gradient: 121 and 126 us.
#pragma once
#include "attention.h"

namespace cpmk {

struct AttentionGrad : Attention {
    AttnTensor dout, dq, dk, dv;
    float *delta, *dout_top;                    // D (batch, heads, tokens), the square of the largest norm of a workgroup's gradients (batch, heads, row_tiles): k_attn_dq's, for k_attn_dkv
    float* table_parts;                         // (batch, heads, row_tiles, entries by distance) or null
    half_t* dtable;
    float natural_scale;
    int64_t batch;
    int32_t query_tiles;
};

constexpr int kGradRows = 128;      // queries (k_attn_dq) or keys (k_attn_dkv) of a workgroup
constexpr float kProbScale = 15.0f;
template <int NT>
constexpr int kGradBuffers = NT <= 4 ? 3 : 2;         // tiles of k_attn_dkv in LDS: three take one barrier a tile (of 256 units two fit)
template <int NT>
constexpr int kDiagonals = (NT <= 4 ? 32 : 4) * 36 + 32;         // floats of a wave's buffer for diagonals: rows of 36, read up to 31 before and behind

// The largest of n numbers, for the whole wave
__device__ __forceinline__ float attn_largest(const float* x, int64_t n, int lane) {
    float m = 0.0f;
    for (int64_t i = lane; i < n; i += 64) m = fmaxf(m, x[i]);
    return wave_max(m);
}
// A bound of the norms of a head's values, squared, from their largest magnitude
__device__ __forceinline__ float attn_value_norm(const AttentionGrad& a, int64_t b, int64_t kvh, int lane) {
    const float m = attn_largest(a.lse + a.rows_in_all + (b * a.held + kvh) * a.splits, a.splits, lane);
    return m * m * (float)a.dim;
}
// log2 of the factor that brings 2 sqrt(squares) to at most 1: with a probability of at most 2^15, ds to at most 2^15
__device__ __forceinline__ int attn_exponent(float dout_square, float value_square) {
    const float bound = 2.0f * (__builtin_sqrtf(dout_square) * __builtin_sqrtf(value_square));
    return bound > 0.0f && bound < __builtin_inff() ? -max(-100, min(__builtin_amdgcn_frexp_expf(bound), 100)) : 0;
}

template <int NT, bool BIAS, bool MASK, int LAY>
__global__ __launch_bounds__(256, NT <= 4 ? 2 : 1) void k_attn_dq(AttentionGrad a) {
    constexpr int D = NT <= 2 ? 64 : NT <= 4 ? 128 : 256, KS = NT * 2, kTileBytes = kAttnTile * D * 2;
    extern __shared__ __attribute__((aligned(128))) int8_t lds[];        // two buffers of keys and values; biases; sums of ds by distance, of each wave
    __shared__ uint32_t bad[3][2];              // tokens of a tile whose keys (and, masked, values) are no finite numbers; those of tile t in t % 3
    __shared__ uint32_t mask_bits[2][kGradRows][2];
    __shared__ float tops[4];
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t inner = (uint32_t)a.group * a.row_tiles;
    uint32_t unit, w;
    attn_deal(blockIdx.x, gridDim.x / inner, inner, unit, w);
    const int64_t b = unit / (uint32_t)a.held;
    const int32_t kvh = unit - (uint32_t)b * a.held;
    const int32_t qt = a.row_tiles - 1 - (int32_t)(w % (uint32_t)a.row_tiles);
    const int32_t h = kvh * a.group + w / (uint32_t)a.row_tiles;
    const AttnRange range = attn_range(a, b);
    const int32_t q_first = qt * kGradRows + wave * 32, q_last_of_all = min(qt * kGradRows + kGradRows - 1, a.tokens - 1);
    const bool real = q_first + col < a.tokens;
    const int32_t query = min(q_first + col, a.tokens - 1);
    const int32_t where = range.pos + query, limit = a.causal ? min(range.len, where + 1) : range.len;
    const int32_t last = min(q_first + 31, a.tokens - 1);
    const int32_t all_see = a.causal ? min(range.len, range.pos + min(q_first, a.tokens - 1) + 1) : range.len;
    const int32_t any_sees = q_first >= a.tokens ? 0 : a.causal ? min(range.len, range.pos + last + 1) : range.len;
    const int32_t every_sees = a.causal ? min(range.len, range.pos + qt * kGradRows + 1) : range.len;
    const int32_t keys_seen = a.causal ? max(0, min(range.len, range.pos + q_last_of_all + 1)) : range.len;
    const int32_t tiles = (keys_seen + kAttnTile - 1) / kAttnTile;
    constexpr bool BY_UNIT = kByUnit<LAY>, ARRIVES = LAY == kDirect || LAY == kTurned;
    const bool masked = MASK && (ARRIVES || a.mask != nullptr), table_wanted = BIAS && a.table_parts != nullptr;
    const float scale = a.scale == 0.0f ? 1.0f : a.scale;
    const uint8_t* const mask = masked ? a.mask + b * a.mask_batch + min(qt * kGradRows + (tid >> 1), a.tokens - 1) * a.mask_token : nullptr;
    const half_t *const keys = a.k.at(b, kvh), *const values = a.v.at(b, kvh);
    const int64_t row = (b * a.heads + h) * a.tokens + query;

    AttnTiles<D, LAY> ks, vs;
    ks.init(keys, a.k, a.length, a.dim, tid, wave, lane);
    vs.init(values, a.v, a.length, a.dim, tid, wave, lane);
    AttnMaskShare<ARRIVES> ms;
    const auto guarded = [&](int32_t t) { return masked || (t + 1) * kAttnTile > every_sees; };       // (a key that is no finite number must not reach the queries that do not see it)
    auto fetch = [&](int32_t t) __attribute__((always_inline)) {
        if (masked) ms.load(mask, t * kAttnTile + (tid & 1) * 32, a.length);
        if (t >= tiles) return;
        int8_t* const buffer = lds + (t & 1) * 2 * kTileBytes;
        ks.fetch(buffer, a.dim, t * kAttnTile, range.len, tid, wave, lane);
        vs.fetch(buffer + kTileBytes, a.dim, t * kAttnTile, range.len, tid, wave, lane);
    };
    auto place = [&](int32_t t) __attribute__((always_inline)) {
        if (t >= tiles) return;
        int8_t* const buffer = lds + (t & 1) * 2 * kTileBytes;
        if (ARRIVES) wait_vmcnt<0>();
        ks.place(buffer, a.dim, t * kAttnTile, range.len, tid, wave, lane, guarded(t) ? bad[(uint32_t)t % 3] : nullptr);
        vs.place(buffer + kTileBytes, a.dim, t * kAttnTile, range.len, tid, wave, lane, masked ? bad[(uint32_t)t % 3] : nullptr);        // (0 times no number is none)
        if (masked) mask_bits[t & 1][tid >> 1][tid & 1] = ms.bits(mask, t * kAttnTile + (tid & 1) * 32, a.length);
        if (tid < 2) bad[(uint32_t)(t + 1) % 3][tid] = 0;
    };
    if (tid < 6) bad[tid >> 1][tid & 1] = 0;
    // (queries that come through LDS themselves take its room first)
    const bool brings = BY_UNIT && a.q.token == 1 && a.out.token == 1 && a.dout.token == 1;
    auto begin = [&]() __attribute__((always_inline)) {
        if (ARRIVES && a.dim < D) {
            attn_clear(lds, 4 * kTileBytes, tid, 256);
            __syncthreads();
        }
        fetch(0);
    };
    if (!ARRIVES || !brings) begin();
    float* const biases = reinterpret_cast<float*>(lds + 4 * kTileBytes);
    const int entries = BIAS ? attn_bias_entries(a) : 0;
    float* const sums = biases + entries + wave * entries;
    if (BIAS) attn_biases(a, h, scale, biases, tid, 256);
    if (table_wanted)
        for (int i = tid; i < 4 * entries; i += 256) biases[entries + i] = 0.0f;
    const int32_t lo_rel = a.first_distance - kBiasPad;
    constexpr int DIAG = NT <= 4 ? 32 : 4;          // rows of a block that are summed along their diagonals at a time (256 units leave no more LDS)
    float* const diagonals = biases + 5 * ((entries + 3) & ~3) + wave * kDiagonals<NT>;

    half8_t q[KS], g[KS];
    float minus_delta, minus_lse, dscale, undo;
    {
        // D from the result and what its rounding left; the factor of ds from the norms
        float square = 0.0f, delta = 0.0f, little = 0.0f;
        auto first = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    square = __builtin_fmaf((float)g[s][e], (float)g[s][e], square);
                    delta = __builtin_fmaf((float)g[s][e], (float)q[s][e], delta);
                }
        };
        auto second = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int e = 0; e < 8; ++e) little = __builtin_fmaf((float)g[s][e], (float)q[s][e], little);
        };
        const half_t *const of_out = a.out.at(b, h), *const of_rest = a.rest + (of_out - a.out.p);
        if (brings) {
            const auto bring = [&](const AttnTensor& x, const half_t* base, int at) __attribute__((always_inline)) {
                attn_bring_columns<D>(x, base, qt * kGradRows, a.tokens, a.dim, tid, lds + at * kTileBytes);
            };
            bring(a.dout, a.dout.at(b, h), 0);
            bring(a.out, of_out, 2);
            __syncthreads();
            attn_keep_columns<D, KS>(g, lds, wave, lane);
            attn_keep_columns<D, KS>(q, lds + 2 * kTileBytes, wave, lane);
            first();
            __syncthreads();
            bring(a.out, of_rest, 0);
            bring(a.q, a.q.at(b, h), 2);
            __syncthreads();
            attn_keep_columns<D, KS>(q, lds, wave, lane);
            second();
            attn_keep_columns<D, KS>(q, lds + 2 * kTileBytes, wave, lane);
        } else {
            attn_keep<KS>(g, a.dout, a.dout.at(b, h) + query * a.dout.token, a.dim, half);
            attn_keep<KS>(q, a.out, of_out + query * a.out.token, a.dim, half);
            first();
            attn_keep<KS>(q, a.out, of_rest + query * a.out.token, a.dim, half);
            second();
            attn_keep<KS>(q, a.q, a.q.at(b, h) + query * a.q.token, a.dim, half);
        }
        delta = __builtin_fmaf(little, 1.0f / kRest, delta);
        square += __shfl_xor(square, 32);
        delta += __shfl_xor(delta, 32);
        if (real && half == 0) a.delta[row] = delta;
        const int exponent = attn_exponent(square, attn_value_norm(a, b, kvh, lane));
        dscale = ldexpf(1.0f, exponent);
        undo = ldexpf(1.0f, -exponent - (int)kProbScale);
        const float lse = real ? a.lse[row] : __builtin_inff();
        // (of queries that see a key, with gradients that are numbers: the others' are none, or make their keys' none, whatever the factor is)
        const float largest = wave_max(lse != __builtin_inff() && square < __builtin_inff() ? square : 0.0f);
        if (lane == 0) tops[wave] = largest;
        minus_lse = kProbScale - lse;
        minus_delta = lse == __builtin_inff() ? 0.0f : -delta * dscale;
        if (lse == __builtin_inff())            // (a query without keys: its result's gradients count for nothing, numbers or none)
#pragma unroll
            for (int s = 0; s < KS; ++s) g[s] = half8_t{0, 0, 0, 0, 0, 0, 0, 0};
    }
    if (a.scale == 0.0f)
#pragma unroll
        for (int s = 0; s < KS; ++s) q[s] *= (half_t)0;
    __syncthreads();
    if (tid == 0) a.dout_top[(b * a.heads + h) * a.row_tiles + qt] = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    if (ARRIVES && brings) begin();
    place(0);
    if (!ARRIVES) fetch(1);
    __syncthreads();
    if (ARRIVES) fetch(1);

    const uint32_t at_rows = attn_rows_at<D, BY_UNIT>(lane), at_units = attn_units_at<D, BY_UNIT>(lane);
    float16_tv acc[NT], s, dp;
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n] = kZero16;
    float far_before = 0.0f, far_behind = 0.0f;         // ds of keys beyond the table's ends: far before the query, far behind it
    half8_t d[2];
    auto scores_of = [&](int32_t t, int blk) __attribute__((always_inline)) {
        const int8_t* const tile = lds + (t & 1) * 2 * kTileBytes;
        s = dp = kZero16;
        if (BIAS) attn_begin(s, 0, attn_window(a, biases, where - t * kAttnTile - blk * 32, half));
#pragma unroll
        for (int u = 0; u < KS; ++u) {
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(attn_rows<D, BY_UNIT>(tile, at_rows, blk, u), q[u], s, 0, 0, 0);
            dp = __builtin_amdgcn_mfma_f32_32x32x16_f16(attn_rows<D, BY_UNIT>(tile + kTileBytes, at_rows, blk, u), g[u], dp, 0, 0, 0);
        }
    };
    auto sums_of = [&](int32_t t, int blk) __attribute__((always_inline)) {
        const int8_t* const tile = lds + (t & 1) * 2 * kTileBytes;
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(attn_units<D, BY_UNIT>(tile, at_units, n, blk, e), d[e], acc[n], 0, 0, 0);
    };
    // ds of a block of 32 keys, as fp16
    auto gradients_of = [&](int32_t t, int blk) __attribute__((always_inline)) {
        const int32_t k0 = t * kAttnTile + blk * 32;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = __builtin_fmaf(s[i], scale, minus_lse);
        if (masked) {
            const uint32_t bits = mask_bits[t & 1][wave * 32 + col][blk];
            if (__builtin_amdgcn_ballot_w64(bits != ~0u)) attn_cap(s, bits >> (half * 4));
        }
        const uint32_t spoilt = bad[(uint32_t)t % 3][blk];
        if (k0 + 32 > all_see || spoilt) {
            const int32_t seen = limit - k0 - half * 4;
            const uint32_t none = spoilt >> (half * 4);        // (a query that sees such a key has no number for a gradient)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int j = (i >> 2) * 8 + (i & 3);
                const bool sees = j < seen && s[i] != -__builtin_inff();
                s[i] = none & (1u << j) ? __builtin_nanf("") : s[i];
                s[i] = sees ? s[i] : -__builtin_inff();
                dp[i] = sees ? dp[i] : 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(s[i]) * __builtin_fmaf(dp[i], dscale, minus_delta);
        if (table_wanted) {
            const int32_t rel_min = range.pos + q_first - (k0 + 31), rel_max = range.pos + last - k0;
            const int32_t rel_of_corner = rel_min - lo_rel;         // of the block's first query from its last key
            const bool before = rel_min >= a.distances - 1;
            if (!before && rel_max > a.first_distance) {
                // Through LDS: a lane writes its 16 keys beside each other, a row a query, and then sums a diagonal, lane l that of distance l - 31 from the block's corner.  (64 float
                // additions in LDS itself, which has an instruction for them, took ten times as long as the block's products.)  All of it is the wave's own.
#pragma unroll
                for (int pass = 0; pass < 32 / DIAG; ++pass) {
                    if (DIAG == 32 || col / DIAG == pass) {
                        float* const p = diagonals + (col % DIAG) * 36 + half * 4;
                        const float f = real ? undo : 0.0f;
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            *reinterpret_cast<float4_t*>(p + c * 8) = float4_t{s[c * 4] * f, s[c * 4 + 1] * f, s[c * 4 + 2] * f, s[c * 4 + 3] * f};
                    }
                    asm volatile("" ::: "memory");
                    float total = 0.0f;
                    const float* const from = diagonals + pass * DIAG + 31 - lane;
#pragma unroll
                    for (int r = 0; r < DIAG; ++r) {
                        const float x = from[r * 37];
                        total += (uint32_t)(pass * DIAG + r + 31 - lane) < 32u ? x : 0.0f;
                    }
                    sums[rel_of_corner + lane] += total;
                    asm volatile("" ::: "memory");
                }
            } else {
                float far = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) far += s[i];
                if (before) far_before += far;
                else far_behind += far;
            }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) d[i >> 3][i & 7] = (half_t)s[i];
    };
    if (0 < any_sees) {
        scores_of(0, 0);
        attn_pace<0, 0, 2 * KS, 2 * KS * (BY_UNIT ? 2 : 1), BIAS ? 8 : 0>();
    }
    for (int32_t t = 0; t < tiles; ++t) {
        const bool one = t * kAttnTile < any_sees;          // (the second block of the tile: scores that nobody sees, or zeros)
        if (one) {
            gradients_of(t, 0);
            sums_of(t, 0);
            scores_of(t, 1);
            attn_pace<2 * NT, 4 * NT, 2 * KS, 2 * KS * (BY_UNIT ? 2 : 1), BIAS ? 8 : 0>();
            gradients_of(t, 1);
            sums_of(t, 1);
            attn_pace<2 * NT, 4 * NT, 0, 0>();
        }
        place(t + 1);
        if (!ARRIVES) fetch(t + 2);
        __syncthreads();
        if (ARRIVES) fetch(t + 2);
        if ((t + 1) * kAttnTile < any_sees) {
            scores_of(t + 1, 0);
            attn_pace<0, 0, 2 * KS, 2 * KS * (BY_UNIT ? 2 : 1), BIAS ? 8 : 0>();
        }
    }
    attn_write<NT>(a.dq, a.dq.at(b, h), acc, undo * a.natural_scale, q_first, a.tokens, a.dim, lane, lds + wave * D * 80);
    if (!table_wanted) return;
    far_before = wave_sum(real ? far_before * undo : 0.0f);
    far_behind = wave_sum(real ? far_behind * undo : 0.0f);
    if (lane == 0) {
        sums[a.distances - 1 - lo_rel] += far_before;
        sums[a.first_distance - lo_rel] += far_behind;
    }
    __syncthreads();
    float* const out = a.table_parts + ((b * a.heads + h) * a.row_tiles + qt) * entries;
    for (int i = tid; i < entries; i += 256) {
        float total = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) total += biases[entries * (1 + j) + i];
        out[i] = total;
    }
}

// The gradient of a head's biases: sums by distance over all tiles of rows, then by bucket, in a fixed order.  A workgroup of k_attn_dkv's launch.
__device__ __forceinline__ void attn_dtable(const AttentionGrad& a, int64_t h, float* by_distance, int tid) {
    const int entries = attn_bias_entries(a), lane = tid & 63, wave = tid >> 6;
    int32_t* const buckets = reinterpret_cast<int32_t*>(by_distance + entries);
    for (int i = tid; i < entries; i += 256) {
        float total = 0.0f;
        for (int64_t b = 0; b < a.batch; ++b) {
            const float* const p = a.table_parts + (b * a.heads + h) * a.row_tiles * entries + i;
#pragma unroll 4
            for (int32_t r = 0; r < a.row_tiles; ++r) total += p[(int64_t)r * entries];
        }
        by_distance[i] = total;
        buckets[i] = attn_bucket(a, max(a.first_distance, min(i + a.first_distance - kBiasPad, a.distances - 1)));
    }
    __syncthreads();
    for (int n = wave; n < a.buckets; n += 4) {
        float total = 0.0f;
        for (int i = lane; i < entries; i += 64) total += buckets[i] == n ? by_distance[i] : 0.0f;
        total = wave_sum(total);
        if (lane == 0) a.dtable[h * a.buckets + n] = (half_t)total;
    }
}

template <int NT, bool BIAS, bool MASK, int LAY>
__global__ __launch_bounds__(256, NT <= 2 ? 2 : 1) void k_attn_dkv(AttentionGrad a, uint32_t blocks) {
    constexpr int D = NT <= 2 ? 64 : NT <= 4 ? 128 : 256, KS = NT * 2, kTileBytes = kAttnTile * D * 2;
    constexpr int BUFS = kGradBuffers<NT>;
    extern __shared__ __attribute__((aligned(128))) int8_t lds[];        // BUFS buffers of queries and their results' gradients; biases of the heads in turn
    __shared__ uint32_t bad[4][2];              // queries of a tile that are no finite numbers, or their gradients; those of tile t in t % 4
    __shared__ __attribute__((aligned(16))) float facts[BUFS][2][kAttnTile];        // 15 - lse and -D of a tile's queries
    __shared__ __attribute__((aligned(16))) uint32_t mask_bits[BUFS][4][kAttnTile];
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (BIAS && blockIdx.x >= blocks) return attn_dtable(a, blockIdx.x - blocks, reinterpret_cast<float*>(lds), tid);
    const uint32_t inner = (uint32_t)ceil_div(a.length, kGradRows);
    uint32_t unit, kt;
    attn_deal(blockIdx.x, blocks / inner, inner, unit, kt);         // (of causal keys the first are seen by most queries)
    const int64_t b = unit / (uint32_t)a.held;
    const int32_t kvh = unit - (uint32_t)b * a.held;
    const AttnRange range = attn_range(a, b);
    const int32_t k_first_of_all = kt * kGradRows, k_first = k_first_of_all + wave * 32, key = k_first + col;
    constexpr bool BY_UNIT = kByUnit<LAY>, ARRIVES = LAY == kDirect || LAY == kTurned;
    const bool masked = MASK && a.mask != nullptr && a.mask_token != 0;         // (by a row for each query)
    constexpr bool kMaskAlways = MASK && ARRIVES;          // read, without a branch
    const uint8_t* const mask = kMaskAlways || masked ? a.mask + b * a.mask_batch : nullptr;
    const float scale = a.scale == 0.0f ? 1.0f : fabsf(a.scale);         // (of keys times its sign: a score of -inf stays one)
    // tiles of queries that see any key of the workgroup
    const int32_t first_query = a.causal ? max(0, k_first_of_all - range.pos) : 0;
    const int32_t first_tile = min(first_query / kAttnTile, a.query_tiles);
    const int32_t of_head = k_first_of_all < range.len && first_query < a.tokens ? a.query_tiles - first_tile : 0;

    half8_t k[KS], v[KS];
    if (BY_UNIT && a.k.token == 1 && a.v.token == 1) {
        attn_bring_columns<D>(a.k, a.k.at(b, kvh), k_first_of_all, a.length, a.dim, tid, lds);
        attn_bring_columns<D>(a.v, a.v.at(b, kvh), k_first_of_all, a.length, a.dim, tid, lds + 2 * kTileBytes);
        __syncthreads();
        attn_keep_columns<D, KS>(k, lds, wave, lane);
        attn_keep_columns<D, KS>(v, lds + 2 * kTileBytes, wave, lane);
    } else {
        const int32_t mine = min(key, a.length - 1);
        attn_keep<KS>(k, a.k, a.k.at(b, kvh) + mine * a.k.token, a.dim, half);
        attn_keep<KS>(v, a.v, a.v.at(b, kvh) + mine * a.v.token, a.dim, half);
    }
    // Keys past the end, and keys that one mask for all queries leaves out: zeros, their scores -inf
    const bool out_of_all = key >= range.len || (MASK && a.mask != nullptr && a.mask_token == 0 && a.mask[b * a.mask_batch + min(key, a.length - 1)] == 0);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        if (out_of_all) k[s] = v[s] = half8_t{0, 0, 0, 0, 0, 0, 0, 0};
        if (!(a.scale > 0.0f)) k[s] *= (half_t)(a.scale < 0.0f ? -1.0f : 0.0f);
    }
    const float of_lane = out_of_all ? -__builtin_inff() : 0.0f;
    const bool some_out = k_first_of_all + kGradRows > range.len || (MASK && a.mask != nullptr && a.mask_token == 0);       // (the same for the whole workgroup)
    const float dout_top = attn_largest(a.dout_top + (b * a.heads + kvh * a.group) * a.row_tiles, (int64_t)a.group * a.row_tiles, lane);
    const int exponent = attn_exponent(dout_top, attn_value_norm(a, b, kvh, lane));
    const float dscale = ldexpf(1.0f, exponent);
    float* const biases = reinterpret_cast<float*>(lds + 2 * BUFS * kTileBytes);
    const int32_t lo_rel = a.first_distance - kBiasPad;
    if (tid < 8) bad[tid >> 1][tid & 1] = 0;
    if (ARRIVES) __syncthreads();
    if (ARRIVES && a.dim < D) {
        attn_clear(lds, 2 * BUFS * kTileBytes, tid, 256);
        __syncthreads();
    }

    AttnTiles<D, LAY> qs, gs;
    qs.init(a.q.at(b, kvh * a.group), a.q, a.tokens, a.dim, tid, wave, lane);
    gs.init(a.dout.at(b, kvh * a.group), a.dout, a.tokens, a.dim, tid, wave, lane);
    AttnMaskShare<ARRIVES> ms;
    float lse = 0.0f, delta = 0.0f;
    int32_t h_fetch = kvh * a.group, t_fetch = 0, t_place = 0;       // head and tile of the head to be fetched next, the tile to be placed next
    int32_t left = of_head * a.group;           // tiles still to be fetched
    uint32_t phase_place = 0;           // of `bad`
    const auto guarded = [&](int32_t q0) { return masked || q0 + kAttnTile > a.tokens || some_out || (a.causal && range.pos + q0 < min(k_first_of_all + kGradRows, range.len) - 1); };
    auto fetch = [&](int buffer) __attribute__((always_inline)) {
        const int32_t q0 = (first_tile + t_fetch) * kAttnTile;
        if (kMaskAlways || masked) ms.load(mask + min(q0 + (tid >> 2), a.tokens - 1) * a.mask_token, k_first_of_all + (tid & 3) * 32, a.length);
        if (left == 0) return;
        int8_t* const at = lds + buffer * 2 * kTileBytes;
        qs.fetch(at, a.dim, q0, a.tokens, tid, wave, lane);
        gs.fetch(at + kTileBytes, a.dim, q0, a.tokens, tid, wave, lane);
        // (as they are, and without a branch: to look at them here would be to wait for the tile)
        const int64_t row = (b * a.heads + h_fetch) * a.tokens + min(q0 + (tid & 63), a.tokens - 1);
        lse = a.lse[row];
        delta = a.delta[row];
        if (++t_fetch == of_head) {
            t_fetch = 0, ++h_fetch;
            qs.advance(a.q.head);
            gs.advance(a.dout.head);
        }
        --left;
    };
    auto place = [&](int buffer) __attribute__((always_inline)) {
        const int32_t q0 = (first_tile + t_place) * kAttnTile;
        uint32_t* const spoilt = guarded(q0) ? bad[phase_place] : nullptr;
        int8_t* const at = lds + buffer * 2 * kTileBytes;
        if (ARRIVES) wait_vmcnt<0>();
        qs.place(at, a.dim, q0, a.tokens, tid, wave, lane, spoilt);
        gs.place(at + kTileBytes, a.dim, q0, a.tokens, tid, wave, lane, spoilt);
        if (masked) mask_bits[buffer][tid & 3][tid >> 2] = ms.bits(mask + min(q0 + (tid >> 2), a.tokens - 1) * a.mask_token, k_first_of_all + (tid & 3) * 32, a.length);
        if (tid < 128) {
            // (a query whose statistics are no numbers, like one that is none itself, must not reach the keys that it does not see)
            const float none = tid < 64 ? -__builtin_inff() : 0.0f;
            const float fact = q0 + (tid & 63) >= a.tokens || lse == __builtin_inff() ? none : tid < 64 ? kProbScale - lse : -delta * dscale;
            const bool spoils = fact != none && !(fabsf(fact) < __builtin_inff());
            facts[buffer][tid >> 6][tid & 63] = spoils ? none : fact;
            if (spoils) atomicOr(&bad[phase_place][(tid & 63) >> 5], 1u << (tid & 31));
        }
        if (++t_place == of_head) t_place = 0;
        phase_place = (phase_place + 1) & 3;
        if (tid < 2) bad[phase_place][tid] = 0;         // (last looked at before the barrier of the tile before)
    };
    const uint32_t at_rows = attn_rows_at<D, BY_UNIT>(lane), at_units = attn_units_at<D, BY_UNIT>(lane);
    constexpr bool ROOM = NT == 3 || NT == 4;         // for registers: one wave a SIMD (65 to 128 units: all of a block's facts before it, operands six ahead; the others, less of both, spill)
    constexpr bool AHEAD = NT <= 4;         // scores of a block beside the one before (256 units leave no registers for that)
    float16_tv dk[NT], dv[NT], s[AHEAD ? 2 : 1], dp[AHEAD ? 2 : 1];
#pragma unroll
    for (int n = 0; n < NT; ++n) dk[n] = dv[n] = kZero16;
    half8_t p[2], d[2];
    auto begin_of = [&](int32_t q0, int blk) __attribute__((always_inline)) {
        s[blk & AHEAD] = dp[blk & AHEAD] = kZero16;
        if (BIAS) {         // (windows beyond the table's ends are moved into the entries of the end that they are beyond)
            const float* const bp = biases + max(0, min(range.pos + q0 + blk * 32 + half * 4 - key - lo_rel, attn_bias_entries(a) - 32));
#pragma unroll
            for (int i = 0; i < 16; ++i) s[blk & AHEAD][i] = bp[(i >> 2) * 8 + (i & 3)];
        }
    };
    auto scores_of = [&](const int8_t* tile, int32_t q0, int blk) __attribute__((always_inline)) {
        begin_of(q0, blk);
#pragma unroll
        for (int u = 0; u < KS; ++u) {
            s[blk & AHEAD] = __builtin_amdgcn_mfma_f32_32x32x16_f16(attn_rows<D, BY_UNIT>(tile, at_rows, blk, u), k[u], s[blk & AHEAD], 0, 0, 0);
            dp[blk & AHEAD] = __builtin_amdgcn_mfma_f32_32x32x16_f16(attn_rows<D, BY_UNIT>(tile + kTileBytes, at_rows, blk, u), v[u], dp[blk & AHEAD], 0, 0, 0);
        }
    };
    // Scores of pairs that do not count become -inf
    auto mask_of = [&](int buffer, uint32_t turn, int32_t q0, int blk) __attribute__((always_inline)) {
        q0 += blk * 32;
        const uint32_t spoilt = bad[turn][blk];
        if (!(masked || spoilt || q0 + 32 > a.tokens || (a.causal && range.pos + q0 - (k_first + 31) < 0))) return;
        // of the block's queries (from the lane's first on) those from `least` on see the key, up to the last one
        const int32_t end = a.tokens - q0 - half * 4;
        const int32_t least = out_of_all ? 64 : a.causal ? key - (range.pos + q0 + half * 4) : -64;
        const uint32_t none = spoilt >> (half * 4);        // (a key that such a query sees has no number for a gradient)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            uint4_t bits = {~0u, ~0u, ~0u, ~0u};
            if (masked) bits = *reinterpret_cast<const uint4_t*>(&mask_bits[buffer][wave][blk * 32 + c * 8 + half * 4]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = c * 4 + e, j = c * 8 + e;
                const bool sees = j >= least && j < end && (bits[e] & (1u << col));
                s[blk & AHEAD][i] = none & (1u << j) ? __builtin_nanf("") : s[blk & AHEAD][i];
                s[blk & AHEAD][i] = sees ? s[blk & AHEAD][i] : -__builtin_inff();
                dp[blk & AHEAD][i] = sees ? dp[blk & AHEAD][i] : 0.0f;
            }
        }
    };
    // A block's p and ds, as fp16, beside the products of the next one's scores, then its sums.  One wave a SIMD is all that 128 units leave registers for, so the order is written out:
    // operands are read kAhead products before theirs, and numbers are dealt out among the products (8 x 64 heads of 512 tokens, dim 64: 151 us with the scores before the numbers, 126 so).
    auto block = [&](int buffer, uint32_t turn, int32_t q0, int blk, const int8_t* next, int32_t next_q0) __attribute__((always_inline)) {
        constexpr int kAhead = ROOM ? 6 : 4, kFacts = ROOM ? 4 : 2, kScores = 2 * KS, kSums = 4 * NT, kPairs = 8;
        const int8_t* const tile = lds + buffer * 2 * kTileBytes;
        float4_t minus_lse[kFacts], minus_delta[kFacts];         // of four queries, and of the next ones
        const auto facts_of = [&](int c) __attribute__((always_inline)) {
            minus_lse[c % kFacts] = *reinterpret_cast<const float4_t*>(&facts[buffer][0][blk * 32 + c * 8 + half * 4]);
            minus_delta[c % kFacts] = *reinterpret_cast<const float4_t*>(&facts[buffer][1][blk * 32 + c * 8 + half * 4]);
        };
        if (!AHEAD) {
            scores_of(tile, q0, blk);
            attn_pace<0, 0, kScores, kScores * (BY_UNIT ? 2 : 1), BIAS ? 8 : 0>();
        }
        mask_of(buffer, turn, q0, blk);
#pragma unroll
        for (int c = 0; c < kFacts - 1; ++c) facts_of(c);
        const int now = blk & AHEAD, then = now ^ AHEAD;
        const auto operand = [&](int i) __attribute__((always_inline)) {
            if (i < kScores) return attn_rows<D, BY_UNIT>(next + (i & 1) * kTileBytes, at_rows, blk ^ 1, i >> 1);
            i -= kScores;
            return attn_units<D, BY_UNIT>(tile + (i & 1 ? 0 : kTileBytes), at_units, (i % (2 * NT)) >> 1, blk, i / (2 * NT));
        };
        const auto numbers = [&](int i) __attribute__((always_inline)) {
            const int c = i >> 1;
            if (i % 2 == 0 && c + kFacts - 1 < 4) facts_of(c + kFacts - 1);
#pragma unroll
            for (int e = 2 * i; e < 2 * i + 2; ++e) {
                const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[now][e], scale, minus_lse[c % kFacts][e & 3] + of_lane));
                p[e >> 3][e & 7] = (half_t)x;
                d[e >> 3][e & 7] = (half_t)(x * __builtin_fmaf(dp[now][e], dscale, minus_delta[c % kFacts][e & 3]));
            }
        };
        constexpr int kFrom = AHEAD ? 0 : kScores;
        if (AHEAD && BIAS) begin_of(next_q0, blk ^ 1);
        half8_t ring[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) ring[i] = operand(kFrom + i);
        if (!AHEAD)
#pragma unroll
            for (int i = 0; i < kPairs; ++i) numbers(i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = kFrom; i < kScores + kSums; ++i) {
            half8_t& x = ring[(i - kFrom) % kAhead];
            if (i < kScores) {
                float16_tv& sum = i & 1 ? dp[then] : s[then];
                sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, (i & 1 ? v : k)[i >> 1], i == 1 || (i == 0 && !BIAS) ? kZero16 : sum, 0, 0, 0);
            } else {
                const int j = i - kScores, e = j / (2 * NT), n = (j % (2 * NT)) >> 1;
                float16_tv& sum = j & 1 ? dk[n] : dv[n];
                sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, (j & 1 ? d : p)[e], sum, 0, 0, 0);
            }
            if (i + kAhead < kScores + kSums) x = operand(i + kAhead);
            if (i < kScores)
#pragma unroll
                for (int j = kPairs * i / kScores; j < kPairs * (i + 1) / kScores; ++j) numbers(j);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    const int32_t total = of_head * a.group;
    fetch(0);
    if (BIAS && total > 0) attn_biases(a, kvh * a.group, scale, biases, tid, 256);
    __syncthreads();
    if (total > 0) place(0);
    if (!ARRIVES) fetch(1);
    __syncthreads();
    if (ARRIVES) fetch(1);
    const auto looked_at = [&](int32_t q0) { return k_first < range.len && (!a.causal || range.pos + q0 + kAttnTile - 1 >= k_first); };
    int buffer = 0;
    int32_t t = 0, g = 0;
    bool active = total > 0 && looked_at(first_tile * kAttnTile);
    if (AHEAD && active) scores_of(lds, first_tile * kAttnTile, 0);
    for (int32_t i = 0; i < total; ++i) {
        const int32_t q0 = (first_tile + t) * kAttnTile;
        if (active) block(buffer, i & 3, q0, 0, lds + buffer * 2 * kTileBytes, q0);
        const int next = buffer + 1 == BUFS ? 0 : buffer + 1;
        if (++t == of_head) t = 0, ++g;
        const bool other_head = BIAS && t == 0 && i + 1 < total;
        if (AHEAD && other_head) {
            __syncthreads();
            attn_biases(a, kvh * a.group + g, scale, biases, tid, 256);
        }
        // (with three buffers the one that is fetched into was last read before this barrier; scores behind the last tile are of what the buffer held, and nobody looks at them)
        const int32_t next_q0 = (first_tile + t) * kAttnTile;
        if (i + 1 < total) place(next);
        if (BUFS == 3 && !ARRIVES) fetch(0);
        __syncthreads();
        if (BUFS == 3 && ARRIVES) fetch(next + 1 == BUFS ? 0 : next + 1);
        if (active) block(buffer, i & 3, q0, 1, lds + next * 2 * kTileBytes, next_q0);
        const bool was = active;
        active = i + 1 < total && looked_at(next_q0);
        if (AHEAD && active && !was) scores_of(lds + next * 2 * kTileBytes, next_q0, 0);
        if (BUFS == 2) {
            if (!ARRIVES) fetch(0);
            __syncthreads();
            if (!AHEAD && other_head) {
                attn_biases(a, kvh * a.group + g, scale, biases, tid, 256);
                __syncthreads();
            }
            if (ARRIVES) fetch(buffer);
        }
        buffer = next;
    }
    __syncthreads();
    int8_t* const own = lds + wave * D * 80;
    attn_write<NT>(a.dk, a.dk.at(b, kvh), dk, ldexpf(a.natural_scale, -exponent - (int)kProbScale), k_first, a.length, a.dim, lane, own);
    attn_write<NT>(a.dv, a.dv.at(b, kvh), dv, ldexpf(1.0f, -(int)kProbScale), k_first, a.length, a.dim, lane, own);
}

template <int NT, bool BIAS, bool MASK, int LAY>
static int dq_launch(const AttentionGrad& a, unsigned grid, hipStream_t st) {
    constexpr int D = NT <= 2 ? 64 : NT <= 4 ? 128 : 256;
    const int entries = a.table ? a.distances - a.first_distance + 2 * kBiasPad : 0;
    const int lds = 4 * kAttnTile * D * 2 + (a.table_parts ? 5 * ((entries + 3) & ~3) + 4 * kDiagonals<NT> : entries) * 4;
    static std::atomic<bool> done[64];
    if (int e = enable_dynamic_lds((const void*)k_attn_dq<NT, BIAS, MASK, LAY>, 156 * 1024, done)) return e;
    hipLaunchKernelGGL((k_attn_dq<NT, BIAS, MASK, LAY>), dim3(grid), dim3(256), lds, st, a);
    return 0;
}
template <int NT, bool BIAS, bool MASK, int LAY>
static int dkv_launch(const AttentionGrad& a, unsigned grid, unsigned more, hipStream_t st) {
    constexpr int D = NT <= 2 ? 64 : NT <= 4 ? 128 : 256;
    const int lds = 2 * kGradBuffers<NT> * kAttnTile * D * 2 + (a.table ? (a.distances - a.first_distance + 2 * kBiasPad) * 4 : 0);
    static std::atomic<bool> done[64];
    if (int e = enable_dynamic_lds((const void*)k_attn_dkv<NT, BIAS, MASK, LAY>, 150 * 1024, done)) return e;
    hipLaunchKernelGGL((k_attn_dkv<NT, BIAS, MASK, LAY>), dim3(grid + more), dim3(256), lds, st, a, grid);
    return 0;
}
// (a mask is looked for in a call's arguments where tiles come through registers)
template <int NT, bool BIAS>
static int grad_launch(const AttentionGrad& a, unsigned dq_grid, unsigned dkv_grid, hipStream_t st) {
    if (dq_grid) {
        const int lay = a.mask && a.length < 32 ? kAnyLayout : attn_layout(a.k, a.v, a.dim, a.length);
        const int e = lay == kDirect    ? a.mask ? dq_launch<NT, BIAS, true, kDirect>(a, dq_grid, st) : dq_launch<NT, BIAS, false, kDirect>(a, dq_grid, st)
                      : lay == kTurned  ? a.mask ? dq_launch<NT, BIAS, true, kTurned>(a, dq_grid, st) : dq_launch<NT, BIAS, false, kTurned>(a, dq_grid, st)
                      : lay == kColumns ? dq_launch<NT, BIAS, true, kColumns>(a, dq_grid, st)
                                        : dq_launch<NT, BIAS, true, kAnyLayout>(a, dq_grid, st);
        if (e) return e;
    }
    const unsigned more = a.dtable ? a.heads : 0;
    if (dkv_grid + more == 0) return 0;
    const int lay = a.mask && a.length < 32 ? kAnyLayout : attn_layout(a.q, a.dout, a.dim, a.tokens);
    return lay == kDirect    ? a.mask ? dkv_launch<NT, BIAS, true, kDirect>(a, dkv_grid, more, st) : dkv_launch<NT, BIAS, false, kDirect>(a, dkv_grid, more, st)
           : lay == kTurned  ? a.mask ? dkv_launch<NT, BIAS, true, kTurned>(a, dkv_grid, more, st) : dkv_launch<NT, BIAS, false, kTurned>(a, dkv_grid, more, st)
           : lay == kColumns ? dkv_launch<NT, BIAS, true, kColumns>(a, dkv_grid, more, st)
                             : dkv_launch<NT, BIAS, true, kAnyLayout>(a, dkv_grid, more, st);
}
template <int NT>
static int grad_launch(const AttentionGrad& a, unsigned dq_grid, unsigned dkv_grid, hipStream_t st) {
    return a.table ? grad_launch<NT, true>(a, dq_grid, dkv_grid, st) : grad_launch<NT, false>(a, dq_grid, dkv_grid, st);
}

// (attention_64.hip and so on)
int attn_grad_launch_64(const AttentionGrad& a, unsigned dq_grid, unsigned dkv_grid, hipStream_t st);
int attn_grad_launch_96(const AttentionGrad& a, unsigned dq_grid, unsigned dkv_grid, hipStream_t st);
int attn_grad_launch_128(const AttentionGrad& a, unsigned dq_grid, unsigned dkv_grid, hipStream_t st);
int attn_grad_launch_256(const AttentionGrad& a, unsigned dq_grid, unsigned dkv_grid, hipStream_t st);

}  // namespace cpmk
