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
// k_attn_facts finds D and the largest norms.
#include <algorithm>
#include "attention.h"

namespace cpmk {

struct AttentionGrad : Attention {
    AttnTensor dout, dq, dk, dv;
    float *delta, *dout_top, *value_top;        // (batch, heads, tokens); squares of the largest norms of 64 tokens: (batch, heads, query_tiles), (batch, held, key_tiles)
    float* table_parts;                         // (batch, heads, row_tiles, entries by distance) or null
    half_t* dtable;
    float natural_scale;
    int32_t query_tiles, key_tiles;
};

constexpr int kGradRows = 128;      // queries (k_attn_dq) or keys (k_attn_dkv) of a workgroup
constexpr float kProbScale = 15.0f;

// D of 64 queries, or nothing, and the largest norm of 64 queries' gradients or of 64 keys' values.
__global__ __launch_bounds__(256) void k_attn_facts(AttentionGrad a, uint32_t query_blocks) {
    __shared__ float sums[2][4][64];
    const int tid = threadIdx.x;
    const bool of_queries = blockIdx.x < query_blocks;
    const uint32_t id = of_queries ? blockIdx.x : blockIdx.x - query_blocks;
    const uint32_t tiles = of_queries ? a.query_tiles : a.key_tiles, heads = of_queries ? a.heads : a.held;
    const uint32_t tile = id % tiles, bh = id / tiles;
    const int64_t b = bh / heads, h = bh % heads;
    const AttnTensor x = of_queries ? a.dout : a.v, y = a.out;
    const int32_t tokens = of_queries ? a.tokens : attn_range(a, b).len;
    // (four threads a token, in the order in which neighbouring ones read neighbouring addresses)
    const bool columns = x.token == 1;
    const int mine = columns ? tid & 63 : tid >> 2, part = columns ? tid >> 6 : tid & 3;
    const int32_t t = tile * 64 + mine;
    float square = 0.0f, dot = 0.0f;
    if (t < tokens) {
        const half_t *const px = x.at(b, h) + t * x.token, *const py = y.at(b, h) + t * y.token, *const pr = a.rest + (py - y.p);
        for (int u = part * 8; u < a.dim; u += 32) {
            half8_t vx, vy = {0, 0, 0, 0, 0, 0, 0, 0}, vr = vy;
            if (x.unit == 1 && u + 8 <= a.dim) vx = load_half8_any(px + u);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) vx[e] = u + e < a.dim ? px[(u + e) * x.unit] : (half_t)0;
            if (of_queries) {
                if (y.unit == 1 && u + 8 <= a.dim) vy = load_half8_any(py + u), vr = load_half8_any(pr + u);
                else
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (u + e < a.dim) vy[e] = py[(u + e) * y.unit], vr[e] = pr[(u + e) * y.unit];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                square = __builtin_fmaf((float)vx[e], (float)vx[e], square);
                dot = __builtin_fmaf((float)vx[e], __builtin_fmaf((float)vr[e], 1.0f / kRest, (float)vy[e]), dot);
            }
        }
    }
    sums[0][part][mine] = square;
    sums[1][part][mine] = dot;
    __syncthreads();
    if (tid >= 64) return;
    square = (sums[0][0][tid] + sums[0][1][tid]) + (sums[0][2][tid] + sums[0][3][tid]);
    if (of_queries && (int32_t)(tile * 64) + tid < tokens) a.delta[(int64_t)bh * a.tokens + tile * 64 + tid] = (sums[1][0][tid] + sums[1][1][tid]) + (sums[1][2][tid] + sums[1][3][tid]);
    square = wave_max(square);
    if (tid == 0) (of_queries ? a.dout_top : a.value_top)[(int64_t)bh * tiles + tile] = square;
}

// The largest of n numbers, for the whole wave
__device__ __forceinline__ float attn_largest(const float* x, int64_t n, int lane) {
    float m = 0.0f;
    for (int64_t i = lane; i < n; i += 64) m = fmaxf(m, x[i]);
    return wave_max(m);
}
// log2 of the factor that brings 2 sqrt(squares) to at most 1: with a probability of at most 2^15, ds to at most 2^15
__device__ __forceinline__ int attn_exponent(float dout_square, float value_square) {
    const float bound = 2.0f * (__builtin_sqrtf(dout_square) * __builtin_sqrtf(value_square));
    return bound > 0.0f && bound < __builtin_inff() ? -max(-100, min(__builtin_amdgcn_frexp_expf(bound), 100)) : 0;
}

template <int NT, bool PLAIN, int LAY>
__global__ __launch_bounds__(256, NT <= 4 ? 2 : 1) void k_attn_dq(AttentionGrad a) {
    constexpr int D = NT <= 2 ? 64 : NT <= 4 ? 128 : 256, KS = NT * 2, kTileBytes = kAttnTile * D * 2;
    extern __shared__ __attribute__((aligned(128))) int8_t lds[];        // two buffers of keys and values; biases; sums of ds by distance, of each wave
    __shared__ int32_t bad[2][kAttnTile + 1];
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
    const bool masked = !PLAIN && a.mask != nullptr, biased = !PLAIN && a.table != nullptr, table_wanted = !PLAIN && a.table_parts != nullptr;
    const uint8_t* const mask = masked ? a.mask + b * a.mask_batch + query * a.mask_token : nullptr;
    const half_t *const keys = a.k.at(b, kvh), *const values = a.v.at(b, kvh);
    const int64_t row = (b * a.heads + h) * a.tokens + query;

    half8_t q[KS], g[KS];
    attn_keep<KS>(q, a.q, a.q.at(b, h) + query * a.q.token, a.dim, half);
    attn_keep<KS>(g, a.dout, a.dout.at(b, h) + query * a.dout.token, a.dim, half);
    const float lse = real ? a.lse[row] : __builtin_inff();
    const float value_top = attn_largest(a.value_top + (b * a.held + kvh) * a.key_tiles, a.key_tiles, lane);
    float square = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) square = __builtin_fmaf((float)g[s][e], (float)g[s][e], square);
    square += __shfl_xor(square, 32);
    const int exponent = attn_exponent(square, value_top);
    const float dscale = ldexpf(1.0f, exponent), undo = ldexpf(1.0f, -exponent - (int)kProbScale);
    const float minus_delta = lse == __builtin_inff() ? 0.0f : -a.delta[row] * dscale, minus_lse = kProbScale - lse;

    float* const biases = reinterpret_cast<float*>(lds + 4 * kTileBytes);
    const int entries = biased ? attn_bias_entries(a) : 0;
    float* const sums = biases + entries + wave * entries;
    if (biased) attn_biases(a, h, biases, tid, 256);
    if (table_wanted)
        for (int i = tid; i < 4 * entries; i += 256) biases[entries + i] = 0.0f;
    const int32_t lo_rel = a.first_distance - kBiasPad;
    if (tid <= kAttnTile) bad[0][tid] = bad[1][tid] = -1;

    AttnShare<D, LAY, 256> ks, vs;
    auto load = [&](int32_t t) {
        ks.load(keys, a.k.token, a.k.unit, a.dim, t * kAttnTile, range.len, tid);
        vs.load(values, a.v.token, a.v.unit, a.dim, t * kAttnTile, range.len, tid);
    };
    auto store = [&](int32_t t) {
        ks.clean(a.dim, t * kAttnTile, range.len, tid, masked || t * kAttnTile + kAttnTile > every_sees, bad[t & 1], t);
        vs.clean(a.dim, t * kAttnTile, range.len, tid, false, nullptr, t);
        int8_t* const buffer = lds + (t & 1) * 2 * kTileBytes;
        ks.store(buffer, tid);
        vs.store(buffer + kTileBytes, tid);
    };
    if (tiles > 0) load(0);
    __syncthreads();
    if (tiles > 0) {
        store(0);
        if (tiles > 1) load(1);
    }
    __syncthreads();

    const uint32_t at_rows = attn_rows_at<D>(lane), at_units = attn_units_at<D>(lane);
    float16_tv acc[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n] = kZero16;
    float far_before = 0.0f, far_behind = 0.0f;         // ds of keys beyond the table's ends: far before the query, far behind it
    for (int32_t t = 0; t < tiles; ++t) {
        const int32_t k0 = t * kAttnTile;
        const int8_t* const key_tile = lds + (t & 1) * 2 * kTileBytes;
        const int8_t* const value_tile = key_tile + kTileBytes;
        if (k0 < any_sees) {
            const int32_t rel_min = range.pos + q_first - (k0 + kAttnTile - 1), rel_max = range.pos + last - k0;
            const bool near = biased && rel_min < a.distances - 1 && rel_max > a.first_distance, before = rel_min >= a.distances - 1;
            float add = minus_lse;
            if (biased && !near) add += biases[(before ? a.distances - 1 : a.first_distance) - lo_rel];
            const bool spoilt = bad[t & 1][kAttnTile] == t;
            const bool partial = masked || near || spoilt || k0 + kAttnTile > all_see;
            float far = 0.0f;
#pragma unroll
            for (int blk = 0; blk < 2; ++blk) {
                float16_tv s = kZero16, dp = kZero16;
#pragma unroll
                for (int u = 0; u < KS; ++u) {
                    s = __builtin_amdgcn_mfma_f32_32x32x16_f16(attn_rows<D>(key_tile, at_rows, blk, u), q[u], s, 0, 0, 0);
                    dp = __builtin_amdgcn_mfma_f32_32x32x16_f16(attn_rows<D>(value_tile, at_rows, blk, u), g[u], dp, 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = __builtin_fmaf(s[i], a.scale, add);
                if (partial) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int32_t key = k0 + blk * 32 + c * 8 + half * 4;
                        uint32_t keep = 0x01010101u;
                        if (masked) keep = attn_mask4(mask, key, a.length);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float x = s[c * 4 + e];
                            if (near) x += biases[where - key - e - lo_rel];
                            if (spoilt && bad[t & 1][key + e - k0] == t) x = __builtin_nanf("");
                            const bool seen = key + e < limit && (keep >> (8 * e) & 0xffu);
                            s[c * 4 + e] = seen ? x : -__builtin_inff();
                            dp[c * 4 + e] = seen ? dp[c * 4 + e] : 0.0f;
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(s[i]) * __builtin_fmaf(dp[i], dscale, minus_delta);
                if (table_wanted) {
                    if (near) {
                        // (32 lanes, 32 distances: no two meet, and no other wave; a wave's operations on LDS keep their order, so each sum's terms do)
                        float* const sum = sums + (where - k0 - blk * 32 - half * 4 - lo_rel);
                        if (real && half == 0)
#pragma unroll
                            for (int i = 0; i < 16; ++i) atomicAdd(sum - (i >> 2) * 8 - (i & 3), s[i] * undo);
                        if (real && half == 1)
#pragma unroll
                            for (int i = 0; i < 16; ++i) atomicAdd(sum - (i >> 2) * 8 - (i & 3), s[i] * undo);
                    } else
#pragma unroll
                        for (int i = 0; i < 16; ++i) far += s[i];
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    half8_t d;
#pragma unroll
                    for (int j = 0; j < 8; ++j) d[j] = (half_t)s[e * 8 + j];
#pragma unroll
                    for (int n = 0; n < NT; ++n) acc[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(attn_units<D>(key_tile, at_units, n, blk, e), d, acc[n], 0, 0, 0);
                }
            }
            if (before) far_before += far;
            else far_behind += far;
        }
        if (t + 1 < tiles) {
            store(t + 1);
            if (t + 2 < tiles) load(t + 2);
        }
        __syncthreads();
    }
    if (real) attn_write<NT>(a.dq, a.dq.at(b, h) + query * a.dq.token, acc, undo * a.natural_scale, a.dim, half);
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

// The gradient of a head's biases: sums by distance over all tiles of rows, then by bucket, in a fixed order.
__global__ __launch_bounds__(1024) void k_attn_dtable(AttentionGrad a, int64_t batch) {
    extern __shared__ float by_distance[];         // four times the entries, then their buckets
    const int tid = threadIdx.x, entries = attn_bias_entries(a), share = tid >> 8;
    int32_t* const buckets = reinterpret_cast<int32_t*>(by_distance + 4 * entries);
    const int64_t h = blockIdx.x, rows = batch * a.row_tiles;
    const int64_t from = rows * share / 4, to = rows * (share + 1) / 4;
    for (int i = tid & 255; i < entries; i += 256) {
        float total = 0.0f;
        for (int64_t r = from; r < to; ++r) total += a.table_parts[((r / a.row_tiles * a.heads + h) * a.row_tiles + r % a.row_tiles) * entries + i];
        by_distance[share * entries + i] = total;
        if (share == 0) buckets[i] = attn_bucket(a, max(a.first_distance, min(i + a.first_distance - kBiasPad, a.distances - 1)));
    }
    __syncthreads();
    for (int i = tid; i < entries; i += 1024) by_distance[i] = (by_distance[i] + by_distance[entries + i]) + (by_distance[2 * entries + i] + by_distance[3 * entries + i]);
    __syncthreads();
    for (int n = tid; n < a.buckets; n += 1024) {
        float total = 0.0f;
        for (int i = 0; i < entries; ++i) total += buckets[i] == n ? by_distance[i] : 0.0f;
        a.dtable[h * a.buckets + n] = (half_t)total;
    }
}

template <int NT, bool PLAIN, int LAY>
__global__ __launch_bounds__(256, NT <= 2 ? 2 : 1) void k_attn_dkv(AttentionGrad a) {
    constexpr int D = NT <= 2 ? 64 : NT <= 4 ? 128 : 256, KS = NT * 2, kTileBytes = kAttnTile * D * 2;
    extern __shared__ __attribute__((aligned(128))) int8_t lds[];        // two buffers of queries and their results' gradients; biases of the heads in turn
    __shared__ int32_t bad[2][kAttnTile + 1];
    __shared__ __attribute__((aligned(16))) float facts[2][2][kAttnTile];        // -lse + 15 and -D of a tile's queries
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t inner = (uint32_t)ceil_div(a.length, kGradRows);
    uint32_t unit, kt;
    attn_deal(blockIdx.x, gridDim.x / inner, inner, unit, kt);         // (of causal keys the first are seen by most queries)
    const int64_t b = unit / (uint32_t)a.held;
    const int32_t kvh = unit - (uint32_t)b * a.held;
    const AttnRange range = attn_range(a, b);
    const int32_t k_first_of_all = kt * kGradRows, k_first = k_first_of_all + wave * 32, key = k_first + col;
    const bool masked = !PLAIN && a.mask != nullptr, biased = !PLAIN && a.table != nullptr;
    // tiles of queries that see any key of the workgroup
    const int32_t first_query = a.causal ? max(0, k_first_of_all - range.pos) : 0;
    const int32_t first_tile = min(first_query / kAttnTile, a.query_tiles);
    const int32_t of_head = k_first_of_all < range.len && first_query < a.tokens ? a.query_tiles - first_tile : 0;
    const int32_t tiles = of_head * a.group;

    half8_t k[KS], v[KS];
    {
        const int32_t mine = min(key, a.length - 1);
        attn_keep<KS>(k, a.k, a.k.at(b, kvh) + mine * a.k.token, a.dim, half);
        attn_keep<KS>(v, a.v, a.v.at(b, kvh) + mine * a.v.token, a.dim, half);
    }
    const float value_top = attn_largest(a.value_top + (b * a.held + kvh) * a.key_tiles, a.key_tiles, lane);
    const float dout_top = attn_largest(a.dout_top + (b * a.heads + kvh * a.group) * a.query_tiles, (int64_t)a.group * a.query_tiles, lane);
    const int exponent = attn_exponent(dout_top, value_top);
    const float dscale = ldexpf(1.0f, exponent);
    float* const biases = reinterpret_cast<float*>(lds + 4 * kTileBytes);
    const int32_t lo_rel = a.first_distance - kBiasPad;
    if (tid <= kAttnTile) bad[0][tid] = bad[1][tid] = -1;

    AttnShare<D, LAY, 256> qs, gs;
    float fact = 0.0f;
    auto load = [&](int32_t t) {
        const int32_t h = kvh * a.group + t / of_head, q0 = (first_tile + t % of_head) * kAttnTile;
        qs.load(a.q.at(b, h), a.q.token, a.q.unit, a.dim, q0, a.tokens, tid);
        gs.load(a.dout.at(b, h), a.dout.token, a.dout.unit, a.dim, q0, a.tokens, tid);
        if (tid < 128) {
            const int32_t query = q0 + (tid & 63);
            const int64_t row = (b * a.heads + h) * a.tokens + min(query, a.tokens - 1);
            const float lse = query < a.tokens ? a.lse[row] : __builtin_inff();
            fact = tid < 64 ? kProbScale - lse : lse == __builtin_inff() ? 0.0f : -a.delta[row] * dscale;
        }
    };
    auto store = [&](int32_t t) {
        const int32_t q0 = (first_tile + t % of_head) * kAttnTile;
        const bool guard = masked || (a.causal && range.pos + q0 < min(k_first_of_all + kGradRows, range.len) - 1);
        qs.clean(a.dim, q0, a.tokens, tid, guard, bad[t & 1], t);
        gs.clean(a.dim, q0, a.tokens, tid, guard, bad[t & 1], t);
        int8_t* const buffer = lds + (t & 1) * 2 * kTileBytes;
        qs.store(buffer, tid);
        gs.store(buffer + kTileBytes, tid);
        if (tid < 128) facts[t & 1][tid >> 6][tid & 63] = fact;
    };
    if (tiles > 0) load(0);
    __syncthreads();
    if (tiles > 0) {
        store(0);
        if (tiles > 1) load(1);
    }
    __syncthreads();

    const uint32_t at_rows = attn_rows_at<D>(lane), at_units = attn_units_at<D>(lane);
    float16_tv dk[NT], dv[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) dk[n] = dv[n] = kZero16;
    for (int32_t t = 0; t < tiles; ++t) {
        const int32_t q0 = (first_tile + t % of_head) * kAttnTile;
        const int8_t* const query_tile = lds + (t & 1) * 2 * kTileBytes;
        const int8_t* const dout_tile = query_tile + kTileBytes;
        if (biased && t % of_head == 0) {
            __syncthreads();
            attn_biases(a, kvh * a.group + t / of_head, biases, tid, 256);
            __syncthreads();
        }
        if (k_first < range.len && (!a.causal || range.pos + q0 + kAttnTile - 1 >= k_first)) {
            const int32_t rel_min = range.pos + q0 - (k_first + 31), rel_max = range.pos + q0 + kAttnTile - 1 - k_first;
            const bool near = biased && rel_min < a.distances - 1 && rel_max > a.first_distance;
            float add = 0.0f;
            if (biased && !near) add = biases[(rel_min >= a.distances - 1 ? a.distances - 1 : a.first_distance) - lo_rel];
            const bool spoilt = bad[t & 1][kAttnTile] == t;
            const bool partial = masked || near || spoilt || k_first + 32 > range.len || (a.causal && rel_min < 0);
#pragma unroll
            for (int blk = 0; blk < 2; ++blk) {
                float16_tv s = kZero16, dp = kZero16;
#pragma unroll
                for (int u = 0; u < KS; ++u) {
                    s = __builtin_amdgcn_mfma_f32_32x32x16_f16(attn_rows<D>(query_tile, at_rows, blk, u), k[u], s, 0, 0, 0);
                    dp = __builtin_amdgcn_mfma_f32_32x32x16_f16(attn_rows<D>(dout_tile, at_rows, blk, u), v[u], dp, 0, 0, 0);
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const float4_t minus_lse = *reinterpret_cast<const float4_t*>(&facts[t & 1][0][blk * 32 + c * 8 + half * 4]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[c * 4 + e] = __builtin_fmaf(s[c * 4 + e], a.scale, minus_lse[e] + add);
                }
                if (partial) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int32_t in_tile = blk * 32 + (i >> 2) * 8 + half * 4 + (i & 3), query = q0 + in_tile, rel = range.pos + query - key;
                        float x = s[i];
                        if (near) x += biases[rel - lo_rel];
                        if (spoilt && bad[t & 1][in_tile] == t) x = __builtin_nanf("");
                        bool seen = key < range.len && query < a.tokens && (!a.causal || rel >= 0);
                        if (masked) seen = seen && a.mask[b * a.mask_batch + min(query, a.tokens - 1) * a.mask_token + min(key, a.length - 1)] != 0;
                        s[i] = seen ? x : -__builtin_inff();
                        dp[i] = seen ? dp[i] : 0.0f;
                    }
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    half8_t p, d;
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const float4_t minus_delta = *reinterpret_cast<const float4_t*>(&facts[t & 1][1][blk * 32 + e * 16 + c * 8 + half * 4]);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float x = __builtin_amdgcn_exp2f(s[e * 8 + c * 4 + j]);
                            p[c * 4 + j] = (half_t)x;
                            d[c * 4 + j] = (half_t)(x * __builtin_fmaf(dp[e * 8 + c * 4 + j], dscale, minus_delta[j]));
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        dv[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(attn_units<D>(dout_tile, at_units, n, blk, e), p, dv[n], 0, 0, 0);
                        dk[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(attn_units<D>(query_tile, at_units, n, blk, e), d, dk[n], 0, 0, 0);
                    }
                }
            }
        }
        if (t + 1 < tiles) {
            store(t + 1);
            if (t + 2 < tiles) load(t + 2);
        }
        __syncthreads();
    }
    if (key >= a.length) return;
    attn_write<NT>(a.dk, a.dk.at(b, kvh) + key * a.dk.token, dk, ldexpf(a.natural_scale, -exponent - (int)kProbScale), a.dim, half);
    attn_write<NT>(a.dv, a.dv.at(b, kvh) + key * a.dv.token, dv, ldexpf(1.0f, -(int)kProbScale), a.dim, half);
}

template <int NT, bool PLAIN, int LAY>
static int dq_launch(const AttentionGrad& a, unsigned grid, hipStream_t st) {
    constexpr int D = NT <= 2 ? 64 : NT <= 4 ? 128 : 256;
    const int lds = 4 * kAttnTile * D * 2 + (a.table ? (a.distances - a.first_distance + 2 * kBiasPad) * 4 * (a.table_parts ? 5 : 1) : 0);
    static std::atomic<bool> done[64];
    if (int e = enable_dynamic_lds((const void*)k_attn_dq<NT, PLAIN, LAY>, 158 * 1024, done)) return e;
    hipLaunchKernelGGL((k_attn_dq<NT, PLAIN, LAY>), dim3(grid), dim3(256), lds, st, a);
    return 0;
}
template <int NT, bool PLAIN, int LAY>
static int dkv_launch(const AttentionGrad& a, unsigned grid, hipStream_t st) {
    constexpr int D = NT <= 2 ? 64 : NT <= 4 ? 128 : 256;
    const int lds = 4 * kAttnTile * D * 2 + (a.table ? (a.distances - a.first_distance + 2 * kBiasPad) * 4 : 0);
    static std::atomic<bool> done[64];
    if (int e = enable_dynamic_lds((const void*)k_attn_dkv<NT, PLAIN, LAY>, 150 * 1024, done)) return e;
    hipLaunchKernelGGL((k_attn_dkv<NT, PLAIN, LAY>), dim3(grid), dim3(256), lds, st, a);
    return 0;
}
template <int NT, bool PLAIN>
static int grad_launch(const AttentionGrad& a, unsigned dq_grid, unsigned dkv_grid, hipStream_t st) {
    if (dq_grid) {
        const int lay = attn_layout(a.k, a.v, a.dim);
        if (int e = lay == kRows ? dq_launch<NT, PLAIN, kRows>(a, dq_grid, st) : lay == kColumns ? dq_launch<NT, PLAIN, kColumns>(a, dq_grid, st) : dq_launch<NT, PLAIN, kAnyLayout>(a, dq_grid, st)) return e;
    }
    if (dkv_grid == 0) return 0;
    const int lay = attn_layout(a.q, a.dout, a.dim);
    return lay == kRows ? dkv_launch<NT, PLAIN, kRows>(a, dkv_grid, st) : lay == kColumns ? dkv_launch<NT, PLAIN, kColumns>(a, dkv_grid, st) : dkv_launch<NT, PLAIN, kAnyLayout>(a, dkv_grid, st);
}
template <int NT>
static int grad_launch(const AttentionGrad& a, unsigned dq_grid, unsigned dkv_grid, hipStream_t st) {
    return a.table || a.mask ? grad_launch<NT, false>(a, dq_grid, dkv_grid, st) : grad_launch<NT, true>(a, dq_grid, dkv_grid, st);
}

}  // namespace cpmk

using namespace cpmk;

extern "C" {

// Workspace, in floats: D, the two kinds of norms, sums by distance
static int64_t attn_workspace(int64_t batch, int64_t heads, int64_t held, int64_t tokens, int64_t length, int64_t entries, int64_t (&at)[4]) {
    const int64_t query_tiles = ceil_div(tokens, kAttnTile), key_tiles = ceil_div(length, kAttnTile);
    at[0] = batch * heads * tokens;
    at[1] = at[0] + batch * heads * query_tiles;
    at[2] = at[1] + batch * held * key_tiles;
    at[3] = at[2] + batch * heads * ceil_div(tokens, kGradRows) * entries;
    return at[3];
}

int64_t cpmk_attention_backward_workspace(int32_t batch, int32_t heads, int32_t kv_heads, int32_t tokens, int32_t length, int32_t max_distance, int bidirectional) {
    if (batch <= 0 || heads <= 0 || kv_heads <= 0 || tokens < 0 || length < 0 || heads % kv_heads || tokens > kAttnLong || length > kAttnLong) return 0;
    if (!grid_fits((int64_t)batch * heads) || max_distance < 0 || (int64_t)max_distance * (bidirectional ? 2 : 1) > 1024) return 0;
    int64_t at[4];
    const int64_t entries = max_distance ? max_distance + (bidirectional ? std::max(max_distance - 1, 1) : 0) + 2 * kBiasPad : 0;
    return attn_workspace(batch, heads, kv_heads, tokens, length, entries, at) * (int64_t)sizeof(float);
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
    a.tokens = tokens, a.dim = dim, a.length = length, a.splits = 1, a.parts = nullptr;
    bool empty;
    if (int e = attn_check(a, batch, heads, kv_heads, bidirectional, empty)) return e;
    if (empty) return 0;
    if ((tokens > 0 && any_null(lse, rest, dout, dq)) || (length > 0 && any_null(dk, dv)) || !workspace || (dbias && !bias)) return CPMK_EBADARG;
    a.row_tiles = (int32_t)ceil_div(tokens, kGradRows), a.query_tiles = (int32_t)ceil_div(tokens, kAttnTile), a.key_tiles = (int32_t)ceil_div(length, kAttnTile);
    const int64_t query_blocks = (int64_t)batch * heads * a.query_tiles, key_blocks = (int64_t)batch * kv_heads * a.key_tiles;
    if (!grid_fits(query_blocks + key_blocks)) return CPMK_ETOOBIG;
    int64_t at[4];
    attn_workspace(batch, heads, kv_heads, tokens, length, dbias ? a.distances - a.first_distance + 2 * kBiasPad : 0, at);
    a.delta = (float*)workspace, a.dout_top = a.delta + at[0], a.value_top = a.delta + at[1], a.table_parts = dbias ? a.delta + at[2] : nullptr;
    hipStream_t st = (hipStream_t)stream;
    if (query_blocks + key_blocks > 0) hipLaunchKernelGGL(k_attn_facts, dim3((unsigned)(query_blocks + key_blocks)), dim3(256), 0, st, a, (uint32_t)query_blocks);
    const unsigned dq_grid = (unsigned)((int64_t)batch * heads * a.row_tiles), dkv_grid = (unsigned)((int64_t)batch * kv_heads * ceil_div(length, kGradRows));
    if (int e = dim <= 64   ? grad_launch<2>(a, dq_grid, dkv_grid, st)
                : dim <= 96 ? grad_launch<3>(a, dq_grid, dkv_grid, st)
                : dim <= 128 ? grad_launch<4>(a, dq_grid, dkv_grid, st)
                             : grad_launch<8>(a, dq_grid, dkv_grid, st))
        return e;
    if (dbias) {
        const int entries = a.distances - a.first_distance + 2 * kBiasPad;
        hipLaunchKernelGGL(k_attn_dtable, dim3((unsigned)heads), dim3(1024), 5 * entries * sizeof(float), st, a, (int64_t)batch);
    }
    return launch_status();
}

}  // extern "C"
