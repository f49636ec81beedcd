// k_attn of attention.hip (the mathematics: there), compiled for each size of heads by itself.
//
// Loop: the values' sums of tile t and the scores of tile t + 1 are issued as one run of products, their operands read eight ahead of them; then the softmax of t + 1.  Keys and masks are
// fetched a tile before the values, each while the tile before it is worked on.
#pragma once
#include "attention.h"

namespace cpmk {

constexpr int kAttnRows = 128, kAttnLeast = 4;       // queries of a workgroup; tiles of a part, at least
constexpr int kLazy = 8;            // log2 of how far the running maximum may lie below the true one
constexpr float kLift = 7.0f;       // log2 of the largest probability's size right behind a change of the maximum

template <int NT, bool BIAS, bool MASK, int LAY, bool TRAIN>
__global__ __launch_bounds__(256, NT <= 4 ? 2 : 1) void k_attn(Attention a) {
    constexpr int D = NT <= 2 ? 64 : NT <= 4 ? 128 : 256, KS = NT * 2, kTileBytes = kAttnTile * D * 2;
    extern __shared__ __attribute__((aligned(128))) int8_t lds[];        // two buffers of keys, two of values, biases
    __shared__ uint32_t bad[3][2];              // tokens of a tile whose values are no finite numbers; those of tile t in t % 3
    __shared__ uint32_t mask_bits[2][kAttnRows][2];
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
    constexpr bool BY_UNIT = kByUnit<LAY>, ARRIVES = LAY == kDirect || LAY == kTurned;
    const bool masked = MASK && (ARRIVES || a.mask != nullptr);
    const half_t *const keys = a.k.at(b, kvh), *const values = a.v.at(b, kvh);
    const uint8_t* const mask = masked ? a.mask + b * a.mask_batch + min(qt * kAttnRows + (tid >> 1), a.tokens - 1) * a.mask_token : nullptr;

    // Keys, and the mask's bits, come a tile before the values: scores of the next tile are formed beside this one's sums.
    const int32_t t_begin = split * parts.per_part, t_end = min(t_begin + parts.per_part, parts.tiles);
    AttnTiles<D, LAY> ks, vs;
    ks.init(keys, a.k, a.length, a.dim, tid, wave, lane);
    vs.init(values, a.v, a.length, a.dim, tid, wave, lane);
    AttnMaskShare<ARRIVES> ms;
    ushort8_t largest = {0, 0, 0, 0, 0, 0, 0, 0};
    const auto guarded = [&](int32_t t) { return masked || (t + 1) * kAttnTile > every_sees; };       // (a value that is no finite number must not reach the queries that do not see it)
    auto fetch = [&](int32_t t) __attribute__((always_inline)) {
        if (t + 1 < t_end) ks.fetch(lds + ((t + 1) & 1) * kTileBytes, a.dim, (t + 1) * kAttnTile, range.len, tid, wave, lane);
        // (without a branch: where paths meet, the compiler waits for what either loads, and for the tiles with it)
        if (masked) ms.load(mask, (t + 1) * kAttnTile + (tid & 1) * 32, a.length);
        if (t >= t_begin && t < t_end) vs.fetch(lds + (2 + (t & 1)) * kTileBytes, a.dim, t * kAttnTile, range.len, tid, wave, lane);
    };
    if (tid < 6) bad[tid >> 1][tid & 1] = 0;
    if (!ARRIVES) fetch(t_begin - 1);
    half8_t q[KS];
    if (BY_UNIT && a.q.token == 1) {
        attn_bring_columns<D>(a.q, a.q.at(b, h), qt * kAttnRows, a.tokens, a.dim, tid, lds + 2 * kTileBytes);
        __syncthreads();
        attn_keep_columns<D, KS>(q, lds + 2 * kTileBytes, wave, lane);
    } else
        attn_keep<KS>(q, a.q, a.q.at(b, h) + query * a.q.token, a.dim, half);
    if (!(a.scale > 0.0f))
#pragma unroll
        for (int s = 0; s < KS; ++s) q[s] *= (half_t)(a.scale < 0.0f ? -1.0f : 0.0f);
    if (BIAS) attn_biases(a, h, scale, biases, tid, 256);
    if (ARRIVES && a.dim < D) {
        __syncthreads();            // (behind the queries that came through LDS)
        attn_clear(lds, 4 * kTileBytes, tid, 256);
    }
    __syncthreads();
    if (ARRIVES) fetch(t_begin - 1);

    const uint32_t at_rows = attn_rows_at<D, BY_UNIT>(lane), at_units = attn_units_at<D, BY_UNIT>(lane);
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
            for (int blk = 0; blk < 2; ++blk) s[blk] = __builtin_amdgcn_mfma_f32_32x32x16_f16(attn_rows<D, BY_UNIT>(tile, at_rows, blk, u), q[u], s[blk], 0, 0, 0);
    };
    auto sums_of = [&](int32_t t) {
        const int8_t* const tile = lds + (2 + (t & 1)) * kTileBytes;
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const half8_t v = attn_units<D, BY_UNIT>(tile, at_units, n, e >> 1, e & 1);
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
                    const uint32_t bits = mask_bits[t & 1][wave * 32 + col][blk];
                    if (__builtin_amdgcn_ballot_w64(bits != ~0u)) attn_cap(s[blk], bits >> (half * 4));
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
        if (ARRIVES) wait_vmcnt<0>();
        if (t + 1 < t_end) {
            ks.place(lds + ((t + 1) & 1) * kTileBytes, a.dim, (t + 1) * kAttnTile, range.len, tid, wave, lane, nullptr);
            if (masked) mask_bits[(t + 1) & 1][tid >> 1][tid & 1] = ms.bits(mask, (t + 1) * kAttnTile + (tid & 1) * 32, a.length);
        }
        if (t >= t_begin) {
            int8_t* const tile = lds + (2 + (t & 1)) * kTileBytes;
            if (looks) largest = vs.largest(largest, tile, range.len - k0, wave, lane);
            vs.place(tile, a.dim, k0, range.len, tid, wave, lane, guarded(t) ? bad[(uint32_t)t % 3] : nullptr);
        }
        if (tid < 2) bad[(uint32_t)(t + 1) % 3][tid] = 0;          // (last looked at two tiles ago)
        if (!ARRIVES) fetch(t + 1);
        __syncthreads();
        if (ARRIVES) fetch(t + 1);
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
            attn_pace<4 * NT * (TRAIN ? 2 : 1), 8 * NT, 2 * KS, 2 * KS * (BY_UNIT ? 2 : 1), BIAS ? 16 : 0>();
        } else if ((t + 1) * kAttnTile < any_sees && t + 1 < t_end) {
            scores_of(t + 1);
            attn_pace<0, 0, 2 * KS, 2 * KS * (BY_UNIT ? 2 : 1), BIAS ? 16 : 0>();
        }
    }
    sum += __shfl_xor(sum, 32);
    __syncthreads();            // (the tiles are done with)
    if (looks) {
        const uint32_t m = wave_max_u32(absbits_max_of(largest));
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

template <int NT, bool BIAS, bool MASK, int LAY, bool TRAIN>
static int attn_launch(const Attention& a, unsigned grid, hipStream_t st) {
    constexpr int D = NT <= 2 ? 64 : NT <= 4 ? 128 : 256;
    const int lds = 4 * kAttnTile * D * 2 + (a.table ? (a.distances - a.first_distance + 2 * kBiasPad) * 4 : 0);
    static std::atomic<bool> done[64];
    if (int e = enable_dynamic_lds((const void*)k_attn<NT, BIAS, MASK, LAY, TRAIN>, 150 * 1024, done)) return e;
    hipLaunchKernelGGL((k_attn<NT, BIAS, MASK, LAY, TRAIN>), dim3(grid), dim3(256), lds, st, a);
    return 0;
}
template <int NT, bool BIAS, bool MASK, int LAY>
static int attn_launch(const Attention& a, unsigned grid, hipStream_t st) {
    return a.lse ? attn_launch<NT, BIAS, MASK, LAY, true>(a, grid, st) : attn_launch<NT, BIAS, MASK, LAY, false>(a, grid, st);
}
// (a mask is looked for in a call's arguments where tiles come through registers: a branch a tile, 15 % of the time where they do not.  Of a mask the others read 32 keys at a time.)
template <int NT, bool BIAS>
static int attn_launch(const Attention& a, unsigned grid, hipStream_t st) {
    const int lay = a.mask && a.length < 32 ? kAnyLayout : attn_layout(a.k, a.v, a.dim, a.length);
    if (lay == kDirect) return a.mask ? attn_launch<NT, BIAS, true, kDirect>(a, grid, st) : attn_launch<NT, BIAS, false, kDirect>(a, grid, st);
    if (lay == kTurned) return a.mask ? attn_launch<NT, BIAS, true, kTurned>(a, grid, st) : attn_launch<NT, BIAS, false, kTurned>(a, grid, st);
    return lay == kColumns ? attn_launch<NT, BIAS, true, kColumns>(a, grid, st) : attn_launch<NT, BIAS, true, kAnyLayout>(a, grid, st);
}
template <int NT>
static int attn_launch(const Attention& a, unsigned grid, hipStream_t st) {
    return a.table ? attn_launch<NT, true>(a, grid, st) : attn_launch<NT, false>(a, grid, st);
}

// (attention_64.hip and so on)
int attn_launch_64(const Attention& a, unsigned grid, hipStream_t st);
int attn_launch_96(const Attention& a, unsigned grid, hipStream_t st);
int attn_launch_128(const Attention& a, unsigned grid, hipStream_t st);
int attn_launch_256(const Attention& a, unsigned grid, hipStream_t st);

}  // namespace cpmk
