// Attention over fp16 keys and values for few rows (the mathematics: attention.hip): a decode step's query, a few drafted tokens, of all heads that share a head of keys.
//
// A row is a query of a head; the rows of a head of keys are dealt out by 16 or 32.  Keys go in tiles of 32 to the waves of a workgroup in turn, from memory straight into registers: a
// lane's 16 bytes of a key are an operand of v_mfma_f32_16x16x32_f16 as they are.  Scores are formed transposed, so that a lane holds eight keys of one row, which is what the second
// product wants of its probabilities; of the values of those eight keys it brings units UL c .. UL c + UL - 1 (c its number in sixteen) and turns them in registers, one v_perm_b32 for two
// halves, into operands of UL products whose rows are units UL c + n.  The next tile is on its way while one is multiplied.  Waves and parts are added up under the largest of their maxima.
//
// Bound by memory: every key and value is read once for each 16 or 32 rows.  One query of 32 x 64 heads of 64, 512 to 1024 keys: 84 us, 4.8 TB/s; of 4 x 64 heads on 8 of 128, 16384 to 32768
// keys: 82 us, 4.9 TB/s.
#include <algorithm>
#include "attention.h"

namespace cpmk {

constexpr int kFewTile = 32, kFewLazy = 8;
constexpr float kFewLift = 7.0f;

// Largest of the four lanes that have the same number in sixteen
__device__ __forceinline__ float across_quads(float x) {
    auto a = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
    uint32_t lo = a[0], hi = a[1];
    x = fmaxf(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
    a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
    lo = a[0], hi = a[1];
    return fmaxf(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
}

// DS: steps of 32 units; CT: groups of 16 rows
template <int DS, int CT, int WAVES, bool PLAIN>
__global__ __launch_bounds__(WAVES * 64, WAVES == 8 || DS * CT <= 4 ? 2 : 1) void k_attn_few(Attention a) {
    constexpr int D = DS * 32, UL = DS <= 2 ? 4 : 8, VB = DS <= 4 ? 1 : DS / 4, NB = UL * VB, ROWS = CT * 16;      // units a lane brings of a value, blocks of them
    extern __shared__ half_t biases[];          // (heads of the rows, distances)
    __shared__ float stats[WAVES][2][ROWS];
    __shared__ float joined[WAVES][ROWS][65];
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, quad = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t inner = (uint32_t)a.row_tiles * a.splits;
    uint32_t unit, w;
    attn_deal(blockIdx.x, gridDim.x / inner, inner, unit, w);
    const int64_t b = unit / (uint32_t)a.held;
    const int32_t kvh = unit - (uint32_t)b * a.held;
    const int32_t split = w % (uint32_t)a.splits, rt = w / (uint32_t)a.splits;
    const int32_t of_head = a.tokens * a.group, r_first = rt * ROWS;
    const AttnRange range = attn_range(a, b);
    const AttnParts parts = attn_parts(a, range, min(r_first + ROWS - 1, of_head - 1) / a.group, WAVES, kFewTile);
    if (split >= parts.parts) return;
    const bool masked = !PLAIN && a.mask != nullptr, biased = !PLAIN && a.table != nullptr;
    const int32_t t_begin = split * parts.per_part, t_end = min(t_begin + parts.per_part, parts.tiles);

    // this lane's rows: of each group of sixteen the c-th
    half8_t q[CT][DS];
    int32_t where[CT], limit[CT], in_table[CT];
    const uint8_t* mask[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        const int32_t r = min(r_first + ct * 16 + c, of_head - 1), query = r / a.group, h = kvh * a.group + r - query * a.group;
        where[ct] = range.pos + query;
        limit[ct] = a.causal ? min(range.len, where[ct] + 1) : range.len;
        mask[ct] = masked ? a.mask + b * a.mask_batch + query * a.mask_token : reinterpret_cast<const uint8_t*>(a.k.at(b, kvh));
        in_table[ct] = (a.group <= ROWS ? h - kvh * a.group : ct * 16 + c) * (a.distances - a.first_distance) - a.first_distance;
        const half_t* const p = a.q.at(b, h) + query * a.q.token;
        if (a.q.unit == 1) {
#pragma unroll
            for (int s = 0; s < DS; ++s) q[ct][s] = load_half8_any(p + min(s * 32 + quad * 8, a.dim - 8));
        } else {
#pragma unroll
            for (int s = 0; s < DS; ++s)
#pragma unroll
                for (int e = 0; e < 8; ++e) q[ct][s][e] = p[(min(s * 32 + quad * 8, a.dim - 8) + e) * a.q.unit];
        }
#pragma unroll
        for (int s = 0; s < DS; ++s) {
            if (s * 32 + quad * 8 >= a.dim) q[ct][s] = half8_t{0, 0, 0, 0, 0, 0, 0, 0};
            if (a.scale < 0.0f) q[ct][s] = -q[ct][s];           // (so that the largest score is the largest product)
        }
    }
    const float scale = fabsf(a.scale);
    // what the rows see all of, the first of them
    const int32_t all_see = a.causal ? min(range.len, range.pos + r_first / a.group + 1) : range.len;

    const half_t *const keys = a.k.at(b, kvh), *const values = a.v.at(b, kvh);
    typedef half_t run_t __attribute__((ext_vector_type(UL)));
    half8_t k[2][DS];
    run_t v[VB][8];
    const int k_unit = quad * 8, v_unit = c * UL;
    auto load_keys = [&](int32_t t) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const half_t* const p = keys + min(t * kFewTile + kb * 16 + c, range.len - 1) * a.k.token;
#pragma unroll
            for (int s = 0; s < DS; ++s) k[kb][s] = load_half8_any(p + min(s * 32 + k_unit, a.dim - 8));
        }
    };
    auto load_values = [&](int32_t t) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const half_t* const p = values + min(t * kFewTile + (j >> 2) * 16 + quad * 4 + (j & 3), range.len - 1) * a.v.token;
#pragma unroll
            for (int vb = 0; vb < VB; ++vb) {
                const half_t* const at = p + min(vb * 16 * UL + v_unit, a.dim - UL);
                if constexpr (UL == 8) v[vb][j] = load_half8_any(at);
                else v[vb][j] = __builtin_bit_cast(half4_t, *reinterpret_cast<const Half4Any*>(at));
            }
        }
    };
    // Four keys' bytes of a mask, on their way with the tile, before it (what is asked for later comes later), and without a branch: without a mask some bytes of the keys
    uint32_t seen[PLAIN ? 1 : CT][2];
    const auto mask_at = [&](int32_t t, int kb) { return min(t * kFewTile + kb * 16 + quad * 4, a.length - 4); };
    auto load_masks = [&](int32_t t) {
        if constexpr (!PLAIN)
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) seen[ct][kb] = reinterpret_cast<const Byte4Any*>(mask[ct] + (masked ? mask_at(t, kb) : 0))->x;
    };
    const int32_t mine = t_begin + wave;
    if (mine < t_end) {
        load_masks(mine);
        load_keys(mine);
        load_values(mine);
    }
    if (biased) {
        // (of heads that have more rows than a tile each row has an entry of its own)
        const int entries = a.distances - a.first_distance, heads = min(a.group, ROWS);
        for (int i = tid; i < heads * entries; i += WAVES * 64) {
            const int g = i / entries, rel = i - g * entries + a.first_distance;
            const int32_t h = kvh * a.group + (a.group <= ROWS ? g : (r_first + g) % a.group);
            biases[i] = a.table[(int64_t)h * a.buckets + attn_bucket(a, rel)];
        }
        __syncthreads();
    }

    float4_t acc[CT][NB];
    float top[CT], sum[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        top[ct] = -__builtin_inff();
        sum[ct] = 0.0f;
#pragma unroll
        for (int n = 0; n < NB; ++n) acc[ct][n] = float4_t{0, 0, 0, 0};
    }
    for (int32_t t = mine; t < t_end; t += WAVES) {
        const int32_t k0 = t * kFewTile;
        const bool guard = masked || k0 + kFewTile > all_see;
        float4_t s[CT][2];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) s[ct][kb] = float4_t{0, 0, 0, 0};
        if (D > a.dim)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int u = 0; u < DS; ++u)
                    if (u * 32 + k_unit >= a.dim) k[kb][u] = half8_t{0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int u = 0; u < DS; ++u)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) s[ct][kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[kb][u], q[ct][u], s[ct][kb], 0, 0, 0);
        const int32_t next = min(t + WAVES, t_end - 1);
        uint32_t keep[CT][2];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const int32_t over = k0 + kb * 16 + quad * 4 - mask_at(t, kb);
                keep[ct][kb] = !masked ? 0x01010101u : over < 4 ? seen[PLAIN ? 0 : ct][kb] >> (8 * over) : 0u;
            }
        load_masks(next);
        load_keys(next);
        // values of the eight keys, turned: x[n] are units UL c + n of the block
        half8_t x[NB];
#pragma unroll
        for (int vb = 0; vb < VB; ++vb)
#pragma unroll
            for (int n = 0; n < UL; ++n)
#pragma unroll
                for (int j = 0; j < 8; ++j) x[vb * UL + n][j] = v[vb][j][n];
        load_values(next);
        uint32_t spoilt = 0;           // keys whose values are no finite numbers: they must not reach the rows that do not see them
        if (guard) {
            half8_t worst = {0, 0, 0, 0, 0, 0, 0, 0};
            const half8_t none = worst;
#pragma unroll
            for (int n = 0; n < NB; ++n) worst = __builtin_elementwise_fma(x[n], none, worst);
            bool any = false;
#pragma unroll
            for (int j = 0; j < 8; ++j) any |= !(worst[j] == (half_t)0);
            if (__builtin_amdgcn_ballot_w64(any)) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if ((__builtin_amdgcn_ballot_w64(!(worst[j] == (half_t)0)) >> (quad * 16)) & 0xffffu) spoilt |= 1u << j;
#pragma unroll
                    for (int n = 0; n < NB; ++n) x[n][j] = x[n][j] * (half_t)0 == (half_t)0 ? x[n][j] : (half_t)0;
                }
            }
        }
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            float factor = scale;
            if (guard || biased) {
                factor = 1.0f;
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    const int32_t key = k0 + kb * 16 + quad * 4;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float y = s[ct][kb][i] * scale;
                        if (biased) y = __builtin_fmaf((float)biases[in_table[ct] + max(a.first_distance, min(where[ct] - key - i, a.distances - 1))], kLog2e, y);
                        if (spoilt >> (kb * 4 + i) & 1) y = __builtin_nanf("");
                        s[ct][kb][i] = key + i < limit[ct] && (keep[ct][kb] >> (8 * i) & 0xffu) ? y : -__builtin_inff();
                    }
                }
            }
            float m = s[ct][0][0];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int i = 0; i < 4; ++i) m = fmaxf(m, s[ct][kb][i]);
            m = across_quads(m * factor);
            if (__builtin_amdgcn_ballot_w64(m > top[ct] + kFewLazy)) {
                const float now = fmaxf(m, top[ct]), f = now == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(top[ct] - now);
                top[ct] = now;
                sum[ct] *= f;
#pragma unroll
                for (int n = 0; n < NB; ++n) acc[ct][n] *= f;
            }
            const float shift = kFewLift - (top[ct] == -__builtin_inff() ? 0.0f : top[ct]);
            half8_t p;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[ct][j >> 2][j & 3], factor, shift));
                sum[ct] += y;
                p[j] = (half_t)y;
            }
#pragma unroll
            for (int n = 0; n < NB; ++n) acc[ct][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[n], p, acc[ct][n], 0, 0, 0);
        }
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        sum[ct] += __shfl_xor(sum[ct], 16);
        sum[ct] += __shfl_xor(sum[ct], 32);
        if (quad == 0) {
            stats[wave][0][ct * 16 + c] = top[ct];
            stats[wave][1][ct * 16 + c] = sum[ct];
        }
    }
    __syncthreads();
    // every wave's sums times the weight of its maximum, 64 units at a time through LDS
    float weight[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        float m = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < WAVES; ++i) m = fmaxf(m, stats[i][0][ct * 16 + c]);
        weight[ct] = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(top[ct] - m);
    }
    float* const part = a.splits > 1 ? a.parts + (((b * a.held + kvh) * a.row_tiles + rt) * a.splits + split) * ROWS * (a.dim + 2) : nullptr;
    // (block n of 16 units a lane's four sums are units vb * 16 UL + UL (4 quad + i) + n of row c)
    constexpr int GROUPS = D / 64 > 0 ? D / 64 : 1;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        if (g) __syncthreads();
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int u = n / UL * 16 * UL + UL * (4 * quad + i) + n % UL;
                    if (u / 64 == g) joined[wave][ct * 16 + c][u % 64] = acc[ct][n][i] * weight[ct];
                }
        __syncthreads();
        for (int i = tid; i < ROWS * 64; i += WAVES * 64) {
            const int r = i >> 6, u = g * 64 + (i & 63);
            if (r_first + r >= of_head || u >= a.dim) continue;
            float m = -__builtin_inff(), total = 0.0f, value = 0.0f;
#pragma unroll
            for (int j = 0; j < WAVES; ++j) m = fmaxf(m, stats[j][0][r]);
#pragma unroll
            for (int j = 0; j < WAVES; ++j) {
                value += joined[j][r][i & 63];
                total = __builtin_fmaf(stats[j][1][r], m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(stats[j][0][r] - m), total);
            }
            if (part) {
                part[r * a.dim + u] = value;
                if (u == 0) {
                    part[ROWS * a.dim + r] = m;
                    part[ROWS * a.dim + ROWS + r] = total;
                }
            } else {
                const int32_t rr = r_first + r, query = rr / a.group;
                a.out.at(b, kvh * a.group + rr - query * a.group)[query * a.out.token + u * a.out.unit] = (half_t)(total == 0.0f ? 0.0f : value / total);
            }
        }
    }
}

template <int DS, int CT, int WAVES>
static int few_launch(const Attention& a, unsigned grid, hipStream_t st) {
    const int lds = a.table ? std::min(a.group, CT * 16) * (a.distances - a.first_distance) * (int)sizeof(half_t) : 0;
    if (a.table || a.mask) {
        static std::atomic<bool> done[64];
        if (int e = enable_dynamic_lds((const void*)k_attn_few<DS, CT, WAVES, false>, 66 * 1024, done)) return e;
        hipLaunchKernelGGL((k_attn_few<DS, CT, WAVES, false>), dim3(grid), dim3(WAVES * 64), lds, st, a);
    } else
        hipLaunchKernelGGL((k_attn_few<DS, CT, WAVES, true>), dim3(grid), dim3(WAVES * 64), 0, st, a);
    return 0;
}
template <int DS, int CT>
static int few_launch(const Attention& a, int waves, unsigned grid, hipStream_t st) {
    if constexpr (DS * CT <= 4)
        if (waves == 8) return few_launch<DS, CT, 8>(a, grid, st);
    return few_launch<DS, CT, 4>(a, grid, st);
}

// How rows and keys of few rows are divided: workgroups of eight waves where there are fewer than two to a compute unit and their registers allow it, of four elsewhere; parts as long
// as all run at once (five queries of four heads each, dim 128: one workgroup to a compute unit by its registers, 44 us in two rounds, 36 in one).
AttnPlan attn_few_plan(int64_t batch, int64_t held, int64_t of_head, int32_t dim, int64_t length) {
    AttnPlan p;
    p.rows = of_head > 16 ? 32 : 16;
    p.row_tiles = (int)ceil_div(of_head, p.rows);
    const int64_t base = batch * held * p.row_tiles, tiles = ceil_div(length, kFewTile), units = compute_units();
    const bool light = dim <= 64 || (dim <= 128 && p.rows == 16);         // two waves to a SIMD
    p.waves = base < 2 * units && light ? 8 : 4;
    p.tile = kFewTile;
    p.least = p.waves;
    p.splits = (int)std::max<int64_t>(1, std::min((light ? 8 / p.waves : 1) * units / base, tiles / p.waves));
    return p;
}

int attn_few_launch(const Attention& a, const AttnPlan& p, int32_t batch, hipStream_t st) {
    const int64_t grid = (int64_t)batch * a.held * a.row_tiles * a.splits;
    if (!grid_fits(grid)) return CPMK_ETOOBIG;
    const unsigned g = (unsigned)grid;
    if (p.rows == 16) return a.dim <= 64 ? few_launch<2, 1>(a, p.waves, g, st) : a.dim <= 128 ? few_launch<4, 1>(a, p.waves, g, st) : few_launch<8, 1>(a, p.waves, g, st);
    return a.dim <= 64 ? few_launch<2, 2>(a, p.waves, g, st) : a.dim <= 128 ? few_launch<4, 2>(a, p.waves, g, st) : few_launch<8, 2>(a, p.waves, g, st);
}

}  // namespace cpmk
