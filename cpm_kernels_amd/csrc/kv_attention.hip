// Attention over the key/value cache in 8 bits (kv_cache.hip): out = softmax(scale q k^T + position bias, over the keys that are left) v.
//
// Rows are the queries of the query heads that share a head of the cache: row r is query r / group of head r % group, sixteen rows to a tile.  Scores are formed transposed,
// keys as the rows and queries as the columns of v_mfma_f32_16x16x32_f16, so that a lane ends up with sixteen neighbouring keys of one query: the integers
// of a key are its A operand as they lie (converted to fp16, exactly), and the lane's own probabilities, rounded to fp16, are the B operand of the second product, whose A operand
// is sixteen neighbouring keys of one unit, 16 bytes of the values as they lie.  Nothing goes through LDS or another lane but the running maximum.
//
// The magnitude of a block of keys multiplies the finished scores.  That of its values is taken into the exponent, p' = exp2(score + log2 s - m'), m' the running maximum of
// that sum: the fp16 of p' then has its full width whatever the magnitudes are, and the sum below takes p' / s in fp32.  (Multiplying p by s instead would leave p' in the
// subnormal numbers beside a block of much larger values.)  Keys of all-zero blocks take s = 2^-34, below the smallest that a block can have.
//
// Rounded to fewer than 32 bits are the probabilities p', to fp16, because the second product takes them as fp16 operands beside the integers (fp32 operands have a sixteenth of that rate), and the result.  The sum
// takes the unrounded ones.  Relative to float64, over all results, the root of the mean square is 2.3 to 2.9 10^-4 where probabilities of 32 bits and the same rounding of the result have 2.1 10^-4.
//
// Work is divided over the keys too where rows are few: a workgroup takes every tile of 64 keys of its part, wave by wave, and its waves join their sums
// through LDS; parts leave theirs in the workspace and a second kernel joins them.
//
// Bound by reading the cache: 32 x 64 heads of 64 units over 512 to 1024 keys (202 MB) 36 us, with nothing but the loads 34; 4 x 64 heads of 128 over 16384 to 32768, eight to a head of the
// cache (201 MB), 41 and 39 us, and 4.7 the joining.  One matrix instruction's sixteen columns hold one query there; conversion, scores and softmax of a tile are 270 operations a wave beside the
// 8 KB that it reads.
#include "kv_attention.h"
#include <algorithm>

namespace cpmk {

// The largest of a value over the four sixteens of lanes (no trip through the LDS crossbar).
__device__ __forceinline__ float quad_max(float m) {
    // (a bit cast of a vector's element itself takes the first one's)
    const auto a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, m), __builtin_bit_cast(uint32_t, m), false, false);
    const uint32_t a0 = a[0], a1 = a[1];
    m = fmaxf(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1));
    const auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, m), __builtin_bit_cast(uint32_t, m), false, false);
    const uint32_t b0 = b[0], b1 = b[1];
    return fmaxf(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
}

// DS: 64-unit steps of a head, CT: sixteens of rows, WAVES of a workgroup.
template <int DS, int CT, int WAVES, bool BIAS, bool MASK>
__global__ __launch_bounds__(WAVES * 64, CT == 2 || DS > 2 ? 2 : DS == 2 ? 3 : 4) void k_kv_attend(KvAttention a) {
    constexpr int ROWS = CT * 16;
    __shared__ float joined[WAVES][ROWS][64 + 4];
    __shared__ float stat[WAVES][2][ROWS];
    extern __shared__ half_t table[];
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, quad = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    uint32_t w, rt_of;
    kv_deal(blockIdx.x, gridDim.x / (uint32_t)a.row_tiles, a.row_tiles, w, rt_of);
    const int32_t rt = rt_of;
    const int32_t split = w % (uint32_t)a.splits;
    w /= (uint32_t)a.splits;
    const int32_t kvh = w % (uint32_t)a.held;
    const int64_t b = w / (uint32_t)a.held;
    const int32_t rows = a.tokens * a.group, r_first = rt * ROWS, r_last = min(r_first + ROWS, rows) - 1;
    const KvRange range = kv_range(a, b, r_last / a.group, WAVES);
    if (split >= range.parts) return;
    const int32_t t_begin = split * range.per_part, t_end = min(t_begin + range.per_part, range.tiles);

    const int64_t head = b * a.held + kvh;
    const int8_t* const keys = a.keys + head * a.length * a.dim;
    const int8_t* const values = a.values + head * a.length * a.dim;
    const half_t* const key_top = a.key_top + (head * a.length >> a.block_shift);
    const half_t* const value_top = a.value_top + (head * a.length >> a.block_shift);
    int32_t query[CT], g[CT], limit[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        const int32_t row = min(r_first + c * 16 + col, r_last);       // (rows past the end repeat the last one)
        query[c] = row / a.group;
        g[c] = row - query[c] * a.group;
        limit[c] = a.causal ? min(range.len, range.pos + query[c] + 1) : range.len;
    }
    // keys that every row sees (without a mask), distances of the first and last of the queries
    const int32_t first_at = range.pos + r_first / a.group;
    const int32_t all_see = a.causal ? min(range.len, first_at + 1) : range.len;

    // A tile's values are on their way during its softmax, the next tile's keys while its values are multiplied: each in the registers that the other has just left, so that more waves
    // fit a SIMD than with both of a tile in flight at once (8 x 32 heads of 256 units over 1024 keys: 33 us for 45, of 128 20 for 21.5).  Row r of the key operand is key
    // 16 (r / 4) + 4 j + r % 4 of the tile, so that a lane's results are neighbours; units past the head's meet zeros of the query.
    const int32_t key_row = (col >> 2) * 16 + (col & 3);
    uint4_t raw[4 * DS], mk[CT];
    half_t kt, vt;
    // Rows of sixteen: up to 128 units they are all that there are, and what they look at is read once (32 x 64 heads over up to 1024 keys 36 us for 42 without the hint, 4 x 64 of 128 over up to 32768 41 for
    // 44.5; 4 x 64 heads on 8 of 256 over 16384 55.0 for 57.4).  Above 128 units CT is 1 with more rows too, which read the keys again, and there the hint costs: 8 x 32 heads of 256 over 1024 keys, 33 queries 63.5 us for
    // 52.4, 64 queries 82.6 for 65.1.
    auto load = [&](const int8_t* p) { return CT == 1 ? __builtin_nontemporal_load(reinterpret_cast<const uint4_t*>(p)) : *reinterpret_cast<const uint4_t*>(p); };
    auto fetch_keys = [&](int32_t t) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t o = (uint32_t)min(t * kTile + key_row + j * 4, a.length - 1) * (uint32_t)a.dim;
#pragma unroll
            for (int d = 0; d < DS; ++d) {
                const int u = d * 64 + quad * 16;
                raw[j * DS + d] = load(keys + (o + (uint32_t)(u < a.dim ? u : 0)));
            }
        }
        const int32_t at = min(t * kTile + quad * 16, a.length - 16);
        kt = key_top[(uint32_t)at >> a.block_shift];
        vt = value_top[(uint32_t)at >> a.block_shift];
        if (MASK)
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                struct __attribute__((packed, aligned(1))) Byte16Any { uint32_t w[4]; };
                mk[c] = __builtin_bit_cast(uint4_t, *reinterpret_cast<const Byte16Any*>(a.mask + b * a.mask_batch + query[c] * a.mask_token + at));
            }
    };
    auto fetch_values = [&](int32_t t) {
        const uint32_t o = (uint32_t)min(t * kTile + quad * 16, a.length - 16) * (uint32_t)a.dim + col * 16;
#pragma unroll
        for (int d = 0; d < 4 * DS; ++d) raw[d] = load(values + (o + (uint32_t)(d * 16 < a.dim ? d * 256 : 0)));
    };
    if (t_begin + wave < t_end) fetch_keys(t_begin + wave);
    half8_t q[CT][2 * DS];
#pragma unroll
    for (int c = 0; c < CT; ++c)
        load_query(q[c], a.q + b * a.q_batch + (int64_t)(kvh * a.group + g[c]) * a.q_head + (int64_t)query[c] * a.q_token, a.q_unit, a.dim,
                   [&](int s) { return (s >> 1) * 64 + quad * 16 + (s & 1) * 8; });
    const int entries = a.distances - a.first_distance;
    const half_t* biases[CT];
    if (BIAS) {
        // the bias of every distance from first_distance on, for each head of the tile
        const int slots = min(a.group, ROWS);
        for (int i = tid; i < slots * entries; i += WAVES * 64) {
            const int slot = i / entries, rel = i - slot * entries + a.first_distance;
            const int head = kvh * a.group + (a.group <= ROWS ? slot : (r_first + slot) % a.group);
            table[i] = kv_bias(a, head, rel);
        }
#pragma unroll
        for (int c = 0; c < CT; ++c) biases[c] = table + (a.group <= ROWS ? g[c] : c * 16 + col) * entries - a.first_distance;
        __syncthreads();
    }

    float4_t acc[CT][4 * DS];
    float top[CT], sum[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
#pragma unroll
        for (int d = 0; d < 4 * DS; ++d) acc[c][d] = float4_t{0, 0, 0, 0};
        top[c] = -__builtin_inff();
        sum[c] = 0.0f;
    }
    for (int32_t t = t_begin + wave; t < t_end; t += WAVES) {
        const int32_t k0 = t * kTile, mine = k0 + quad * 16;
        float4_t s[CT][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int c = 0; c < CT; ++c) s[c][j] = float4_t{0, 0, 0, 0};
#pragma unroll
            for (int d = 0; d < DS; ++d) {
                half8_t lo, hi;
                halves_of(raw[j * DS + d], lo, hi);
#pragma unroll
                for (int c = 0; c < CT; ++c) {
                    s[c][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, q[c][2 * d], s[c][j], 0, 0, 0);
                    s[c][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, q[c][2 * d + 1], s[c][j], 0, 0, 0);
                }
            }
        }
        const float factor = (float)kt * (1.0f / 127.0f) * a.scale, vs = kv_scale(vt), add = __builtin_amdgcn_logf(vs), inverse = __builtin_amdgcn_rcpf(vs);
        fetch_values(t);
        half8_t p[CT][2];
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            float x[16];
            // (one bias for the whole tile where all its distances lie beyond the table's end)
            const bool far = BIAS && first_at - (k0 + kTile - 1) >= a.distances - 1;
            if (BIAS && !far) {
                const int32_t where = range.pos + query[c];
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float bias = (float)biases[c][max(a.first_distance, min(where - (mine + j), a.distances - 1))];
                    x[j] = __builtin_fmaf(s[c][j >> 2][j & 3], factor, __builtin_fmaf(bias, kLog2e, add));
                }
            } else {
                const float shift = BIAS ? __builtin_fmaf((float)biases[c][a.distances - 1], kLog2e, add) : add;
#pragma unroll
                for (int j = 0; j < 16; ++j) x[j] = __builtin_fmaf(s[c][j >> 2][j & 3], factor, shift);
            }
            if (k0 + kTile > all_see) {
                const int32_t left = limit[c] - mine;
#pragma unroll
                for (int j = 0; j < 16; ++j) x[j] = j < left ? x[j] : -__builtin_inff();
            }
            if (MASK)
#pragma unroll
                for (int j = 0; j < 16; ++j) x[j] = (mk[c][j >> 2] >> ((j & 3) * 8) & 0xffu) ? x[j] : -__builtin_inff();
            float m = x[0];
#pragma unroll
            for (int j = 1; j < 16; ++j) m = fmaxf(m, x[j]);
            m = quad_max(m);
            if (__builtin_amdgcn_ballot_w64(m > top[c] + kLazy)) {
                const float now = fmaxf(m, top[c]);
                const float f = now == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(top[c] - now);
                top[c] = now;
                sum[c] *= f;
#pragma unroll
                for (int d = 0; d < 4 * DS; ++d) acc[c][d] *= f;
            }
            const float base = top[c] == -__builtin_inff() ? 0.0f : top[c];
            float part = 0.0f;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float e = __builtin_amdgcn_exp2f(x[j] - base);
                part += e;
                p[c][j >> 3][j & 7] = (half_t)e;
            }
            sum[c] = __builtin_fmaf(part, inverse, sum[c]);
        }
#pragma unroll
        for (int d = 0; d < 4 * DS; ++d) {
            half8_t lo, hi;
            halves_of(raw[d], lo, hi);
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                acc[c][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, p[c][0], acc[c][d], 0, 0, 0);
                acc[c][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, p[c][1], acc[c][d], 0, 0, 0);
            }
        }
        if (t + WAVES < t_end) fetch_keys(t + WAVES);
    }
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        sum[c] += __shfl_xor(sum[c], 16);
        sum[c] += __shfl_xor(sum[c], 32);
        if (quad == 0) {
            stat[wave][0][c * 16 + col] = top[c];
            stat[wave][1][c * 16 + col] = sum[c];
        }
    }
    // the waves' sums under the largest of their maxima, 64 units at a time
    float* const part = a.parts + ((head * a.row_tiles + rt) * a.splits + split) * ROWS * (a.dim + 2);
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) {
        if (ds) __syncthreads();
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int d = 0; d < 4; ++d) *reinterpret_cast<float4_t*>(&joined[wave][c * 16 + col][d * 16 + quad * 4]) = acc[c][ds * 4 + d];
        __syncthreads();
        for (int i = tid; i < ROWS * 64; i += WAVES * 64) {
            const int r = i >> 6, u = ds * 64 + (i & 63);
            if (r_first + r > r_last || u >= a.dim) continue;
            float m = stat[0][0][r];
#pragma unroll
            for (int v = 1; v < WAVES; ++v) m = fmaxf(m, stat[v][0][r]);
            const float base = m == -__builtin_inff() ? 0.0f : m;
            float value = 0.0f, total = 0.0f;
#pragma unroll
            for (int v = 0; v < WAVES; ++v) {
                const float f = __builtin_amdgcn_exp2f(stat[v][0][r] - base);
                value = __builtin_fmaf(joined[v][r][i & 63], f, value);
                total = __builtin_fmaf(stat[v][1][r], f, total);
            }
            if (a.splits > 1) {
                part[r * a.dim + u] = value;
                if (u == 0) {
                    part[ROWS * a.dim + r] = m;
                    part[ROWS * a.dim + ROWS + r] = total;
                }
            } else {
                const int32_t rr = r_first + r, qq = rr / a.group;
                a.out[b * a.out_batch + (int64_t)(kvh * a.group + rr - qq * a.group) * a.out_head + (int64_t)qq * a.out_token + (int64_t)u * a.out_unit] =
                    (half_t)(total == 0.0f ? 0.0f : value / total);
            }
        }
    }
}

// Parts joined under the largest of their maxima: a wave a row, its lanes along the units.  `rows` of them lie together (sixteen rows of a head of the cache, or queries of a query head).
__global__ __launch_bounds__(256) void k_kv_join(KvAttention a, int rows, int chunks, int least, uint32_t total_rows) {
    const int lane = threadIdx.x & 63;
    const uint32_t id = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= total_rows) return;
    const int32_t group = chunks ? 1 : a.group, heads = chunks ? a.heads : a.held, of_head = a.tokens * group;
    const int32_t r = id % (uint32_t)of_head;
    const uint32_t w = id / (uint32_t)of_head;
    const int32_t h = w % (uint32_t)heads;
    const int64_t b = w / (uint32_t)heads;
    const int32_t rt = r / rows, in_tile = r - rt * rows, query = r / group, g = r - query * group;
    const KvRange range = kv_range(a, b, min(rt * rows + rows - 1, of_head - 1) / group, least);
    const int64_t size = (int64_t)rows * (a.dim + 2);
    const float* const part = a.parts + ((b * heads + h) * a.row_tiles + rt) * a.splits * size;
    const float* const tops = part + rows * a.dim + in_tile;
    float m = -__builtin_inff();
    for (int i = lane; i < range.parts; i += 64) m = fmaxf(m, tops[i * size]);
    m = wave_max(m);
    const float base = m == -__builtin_inff() ? 0.0f : m;
    float total = 0.0f, value[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int first = 0; first < range.parts; first += 64) {
        // a lane a part: its weight; then eight parts' sums at a time, all on their way together
        const bool real = first + lane < range.parts;
        const float* const mine = tops + (first + (real ? lane : 0)) * size;
        const float weight = real ? __builtin_amdgcn_exp2f(mine[0] - base) : 0.0f;
        total = __builtin_fmaf(real ? mine[rows] : 0.0f, weight, total);
        const int n = min(64, range.parts - first);
        for (int i = 0; i < n; i += 8) {
            float x[8][4];
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (c * 64 < a.dim) x[k][c] = part[(first + min(i + k, n - 1)) * size + in_tile * a.dim + min(c * 64 + lane, a.dim - 1)];
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
    half_t* const out = a.out + b * a.out_batch + (int64_t)(h * group + g) * a.out_head + (int64_t)query * a.out_token;
#pragma unroll
    for (int c = 0; c < 4; ++c)
        if (c * 64 + lane < a.dim) out[(int64_t)(c * 64 + lane) * a.out_unit] = (half_t)(total == 0.0f ? 0.0f : value[c] / total);
}

// Which kernel a call takes, and into how many parts its keys are cut.
//   Up to 64 queries on k_kv_attend, more on k_kv_chunk: 32 heads over 1024 (8 sequences) and 8192 keys (one), us, the one and the other: 33 queries of 64 units 21.4, 24.5 and 25.4, 29.7,
//   64 21.5, 24.7 and 25.8, 30.3, 96 26.2, 32.9 and 26.6, 32.1; of 128 units 33 31.3, 32.4 and 33.1, 37.3, 64 31.9, 33.2 and 34.0, 38.8, 96 42.9, 44.3 and 36.0, 41.8; of 256 units 33 67.2,
//   79.4 and 73.3, 78.8, 64 84.8, 81.7 and 75.1, 81.4, 96 112, 122 and 77.4, 85.0.
//   Workgroups of eight waves where there are fewer than two to a compute unit (8 x 32 heads over 1024 keys, in fours and eights: 64 units 17.2 and 14.2 us, 128 24.0 and 20.0, 256 36.9 and 32.9), of
//   four elsewhere (16 x 32 heads of 256 53 and 57, 32 x 64 of 64 over up to 1024 36 and 38).
//   Parts as long as all workgroups run at once, one a compute unit of eight waves, two of four: with twice as many the joining grows by more than the reading shrinks (4 x 64 heads on 8 of 256
//   units over up to 16384 keys 58 us, with twice the parts 65; 32 on 8 of 128 over up to 65536 38 and 43).  Chunks: one a compute unit, two where the parts keep 16 tiles (96 queries, 8 x 32 heads
//   over 1024 keys in one part 26.6 us, in two 45.2).
struct KvPlan {
    int rows, row_tiles, splits, waves;
    bool chunks;
};
static KvPlan kv_plan(int64_t batch, int64_t heads, int64_t held, int64_t tokens, int32_t dim, int64_t length) {
    KvPlan p;
    p.chunks = tokens > 64;
    p.rows = p.chunks ? kChunkRows : tokens * (heads / held) > 16 && dim <= 128 ? 32 : 16;
    p.row_tiles = (int)ceil_div(p.chunks ? tokens : tokens * (heads / held), p.rows);
    const int64_t base = batch * (p.chunks ? heads : held) * p.row_tiles, tiles = ceil_div(length, kTile), units = compute_units();
    p.waves = base < 2 * units ? 8 : 4;
    const int64_t splits = p.chunks ? std::max(std::min(2 * units / base, tiles / 16), std::min(units / base, tiles / kChunkLeast)) : std::min(8 / p.waves * units / base, tiles / p.waves);
    p.splits = (int)std::max<int64_t>(1, splits);
    return p;
}

template <int DS, int CT, int WAVES, bool BIAS, bool MASK>
static int kv_launch(const KvAttention& a, unsigned grid, hipStream_t st) {
    const size_t lds = BIAS ? (size_t)(a.group < CT * 16 ? a.group : CT * 16) * (a.distances - a.first_distance) * sizeof(half_t) : 0;
    static std::atomic<bool> done[64];
    if (BIAS)
        if (int e = enable_dynamic_lds((const void*)k_kv_attend<DS, CT, WAVES, BIAS, MASK>, 32 * 1024 * (int)sizeof(half_t), done)) return e;
    hipLaunchKernelGGL((k_kv_attend<DS, CT, WAVES, BIAS, MASK>), dim3(grid), dim3(WAVES * 64), lds, st, a);
    return 0;
}

template <int DS, int CT, int WAVES>
static int kv_launch(const KvAttention& a, unsigned grid, hipStream_t st) {
    if (a.table) return a.mask ? kv_launch<DS, CT, WAVES, true, true>(a, grid, st) : kv_launch<DS, CT, WAVES, true, false>(a, grid, st);
    return a.mask ? kv_launch<DS, CT, WAVES, false, true>(a, grid, st) : kv_launch<DS, CT, WAVES, false, false>(a, grid, st);
}

template <int DS, int CT>
static int kv_launch(const KvAttention& a, int waves, unsigned grid, hipStream_t st) {
    return waves == 8 ? kv_launch<DS, CT, 8>(a, grid, st) : kv_launch<DS, CT, 4>(a, grid, st);
}

}  // namespace cpmk

using namespace cpmk;

extern "C" {

int64_t cpmk_kv_attention_int8_workspace(int32_t batch, int32_t heads, int32_t kv_heads, int32_t tokens, int32_t dim, int32_t length) {
    if (batch <= 0 || heads <= 0 || kv_heads <= 0 || tokens <= 0 || dim <= 0 || length <= 0 || heads % kv_heads) return 0;
    if ((int64_t)tokens * (heads / kv_heads) > kFar || !grid_fits((int64_t)batch * heads)) return 0;
    const KvPlan p = kv_plan(batch, heads, kv_heads, tokens, dim, length);
    return p.splits > 1 ? (int64_t)batch * (p.chunks ? heads : kv_heads) * p.row_tiles * p.splits * p.rows * (dim + 2) * (int64_t)sizeof(float) : 0;
}

int cpmk_kv_attention_int8(int32_t batch, int32_t heads, int32_t kv_heads, int32_t tokens, int32_t dim, int32_t length, int32_t block, const void* q,
                           int64_t q_batch, int64_t q_head, int64_t q_token, int64_t q_unit, const void* keys, const void* values,
                           const void* key_absmax, const void* value_absmax, const void* lens_each, int32_t len, const void* pos_each, int32_t pos,
                           int causal, float scale, const void* bias, const void* mapping, int32_t num_buckets, int32_t max_distance,
                           int bidirectional, const void* mask, int64_t mask_batch, int64_t mask_token, void* out, int64_t out_batch,
                           int64_t out_head, int64_t out_token, int64_t out_unit, void* workspace, void* stream) {
    clear_stale_error();
    if (batch < 0 || heads < 0 || kv_heads < 0 || tokens < 0 || dim < 0 || length < 0) return CPMK_EBADARG;
    if (block != 16 && block != 32 && block != 64 && block != 128) return CPMK_EBADARG;
    if (dim % 16 || length % block) return CPMK_EALIGN;
    if (batch == 0 || heads == 0 || tokens == 0 || dim == 0) return 0;
    if (!grid_fits((int64_t)batch * heads)) return CPMK_ETOOBIG;         // (a row each at least; what is multiplied by it below stays below 2^63)
    if (kv_heads == 0 || heads % kv_heads || length == 0) return CPMK_EBADARG;
    if (any_null(q, keys, values, key_absmax, value_absmax, out)) return CPMK_EBADARG;
    if (!lens_each && (len < 0 || len > length)) return CPMK_EBADARG;
    if (bias && (!mapping || num_buckets <= 0 || max_distance <= 0)) return CPMK_EBADARG;
    if (dim > 256 || (int64_t)length * dim > 0x7fffffffll || (int64_t)tokens * (heads / kv_heads) > kFar) return CPMK_ETOOBIG;
    if (bias && (int64_t)max_distance * (bidirectional ? 2 : 1) > 1024) return CPMK_ETOOBIG;
    if (!aligned16(keys) || !aligned16(values)) return CPMK_EALIGN;
    KvAttention a;
    a.q = (const half_t*)q, a.q_batch = q_batch, a.q_head = q_head, a.q_token = q_token, a.q_unit = q_unit;
    a.keys = (const int8_t*)keys, a.values = (const int8_t*)values, a.key_top = (const half_t*)key_absmax, a.value_top = (const half_t*)value_absmax;
    a.lens_each = (const int32_t*)lens_each, a.pos_each = (const int32_t*)pos_each, a.len = len, a.pos = pos;
    a.table = (const half_t*)bias, a.mapping = (const int32_t*)mapping, a.buckets = num_buckets, a.distances = max_distance;
    a.first_distance = bidirectional ? std::min(1 - max_distance, -1) : 0;
    a.mask = (const uint8_t*)mask, a.mask_batch = mask_batch, a.mask_token = mask_token;
    a.out = (half_t*)out, a.out_batch = out_batch, a.out_head = out_head, a.out_token = out_token, a.out_unit = out_unit;
    a.parts = (float*)workspace, a.scale = scale * kLog2e, a.causal = causal != 0;
    a.heads = heads, a.held = kv_heads, a.group = heads / kv_heads, a.tokens = tokens, a.dim = dim, a.length = length;
    a.block_shift = __builtin_ctz((unsigned)block);
    const KvPlan plan = kv_plan(batch, heads, kv_heads, tokens, dim, length);
    a.row_tiles = plan.row_tiles, a.splits = plan.splits;
    if (a.splits > 1 && !workspace) return CPMK_EBADARG;
    const int64_t grid = (int64_t)batch * kv_heads * a.row_tiles * a.splits, rows = (int64_t)batch * heads * tokens;
    if (!grid_fits(grid) || !grid_fits(rows)) return CPMK_ETOOBIG;
    hipStream_t st = (hipStream_t)stream;
    const unsigned g = (unsigned)grid;
    int e;
    if (plan.chunks) e = kv_chunk_launch(a, batch, st);
    else if (plan.rows == 32) e = dim <= 64 ? kv_launch<1, 2>(a, plan.waves, g, st) : kv_launch<2, 2>(a, plan.waves, g, st);
    else if (dim <= 128) e = dim <= 64 ? kv_launch<1, 1>(a, plan.waves, g, st) : kv_launch<2, 1>(a, plan.waves, g, st);
    else e = dim <= 192 ? kv_launch<3, 1>(a, plan.waves, g, st) : kv_launch<4, 1>(a, plan.waves, g, st);
    if (e) return e;
    if (a.splits > 1)
        hipLaunchKernelGGL(k_kv_join, dim3((unsigned)ceil_div(rows, 4)), dim3(256), 0, st, a, plan.rows, (int)plan.chunks, plan.chunks ? kChunkLeast : plan.waves,
                           (uint32_t)rows);
    return launch_status();
}

}  // extern "C"
