// Attention over the 8-bit key/value cache for chunks of queries (the mathematics: kv_attention.hip).
//
// A workgroup has 32 queries a wave of one head and goes over its keys in tiles of 64.  It turns a tile's integers into fp16 once, for all its waves, into LDS, two tiles in turn:
// while one is multiplied the next is converted and the one behind it is on its way from memory.  Scores are formed transposed with v_mfma_f32_32x32x16_f16, keys as
// the rows in an order that leaves each lane sixteen neighbouring keys (one block of magnitudes) of one query twice, so the probabilities go from the lane's registers
// straight into the second product.  The running maximum follows the true one at a distance of up to 2^8: fp16 keeps the probabilities' bits either way, and the sums are rescaled
// in the first tiles only.
//
// A workgroup of four waves meets at one barrier a tile, between the softmax (with the conversion and the loads) and the products (values of this tile, scores of the next); what fills the
// matrix pipe meanwhile are the other workgroups of the compute unit, three of them for heads of up to 64 units, two up to 128.  One workgroup of eight waves, half of them a
// phase behind the others, was 20 % slower with 64 units (8 x 64 heads of 512 queries over 1024 keys: 138 against 114 us) and between 3 % slower and 6 % faster with 128.
//
// Bound by the vector and the matrix instructions together: 32 heads of 2000 queries over 8011 keys of 128 units (230 GFLOP) take 270 to 296 us, in which a SIMD's matrix pipe is busy for 223 thousand cycles of 550 and its vector
// instructions issue for 296 (a wave and tile: 32 products, 130 operations of the softmax, 32 of them exponentials, 96 of the conversion); a wave of each side by side reaches two thirds of the sum at
// best.  8 x 64 heads of 512 queries over 1024 of 64 units with a position bias (52 GFLOP) 108 us.  The scores of the next tile between the exponentials of this one, in the same wave, took 329 us for 296 and
// 144 for 110: both tiles' scores do not fit the registers beside the sums.
//
// Registers: with a bias and a mask, heads of up to 64 units have 27 registers a lane in scratch under the bound of three waves a SIMD (8 x 64 heads of 512 queries over 1024 keys 164 us; the bias alone 109,
// the mask alone 130, neither 99), and with a mask heads of more than 128 units three (8 x 32 heads of 256, the same lengths, 301 us; without 292).  Above 128 units there is one form, of 256 units and one wave a SIMD.
//
// LDS, in pieces of 16 bytes: keys (unit step u, half h, row r) at 129 u + 64 h + r, read along r; the odd distance spreads the eight unit steps that
// neighbouring lanes write over the banks.  Values (group of sixteen keys g, half s, unit) at (2 g + s) D + unit.
#include "kv_attention.h"

namespace cpmk {

constexpr int kChunkWaves = kChunkRows / 32;

// N products whose operands come from LDS one each: so many reads ahead that a read's latency lies behind products (the compiler keeps two ahead).
template <int N>
__device__ __forceinline__ void products_in_step() {
    constexpr int kAhead = 6;
    __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
    for (int i = 0; i < N - kAhead; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, kAhead, 0);
}

// NT: 32-unit steps of a head
template <int NT, bool BIAS, bool MASK>
__global__ __launch_bounds__(kChunkWaves * 64, NT == 2 ? 3 : NT <= 4 ? 2 : 1) void k_kv_chunk(KvAttention a) {
    constexpr int D = NT * 32, KS = NT * 2, NTHR = kChunkWaves * 64, PIECES = (8 * D + NTHR - 1) / NTHR, ROWS = kChunkRows;
    constexpr int kKeyBytes = KS * 129 * 16, kBuffer = kKeyBytes + 64 * D * 2;
    extern __shared__ __attribute__((aligned(16))) int8_t lds[];
    __shared__ float4_t facts[16][4];           // of the groups of keys of sixteen tiles, in a ring: factor of the scores, log2 and inverse of the values' scale
    float* const biases = reinterpret_cast<float*>(lds + 2 * kBuffer);
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t inner = (uint32_t)a.group * a.row_tiles * a.splits;
    uint32_t unit, w;
    kv_deal(blockIdx.x, gridDim.x / inner, inner, unit, w);
    const int64_t b = unit / (uint32_t)a.held;
    const int32_t split = w % (uint32_t)a.splits;
    w /= (uint32_t)a.splits;
    // (of a causal chunk the last queries see most keys: their workgroups come first)
    const int32_t qt = a.row_tiles - 1 - (int32_t)(w % (uint32_t)a.row_tiles);
    const int32_t h = (unit - (uint32_t)b * a.held) * a.group + w / (uint32_t)a.row_tiles;
    const int64_t tile_of = (b * a.heads + h) * a.row_tiles + qt;
    const KvRange range = kv_range(a, b, min(qt * ROWS + ROWS - 1, a.tokens - 1), kChunkLeast);
    if (split >= range.parts) return;

    const int32_t q_first = qt * ROWS + wave * 32;
    const int32_t query = min(q_first + col, a.tokens - 1);         // (queries past the end repeat the last one)
    const int32_t where = range.pos + query, limit = a.causal ? min(range.len, where + 1) : range.len;
    // what all and what any of the wave's queries see
    const int32_t last = min(q_first + 31, a.tokens - 1);
    const int32_t all_see = a.causal ? min(range.len, range.pos + min(q_first, a.tokens - 1) + 1) : range.len;
    const int32_t any_sees = q_first >= a.tokens ? 0 : a.causal ? min(range.len, range.pos + last + 1) : range.len;
    const bool flip = a.scale < 0.0f;           // (so that the largest score is the largest product)
    const float scale = flip ? -a.scale : a.scale;

    const int64_t head = b * a.held + h / a.group;
    const int8_t* const keys = a.keys + head * a.length * a.dim;
    const int8_t* const values = a.values + head * a.length * a.dim;
    const half_t* const key_top = a.key_top + (head * a.length >> a.block_shift);
    const half_t* const value_top = a.value_top + (head * a.length >> a.block_shift);
    const uint8_t* const mask = MASK ? a.mask + b * a.mask_batch + query * a.mask_token : nullptr;

    // the pieces of a tile that this thread brings: keys first, a token's units side by side, then values as they lie (a wave has one kind)
    const int runs = a.dim >> 4;
    uint32_t at_lds[PIECES], offset[PIECES], last_offset[PIECES];
    bool is_key[PIECES], real[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int p = tid + i * NTHR;
        real[i] = wave * 64 + i * NTHR < 8 * a.dim;
        is_key[i] = wave * 64 + i * NTHR < 4 * a.dim;
        if (is_key[i]) {
            const int key = p / runs, u = p - key * runs;
            const int r = (key & 32) | ((key >> 2) & 3) << 3 | ((key >> 4) & 1) << 2 | (key & 3);
            offset[i] = key * a.dim + u * 16;
            last_offset[i] = (a.length - 1) * a.dim + u * 16;
            at_lds[i] = (u * 129 + r) * 16;
        } else {
            const int v = p - 4 * a.dim, g = min(v / a.dim, 3), unit = min(v - g * a.dim, a.dim - 1);
            offset[i] = g * 16 * a.dim + unit * 16;
            last_offset[i] = (a.length - 16) * a.dim + unit * 16;
            at_lds[i] = kKeyBytes + (g * 2 * D + unit) * 16;
        }
    }
    const int32_t t_begin = split * range.per_part, t_end = min(t_begin + range.per_part, range.tiles);
    uint4_t raw[PIECES];
    half_t key_raw = 0, value_raw = 0;
    // Keys of tile t + 1 and values of tile t.  (Tiles past the end: the last keys again, into buffers that nobody reads.)
    auto fetch = [&](int32_t t) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
            if (PIECES * NTHR == 8 * D || real[i]) {
                const uint32_t o = min(offset[i] + (uint32_t)max(t + is_key[i], 0) * (uint32_t)(kTile * a.dim), last_offset[i]);
                raw[i] = *reinterpret_cast<const uint4_t*>((is_key[i] ? keys : values) + o);
            }
    };
    uint4_t keep[2];
    auto fetch_mask = [&](int32_t t) {
#pragma unroll
        for (int su = 0; su < 2; ++su) {
            struct __attribute__((packed, aligned(1))) Byte16Any { uint32_t w[4]; };
            keep[su] = __builtin_bit_cast(uint4_t, *reinterpret_cast<const Byte16Any*>(mask + min(t * (int64_t)kTile + su * 32 + half * 16, (int64_t)a.length - 16)));
        }
    };
    auto fetch_tops = [&](int32_t t) {      // a lane a group of keys from tile t on
        const uint32_t at = (uint32_t)min(t * (int64_t)kTile + lane * 16, (int64_t)a.length - 16) >> a.block_shift;
        key_raw = key_top[at];
        value_raw = value_top[at];
    };
    auto convert_tops = [&](int32_t t) {
        const float vs = kv_scale(value_raw);
        facts[(t - t_begin + (lane >> 2)) & 15][lane & 3] = float4_t{(float)key_raw * (1.0f / 127.0f) * scale, __builtin_amdgcn_logf(vs), __builtin_amdgcn_rcpf(vs), 0.0f};
    };
    auto convert = [&](int32_t t) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
            if (PIECES * NTHR == 8 * D || real[i]) {
                half8_t lo, hi;
                halves_of(raw[i], lo, hi);
                int8_t* const p = lds + ((t + is_key[i] - t_begin) & 1) * kBuffer + at_lds[i];
                *reinterpret_cast<half8_t*>(p) = lo;
                *reinterpret_cast<half8_t*>(p + (is_key[i] ? 64 : D) * 16) = hi;
            }
    };
    if (t_begin < t_end) {
        fetch(t_begin - 1);
        if (wave == 0) fetch_tops(t_begin);
        if (MASK) fetch_mask(t_begin);
    }
    half8_t q[KS];
    {
        // (steps of sixteen units lie in the head or behind it as a whole, and their distances are the same for all lanes: one addition a load)
        const half_t* const p = a.q + b * a.q_batch + (int64_t)h * a.q_head + (int64_t)query * a.q_token + half * 8 * a.q_unit;
        if (a.q_unit == 1) {
#pragma unroll
            for (int s = 0; s < KS; ++s) q[s] = load_half8_any(p + min(s * 16, a.dim - 16));
        } else {
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int e = 0; e < 8; ++e) q[s][e] = p[(min(s * 16, a.dim - 16) + e) * a.q_unit];
        }
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            if (s * 16 >= a.dim) q[s] = half8_t{0, 0, 0, 0, 0, 0, 0, 0};
            if (flip) q[s] = -q[s];
        }
    }
    const int32_t lo_rel = a.first_distance - kChunkPad;
    if (BIAS)
        for (int i = tid; i < a.distances - a.first_distance + 2 * kChunkPad; i += NTHR) biases[i] = (float)kv_bias(a, h, max(a.first_distance, min(i + lo_rel, a.distances - 1))) * kLog2e;

    if (t_begin < t_end) {
        if (a.dim < D) {        // (units past the head's: zeros)
            for (int i = tid; i < 2 * kBuffer / 16; i += NTHR) reinterpret_cast<uint4_t*>(lds)[i] = uint4_t{0, 0, 0, 0};
            __syncthreads();
        }
        convert(t_begin - 1);
        fetch(t_begin);
        if (wave == 0) convert_tops(t_begin);
        __syncthreads();
    }

    float16_tv acc[NT], s[2];
    float4_t fact[2];
    half8_t p[2][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n] = float16_tv{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    float top = -__builtin_inff(), sum = 0.0f;
    auto values_of = [&](int32_t t) {       // the values of tile t by their probabilities
        const int8_t* const vl = lds + ((t - t_begin) & 1) * kBuffer + kKeyBytes + (half * 2 * D + col) * 16;
#pragma unroll
        for (int su = 0; su < 2; ++su)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const half8_t v = *reinterpret_cast<const half8_t*>(vl + ((su * 4 + e) * D + n * 32) * 16);
                    acc[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[su][e], acc[n], 0, 0, 0);
                }
    };
    auto scores_of = [&](int32_t t) {
        const int8_t* const kl = lds + ((t - t_begin) & 1) * kBuffer + (half * 64 + col) * 16;
#pragma unroll
        for (int su = 0; su < 2; ++su) {
            fact[su] = facts[(t - t_begin) & 15][su * 2 + half];
            s[su] = float16_tv{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
        }
#pragma unroll
        for (int u = 0; u < KS; ++u)
#pragma unroll
            for (int su = 0; su < 2; ++su) {
                const half8_t k = *reinterpret_cast<const half8_t*>(kl + (u * 129 + su * 32) * 16);
                s[su] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, q[u], s[su], 0, 0, 0);
            }
    };
    if (t_begin < t_end && t_begin * kTile < any_sees) scores_of(t_begin);
    for (int32_t t = t_begin; t < t_end; ++t) {
        const int32_t k0 = t * kTile;
        const bool active = k0 < any_sees;
        if (active) {
            float factor[2] = {fact[0][0], fact[1][0]}, add[2] = {fact[0][1], fact[1][1]};
            // one bias for the whole tile where all its distances lie beyond the table's end
            const int32_t rel_min = range.pos + q_first - (k0 + kTile - 1), rel_max = range.pos + last - k0;
            const bool near = BIAS && rel_min < a.distances - 1 && rel_max > a.first_distance;
            if (BIAS && !near) {
                const float one = biases[(rel_min >= a.distances - 1 ? a.distances - 1 : a.first_distance) - lo_rel];
                add[0] += one;
                add[1] += one;
            }
            float m;
            if (!MASK && !near && k0 + kTile <= all_see) {
                float g[2];
#pragma unroll
                for (int su = 0; su < 2; ++su) {
                    g[su] = s[su][0];
#pragma unroll
                    for (int j = 1; j < 16; ++j) g[su] = fmaxf(g[su], s[su][j]);
                }
                m = fmaxf(__builtin_fmaf(g[0], factor[0], add[0]), __builtin_fmaf(g[1], factor[1], add[1]));
            } else {
#pragma unroll
                for (int su = 0; su < 2; ++su) {
                    const int32_t mine = k0 + su * 32 + half * 16;
                    if (BIAS && near) {
                        const float* const bp = biases + (where - mine - 15 - lo_rel);
#pragma unroll
                        for (int j = 0; j < 16; ++j) s[su][j] = __builtin_fmaf(s[su][j], factor[su], add[su] + bp[15 - j]);
                    } else
#pragma unroll
                        for (int j = 0; j < 16; ++j) s[su][j] = __builtin_fmaf(s[su][j], factor[su], add[su]);
                    if (k0 + kTile > all_see) {
                        const int32_t left = limit - mine;
#pragma unroll
                        for (int j = 0; j < 16; ++j) s[su][j] = j < left ? s[su][j] : -__builtin_inff();
                    }
                    if (MASK)
#pragma unroll
                        for (int j = 0; j < 16; ++j) s[su][j] = (keep[su][j >> 2] >> ((j & 3) * 8) & 0xffu) ? s[su][j] : -__builtin_inff();
                    factor[su] = 1.0f;
                    add[su] = 0.0f;
                }
                m = s[0][0];
#pragma unroll
                for (int su = 0; su < 2; ++su)
#pragma unroll
                    for (int j = 0; j < 16; ++j) m = fmaxf(m, s[su][j]);
            }
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
            const float base = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
            for (int su = 0; su < 2; ++su) {
                const float shift = add[su] - base;
                float part = 0.0f;         // (of the unrounded ones: beside much larger values the rounded ones may have no bits left, and still be most of the sum)
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[su][j], factor[su], shift));
                    part += e;
                    p[su][j >> 3][j & 7] = (half_t)e;           // (an operand of the second product: kv_attention.hip)
                }
                sum = __builtin_fmaf(part, fact[su][2], sum);
            }
        }
        if (MASK) fetch_mask(t + 1);
        convert(t);
        fetch(t + 1);
        if (wave == 0 && t - t_begin >= 8) {        // eight tiles' magnitudes at a time, into the half of the ring that has been read
            if (((t - t_begin) & 7) == 0 && lane < 32) fetch_tops(t + 8);
            if (((t - t_begin) & 7) == 1 && lane < 32) convert_tops(t + 7);
        }
        __syncthreads();
        if (active) {           // (behind the last tile: scores that nobody looks at)
            values_of(t);
            scores_of(t + 1);
            products_in_step<4 * NT + 2 * KS>();
        }
    }
    sum += __shfl_xor(sum, 32);
    if (q_first + col >= a.tokens) return;
    if (a.splits > 1) {
        struct __attribute__((packed, aligned(4))) Float4Any { float x, y, z, w; };         // (a workspace is aligned to 4 bytes)
        float* const part = a.parts + (tile_of * a.splits + split) * ROWS * (a.dim + 2);
        const int r = wave * 32 + col;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int u = n * 32 + c * 8 + half * 4;
                if (u < a.dim) *reinterpret_cast<Float4Any*>(part + r * a.dim + u) = Float4Any{acc[n][c * 4], acc[n][c * 4 + 1], acc[n][c * 4 + 2], acc[n][c * 4 + 3]};
            }
        if (half == 0) {
            part[ROWS * a.dim + r] = top;
            part[ROWS * a.dim + ROWS + r] = sum;
        }
        return;
    }
    half_t* const out = a.out + b * a.out_batch + (int64_t)h * a.out_head + (int64_t)query * a.out_token + half * 4 * a.out_unit;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    if (a.out_unit == 1) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                half4_t v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = (half_t)(acc[n][c * 4 + e] * inv);
                if (n * 32 + c * 8 < a.dim) *reinterpret_cast<Half4Any*>(out + n * 32 + c * 8) = __builtin_bit_cast(Half4Any, v);
            }
    } else {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (n * 32 + c * 8 < a.dim)
#pragma unroll
                    for (int e = 0; e < 4; ++e) out[(n * 32 + c * 8 + e) * a.out_unit] = (half_t)(acc[n][c * 4 + e] * inv);
    }
}

template <int NT, bool BIAS, bool MASK>
static int chunk_launch(const KvAttention& a, unsigned grid, hipStream_t st) {
    const int lds = 2 * (NT * 2 * 129 * 16 + 64 * NT * 32 * 2) + (BIAS ? (a.distances - a.first_distance + 2 * kChunkPad) * 4 : 0);
    static std::atomic<bool> done[64];
    if (int e = enable_dynamic_lds((const void*)k_kv_chunk<NT, BIAS, MASK>, 158 * 1024, done)) return e;
    hipLaunchKernelGGL((k_kv_chunk<NT, BIAS, MASK>), dim3(grid), dim3(kChunkWaves * 64), lds, st, a);
    return 0;
}

template <int NT>
static int chunk_launch(const KvAttention& a, unsigned grid, hipStream_t st) {
    if (a.table) return a.mask ? chunk_launch<NT, true, true>(a, grid, st) : chunk_launch<NT, true, false>(a, grid, st);
    return a.mask ? chunk_launch<NT, false, true>(a, grid, st) : chunk_launch<NT, false, false>(a, grid, st);
}

int kv_chunk_launch(const KvAttention& a, int32_t batch, hipStream_t st) {
    const int64_t grid = (int64_t)batch * a.heads * a.row_tiles * a.splits;
    if (!grid_fits(grid)) return CPMK_ETOOBIG;
    const unsigned g = (unsigned)grid;
    return a.dim <= 64 ? chunk_launch<2>(a, g, st) : a.dim <= 96 ? chunk_launch<3>(a, g, st) : a.dim <= 128 ? chunk_launch<4>(a, g, st) : chunk_launch<8>(a, g, st);
}

}  // namespace cpmk
