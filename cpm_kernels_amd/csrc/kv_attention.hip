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
// Work is divided over the keys too where rows are few: a workgroup takes every tile of 64 keys of its part, wave by wave, and its waves join their sums
// through LDS; parts leave theirs in the workspace and a second kernel joins them.
#include "kv_attention.h"

namespace cpmk {

constexpr int kWaves = 4;

// DS: 64-unit steps of a head.
template <int DS, int WAVES, bool BIAS, bool MASK>
__global__ __launch_bounds__(WAVES * 64) void k_kv_attend(KvAttention a) {
    __shared__ float joined[WAVES][16][64 + 4];
    __shared__ float stat[WAVES][2][16];
    extern __shared__ half_t table[];
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, quad = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    uint32_t w = blockIdx.x;
    const int32_t split = w % (uint32_t)a.splits;
    w /= (uint32_t)a.splits;
    const int32_t rt = w % (uint32_t)a.row_tiles;
    w /= (uint32_t)a.row_tiles;
    const int32_t kvh = w % (uint32_t)a.held;
    const int64_t b = w / (uint32_t)a.held;
    const int64_t tile_of = blockIdx.x / (uint32_t)a.splits;
    const int32_t rows = a.tokens * a.group;
    const int32_t row = min(rt * 16 + col, rows - 1);       // (rows past the end repeat the last one)
    const int32_t query = row / a.group, g = row - query * a.group;
    const KvRange range = kv_range(a, b, min(rt * 16 + 15, rows - 1) / a.group, WAVES);
    if (split >= range.parts) return;
    const int32_t where = range.pos + query;                // position of the query
    const int32_t limit = a.causal ? min(range.len, where + 1) : range.len;

    half8_t q[2 * DS];
    load_query(q, a.q + b * a.q_batch + (int64_t)(kvh * a.group + g) * a.q_head + (int64_t)query * a.q_token, a.q_unit, a.dim,
               [&](int s) { return (s >> 1) * 64 + quad * 16 + (s & 1) * 8; });
    const int entries = a.distances - a.first_distance;
    if (BIAS) {
        // the bias of every distance from first_distance on, for each head of the tile
        const int slots = min(a.group, 16);
        for (int i = tid; i < slots * entries; i += WAVES * 64) {
            const int slot = i / entries, rel = i - slot * entries + a.first_distance;
            const int head = kvh * a.group + (a.group <= 16 ? slot : (rt * 16 + slot) % a.group);
            const int bucket = a.mapping[rel < 0 ? -rel : rel] + (rel < 0 ? a.buckets / 2 : 0);
            table[i] = a.table[(int64_t)head * a.buckets + max(0, min(bucket, a.buckets - 1))];
        }
        __syncthreads();
    }
    const half_t* const biases = table + (a.group <= 16 ? g : col) * entries;

    const int64_t head = b * a.held + kvh;
    const int8_t* const keys = a.keys + head * a.length * a.dim;
    const int8_t* const values = a.values + head * a.length * a.dim;
    const half_t* const key_top = a.key_top + (head * a.length >> a.block_shift);
    const half_t* const value_top = a.value_top + (head * a.length >> a.block_shift);
    const uint8_t* const mask = MASK ? a.mask + b * a.mask_batch + query * a.mask_token : nullptr;

    float4_t acc[4 * DS];
#pragma unroll
    for (int d = 0; d < 4 * DS; ++d) acc[d] = float4_t{0, 0, 0, 0};
    float top = -__builtin_inff(), sum = 0.0f;
    const int32_t t_begin = split * range.per_part, t_end = min(t_begin + range.per_part, range.tiles);
    for (int32_t t = t_begin + wave; t < t_end; t += WAVES) {
        const int32_t k0 = t * kTile;
        float4_t s[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // row r of this operand is key 16 (r / 4) + 4 j + r % 4, so that a lane's results are neighbours
            const int32_t key = min(k0 + (col >> 2) * 16 + j * 4 + (col & 3), a.length - 1);
            s[j] = float4_t{0, 0, 0, 0};
#pragma unroll
            for (int d = 0; d < DS; ++d) {
                const int u = d * 64 + quad * 16;       // (units past the head's meet zeros of the query)
                half8_t lo, hi;
                halves_of(*reinterpret_cast<const uint4_t*>(keys + (int64_t)key * a.dim + (u < a.dim ? u : 0)), lo, hi);
                s[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, q[2 * d], s[j], 0, 0, 0);
                s[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, q[2 * d + 1], s[j], 0, 0, 0);
            }
        }
        const int32_t mine = k0 + quad * 16, at = min(mine, a.length - 16);
        const float factor = (float)key_top[at >> a.block_shift] * (1.0f / 127.0f) * a.scale;
        const float vs = kv_scale(value_top[at >> a.block_shift]), add = __builtin_log2f(vs);
        float x[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            float bias = add;
            if (BIAS) bias = __builtin_fmaf((float)biases[max(a.first_distance, min(where - (mine + j), a.distances - 1)) - a.first_distance], kLog2e, add);
            x[j] = __builtin_fmaf(s[j >> 2][j & 3], factor, bias);
            if (mine + j >= limit) x[j] = -__builtin_inff();
        }
        if (MASK) {
            struct __attribute__((packed, aligned(1))) Byte16Any { uint32_t w[4]; };
            const Byte16Any keep = *reinterpret_cast<const Byte16Any*>(mask + at);
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (!(keep.w[j >> 2] >> ((j & 3) * 8) & 0xffu)) x[j] = -__builtin_inff();
        }
        float m = x[0];
#pragma unroll
        for (int j = 1; j < 16; ++j) m = fmaxf(m, x[j]);
        m = fmaxf(m, __shfl_xor(m, 16));
        m = fmaxf(m, __shfl_xor(m, 32));
        if (__builtin_amdgcn_ballot_w64(m > top)) {
            const float now = fmaxf(m, top);
            const float f = now == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(top - now);
            top = now;
            sum *= f;
#pragma unroll
            for (int d = 0; d < 4 * DS; ++d) acc[d] *= f;
        }
        const float base = top == -__builtin_inff() ? 0.0f : top;
        float part = 0.0f;
        half8_t p[2];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const float e = __builtin_amdgcn_exp2f(x[j] - base);
            part += e;
            p[j >> 3][j & 7] = (half_t)e;
        }
        sum = __builtin_fmaf(part, 1.0f / vs, sum);
#pragma unroll
        for (int d = 0; d < 4 * DS; ++d) {
            const int u = d * 16;
            half8_t lo, hi;
            halves_of(*reinterpret_cast<const uint4_t*>(values + (int64_t)at * a.dim + ((u < a.dim ? u : 0) + col) * 16), lo, hi);
            acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, p[0], acc[d], 0, 0, 0);
            acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, p[1], acc[d], 0, 0, 0);
        }
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (quad == 0) {
        stat[wave][0][col] = top;
        stat[wave][1][col] = sum;
    }
    // the waves' sums under the largest of their maxima, 64 units at a time
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) {
    if (ds) __syncthreads();
#pragma unroll
    for (int d = 0; d < 4; ++d) *reinterpret_cast<float4_t*>(&joined[wave][col][d * 16 + quad * 4]) = acc[ds * 4 + d];
    __syncthreads();
    for (int i = tid; i < 16 * 64; i += WAVES * 64) {
        const int r = i >> 6, u = ds * 64 + (i & 63);
        if (rt * 16 + r >= rows || u >= a.dim) continue;
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
            float* const part = a.parts + (tile_of * a.splits + split) * 16 * (a.dim + 2);
            part[r * a.dim + u] = value;
            if (u == 0) {
                part[16 * a.dim + r] = m;
                part[16 * a.dim + 16 + r] = total;
            }
        } else {
            const int32_t rr = rt * 16 + r, qq = rr / a.group;
            a.out[b * a.out_batch + (int64_t)(kvh * a.group + rr - qq * a.group) * a.out_head + (int64_t)qq * a.out_token + (int64_t)u * a.out_unit] =
                (half_t)(total == 0.0f ? 0.0f : value / total);
        }
    }
    }
}

// Parts joined under the largest of their maxima: a wave a row, its lanes along the units.  `rows` of them lie together (sixteen rows of a head of the cache, or queries of a query head).
__global__ __launch_bounds__(256) void k_kv_join(KvAttention a, int rows, int chunks, uint32_t total_rows) {
    const int lane = threadIdx.x & 63;
    const uint32_t id = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= total_rows) return;
    const int32_t group = chunks ? 1 : a.group, heads = chunks ? a.heads : a.held, of_head = a.tokens * group;
    const int32_t r = id % (uint32_t)of_head;
    const uint32_t w = id / (uint32_t)of_head;
    const int32_t h = w % (uint32_t)heads;
    const int64_t b = w / (uint32_t)heads;
    const int32_t rt = r / rows, in_tile = r - rt * rows, query = r / group, g = r - query * group;
    const KvRange range = kv_range(a, b, min(rt * rows + rows - 1, of_head - 1) / group, chunks ? kChunkLeast : kWaves);
    const int64_t size = (int64_t)rows * (a.dim + 2);
    const float* const part = a.parts + ((b * heads + h) * a.row_tiles + rt) * a.splits * size;
    const float* const tops = part + rows * a.dim + in_tile;
    float m = -__builtin_inff();
    for (int i = lane; i < range.parts; i += 64) m = fmaxf(m, tops[i * size]);
    m = wave_max(m);
    const float base = m == -__builtin_inff() ? 0.0f : m;
    float total = 0.0f, value[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = 0; i < range.parts; ++i) {
        const float f = __builtin_amdgcn_exp2f(tops[i * size] - base);
        total = __builtin_fmaf(tops[i * size + rows], f, total);
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (c * 64 + lane < a.dim) value[c] = __builtin_fmaf(part[i * size + in_tile * a.dim + c * 64 + lane], f, value[c]);
    }
    half_t* const out = a.out + b * a.out_batch + (int64_t)(h * group + g) * a.out_head + (int64_t)query * a.out_token;
#pragma unroll
    for (int c = 0; c < 4; ++c)
        if (c * 64 + lane < a.dim) out[(int64_t)(c * 64 + lane) * a.out_unit] = (half_t)(total == 0.0f ? 0.0f : value[c] / total);
}

// Which kernel a call takes, and into how many parts its keys are cut.
struct KvPlan {
    int rows, row_tiles, splits;
    bool chunks;
};
static KvPlan kv_plan(int64_t batch, int64_t heads, int64_t held, int64_t tokens, int32_t dim, int64_t length) {
    KvPlan p;
    p.chunks = tokens > 32;
    p.rows = p.chunks ? kChunkRows : 16;
    p.row_tiles = (int)ceil_div(p.chunks ? tokens : tokens * (heads / held), p.rows);
    const int64_t base = batch * (p.chunks ? heads : held) * p.row_tiles, most = ceil_div(length, kTile * (p.chunks ? kChunkLeast : kWaves));
    const int64_t want = ceil_div((p.chunks ? 1 : 4) * (int64_t)compute_units(), base);
    p.splits = (int)(want < 1 ? 1 : want > most ? most : want);
    return p;
}

template <int DS>
static void kv_launch(const KvAttention& a, unsigned grid, hipStream_t st) {
    const size_t lds = a.table ? (size_t)(a.group < 16 ? a.group : 16) * (a.distances - a.first_distance) * sizeof(half_t) : 0;
    const dim3 g(grid), t(kWaves * 64);
    if (a.table && a.mask) hipLaunchKernelGGL((k_kv_attend<DS, kWaves, true, true>), g, t, lds, st, a);
    else if (a.table) hipLaunchKernelGGL((k_kv_attend<DS, kWaves, true, false>), g, t, lds, st, a);
    else if (a.mask) hipLaunchKernelGGL((k_kv_attend<DS, kWaves, false, true>), g, t, lds, st, a);
    else hipLaunchKernelGGL((k_kv_attend<DS, kWaves, false, false>), g, t, lds, st, a);
}

}  // namespace cpmk

using namespace cpmk;

extern "C" {

int64_t cpmk_kv_attention_int8_workspace(int32_t batch, int32_t heads, int32_t kv_heads, int32_t tokens, int32_t dim, int32_t length) {
    if (batch <= 0 || heads <= 0 || kv_heads <= 0 || tokens <= 0 || dim <= 0 || length <= 0 || heads % kv_heads) return 0;
    if ((int64_t)tokens * (heads / kv_heads) > kFar) return 0;
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
    if ((int64_t)batch * heads * tokens * dim == 0) return 0;
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
    a.first_distance = bidirectional ? 1 - max_distance : 0;
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
    if (plan.chunks) {
        if (int e = kv_chunk_launch(a, batch, st)) return e;
    } else if (dim <= 64) kv_launch<1>(a, (unsigned)grid, st);
    else if (dim <= 128) kv_launch<2>(a, (unsigned)grid, st);
    else if (dim <= 192) kv_launch<3>(a, (unsigned)grid, st);
    else kv_launch<4>(a, (unsigned)grid, st);
    if (a.splits > 1)
        hipLaunchKernelGGL(k_kv_join, dim3((unsigned)ceil_div(rows, 4)), dim3(256), 0, st, a, plan.rows, (int)plan.chunks, (uint32_t)rows);
    return launch_status();
}

}  // extern "C"
