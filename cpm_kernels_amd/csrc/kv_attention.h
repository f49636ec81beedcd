// What the kernels of the attention over the 8-bit key/value cache share (kv_attention.hip: few queries, kv_chunk.hip: many).
#pragma once
#include "kv_ints.h"

namespace cpmk {

struct KvAttention {
    const half_t* q;
    int64_t q_batch, q_head, q_token, q_unit;
    const int8_t *keys, *values;
    const half_t *key_top, *value_top;
    const int32_t *lens_each, *pos_each;
    const half_t* table;            // (heads, buckets) or null
    const int32_t* mapping;
    const uint8_t* mask;
    int64_t mask_batch, mask_token;
    half_t* out;
    int64_t out_batch, out_head, out_token, out_unit;
    float* parts;
    float scale;                    // with log2(e)
    int32_t len, pos;               // pos < 0: the queries are the last of the keys
    int32_t heads, held, group, tokens, dim, length, block_shift, buckets, distances, first_distance;
    int32_t causal;
    int32_t row_tiles, splits;
};

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kTile = 64;           // keys a wave takes at a time
constexpr int32_t kFar = 1 << 30;   // positions and rows stay below
constexpr int kLazy = 8;             // log2 of how far the running maximum may lie below the true one
constexpr int kChunkRows = 128;     // queries of a workgroup (kv_chunk.hip)
constexpr int kChunkLeast = 4;       // tiles of a part, at least (kv_chunk.hip)
constexpr int kChunkPad = 96;        // distances beyond the table's ends that a tile of 32 queries and 64 keys can reach into

__device__ __forceinline__ float kv_scale(half_t top) { return fmaxf((float)top * (1.0f / 127.0f), 0x1p-34f); }

// The keys that a tile of rows looks at: how many, and the parts they are cut into (the same here and where the parts are joined).
struct KvRange {
    int32_t len, pos, keys, tiles, per_part, parts;
};
__device__ __forceinline__ KvRange kv_range(const KvAttention& a, int64_t b, int32_t last_query, int least) {
    KvRange r;
    r.len = max(0, min(a.lens_each ? a.lens_each[b] : a.len, a.length));
    r.pos = a.pos_each ? max(-kFar, min(a.pos_each[b], kFar - 1)) : a.pos < 0 ? r.len - a.tokens : min(a.pos, kFar - 1);
    r.keys = a.causal ? max(0, min(r.len, r.pos + last_query + 1)) : r.len;
    r.tiles = (r.keys + kTile - 1) / kTile;
    r.per_part = max((r.tiles + a.splits - 1) / a.splits, min(least, max(r.tiles, 1)));
    r.parts = max(1, (r.tiles + r.per_part - 1) / r.per_part);
    return r;
}

// The bias of a head at a distance first_distance .. distances - 1 (others are as those at the ends).  With biases for both signs first_distance is -1 at least, where the table has
// one distance only: a key behind the query takes the upper half of the buckets however short the table is.  Numbers of buckets that the table does not have (position_embedding_init
// gives such where the distances are no multiple of the buckets that are exact) count as the nearest that it has.
__device__ __forceinline__ half_t kv_bias(const KvAttention& a, int32_t head, int32_t rel) {
    const int32_t bucket = min(a.mapping[min(abs(rel), a.distances - 1)], a.buckets) + (rel < 0 ? a.buckets / 2 : 0);
    return a.table[(int64_t)head * a.buckets + max(0, min(bucket, a.buckets - 1))];
}

// Workgroup x of units * inner ones: the `inner` workgroups of a unit, which read the same keys, follow one another on one XCD, and units are dealt to the XCDs in turn (of sequences of
// unequal length no XCD gets the long ones).
__device__ __forceinline__ void kv_deal(uint32_t x, uint32_t units, uint32_t inner, uint32_t& unit, uint32_t& in) {
    const uint32_t whole = units & ~7u;
    if (x < whole * inner) {
        const uint32_t y = x >> 3, u = y / inner;
        unit = u * 8 + (x & 7);
        in = y - u * inner;
    } else {
        x -= whole * inner;
        in = x / (units - whole);
        unit = whole + (x - in * (units - whole));
    }
}

// Eight units of a query from each of `first[]` on, zeros past the head's last one.  Every load is made, inside the row, so that none waits for another.
template <int N, class First>
__device__ __forceinline__ void load_query(half8_t (&q)[N], const half_t* p, int64_t stride, int dim, First first) {
    if (stride == 1) {
#pragma unroll
        for (int s = 0; s < N; ++s) q[s] = load_half8_any(p + min(first(s), dim - 8));
    } else {
#pragma unroll
        for (int s = 0; s < N; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) q[s][e] = p[(min(first(s), dim - 8) + e) * stride];
    }
#pragma unroll
    for (int s = 0; s < N; ++s)
        if (first(s) >= dim) q[s] = half8_t{0, 0, 0, 0, 0, 0, 0, 0};
}

// Many queries (kv_chunk.hip): 0 or an error code.
int kv_chunk_launch(const KvAttention& a, int32_t batch, hipStream_t st);

}  // namespace cpmk
