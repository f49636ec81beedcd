// What the kernels of the attention over fp16 keys and values share (attention.hip: forward, attention_bwd.hip: gradients).
#pragma once
#include "common.h"

namespace cpmk {

// (batch, heads, tokens, dim) fp16 under any strides, in elements
struct AttnTensor {
    half_t* p;
    int64_t batch, head, token, unit;
    __device__ __forceinline__ half_t* at(int64_t b, int64_t h) const { return p + b * batch + h * head; }
};

struct Attention {
    AttnTensor q, k, v, out;
    const int32_t *lens_each, *pos_each;
    const half_t* table;            // (heads, buckets) or null
    const int32_t* mapping;
    const uint8_t* mask;
    int64_t mask_batch, mask_token;
    float* lse;                     // (batch, heads, tokens): log2 of the sum of exp2(score), +inf of a query without keys; behind them (batch, held, parts): the largest magnitude
                                    // of a part's finite values, masked or not, up to the last key of any query; or null
    int64_t rows_in_all;
    half_t* rest;                   // with lse: what the rounding of `out` left, times 2^11, under the same strides
    float* parts;
    float scale;                    // with log2(e)
    int32_t len, pos;               // pos < 0: the queries are the last of the keys
    int32_t heads, held, group, tokens, dim, length, buckets, distances, first_distance;
    int32_t causal;
    int32_t row_tiles, splits;
};

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kAttnTile = 64;       // tokens a workgroup stages at a time
constexpr int32_t kAttnFar = 1 << 30, kAttnLong = 1 << 29;       // positions stay below the one, numbers of tokens and keys up to the other: distances fit 32 bits
constexpr int kBiasPad = 96;        // distances beyond the table's ends that a tile of 64 tokens and the 32 of a wave can reach into

// How tiles come: units beside each other or tokens beside each other, straight into LDS (kDirect, kTurned) or through registers (kAnyLayout, kColumns); rotary.hip: kRows
enum { kDirect = 0, kColumns = 1, kAnyLayout = 2, kTurned = 3, kRows = 4 };

struct AttnRange {
    int32_t len, pos;
};
__device__ __forceinline__ AttnRange attn_range(const Attention& a, int64_t b) {
    AttnRange r;
    r.len = max(0, min(a.lens_each ? a.lens_each[b] : a.len, a.length));
    r.pos = a.pos_each ? max(-kAttnFar, min(a.pos_each[b], kAttnFar - 1)) : a.pos < 0 ? r.len - a.tokens : min(a.pos, kAttnFar - 1);
    return r;
}

// The keys that a tile of rows looks at, and the parts they are cut into (the same here and where the parts are joined): `least` tiles each at least.
struct AttnParts {
    int32_t keys, tiles, per_part, parts;
};
__device__ __forceinline__ AttnParts attn_parts(const Attention& a, const AttnRange& r, int32_t last_query, int least, int tile) {
    AttnParts p;
    p.keys = a.causal ? max(0, min(r.len, r.pos + last_query + 1)) : r.len;
    p.tiles = (p.keys + tile - 1) / tile;
    p.per_part = max((p.tiles + a.splits - 1) / a.splits, min(least, max(p.tiles, 1)));
    p.parts = max(1, (p.tiles + p.per_part - 1) / p.per_part);
    return p;
}

// How a call is divided: rows of a workgroup, workgroups of rows, parts of the keys (of `least` tiles of `tile` keys at least), waves of a workgroup; few: attention_few.hip.
struct AttnPlan {
    int rows, row_tiles, splits, tile, least, waves;
    bool few;
};
AttnPlan attn_plan(int64_t batch, int64_t heads, int64_t held, int64_t tokens, int32_t dim, int64_t length, bool rows_of_keys, bool train);
AttnPlan attn_few_plan(int64_t batch, int64_t held, int64_t of_head, int32_t dim, int64_t length);
int attn_few_launch(const Attention& a, const AttnPlan& p, int32_t batch, hipStream_t st);

// The bucket of a distance (query - key) first_distance .. distances - 1; others are as those at the ends.  With biases for both signs first_distance is -1 at least: a key behind
// the query takes the upper half of the buckets however short the table is.  Numbers of buckets that the table does not have count as the nearest that it has.
__device__ __forceinline__ int32_t attn_bucket(const Attention& a, int32_t rel) {
    const int32_t bucket = min(a.mapping[min(abs(rel), a.distances - 1)], a.buckets) + (rel < 0 ? a.buckets / 2 : 0);
    return max(0, min(bucket, a.buckets - 1));
}

// The biases of a head by distance over the scores' scale, in LDS: where a product's sums begin.  Entry i is that of the distance i + first_distance - kBiasPad, clamped to the table's ends.
__device__ __forceinline__ int attn_bias_entries(const Attention& a) { return a.distances - a.first_distance + 2 * kBiasPad; }
__device__ __forceinline__ void attn_biases(const Attention& a, int32_t head, float scale, float* biases, int tid, int threads) {
    const float factor = kLog2e / scale;
    const half_t* const row = a.table + (int64_t)head * a.buckets;
    for (int i = tid; i < attn_bias_entries(a); i += threads)
        biases[i] = (float)row[attn_bucket(a, max(a.first_distance, min(i + a.first_distance - kBiasPad, a.distances - 1)))] * factor;
}

// Workgroup x of units * inner ones: the `inner` workgroups of a unit, which read the same keys, follow one another on one XCD, and units are dealt to the XCDs in turn.
__device__ __forceinline__ void attn_deal(uint32_t x, uint32_t units, uint32_t inner, uint32_t& unit, uint32_t& in) {
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

// ---- tiles of 64 tokens in LDS -----------------------------------------------------------------------------------------------
// A tile lies token by token, D units (64, 128 or 256) each, in pieces of eight units; piece c of token t at place c ^ swizzle(t) within its group of 16 (8 of 64 units): the 64 banks hold one
// token of 128 units or two of 64.  An operand of the matrix instructions is read in one of two ways, each free of conflicts: eight units of a token a lane (16 bytes; sixteen neighbouring
// lanes have neighbouring tokens, whose places differ), or, transposed, four tokens of a unit a lane (ds_read_b64_tr_b16: 16 lanes hand in the addresses of four tokens' 32 bytes; the places
// of 32 lanes' four tokens differ in the bits above the lowest two).  A thread that brings eight tokens of some units writes to them one after another, beside its neighbours', whose tokens
// are 8 apart: their places differ above the lowest bit.
template <int D>
__device__ __forceinline__ int attn_swizzle(int t) {
    const int r0 = t & 1, r1 = t >> 1 & 1, r2 = t >> 2 & 1, r3 = t >> 3 & 1, r4 = t >> 4 & 1, r5 = t >> 5 & 1;
    return D == 64 ? (r1 ^ r4) << 2 | r3 << 1 | (r2 ^ r5) : (r1 ^ r4) << 3 | (r0 ^ r5) << 2 | r3 << 1 | r2;
}
template <int D>
__device__ __forceinline__ int attn_place(int token, int piece) {
    constexpr int W = D == 64 ? 8 : 16;
    return token * D * 2 + (((piece & ~(W - 1)) | ((piece ^ attn_swizzle<D>(token)) & (W - 1))) << 4);
}

// Tiles of tensors whose tokens are neighbours lie unit by unit instead, as in memory, 64 tokens each, piece c of eight tokens of unit u at place c ^ turned(u).  The two ways of reading change
// places: tokens of the lanes through the transposing read, units of the lanes as they lie (8 bytes; u and u + 16 share banks).
__device__ __forceinline__ int attn_turned(int u) { return (u >> 1 & 1) << 2 | (u >> 3 & 1) << 1 | (u >> 2 & 1); }

typedef short short4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ half8_t attn_join(short4_t lo, short4_t hi) { return __builtin_bit_cast(half8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7)); }
__device__ __forceinline__ short4_t attn_read_turning(const int8_t* p) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(uintptr_t)p); }

template <int LAY>
constexpr bool kByUnit = LAY == kTurned || LAY == kColumns;

// Lane's address for operands of rows = tokens, units 16 s + 8 half + {0..7} of token (lane & 31) + 32 blk
template <int D, bool BY_UNIT = false>
__device__ __forceinline__ uint32_t attn_rows_at(int lane) {
    const int t = lane & 31, half = lane >> 5;
    if (BY_UNIT) {
        const int j = lane & 15, u = 8 * half + (j >> 2);
        return u * 128 + (((((lane >> 4) & 1) * 2 + ((j & 3) >> 1)) ^ attn_turned(u)) << 4) + (j & 1) * 8;
    }
    return t * D * 2 + ((half ^ attn_swizzle<D>(t)) << 4);
}
template <int D, bool BY_UNIT = false>
__device__ __forceinline__ half8_t attn_rows(const int8_t* tile, uint32_t at, int blk, int s) {
    if (BY_UNIT) {
        const int8_t* const p = tile + s * 16 * 128;
        return attn_join(attn_read_turning(p + (at ^ (blk << 6))), attn_read_turning(p + 4 * 128 + (at ^ (blk << 6) ^ 16)));
    }
    const int x = D == 64 ? (2 * s) ^ blk : ((2 * s) & 15) ^ (blk << 2);
    return *reinterpret_cast<const half8_t*>(tile + ((at ^ (x << 4)) + blk * 32 * D * 2 + (D == 256 ? (s >> 3) * 256 : 0)));
}
// Lane's address for operands of rows = units: of unit block n (32 units), tokens 32 blk + 16 e + 4 half + {0..3, 8..11}: the order in which the results of a product with tokens as
// rows lie in a lane's registers 8 e .. 8 e + 7.
template <int D, bool BY_UNIT = false>
__device__ __forceinline__ uint32_t attn_units_at(int lane) {
    const int half = lane >> 5, j = lane & 15, c = ((lane >> 4) & 1) * 2 + ((j & 3) >> 1), t = 4 * half + (j >> 2);
    if (BY_UNIT) return (lane & 31) * 128 + (attn_turned(lane & 31) << 4) + half * 8;
    return t * D * 2 + ((c ^ attn_swizzle<D>(t)) << 4) + (j & 1) * 8;
}
template <int D, bool BY_UNIT = false>
__device__ __forceinline__ half8_t attn_units(const int8_t* tile, uint32_t at, int n, int blk, int e) {
    if (BY_UNIT) {
        const int8_t* const p = tile + n * 32 * 128;
        const int x = blk * 4 + e * 2;
        return attn_join(*reinterpret_cast<const short4_t*>(p + (at ^ (x << 4))), *reinterpret_cast<const short4_t*>(p + (at ^ ((x + 1) << 4))));
    }
    const int x = D == 64 ? (n << 2) ^ (e << 2) ^ blk : ((n & 3) << 2) ^ (e << 3) ^ (blk << 2);
    const int8_t* const p = tile + (blk * 32 + e * 16) * D * 2 + (D == 256 ? (n >> 2) * 256 : 0);
    return attn_join(attn_read_turning(p + (at ^ (x << 4))), attn_read_turning(p + 8 * D * 2 + (at ^ ((x ^ 2) << 4))));
}

// Magnitudes, as bits, of finite numbers (the others make their queries' results no numbers whatever the gradients' factor is)
__device__ __forceinline__ ushort8_t attn_larger(ushort8_t m, half8_t v) {
    const ushort8_t b = __builtin_bit_cast(ushort8_t, v) & (uint16_t)0x7fff;
    return __builtin_elementwise_max(m, b & (ushort8_t)(b < (uint16_t)0x7c00));
}

// A thread's share of a tile on its way from memory to LDS through registers.  kColumns: eight tokens of PIECES neighbouring units, turned there.  Else pieces of eight units, unit by unit
// where they are not neighbours.  Tokens past the last one and units past the head's are zeros.
template <int D, int LAY, int THREADS>
struct AttnShare {
    static constexpr int PIECES = 64 * D / 8 / THREADS, RUN = D / 8, STEP = THREADS / RUN;      // (rows: a pass of the workgroup brings STEP tokens)
    static_assert(PIECES >= 1 && (LAY != kColumns || PIECES <= 8), "share of a tile");
    half8_t r[PIECES];

    __device__ __forceinline__ void load(const half_t* base, int64_t token, int64_t unit, int dim, int32_t t0, int32_t tokens, int tid) {
        if constexpr (LAY == kColumns) {
            const int tb = (tid & 7) * 8, u0 = (tid >> 3) * PIECES;
            const half_t* p[PIECES];
#pragma unroll
            for (int i = 0; i < PIECES; ++i) p[i] = base + min(u0 + i, dim - 1) * unit + tb;
            load_columns(p, t0, tokens, tb);
        } else if (unit == 1 && dim % 8 == 0) {
            const int row = tid / RUN, u = min((tid % RUN) * 8, dim - 8);
#pragma unroll
            for (int i = 0; i < PIECES; ++i) r[i] = load_half8_any(base + min(t0 + row + i * STEP, tokens - 1) * token + u);
        } else {
            const int row = tid / RUN, u = (tid % RUN) * 8;
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                half_t y[8];            // (element by element into the vector itself leaves it in scratch memory)
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = base[min(t0 + row + i * STEP, tokens - 1) * token + min(u + e, dim - 1) * unit];
                r[i] = half8_t{y[0], y[1], y[2], y[3], y[4], y[5], y[6], y[7]};
            }
        }
    }
    // p: the thread's units at its first token of the tensor's first tile, the tb-th
    __device__ __forceinline__ void load_columns(const half_t* const (&p)[PIECES], int32_t t0, int32_t tokens, int tb) {
        if (t0 + kAttnTile <= tokens) {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) r[i] = load_half8_any(p[i] + t0);
        } else {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                half_t y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = p[i][min(t0 + tb + e, tokens - 1) - tb];
                r[i] = half8_t{y[0], y[1], y[2], y[3], y[4], y[5], y[6], y[7]};
            }
        }
    }

    // Into LDS, zeros where there is nothing.  With `guard` numbers that are none or infinite become zeros as well, and their tokens' bits are set in `bad`: a product with a probability
    // of 0 would not be 0, and must not reach the tokens that do not see these.
    __device__ __forceinline__ void store(int8_t* tile, int dim, int32_t t0, int32_t tokens, int tid, bool guard, uint32_t* bad) {
        const bool whole = t0 + kAttnTile <= tokens && D == dim;
        const half8_t none = {0, 0, 0, 0, 0, 0, 0, 0};
        const int run = tid % RUN, first = LAY == kColumns ? (tid & 7) * 8 : tid / RUN, u0 = (tid >> 3) * PIECES;
        if (!whole)
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int units = LAY == kColumns ? (u0 + i < dim ? tokens - t0 - first : 0) : (t0 + first + i * STEP < tokens ? dim - run * 8 : 0);       // how many of the eight are real
                r[i] = half8_fill(r[i], half8_keep(units), none);
            }
        bool any = false;
        if (guard) {
            half8_t worst = none;
#pragma unroll
            for (int i = 0; i < PIECES; ++i) worst = __builtin_elementwise_fma(r[i], none, worst);
            const uint4_t w = __builtin_bit_cast(uint4_t, worst);
            any = ((w[0] | w[1] | w[2] | w[3]) & 0x7fff7fffu) != 0;
        }
        if constexpr (LAY == kColumns) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                run_t v;
#pragma unroll
                for (int i = 0; i < PIECES; ++i) v[i] = r[i][e];
                *reinterpret_cast<run_t*>(tile + attn_place<D>(first + e, u0 >> 3) + (u0 & 7) * 2) = v;
            }
        } else {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) *reinterpret_cast<half8_t*>(tile + attn_place<D>(first + i * STEP, run)) = r[i];
        }
        if (any) {          // (rare: what the thread has just written is looked through again)
#pragma unroll 1
            for (int i = 0; i < (LAY == kColumns ? 8 : PIECES); ++i) {
                const int token = LAY == kColumns ? first + i : first + i * STEP;
                half_t* const p = reinterpret_cast<half_t*>(tile + attn_place<D>(token, LAY == kColumns ? u0 >> 3 : run)) + (LAY == kColumns ? u0 & 7 : 0);
#pragma unroll 1
                for (int e = 0; e < (LAY == kColumns ? PIECES : 8); ++e)
                    if (!(p[e] * (half_t)0 == (half_t)0)) {
                        p[e] = (half_t)0;
                        atomicOr(bad + (token >> 5), 1u << (token & 31));
                    }
            }
        }
    }
    __device__ __forceinline__ ushort8_t largest(ushort8_t m) const {        // of the magnitudes, as bits
#pragma unroll
        for (int i = 0; i < PIECES; ++i) m = attn_larger(m, r[i]);
        return m;
    }
    typedef half_t run_t __attribute__((ext_vector_type(PIECES)));
};

// The same without registers, 16 bytes a lane straight into LDS: tensors whose units are neighbours, every token on a 16-byte boundary.  A wave brings sixteen tokens, 1 KB an
// instruction; which piece a lane fetches makes up for LDS being written in the order of the lanes.  Tokens past the last one are copies of it, places of units past the head's are left
// alone (attn_clear has made them zeros).
template <int D>
struct AttnDirect {
    static constexpr int PIECES = D / 32, EACH = 512 / D;       // instructions a wave and tile, tokens of one
    uint32_t off[PIECES];

    __device__ __forceinline__ void init(int64_t token, int wave, int lane) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) off[i] = (uint32_t)((wave * 16 + i * EACH + lane / (D / 8)) * (int32_t)token + piece(i, wave, lane) * 8) * 2;
    }
    static __device__ __forceinline__ int piece(int i, int wave, int lane) {
        constexpr int W = D == 64 ? 8 : 16;
        const int place = lane % (D / 8);
        return (place & ~(W - 1)) | ((place ^ attn_swizzle<D>(wave * 16 + i * EACH + lane / (D / 8))) & (W - 1));
    }
    __device__ __forceinline__ void issue(const half_t* tile, int64_t token, int32_t count, int8_t* lds, int dim, int wave, int lane) const {
        const uint32_t to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) int8_t*)lds + wave * 16 * D * 2;
        if (dim == D && count >= kAttnTile) {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) lds_dma16(off[i], reinterpret_cast<const int8_t*>(tile), to + i * 1024);
        } else {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int over = max(0, wave * 16 + i * EACH + lane / (D / 8) - (count - 1));
                if (piece(i, wave, lane) * 8 < dim) lds_dma16(off[i] - (uint32_t)(over * (int32_t)token) * 2, reinterpret_cast<const int8_t*>(tile), to + i * 1024);
            }
        }
    }
    // Numbers that are none or infinite among what the wave has brought become zeros, their tokens' bits are set
    static __device__ __forceinline__ void guard(int8_t* lds, int wave, int lane, uint32_t* bad) {
        half_t* const p = reinterpret_cast<half_t*>(lds + wave * 16 * D * 2 + lane * 16);
        const half8_t none = {0, 0, 0, 0, 0, 0, 0, 0};
        half8_t worst = none;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) worst = __builtin_elementwise_fma(*reinterpret_cast<const half8_t*>(p + i * 512), none, worst);
        const uint4_t w = __builtin_bit_cast(uint4_t, worst);
        if ((w[0] | w[1] | w[2] | w[3]) & 0x7fff7fffu) {
#pragma unroll 1
            for (int i = 0; i < PIECES * 8; ++i) {
                half_t* const x = p + (i >> 3) * 512 + (i & 7);
                const int t = wave * 16 + (i >> 3) * EACH + lane / (D / 8);
                if (!(*x * (half_t)0 == (half_t)0)) {
                    *x = (half_t)0;
                    atomicOr(bad + (t >> 5), 1u << (t & 31));
                }
            }
        }
    }
    static __device__ __forceinline__ ushort8_t largest(ushort8_t m, const int8_t* lds, int wave, int lane) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) m = attn_larger(m, *reinterpret_cast<const half8_t*>(lds + wave * 16 * D * 2 + i * 1024 + lane * 16));
        return m;
    }
};
// Zeros in tiles' buffers, where a head has fewer units than they have room for
__device__ __forceinline__ void attn_clear(int8_t* lds, int bytes, int tid, int threads) {
    for (int i = tid; i < bytes / 16; i += threads) reinterpret_cast<uint4_t*>(lds)[i] = uint4_t{0, 0, 0, 0};
}

// Pieces of eight tokens from `token` on, `step` bytes apart: numbers that are none or infinite become zeros, their tokens' bits are set
__device__ __forceinline__ void attn_clean_turned(int8_t* p, int step, int pieces, int token, uint32_t* bad) {
#pragma unroll 1
    for (int i = 0; i < pieces * 8; ++i) {
        half_t* const x = reinterpret_cast<half_t*>(p + (i >> 3) * step) + (i & 7);
        const int t = token + (i & 7);
        if (!(*x * (half_t)0 == (half_t)0)) {
            *x = (half_t)0;
            atomicOr(bad + (t >> 5), 1u << (t & 31));
        }
    }
}

// A tensor's tiles, one after another (largest: of the magnitudes of a tile's first `count` tokens, or copies of them): `fetch` asks for one, `place`, when it has arrived, puts it into LDS (kDirect: it is there, behind wait_vmcnt); bad: to be guarded (AttnShare::store),
// or null.  kDirect writes the buffer from `fetch` on.
template <int D, int LAY>
struct AttnTiles {
    const half_t* base;
    int64_t token, unit;
    AttnShare<D, LAY, 256> share;
    __device__ __forceinline__ void init(const half_t* b, const AttnTensor& t, int32_t, int, int, int, int) { base = b, token = t.token, unit = t.unit; }
    __device__ __forceinline__ void advance(int64_t by) { base += by; }
    __device__ __forceinline__ void fetch(int8_t*, int dim, int32_t t0, int32_t tokens, int tid, int, int) { share.load(base, token, unit, dim, t0, tokens, tid); }
    __device__ __forceinline__ void place(int8_t* lds, int dim, int32_t t0, int32_t tokens, int tid, int, int, uint32_t* bad) { share.store(lds, dim, t0, tokens, tid, bad != nullptr, bad); }
    __device__ __forceinline__ ushort8_t largest(ushort8_t m, const int8_t*, int32_t, int, int) const { return share.largest(m); }
};
// (pieces of eight tokens of a unit, beside each other in memory: PIECES units of a thread, 32 apart)
template <int D>
struct AttnTiles<D, kColumns> {
    static constexpr int PIECES = D / 32;
    const half_t* p;
    int64_t unit;
    half8_t r[PIECES];
    __device__ __forceinline__ void init(const half_t* b, const AttnTensor& t, int32_t, int dim, int tid, int, int) { p = b + min(tid >> 3, dim - 1) * t.unit + (tid & 7) * 8, unit = t.unit; }
    __device__ __forceinline__ void advance(int64_t by) { p += by; }
    __device__ __forceinline__ void fetch(int8_t*, int dim, int32_t t0, int32_t tokens, int tid, int, int) {
        const int tb = (tid & 7) * 8, u = tid >> 3;
        const half8_t none = {0, 0, 0, 0, 0, 0, 0, 0};
        if (t0 + kAttnTile <= tokens) {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) r[i] = load_half8_any(p + (u + i * 32 < dim ? i * 32 : 0) * unit + t0);
        } else {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                half_t y[8];
                const half_t* const q = p + (u + i * 32 < dim ? i * 32 : 0) * unit - tb;
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = q[min(t0 + tb + e, tokens - 1)];
                r[i] = half8_fill(half8_t{y[0], y[1], y[2], y[3], y[4], y[5], y[6], y[7]}, half8_keep(tokens - t0 - tb), none);
            }
        }
    }
    __device__ __forceinline__ void place(int8_t* lds, int dim, int32_t, int32_t, int tid, int, int, uint32_t* bad) {
        const int u = tid >> 3, c = tid & 7;
        const half8_t none = {0, 0, 0, 0, 0, 0, 0, 0};
        if (dim < D)
#pragma unroll
            for (int i = 0; i < PIECES; ++i)
                if (u + i * 32 >= dim) r[i] = none;
        half8_t worst = none;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            *reinterpret_cast<half8_t*>(lds + (u + i * 32) * 128 + ((c ^ attn_turned(u)) << 4)) = r[i];
            worst = __builtin_elementwise_fma(r[i], none, worst);
        }
        if (bad == nullptr) return;
        const uint4_t w = __builtin_bit_cast(uint4_t, worst);
        if ((w[0] | w[1] | w[2] | w[3]) & 0x7fff7fffu) attn_clean_turned(lds + u * 128 + ((c ^ attn_turned(u)) << 4), 32 * 128, PIECES, c * 8, bad);
    }
    __device__ __forceinline__ ushort8_t largest(ushort8_t m, const int8_t*, int32_t, int, int) const {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) m = attn_larger(m, r[i]);
        return m;
    }
};
// Straight into LDS: a wave brings D / 4 units, eight an instruction.  Whole pieces of tokens: their number is a multiple of eight, and pieces past the end are copies of the last one.
template <int D>
struct AttnTiles<D, kTurned> {
    static constexpr int PIECES = D / 32;
    const half_t* base;
    int64_t unit;
    int32_t all;            // tokens of the tensor
    uint32_t off;           // (units 8 apart have the same places but for bit 1)
    __device__ __forceinline__ void init(const half_t* b, const AttnTensor& t, int32_t tokens, int, int, int wave, int lane) {
        base = b, unit = t.unit, all = tokens;
        off = (uint32_t)((lane >> 3) * (int32_t)unit) * 2;
    }
    __device__ __forceinline__ void advance(int64_t by) { base += by; }
    __device__ __forceinline__ void fetch(int8_t* lds, int dim, int32_t t0, int32_t, int, int wave, int lane) {
        const uint32_t to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) int8_t*)lds + wave * (D / 4) * 128;
        const int most = min(7, ((all - t0) >> 3) - 1);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int u = wave * (D / 4) + i * 8 + (lane >> 3), c = (lane & 7) ^ attn_turned(u);
            if (dim == D || u < dim) lds_dma16(off + min(c, most) * 16, reinterpret_cast<const int8_t*>(base + (int64_t)(wave * (D / 4) + i * 8) * unit + t0), to + i * 1024);
        }
    }
    __device__ __forceinline__ void place(int8_t* lds, int, int32_t, int32_t, int, int wave, int lane, uint32_t* bad) {
        if (bad == nullptr) return;
        const half8_t none = {0, 0, 0, 0, 0, 0, 0, 0};
        half8_t worst = none;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) worst = __builtin_elementwise_fma(*reinterpret_cast<const half8_t*>(lds + wave * (D / 4) * 128 + i * 1024 + lane * 16), none, worst);
        const uint4_t w = __builtin_bit_cast(uint4_t, worst);
        if ((w[0] | w[1] | w[2] | w[3]) & 0x7fff7fffu)
#pragma unroll 1
            for (int i = 0; i < PIECES; ++i) attn_clean_turned(lds + wave * (D / 4) * 128 + i * 1024 + lane * 16, 0, 1, ((lane & 7) ^ attn_turned(wave * (D / 4) + i * 8 + (lane >> 3))) * 8, bad);
    }
    __device__ __forceinline__ ushort8_t largest(ushort8_t m, const int8_t* lds, int32_t count, int wave, int lane) const {
        const half8_t none = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int c = (lane & 7) ^ attn_turned(wave * (D / 4) + i * 8 + (lane >> 3));
            const half8_t x = *reinterpret_cast<const half8_t*>(lds + wave * (D / 4) * 128 + i * 1024 + lane * 16);
            m = attn_larger(m, count < kAttnTile ? half8_fill(x, half8_keep(count - c * 8), none) : x);
        }
        return m;
    }
};
template <int D>
struct AttnTiles<D, kDirect> {
    const half_t* base;
    int64_t token;
    AttnDirect<D> direct;
    __device__ __forceinline__ void init(const half_t* b, const AttnTensor& t, int32_t, int, int, int wave, int lane) {
        base = b, token = t.token;
        direct.init(token, wave, lane);
    }
    __device__ __forceinline__ void advance(int64_t by) { base += by; }
    __device__ __forceinline__ void fetch(int8_t* lds, int dim, int32_t t0, int32_t tokens, int, int wave, int lane) { direct.issue(base + t0 * token, token, tokens - t0, lds, dim, wave, lane); }
    __device__ __forceinline__ void place(int8_t* lds, int, int32_t, int32_t, int, int wave, int lane, uint32_t* bad) {
        if (bad != nullptr) AttnDirect<D>::guard(lds, wave, lane, bad);
    }
    __device__ __forceinline__ ushort8_t largest(ushort8_t m, const int8_t* lds, int32_t, int wave, int lane) const { return AttnDirect<D>::largest(m, lds, wave, lane); }
};

// Operands that the waves keep of tensors whose tokens are neighbours in memory, of 128 tokens from t0 on: through two tiles in LDS (`bring`, then, behind a barrier, `keep`).
template <int D>
__device__ __forceinline__ void attn_bring_columns(const AttnTensor& t, const half_t* base, int32_t t0, int32_t tokens, int dim, int tid, int8_t* tiles) {
    AttnShare<D, kColumns, 256> share[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) share[i].load(base, t.token, t.unit, dim, t0 + i * kAttnTile, tokens, tid);
#pragma unroll
    for (int i = 0; i < 2; ++i) share[i].store(tiles + i * kAttnTile * D * 2, dim, t0 + i * kAttnTile, tokens, tid, false, nullptr);
}
template <int D, int KS>
__device__ __forceinline__ void attn_keep_columns(half8_t (&x)[KS], const int8_t* tiles, int wave, int lane) {
    const uint32_t at = attn_rows_at<D>(lane);
#pragma unroll
    for (int s = 0; s < KS; ++s) x[s] = attn_rows<D>(tiles + (wave >> 1) * kAttnTile * D * 2, at, wave & 1, s);
}

// 32 bytes of a row of a mask, on their way from memory, as bits.  LONG: rows of 32 at least
template <bool LONG>
struct AttnMaskShare {
    uint4_t raw[2];
    __device__ __forceinline__ void load(const uint8_t* row, int32_t key, int32_t length) {
        struct __attribute__((packed, aligned(1))) Byte16Any { uint32_t w[4]; };
        if (!LONG && length < 32) return;
        const uint8_t* const p = row + min(key, length - 32);
        raw[0] = __builtin_bit_cast(uint4_t, *reinterpret_cast<const Byte16Any*>(p));
        raw[1] = __builtin_bit_cast(uint4_t, *reinterpret_cast<const Byte16Any*>(p + 16));
    }
    __device__ __forceinline__ uint32_t bits(const uint8_t* row, int32_t key, int32_t length) const {
        uint32_t all = 0;
        if (!LONG && length < 32) {
#pragma unroll 1
            for (int i = 0; key + i < length; ++i) all |= (row[key + i] != 0 ? 1u : 0u) << i;
            return all;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            uint32_t m = raw[i >> 2][i & 3];
            m |= m >> 4;
            m |= m >> 2;
            m |= m >> 1;                    // the lowest bit of a byte: whether any was set
            all |= ((m & 0x01010101u) * 0x10204080u >> 28) << (4 * i);
        }
        const int over = key - min(key, length - 32);
        return over < 32 ? all >> over : 0u;
    }
};

// An operand that a wave keeps: eight units from 16 s + 8 half on of the lane's token, zeros past the head's last unit.
template <int KS>
__device__ __forceinline__ void attn_keep(half8_t (&x)[KS], const AttnTensor& t, const half_t* row, int dim, int half) {
    if (t.unit == 1 && dim % 8 == 0) {
#pragma unroll
        for (int s = 0; s < KS; ++s) x[s] = load_half8_any(row + min(s * 16 + half * 8, dim - 8));
    } else {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            half_t y[8];            // (element by element into the operand itself leaves it in scratch memory)
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = row[min(s * 16 + half * 8 + e, dim - 1) * t.unit];
            x[s] = half8_t{y[0], y[1], y[2], y[3], y[4], y[5], y[6], y[7]};
        }
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) x[s] = half8_fill(x[s], half8_keep(dim - s * 16 - half * 8), half8_t{0, 0, 0, 0, 0, 0, 0, 0});
}

constexpr float kRest = 2048.0f;        // fp16 has 11 bits: what a rounding leaves, times this, is as large as the number at most

// A wave's results, transposed (units n * 32 + 8 c + 4 half + {0..3} in registers 4 c .., a token a lane), times the lane's f, as fp16 to the tokens first .. first + 31 below `tokens`; or,
// REST, what that rounding leaves.  Through LDS of the wave's own (80 D bytes), so that 16 bytes a lane go out side by side, units or tokens, whichever are neighbours in memory.
template <int NT, bool REST = false>
__device__ __forceinline__ void attn_write(const AttnTensor& t, half_t* base, const float16_tv (&acc)[NT], float f, int32_t first, int32_t tokens, int dim, int lane, int8_t* lds) {
    constexpr int D = NT <= 2 ? 64 : NT <= 4 ? 128 : 256;
    const int col = lane & 31, half = lane >> 5, count = min(32, tokens - first);
    if (count <= 0) return;
    const auto rounded = [&](float x) {
        x *= f;
        const half_t r = round_f16(x);
        return REST ? (half_t)((x - (float)r) * kRest) : r;
    };
    if (t.unit == 1 && dim % 8 == 0) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                half4_t v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = rounded(acc[n][c * 4 + e]);
                *reinterpret_cast<half4_t*>(lds + attn_place<D>(col, n * 4 + c) + half * 8) = v;
            }
        asm volatile("" ::: "memory");
        const int piece = lane % (D / 8);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            const int token = i * (512 / D) + lane / (D / 8);
            const half8_t v = *reinterpret_cast<const half8_t*>(lds + attn_place<D>(token, piece));
            if (token < count && piece * 8 < dim) store_half8_any(base + (first + token) * t.token + piece * 8, v);
        }
    } else if (t.token == 1) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) *reinterpret_cast<half_t*>(lds + (n * 32 + (i >> 2) * 8 + half * 4 + (i & 3)) * 80 + col * 2) = rounded(acc[n][i]);
        asm volatile("" ::: "memory");
        const int at = (lane & 3) * 8;
#pragma unroll
        for (int i = 0; i < NT * 2; ++i) {
            const int unit = i * 16 + (lane >> 2);
            const half8_t v = *reinterpret_cast<const half8_t*>(lds + unit * 80 + at * 2);
            half_t* const p = base + unit * t.unit + first + at;
            if (unit < dim && at < count) {
                if (at + 8 <= count) store_half8_any(p, v);
                else
#pragma unroll 1
                    for (int e = 0; at + e < count; ++e) p[e] = reinterpret_cast<const half_t*>(lds + unit * 80 + at * 2)[e];
            }
        }
    } else if (col < count) {
        half_t* const row = base + (first + col) * t.token;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int u = n * 32 + (i >> 2) * 8 + half * 4 + (i & 3);
                if (u < dim) row[u * t.unit] = rounded(acc[n][i]);
            }
    }
    asm volatile("" ::: "memory");
}

// The order of a stretch of products whose operands come from LDS, first M1 of R1 reads, then M2 of M2: eight reads ahead, so that their latency lies behind products (the compiler by
// itself reads an operand right before its product and waits).
// With B: before M2, B other reads (where its sums begin).
template <int M1, int R1, int M2, int R2, int B = 0>
__device__ __forceinline__ void attn_pace() {
    constexpr int kEach1 = M1 ? R1 / M1 : 1, kEach2 = M2 ? R2 / M2 : 1, kAhead = M2 == 0 || R2 >= 8 ? 8 : R2;
    static_assert((M1 == 0 || R1 % M1 == 0) && (M2 == 0 || R2 % M2 == 0), "reads of a product");
    if (B) __builtin_amdgcn_sched_group_barrier(0x100, B, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
    for (int i = 0; i < M1; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        if (M2 > 0 || i < M1 - kAhead / kEach1) __builtin_amdgcn_sched_group_barrier(0x100, kEach1, 0);
    }
#pragma unroll
    for (int i = 0; i < M2; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        if (i < M2 - kAhead / kEach2) __builtin_amdgcn_sched_group_barrier(0x100, kEach2, 0);
    }
}

// Where the sums of a tile's scores begin, for a wave with keys as rows: the biases' entries from `first` on downwards
__device__ __forceinline__ void attn_begin(float16_tv& s, int blk, const float* first) {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = first[-(blk * 32 + (i >> 2) * 8 + (i & 3))];
}
// The lane's entry for key 0 of a tile of 64 (or 32) keys, its query being `rel` behind it: windows beyond the table's ends are moved into the entries of the end that they are beyond
__device__ __forceinline__ const float* attn_window(const Attention& a, const float* biases, int32_t rel, int half) {
    return biases + max(63, min(rel - half * 4 - (a.first_distance - kBiasPad), attn_bias_entries(a) - 1));
}
// Scores of keys that a query's mask leaves out: -inf (whatever they are).  bits: the half's first key lowest
__device__ __forceinline__ void attn_cap(float16_tv& s, uint32_t bits) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const uint32_t keep = (int32_t)(bits << (31 - ((i >> 2) * 8 + (i & 3)))) >> 31;
        const float x = s[i];           // (a bit cast of a vector's element itself takes the first one's)
        s[i] = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, x) & keep) | (0xff800000u & ~keep));
    }
}

constexpr float16_tv kZero16 = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};

// The layout by which tiles of two tensors are brought: straight into LDS where every piece of 16 bytes is on its boundary, through registers elsewhere (columns, gradients of 64 heads of 64
// units, 4 x 1024 tokens and 4 x 1025: 340 and 650 us; 32 of 128: 360 and 610)
inline bool attn_direct(const AttnTensor& x, int32_t dim) {
    return x.unit == 1 && dim % 8 == 0 && aligned16(x.p) && x.batch % 8 == 0 && x.head % 8 == 0 && x.token % 8 == 0 && x.token >= 0 && x.token < (1 << 23);        // (64 tokens: offsets of 32 bits)
}
inline bool attn_turnable(const AttnTensor& x, int32_t tokens) {
    return x.token == 1 && tokens % 8 == 0 && aligned16(x.p) && x.batch % 8 == 0 && x.head % 8 == 0 && x.unit % 8 == 0 && x.unit >= 0 && x.unit < (1 << 26);         // (eight units: the same)
}
inline int attn_layout(const AttnTensor& x, const AttnTensor& y, int32_t dim, int32_t tokens) {
    if (attn_direct(x, dim) && attn_direct(y, dim)) return kDirect;
    if (attn_turnable(x, tokens) && attn_turnable(y, tokens)) return kTurned;
    return x.token == 1 && y.token == 1 ? kColumns : kAnyLayout;
}

// What forward and backward refuse; sets heads and the table's first distance.  0 or an error code; `empty`: tensors without elements whatever the numbers of tokens and keys.
inline int attn_check(Attention& a, int32_t batch, int32_t heads, int32_t kv_heads, int bidirectional, bool& empty) {
    empty = false;
    if (batch < 0 || heads < 0 || kv_heads < 0 || a.tokens < 0 || a.dim < 0 || a.length < 0) return CPMK_EBADARG;
    if (!a.lens_each && (a.len < 0 || a.len > a.length)) return CPMK_EBADARG;
    if (batch == 0 || heads == 0 || a.dim == 0) {
        empty = true;
        return 0;
    }
    if (kv_heads == 0 || heads % kv_heads) return CPMK_EBADARG;
    if (a.dim > 256 || a.tokens > kAttnLong || a.length > kAttnLong || !grid_fits((int64_t)batch * heads)) return CPMK_ETOOBIG;
    if (!(fabsf(a.scale) < __builtin_inff())) return CPMK_EBADARG;
    // (products of fp16 numbers sum up to 2^40 at most: times this they are nothing beside 1, while biases over it would leave fp32)
    if (fabsf(a.scale) < 0x1p-100f) a.scale = 0.0f;
    if (a.table && (!a.mapping || a.buckets <= 0 || a.distances <= 0)) return CPMK_EBADARG;
    if (a.table && (int64_t)a.distances * (bidirectional ? 2 : 1) > 1024) return CPMK_ETOOBIG;
    a.heads = heads, a.held = kv_heads, a.group = heads / kv_heads;
    a.first_distance = bidirectional ? (a.distances > 1 ? 1 - a.distances : -1) : 0;
    if ((a.tokens > 0 && any_null(a.q.p, a.out.p)) || (a.length > 0 && any_null(a.k.p, a.v.p))) return CPMK_EBADARG;
    return 0;
}

}  // namespace cpmk
