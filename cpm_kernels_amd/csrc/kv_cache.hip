// The key/value cache in 8 bits: tokens in (quantised as they are written) and out again.
//
// A block of `block` tokens of one head keeps its largest magnitude a = max |x| beside it (fp16: the value itself, so it is exact) and every element as
//     q = round(127 x / a),  halves away from zero,            and stands for q a / 127.
// (The row quantisers keep fp16(a / 127) instead; that is a subnormal number for a < 2^-7, and a block of small values would lose its bits with it.)
// An infinity counts as +-65504, a NaN as 0: one bad element would take its block with it.  A write that begins inside a block meets the older tokens of its sequence there: the
// block's magnitude becomes a' = max(a, max |new x|) and the older integers q' = round(q a / a').  Bytes behind the last token that is written stay as they are.
//
// One fused product and addition an element gives the rounded quotient (kv_round.h; tests/native/kv_round_fma_check.cpp goes through every pair with that header's own functions).
//
// Storage: keys (batch, heads, length, dim), values (batch, heads, length / 16, dim, 16): what the attention reads as matrix operands is 16 contiguous
// bytes in both, sixteen units of a token and sixteen tokens of a unit.  Such a run is the "minor" axis here, and a lane takes a piece of 4 (major) x 16 (minor) elements:
// four 16-byte accesses to the cache; to and from the fp16 side 32 contiguous bytes four times where the minor axis is contiguous there too ("straight"), 8 bytes sixteen
// times where the major axis is ("crossed"), single halves otherwise and at the ends of a range.
//
// Bound by memory.  Writing 8 x 64 heads x 512 tokens of 64 units (101 MB) takes 25 us: all loads, a barrier, then all stores, two rounds of workgroups (124 registers, so 1024 of 2048 at once); with the
// pieces at a range's ends read twice instead of kept, 85 registers (1280 at once), the same took 24 us and ragged prompts 27 instead of 15.6 (1280 workgroups: a round and a quarter here).  A block that the range cuts is
// loaded element by element and written as a whole: 5 tokens in the middle of a block of 64 take 14.2 us for 32 x 64 heads of 64 units, 16 take 18.5, where one takes 4.2 (k_kv_write_token).
// Reading 16 x 64 x 1024 (403 MB) takes 85 us, 4.7 TB/s: the hint for data that is not read again, which the loads carry, changes neither loads nor stores (83 to 87), nor do rows of 256 or 512 bytes a wave
// instead of 128 (82 to 87).
#include "kv_ints.h"
#include "kv_round.h"

namespace cpmk {

enum { kStraight = 0, kCrossed = 1, kAnyStride = 2 };

struct KvSide {             // keys or values
    const half_t* x;        // write: tokens in, read: tokens out (element strides below)
    int64_t batch, head, token, unit;
    int8_t* ints;
    half_t* top;            // (batch, heads, length / block)
    int mode;
};

struct KvArgs {
    KvSide side[2];
    const int32_t *pos_each, *count_each;
    int32_t pos, tokens, heads, dim, length, block;
    int32_t block_shift;
    int32_t span;           // tokens of a workgroup: whole blocks (write), a multiple of 16 (read)
    int32_t pieces;         // of a workgroup, span * dim / 64
    uint32_t chunks;        // workgroups of a head
};

// Where a lane's piece lies: `major[e]` and the first of the sixteen minors, in tokens from the workgroup's first one and units.  The four majors are as far apart
// as the accesses of a wave are best served by: four neighbours where they are read together, else a quarter of `apart` (of the units) from one to the next.
template <bool V>
__device__ __forceinline__ void piece_of(int idx, int dim, int apart, bool neighbours, int (&major)[4], int& minor) {
    if (V) {
        const int quads = dim >> 2, group = idx / quads, u = idx - group * quads;
        minor = group * 16;
#pragma unroll
        for (int e = 0; e < 4; ++e) major[e] = neighbours ? u * 4 + e : u + e * quads;
    } else {
        const int runs = dim >> 4, r = idx / runs;
        minor = (idx - r * runs) * 16;
        const int q = apart >> 2, blk = r / q;
#pragma unroll
        for (int e = 0; e < 4; ++e) major[e] = neighbours ? r * 4 + e : blk * apart + (r - blk * q) + e * q;
    }
}

// The nearest integer of x times a factor of kv_factor, halves away from zero: its low byte in the low byte of the bits.
__device__ __forceinline__ uint32_t nearest_bits(float x, float factor) {
    float t = kv_shifted(x, factor);
    asm("" : "+v"(t));
    return __builtin_bit_cast(uint32_t, t);
}

template <bool V>
__device__ __forceinline__ void write_piece(const KvArgs& a, const KvSide& s, uint32_t* tops, int64_t b, int32_t h, int32_t first, int32_t pos, int32_t end) {
    const int tid = threadIdx.x;
    const int64_t head = b * a.heads + h;
    half_t* const top = s.top + head * (a.length / a.block) + first / a.block;
    // tops[0 ..]: the blocks' magnitudes (bit patterns); behind them the first block's old one, if it holds older tokens
    const int blocks = a.span / a.block;
    for (int i = tid; i <= blocks; i += blockDim.x) {
        uint32_t old = 0;
        if ((i == 0 || i == blocks) && first < pos) old = min((uint32_t)(__builtin_bit_cast(uint16_t, top[0]) & 0x7fff), 0x7bffu);
        tops[i] = old;
    }
    const bool mine = tid < a.pieces;
    int major[4], minor;
    piece_of<V>(mine ? tid : 0, a.dim, a.block, s.mode != kStraight, major, minor);
    const int32_t t_lo = first + (V ? minor : major[0]), t_hi = first + (V ? minor + 15 : major[3]);
    const bool whole = t_lo >= pos && t_hi < end && s.mode != kAnyStride;
    const bool some = mine && t_lo < end;                 // (a piece behind the end, in a block of its own or not, stays as it is)
    const half_t* const x = s.x + b * s.batch + h * s.head - (int64_t)pos * s.token;
    int8_t* const ints = s.ints + head * a.length * a.dim + (int64_t)first * a.dim;
    auto place = [&](int e) { return V ? ints + (int64_t)minor * a.dim + major[e] * 16 : ints + (int64_t)major[e] * a.dim + minor; };
    half8_t v[4][2];
    uint4_t old[4];
    if (some) {
        if (whole && s.mode == kStraight) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const half_t* p = V ? x + (int64_t)(first + minor) * s.token + major[e] * s.unit : x + (int64_t)(first + major[e]) * s.token + minor * s.unit;
                v[e][0] = load_half8_any(p);
                v[e][1] = load_half8_any(p + 8);
            }
        } else if (whole) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const half_t* p = V ? x + (int64_t)(first + minor + i) * s.token + major[0] * s.unit : x + (int64_t)(first + major[0]) * s.token + (minor + i) * s.unit;
                const half4_t q = __builtin_bit_cast(half4_t, *reinterpret_cast<const Half4Any*>(p));
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e][i >> 3][i & 7] = q[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                old[e] = *reinterpret_cast<const uint4_t*>(place(e));
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int32_t t = first + (V ? minor + i : major[e]), u = V ? major[e] : minor + i;
                    v[e][i >> 3][i & 7] = t >= pos && t < end ? x[(int64_t)t * s.token + (int64_t)u * s.unit] : (half_t)0.0f;
                }
            }
        }
    }
    __syncthreads();
    const int slot = (V ? minor : major[0]) / a.block;
    if (some) {
        ushort8_t mb = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e) mb = absbits_max(absbits_max(mb, v[e][0]), v[e][1]);
        uint32_t m = absbits_max_of(mb);
        if (m >= 0x7c00u) {             // an infinity or a NaN among them
            m = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const half_t one = v[e][i >> 3][i & 7];         // (a bit cast of the vector's element itself takes the first one's)
                    const uint16_t w = __builtin_bit_cast(uint16_t, one), w0 = w & 0x7fff;
                    const uint16_t r = w0 > 0x7c00 ? (uint16_t)0 : w0 == 0x7c00 ? (uint16_t)(w - 1) : w;
                    v[e][i >> 3][i & 7] = __builtin_bit_cast(half_t, r);
                    m = max(m, (uint32_t)(r & 0x7fff));
                }
        }
        atomicMax(&tops[slot], m);
    }
    __syncthreads();
    for (int i = tid; i < blocks; i += blockDim.x)
        if (first + i * a.block < end) top[i] = __builtin_bit_cast(half_t, (uint16_t)tops[i]);
    if (!some) return;
    const float now = (float)__builtin_bit_cast(half_t, (uint16_t)tops[slot]);
    const float was = (float)__builtin_bit_cast(half_t, (uint16_t)tops[blocks]);
    const float y = now > 0.0f ? kv_factor(127.0f, now) : 0.0f;
    const float again = now > 0.0f ? kv_factor(was, now) : 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        uint4_t out;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            uint32_t q[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = d * 4 + k;
                q[k] = nearest_bits((float)v[e][i >> 3][i & 7], y);
                if (!whole) {
                    const int32_t t = first + (V ? minor + i : major[e]);
                    const int32_t byte = (int32_t)(old[e][d] << (24 - 8 * k)) >> 24;
                    if (t < pos) q[k] = nearest_bits((float)byte, again);
                    if (t >= end) q[k] = (uint32_t)byte;
                }
            }
            out[d] = pack4_i8(q[0], q[1], q[2], q[3]);
        }
        *reinterpret_cast<uint4_t*>(place(e)) = out;
    }
}

// One token a sequence, the decode step: a wave a head's key or value, whose units its lanes hold.  Its integers are all that is written unless the token is larger than what its block holds, in which case
// the block's older ones are read and rounded again, a wave's loads one behind another's store.  Bound by latency: 32 x 64 heads of 64 take 4.2 us where no block grows, 5.0 where one in fourteen does (as many
// as do on average while a block of 64 fills), and where all do 6.5 in the middle of a block of 64 and 10.3 at its end; 32 x 8 heads of 256 in blocks of 128 take 3.9, and up to 16.8 where all grow.  Of the general kernel, which passes over the
// whole block either way, 32 x 64 heads of 64 took 13.2 us.
template <bool V>
__device__ __forceinline__ void write_token(const KvArgs& a, const KvSide& s, int64_t b, int32_t h, int32_t pos) {
    const int lane = threadIdx.x & 63;
    const int64_t head = b * a.heads + h;
    const half_t* const x = s.x + b * s.batch + h * s.head;
    const int32_t first = pos & -a.block;
    half_t* const top = s.top + head * (a.length / a.block) + pos / a.block;
    const uint32_t old = first < pos ? min((uint32_t)(__builtin_bit_cast(uint16_t, *top) & 0x7fff), 0x7bffu) : 0u;
    half_t v[4];
    uint32_t m = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        v[c] = 0;
        if (c * 64 + lane < a.dim) v[c] = x[(int64_t)(c * 64 + lane) * s.unit];
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const uint16_t w = __builtin_bit_cast(uint16_t, v[c]), w0 = w & 0x7fff;
        const uint16_t r = w0 > 0x7c00 ? (uint16_t)0 : w0 == 0x7c00 ? (uint16_t)(w - 1) : w;
        v[c] = __builtin_bit_cast(half_t, r);
        m = max(m, (uint32_t)(r & 0x7fff));
    }
    m = max(wave_max_u32_uniform(m), old);
    const float now = (float)__builtin_bit_cast(half_t, (uint16_t)m);
    const float y = now > 0.0f ? kv_factor(127.0f, now) : 0.0f;
    int8_t* const ints = s.ints + head * a.length * a.dim;
    int8_t* const at = V ? ints + (int64_t)(pos >> 4) * 16 * a.dim + (pos & 15) : ints + (int64_t)pos * a.dim;
#pragma unroll
    for (int c = 0; c < 4; ++c)
        if (c * 64 + lane < a.dim) at[(c * 64 + lane) * (V ? 16 : 1)] = (int8_t)nearest_bits((float)v[c], y);
    if (m == old && first < pos) return;         // (at a block's start what the magnitude was does not count, not even where it is 0 now)
    if (lane == 0) *top = __builtin_bit_cast(half_t, (uint16_t)m);
    if (first == pos) return;
    const float again = kv_factor((float)__builtin_bit_cast(half_t, (uint16_t)old), now);
    // sixteen bytes at a time: whole keys; whole groups of values, of the last one the bytes before the token
    const int32_t part = V ? pos & 15 : 0, pieces = ((V ? (pos + 15) & -16 : pos) - first) * a.dim / 16, partial = V && part ? pieces - a.dim : pieces;
    uint4_t* const p = reinterpret_cast<uint4_t*>(ints + (int64_t)first * a.dim);
    for (int i = lane; i < pieces; i += 64) {
        const uint4_t w = p[i];
        uint4_t r;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            uint32_t q[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) q[k] = nearest_bits((float)((int32_t)(w[d] << (24 - 8 * k)) >> 24), again);
            r[d] = pack4_i8(q[0], q[1], q[2], q[3]);
        }
        if (i < partial) p[i] = r;
        else
            for (int k = 0; k < part; ++k) reinterpret_cast<int8_t*>(p + i)[k] = (int8_t)(r[k >> 2] >> (8 * (k & 3)));
    }
}

__global__ __launch_bounds__(256) void k_kv_write_token(KvArgs a, uint32_t waves) {
    const uint32_t w = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (w >= waves) return;
    const uint32_t head = w >> 1;
    const int64_t b = head / (uint32_t)a.heads;
    const int32_t h = head - (uint32_t)b * a.heads, pos = a.pos_each ? a.pos_each[b] : a.pos;
    if (pos < 0 || pos >= a.length || (a.count_each && a.count_each[b] <= 0)) return;
    if (w & 1) write_token<true>(a, a.side[1], b, h, pos);
    else write_token<false>(a, a.side[0], b, h, pos);
}

// grid: chunks x heads x batch x (keys, values)
__global__ __launch_bounds__(512) void k_kv_write(KvArgs a) {
    __shared__ uint32_t tops[65];
    uint32_t w = blockIdx.x;
    const bool values = w & 1;
    w >>= 1;
    const uint32_t chunk = w % a.chunks;
    w /= a.chunks;
    const int32_t h = w % (uint32_t)a.heads;
    const int64_t b = w / (uint32_t)a.heads;
    const int32_t pos = a.pos_each ? a.pos_each[b] : a.pos;
    const int32_t count = a.count_each ? min(a.count_each[b], a.tokens) : a.tokens;
    if (pos < 0 || pos >= a.length || count <= 0) return;
    const int32_t end = (int32_t)min((int64_t)pos + count, (int64_t)a.length);
    const int64_t first = (int64_t)(pos / a.block) * a.block + (int64_t)chunk * a.span;
    if (first >= end) return;
    if (values) write_piece<true>(a, a.side[1], tops, b, h, (int32_t)first, pos, end);
    else write_piece<false>(a, a.side[0], tops, b, h, (int32_t)first, pos, end);
}

template <bool V>
__device__ __forceinline__ void read_piece(const KvArgs& a, const KvSide& s, int64_t b, int32_t h, int64_t first, int32_t from) {
    if ((int)threadIdx.x >= a.pieces) return;
    const int64_t head = b * a.heads + h, end = (int64_t)from + a.tokens;
    int major[4], minor;
    piece_of<V>(threadIdx.x, a.dim, 16, s.mode != kStraight, major, minor);
    // (a piece's tokens lie in one group of sixteen, which lies in the cache or outside of it)
    const int64_t group = first + ((V ? minor : major[0]) & -16);
    const int64_t t_lo = first + (V ? minor : major[0]), t_hi = first + (V ? minor + 15 : major[3]);
    if (t_lo >= end || t_hi < from) return;
    const bool inside = group >= 0 && group < a.length;
    const int8_t* const ints = s.ints + (head * a.length + (inside ? group : 0)) * a.dim;
    const int skip = inside ? (int)(first - group) : 0;                    // tokens from the group to the workgroup's first one
    uint4_t p[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int o = V ? major[e] * 16 : (inside ? major[e] + skip : 0) * a.dim + minor;
        p[e] = __builtin_nontemporal_load(reinterpret_cast<const uint4_t*>(ints + o));
        if (!inside) p[e] = uint4_t{0, 0, 0, 0};
    }
    const half_t top = s.top[head * (a.length >> a.block_shift) + ((inside ? group : 0) >> a.block_shift)];
    const float f = inside ? (float)top / 127.0f : 0.0f;
    half8_t v[4][2];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        half8_t lo, hi;
        halves_of(p[e], lo, hi);
#pragma unroll
        for (int i = 0; i < 8; ++i) {       // (a product rounded once, to fp16)
            v[e][0][i] = (half_t)((float)lo[i] * f);
            v[e][1][i] = (half_t)((float)hi[i] * f);
        }
    }
    half_t* const x = const_cast<half_t*>(s.x) + b * s.batch + h * s.head + (first - from) * s.token;
    auto place = [&](int t, int u) { return x + t * s.token + u * s.unit; };
    const bool whole = t_lo >= from && t_hi < end;
    if (whole && s.mode == kStraight) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            half_t* o = V ? place(minor, major[e]) : place(major[e], minor);
            store_half8_any(o, v[e][0]);
            store_half8_any(o + 8, v[e][1]);
        }
    } else if (whole && s.mode == kCrossed) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            half4_t q;
#pragma unroll
            for (int e = 0; e < 4; ++e) q[e] = v[e][i >> 3][i & 7];
            *reinterpret_cast<Half4Any*>(V ? place(minor + i, major[0]) : place(major[0], minor + i)) = __builtin_bit_cast(Half4Any, q);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int64_t t = first + (V ? minor + i : major[e]);
                if (t >= from && t < end) *place(V ? minor + i : major[e], V ? major[e] : minor + i) = v[e][i >> 3][i & 7];
            }
    }
}

__global__ __launch_bounds__(256) void k_kv_read(KvArgs a) {
    uint32_t w = blockIdx.x;
    const bool values = w & 1;
    w >>= 1;
    const uint32_t chunk = w % a.chunks;
    w /= a.chunks;
    const int32_t h = w % (uint32_t)a.heads;
    const int64_t b = w / (uint32_t)a.heads;
    const int32_t from = a.pos_each ? a.pos_each[b] : a.pos;
    const int64_t first = (int64_t)(from >> 4) * 16 + (int64_t)chunk * a.span;
    if (values) read_piece<true>(a, a.side[1], b, h, first, from);
    else read_piece<false>(a, a.side[0], b, h, first, from);
}

// What the two have in common: 0, an error code, or -1 for nothing to do.
static int kv_check(int32_t batch, int32_t heads, int32_t tokens, int32_t dim, int32_t length, int32_t block) {
    if (batch < 0 || heads < 0 || tokens < 0 || dim < 0 || length < 0) return CPMK_EBADARG;
    if (block != 16 && block != 32 && block != 64 && block != 128) return CPMK_EBADARG;
    if (dim % 16 || length % block) return CPMK_EALIGN;
    if (dim > 256 || (int64_t)length * dim > 0x7fffffffll) return CPMK_ETOOBIG;
    if ((int64_t)batch * heads == 0 || tokens == 0 || dim == 0) return -1;
    if (!grid_fits((int64_t)batch * heads)) return CPMK_ETOOBIG;         // (two workgroups a head at least; what is multiplied by it below stays below 2^63)
    return length == 0 ? CPMK_EBADARG : 0;
}

static int kv_mode(bool values, int64_t token, int64_t unit) {
    if ((values ? token : unit) == 1) return kStraight;
    return (values ? unit : token) == 1 ? kCrossed : kAnyStride;
}

}  // namespace cpmk

using namespace cpmk;

extern "C" {

int cpmk_kv_write_int8(int32_t batch, int32_t heads, int32_t tokens, int32_t dim, int32_t length, int32_t block, const void* k, int64_t k_batch,
                       int64_t k_head, int64_t k_token, int64_t k_unit, const void* v, int64_t v_batch, int64_t v_head, int64_t v_token,
                       int64_t v_unit, const void* pos_each, int32_t pos, const void* count_each, void* keys, void* values, void* key_absmax,
                       void* value_absmax, void* stream) {
    clear_stale_error();
    if (int e = kv_check(batch, heads, tokens, dim, length, block)) return e < 0 ? 0 : e;
    if (any_null(k, v, keys, values, key_absmax, value_absmax)) return CPMK_EBADARG;
    if (!pos_each && (pos < 0 || (int64_t)pos + tokens > length)) return CPMK_EBADARG;
    if (!aligned16(keys) || !aligned16(values)) return CPMK_EALIGN;
    KvArgs a;
    a.side[0] = {(const half_t*)k, k_batch, k_head, k_token, k_unit, (int8_t*)keys, (half_t*)key_absmax, kv_mode(false, k_token, k_unit)};
    a.side[1] = {(const half_t*)v, v_batch, v_head, v_token, v_unit, (int8_t*)values, (half_t*)value_absmax, kv_mode(true, v_token, v_unit)};
    a.pos_each = (const int32_t*)pos_each;
    a.count_each = (const int32_t*)count_each;
    a.pos = pos, a.tokens = tokens, a.heads = heads, a.dim = dim, a.length = length, a.block = block, a.block_shift = __builtin_ctz((unsigned)block);
    if (tokens == 1) {
        const int64_t waves = (int64_t)batch * heads * 2;
        if (waves > 0x7fffffffll) return CPMK_ETOOBIG;
        hipLaunchKernelGGL(k_kv_write_token, dim3((unsigned)ceil_div(waves, 4)), dim3(256), 0, (hipStream_t)stream, a, (uint32_t)waves);
        return launch_status();
    }
    // blocks that a sequence's tokens can lie in, 64 elements a lane, about 256 lanes a workgroup
    const int64_t behind = pos_each ? block - 1 : pos % block;
    int64_t blocks = ceil_div(behind + tokens, block);
    if (blocks > length / block) blocks = length / block;
    int64_t some = 16384 / dim / block;
    some = some < 1 ? 1 : some > blocks ? blocks : some;
    a.span = (int32_t)some * block;
    a.pieces = a.span * dim / 64;
    const int64_t chunks = ceil_div(blocks, some), grid = chunks * heads * batch * 2;
    if (!grid_fits(grid)) return CPMK_ETOOBIG;
    a.chunks = (uint32_t)chunks;
    hipLaunchKernelGGL(k_kv_write, dim3((unsigned)grid), dim3((unsigned)ceil_div(a.pieces, 64) * 64), 0, (hipStream_t)stream, a);
    return launch_status();
}

int cpmk_kv_read_int8(int32_t batch, int32_t heads, int32_t tokens, int32_t dim, int32_t length, int32_t block, const void* keys, const void* values,
                      const void* key_absmax, const void* value_absmax, const void* from_each, int32_t from, void* k, void* v, int64_t out_batch,
                      int64_t out_head, int64_t out_token, int64_t out_unit, void* stream) {
    clear_stale_error();
    if (int e = kv_check(batch, heads, tokens, dim, length, block)) return e < 0 ? 0 : e;
    if (any_null(k, v, keys, values, key_absmax, value_absmax)) return CPMK_EBADARG;
    if (!aligned16(keys) || !aligned16(values)) return CPMK_EALIGN;
    KvArgs a;
    a.side[0] = {(const half_t*)k, out_batch, out_head, out_token, out_unit, (int8_t*)keys, (half_t*)key_absmax, kv_mode(false, out_token, out_unit)};
    a.side[1] = {(const half_t*)v, out_batch, out_head, out_token, out_unit, (int8_t*)values, (half_t*)value_absmax, kv_mode(true, out_token, out_unit)};
    a.pos_each = (const int32_t*)from_each;
    a.count_each = nullptr;
    a.pos = from, a.tokens = tokens, a.heads = heads, a.dim = dim, a.length = length, a.block = block, a.block_shift = __builtin_ctz((unsigned)block);
    const int64_t groups = ceil_div((from_each ? 15 : from & 15) + (int64_t)tokens, 16);
    int64_t some = 16384 / dim / 16;
    some = some > groups ? groups : some;
    a.span = (int32_t)some * 16;
    a.pieces = a.span * dim / 64;
    const int64_t chunks = ceil_div(groups, some), grid = chunks * heads * batch * 2;
    if (!grid_fits(grid)) return CPMK_ETOOBIG;
    a.chunks = (uint32_t)chunks;
    hipLaunchKernelGGL(k_kv_read, dim3((unsigned)grid), dim3((unsigned)ceil_div(a.pieces, 64) * 64), 0, (hipStream_t)stream, a);
    return launch_status();
}

}  // extern "C"
