// Rotary positions: pair i of `part` units of a head turned by the angle of its token's position,
//
//     (x, y) -> magnitude (x cos a - y sin a, x sin a + y cos a),   a = position * turns[i] of a whole turn,
//
// units 2 i and 2 i + 1 (interleaved) or i and i + part / 2; the head's other units are copied.  The gradient is turned by -a.
//
// Angles are formed here, in fp64 up to the fraction of a turn that is left (a position of 2^31 keeps 2^-22 of a turn; in fp32 one of 10^6 would keep 2^-4) and in fp32 from there; a
// thread uses its eight for several heads.  No table of them is read, and there is no longest position.
//
// Bound by memory, each element read and written once: 8 x 512 tokens of 64 heads of 64, twice, columns, interleaved: 26 us, 5.2 TB/s; 2 x 8191 tokens of 40 heads of 128, rows, half of the
// units turned: 72 us, 4.7 TB/s.
#include <algorithm>
#include "attention.h"

namespace cpmk {

struct Rotary {
    AttnTensor x[2], y[2];          // queries, keys
    int32_t heads[2];
    const double* turns;
    const int32_t* positions;       // at b * pos_batch + t * pos_token, or null: pos + t (a pos_token of 0: + t as well)
    int64_t pos_batch, pos_token;
    int32_t pos, tokens, dim, part;
    int32_t slots, groups;          // shares of a token's head, of the heads
    float magnitude, sign;
    int interleaved, copies;        // copies: whether units that are not turned have to be copied
};

__device__ __forceinline__ void rotary_angle(const Rotary& a, int64_t b, int32_t t, int32_t pair, float& c, float& s) {
    const double position = a.positions == nullptr ? (double)a.pos + t : (double)a.positions[b * a.pos_batch + t * a.pos_token] + (a.pos_token == 0 ? t : 0);
    const double turn = position * a.turns[pair];
    sincospif(2.0f * (float)(turn - __builtin_rint(turn)), &s, &c);
    c *= a.magnitude;
    s *= a.magnitude * a.sign;
}
__device__ __forceinline__ void rotary_turn(half_t& x, half_t& y, float c, float s) {
    const float p = x, q = y;
    x = round_f16(__builtin_fmaf(p, c, -(q * s)));         // (by name: the same bits in every layout)
    y = round_f16(__builtin_fmaf(p, s, q * c));
}

// A thread has one slot of a token (kRows: eight pairs, or sixteen units to copy; kAnyLayout: one pair or two units) or of eight tokens (kColumns: one pair or two units), and every
// a.groups-th head from its own on.
template <int LAY>
__global__ __launch_bounds__(256) void k_rotary(Rotary a, int64_t b0) {
    constexpr int N = LAY == kAnyLayout ? 1 : 8, PAIRS = LAY == kRows ? 8 : 1, TOKENS = LAY == kColumns ? 8 : 1;
    const uint32_t id = blockIdx.x * 256u + threadIdx.x;
    const int64_t b = b0 + blockIdx.y;
    int32_t slot, group, t;
    if (LAY == kColumns) {
        const uint32_t runs = ((uint32_t)a.tokens + 7) / 8, rest = id / runs;
        t = (id - rest * runs) * 8;
        group = rest / (uint32_t)a.slots;
        slot = rest - (uint32_t)group * a.slots;
        if (group >= a.groups) return;
    } else {
        const uint32_t rest = id / (uint32_t)a.slots;
        slot = id - rest * a.slots;
        t = rest / (uint32_t)a.groups;
        group = rest - (uint32_t)t * a.groups;
        if (t >= a.tokens) return;
    }
    const int turned = a.part / (2 * PAIRS);        // slots that are
    const bool copy = slot >= turned;
    const int count = LAY == kColumns ? min(8, a.tokens - t) : LAY == kRows && copy ? min(16, a.dim - a.part - (slot - turned) * 16) : 8;
    // the two runs of units: their first ones, and the distance inside of a run
    int u0, u1;
    if (copy) u0 = a.part + (slot - turned) * 2 * PAIRS, u1 = u0 + PAIRS;
    else if (a.interleaved) u0 = slot * 2 * PAIRS, u1 = u0 + PAIRS;
    else u0 = slot * PAIRS, u1 = u0 + a.part / 2;
    float c[N], s[N];
    if (!copy)
#pragma unroll
        for (int i = 0; i < N; ++i) rotary_angle(a, b, LAY == kColumns ? min(t + i, a.tokens - 1) : t, LAY == kRows ? slot * 8 + i : slot, c[i], s[i]);
    const int32_t all = a.heads[0] + a.heads[1];
    for (int32_t head = group; head < all; head += a.groups) {
        const int which = head >= a.heads[0];
        const AttnTensor &x = a.x[which], &y = a.y[which];
        const int64_t h = which ? head - a.heads[0] : head;
        const half_t* const px = x.at(b, h) + t * x.token;
        half_t* const py = y.at(b, h) + t * y.token;
        if (LAY == kAnyLayout) {
            half_t p = px[u0 * x.unit], q = u1 < a.dim ? px[u1 * x.unit] : (half_t)0;
            if (!copy) rotary_turn(p, q, c[0], s[0]);
            py[u0 * y.unit] = p;
            if (u1 < a.dim) py[u1 * y.unit] = q;
        } else if (LAY == kRows) {
            if (copy && count < 16) {
                for (int i = 0; i < count; ++i) py[u0 + i] = px[u0 + i];
                continue;
            }
            half8_t p = load_half8_any(px + u0), q = load_half8_any(px + u1);
            if (!copy) {
                if (a.interleaved) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        half_t v[4] = {p[2 * i], p[2 * i + 1], q[2 * i], q[2 * i + 1]};
                        rotary_turn(v[0], v[1], c[i], s[i]);
                        rotary_turn(v[2], v[3], c[4 + i], s[4 + i]);
                        p[2 * i] = v[0], p[2 * i + 1] = v[1], q[2 * i] = v[2], q[2 * i + 1] = v[3];
                    }
                } else
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        half_t v0 = p[i], v1 = q[i];
                        rotary_turn(v0, v1, c[i], s[i]);
                        p[i] = v0, q[i] = v1;
                    }
            }
            store_half8_any(py + u0, p);
            store_half8_any(py + u1, q);
        } else {
            const bool both = u1 < a.dim;
            const int64_t x0 = u0 * x.unit, x1 = (both ? u1 : u0) * x.unit, y0 = u0 * y.unit, y1 = u1 * y.unit;
            half8_t p = {0, 0, 0, 0, 0, 0, 0, 0}, q = p;
            if (count == 8) p = load_half8_any(px + x0), q = load_half8_any(px + x1);
            else
                for (int i = 0; i < 7; ++i)
                    if (i < count) p[i] = px[x0 + i], q[i] = px[x1 + i];
            if (!copy)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    half_t v0 = p[i], v1 = q[i];
                    rotary_turn(v0, v1, c[i], s[i]);
                    p[i] = v0, q[i] = v1;
                }
            if (count == 8) {
                store_half8_any(py + y0, p);
                if (both) store_half8_any(py + y1, q);
            } else
                for (int i = 0; i < 7; ++i)
                    if (i < count) {
                        py[y0 + i] = p[i];
                        if (both) py[y1 + i] = q[i];
                    }
        }
    }
}

}  // namespace cpmk

using namespace cpmk;

extern "C" {

int cpmk_rotary(int32_t batch, int32_t tokens, int32_t dim, int32_t part, int interleaved, int32_t heads_q, const void* q, int64_t q_batch, int64_t q_head, int64_t q_token, int64_t q_unit,
                void* q_out, int64_t qo_batch, int64_t qo_head, int64_t qo_token, int64_t qo_unit, int32_t heads_k, const void* k, int64_t k_batch, int64_t k_head, int64_t k_token,
                int64_t k_unit, void* k_out, int64_t ko_batch, int64_t ko_head, int64_t ko_token, int64_t ko_unit, const void* turns, const void* positions, int64_t pos_batch,
                int64_t pos_token, int32_t pos, float magnitude, int inverse, void* stream) {
    clear_stale_error();
    if (batch < 0 || tokens < 0 || dim < 0 || heads_q < 0 || heads_k < 0 || part < 0 || part > dim) return CPMK_EBADARG;
    if (part % 2) return CPMK_EALIGN;
    const int64_t all = (int64_t)heads_q + heads_k;
    if (batch == 0 || tokens == 0 || dim == 0 || all == 0) return 0;
    if ((heads_q > 0 && any_null(q, q_out)) || (heads_k > 0 && any_null(k, k_out)) || (part > 0 && !turns)) return CPMK_EBADARG;
    if (all > 0x7fffffffll) return CPMK_ETOOBIG;
    Rotary a;
    a.x[0] = {(half_t*)q, q_batch, q_head, q_token, q_unit}, a.y[0] = {(half_t*)q_out, qo_batch, qo_head, qo_token, qo_unit};
    a.x[1] = {(half_t*)k, k_batch, k_head, k_token, k_unit}, a.y[1] = {(half_t*)k_out, ko_batch, ko_head, ko_token, ko_unit};
    a.heads[0] = heads_q, a.heads[1] = heads_k;
    a.turns = (const double*)turns, a.positions = (const int32_t*)positions, a.pos_batch = pos_batch, a.pos_token = pos_token, a.pos = pos;
    a.tokens = tokens, a.dim = dim, a.part = part, a.magnitude = magnitude, a.sign = inverse ? -1.0f : 1.0f, a.interleaved = interleaved != 0;
    bool rows = part % 16 == 0, columns = true, in_place = true;
    for (int i = 0; i < 2; ++i) {
        if (a.heads[i] == 0) continue;
        rows = rows && a.x[i].unit == 1 && a.y[i].unit == 1;
        columns = columns && a.x[i].token == 1 && a.y[i].token == 1;
        in_place = in_place && a.x[i].p == a.y[i].p && a.x[i].batch == a.y[i].batch && a.x[i].head == a.y[i].head && a.x[i].token == a.y[i].token && a.x[i].unit == a.y[i].unit;
    }
    const int pairs = rows ? 8 : 1;
    // one layout or the other where both fit (one token, one unit): units
    const int lay = rows ? kRows : columns ? kColumns : kAnyLayout;
    if (in_place && part == 0) return 0;
    a.slots = part / (2 * pairs) + (in_place ? 0 : (int32_t)ceil_div(dim - part, 2 * pairs));
    // as many heads a thread as leave every compute unit 2048 threads, up to eight
    const int64_t shares = (lay == kColumns ? ceil_div(tokens, 8) : (int64_t)tokens) * a.slots, threads = shares * batch;
    const int64_t each = std::max<int64_t>(1, std::min<int64_t>(8, threads * all / (2048ll * compute_units())));
    a.groups = (int32_t)ceil_div(all, each);
    if (shares > 0x7fffffffll / a.groups) return CPMK_ETOOBIG;
    const unsigned grid = (unsigned)ceil_div(shares * a.groups, 256);
    for (int64_t b0 = 0; b0 < batch; b0 += 65535) {
        const dim3 blocks(grid, (unsigned)std::min<int64_t>(65535, batch - b0));
        if (lay == kRows) hipLaunchKernelGGL(k_rotary<kRows>, blocks, dim3(256), 0, (hipStream_t)stream, a, b0);
        else if (lay == kColumns) hipLaunchKernelGGL(k_rotary<kColumns>, blocks, dim3(256), 0, (hipStream_t)stream, a, b0);
        else hipLaunchKernelGGL(k_rotary<kAnyLayout>, blocks, dim3(256), 0, (hipStream_t)stream, a, b0);
    }
    return launch_status();
}

}  // extern "C"
