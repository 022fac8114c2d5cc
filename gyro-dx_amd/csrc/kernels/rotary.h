// Heads turned by their positions, and new tokens' keys and values on their way into a paged cache:
//   (y1, y2) = scale (x1 cos a - x2 sin a, x1 sin a + x2 cos a),  a = position * frequency of the pair
// Rows of up to three kinds in one launch: queries (turned, to rows), keys (turned, to the cache's slots) and values
// (as they are, to the slots). A thread takes one unit of 8 pairs (or 16 values that do not turn) of a token and the
// same unit of several heads, so that the angles are formed once for them.
//
// Angles: a frequency is a fraction of a turn in 64 bits, whole turns dropped; its product with the position modulo 2^64 is the
// angle's fraction of a turn, exact but for the frequency's own last place. Its top two bits, rounded, are the quadrant; what is
// left, at most an eighth of a turn, goes to fp32 and through the series of sine and cosine up to x^9 and x^10 (a remainder
// below 2e-9). fp32 angles would be wrong in the first digit at a position of 10^6.
//
// Constants: 0 q 2 q stride 4 q_out 6 q_out stride 8 k 10 k stride 12 v 14 v stride 16 cache k 18 cache v 20 page stride
// 22 head stride 24 token stride (bytes) 26 frequencies (0: nothing turns) 28 positions 30 slots 32 D 33 pairs 34 query heads
// 35 kv heads (0: no cache) 36 tokens 37 types (q_out | cache << 4) 38 flags (1 interleaved, 2 positions in 64 bits, 4 slots
// in 64 bits) 39 scale 40 page size 41 pages * page size 42 heads per thread 43 threads' groups of heads per token 44 units per
// head
#pragma once
#include "rows.h"

// The position or slot t of an array of 32- or 64-bit integers.
__device__ __forceinline__ int64_t ro_index(uint64_t base, uint64_t t, bool wide) {
    return wide ? gd_at<const int64_t>(base)[t] : (int64_t)gd_at<const int32_t>(base)[t];
}

// scale times cosine and sine of a fraction of a turn (2^64: a whole one).
__device__ __forceinline__ void ro_turn(uint64_t fraction, float scale, float &c, float &s) {
    const uint64_t q = (fraction + (1ull << 61)) >> 62;
    const float x = (float)(int32_t)((fraction - (q << 62)) >> 32) * 1.46291807926715968e-9f;  // 2 pi 2^-32; at most pi / 4
    const float z = x * x;
    const float sine = x + x * z * (-1.f / 6 + z * (1.f / 120 + z * (-1.f / 5040 + z * (1.f / 362880))));
    const float cosine = 1.f + z * (-0.5f + z * (1.f / 24 + z * (-1.f / 720 + z * (1.f / 40320 - z * (1.f / 3628800)))));
    const bool odd = q & 1u;
    const float a = odd ? sine : cosine, b = odd ? cosine : sine;
    c = scale * ((q + 1u) & 2u ? -a : a);
    s = scale * (q & 2u ? -b : b);
}

// Values i .. i + m - 1 of a head, m <= 8, the others zeros.
template <uint32_t TYPE>
__device__ __forceinline__ void ro_load(uint64_t head, uint32_t i, uint32_t m, float (&v)[8]) {
    if (m == 8u) return row_load8<TYPE>(head, i, v);
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) v[j] = j < m ? row_load(head, i + j, TYPE) : 0.f;
}
__device__ __forceinline__ void ro_store(uint64_t head, uint32_t i, uint32_t m, uint32_t type, const float (&v)[8]) {
    row_store8(head, i, i + m, type, v);
}

template <uint32_t TYPE>
__device__ __forceinline__ void rotary_body(const GdArgs &a) {
    const uint32_t D = a.c[32], pairs = a.c[33], QH = a.c[34], KVH = a.c[35], n = a.c[36], types = a.c[37], flags = a.c[38];
    const uint32_t per = a.c[42], groups = a.c[43], units = a.c[44], heads = QH + 2u * KVH;
    const uint64_t FREQ = gd_addr(a, 26);
    const uint32_t own = threadIdx.x / units, u = threadIdx.x - own * units, at_once = 256u / units;
    if (own >= at_once) return;
    const uint64_t item = ((uint64_t)blockIdx.y * gridDim.x + blockIdx.x) * at_once + own;
    if (item >= (uint64_t)n * groups) return;
    const uint32_t t = (uint32_t)item / groups, head0 = ((uint32_t)item - t * groups) * per;
    const uint32_t turning = (pairs + 7u) / 8u;  // units of pairs; the others' values are copied
    // Where the two halves of a unit lie in a head, and how many values of each there are.
    uint32_t at1, at2, m1, m2;
    if (u < turning) {
        const uint32_t m = min(8u, pairs - 8u * u);
        if (flags & 1u) {
            at1 = 16u * u;
            at2 = at1 + 8u;
            m1 = min(8u, 2u * m);
            m2 = 2u * m - m1;
        } else {
            at1 = 8u * u;
            at2 = pairs + at1;
            m1 = m2 = m;
        }
    } else {
        at1 = 2u * pairs + 16u * (u - turning);
        at2 = at1 + 8u;
        m1 = at1 < D ? min(8u, D - at1) : 0u;
        m2 = at2 < D ? min(8u, D - at2) : 0u;
    }
    // Units of the values' heads, which have nothing that turns.
    const uint32_t v1 = 16u * u, v2 = v1 + 8u, mv1 = v1 < D ? min(8u, D - v1) : 0u, mv2 = v2 < D ? min(8u, D - v2) : 0u;

    float c[8], s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        c[j] = 1.f;
        s[j] = 0.f;
    }
    if (u < turning && head0 < QH + KVH) {
        const int64_t position = ro_index(gd_addr(a, 28), t, flags & 2u);
        const float scale = gd_bits_f32(a.c[39]);
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j)  // the table's last pair is read again behind the end
            ro_turn((uint64_t)position * gd_at<const uint64_t>(FREQ)[min(8u * u + j, pairs - 1u)], scale, c[j], s[j]);
    }
    uint64_t slot_offset = 0;
    bool kept = false;
    if (head0 + per > QH && KVH) {
        const int64_t slot = ro_index(gd_addr(a, 30), t, flags & 4u);
        kept = (uint64_t)slot < a.c[41];
        const uint32_t where = kept ? (uint32_t)slot : 0u, page = where / a.c[40];
        slot_offset = page * gd_addr(a, 20) + (where - page * a.c[40]) * gd_addr(a, 24);
    }
#pragma unroll 1
    for (uint32_t h = head0; h < min(head0 + per, heads); ++h) {
        const bool value = h >= QH + KVH, query = h < QH;
        if (!query && !kept) continue;
        const uint32_t in_row = query ? h : value ? h - QH - KVH : h - QH;
        const uint64_t from = query ? gd_addr(a, 0) : value ? gd_addr(a, 12) : gd_addr(a, 8);
        const uint64_t stride = query ? gd_addr(a, 2) : value ? gd_addr(a, 14) : gd_addr(a, 10);
        const uint64_t x = from + ((t * stride + (uint64_t)in_row * D) << row_shift(TYPE));
        const uint32_t to = query ? types & 15u : types >> 4;
        const uint64_t y = query ? gd_addr(a, 4) + ((t * gd_addr(a, 6) + (uint64_t)in_row * D) << row_shift(to))
                                 : (value ? gd_addr(a, 18) : gd_addr(a, 16)) + slot_offset + in_row * gd_addr(a, 22);
        const uint32_t f1 = value ? v1 : at1, f2 = value ? v2 : at2, n1 = value ? mv1 : m1, n2 = value ? mv2 : m2;
        float p[8], q[8];
        ro_load<TYPE>(x, f1, n1, p);
        ro_load<TYPE>(x, f2, n2, q);
        if (!value && u < turning) {
            if (flags & 1u) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float p1 = p[2 * j], q1 = q[2 * j];
                    p[2 * j] = p1 * c[j] - p[2 * j + 1] * s[j];
                    p[2 * j + 1] = p1 * s[j] + p[2 * j + 1] * c[j];
                    q[2 * j] = q1 * c[4 + j] - q[2 * j + 1] * s[4 + j];
                    q[2 * j + 1] = q1 * s[4 + j] + q[2 * j + 1] * c[4 + j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float p1 = p[j];
                    p[j] = p1 * c[j] - q[j] * s[j];
                    q[j] = p1 * s[j] + q[j] * c[j];
                }
            }
        }
        ro_store(y, f1, n1, to, p);
        ro_store(y, f2, n2, to, q);
    }
}
