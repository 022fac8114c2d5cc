// Heads turned by their positions, and new tokens' keys and values on their way into a paged cache:
//   (y1, y2) = scale (x1 cos a - x2 sin a, x1 sin a + x2 cos a),  a = position * frequency of the pair
// Rows of up to three kinds in one launch: queries (turned, to rows), keys (turned, to the cache's slots) and values (as they
// are, to the slots). A group takes a token, or a part of one, forms its sines and cosines once, a pair a thread, and turns its
// heads by them; of many tokens a wave takes one, if its turns cover the heads. A thread takes units of 8 pairs (or 16 values
// that do not turn) of a head.
//
// Angles: a frequency is a fraction of a turn in 64 bits, whole turns dropped; its product with the position modulo 2^64 is the
// angle's fraction of a turn, exact but for the frequency's own last place. Its top two bits, rounded, are the quadrant; what is
// left, at most an eighth of a turn, goes to fp32 and through the series of sine and cosine up to x^9 and x^10 (a remainder
// below 2e-9). fp32 angles would be wrong in the first digit at a position of 10^6.
//
// Bound by memory where there are many tokens: 4096 of 32 + 2 x 8 heads of 128 bf16 values, 101 MB in and out, take 18.7 us
// (5.4 TB/s; a call in a loop 21.3, a copy of as many bytes 21.7), 1023 of 40 heads 7.3; of one token the launch, 3.8.
//
// Constants: 0 q 2 q stride 4 q_out 6 q_out stride 8 k 10 k stride 12 v 14 v stride 16 cache k 18 cache v 20 page stride 22
// head stride 24 token stride (bytes) 26 frequencies (0: nothing turns) 28 positions 30 slots 32 D 33 pairs 34 query heads 35
// kv heads (0: no cache) 36 tokens 37 types (q_out | cache << 4) 38 flags (1 interleaved, 2 positions in 64 bits, 4 slots in 64
// bits, 8 q in place) 39 scale 40 page size 41 pages * page size 42 groups that share a token 43 units per head 44 turns of two
// heads of a thread 45 a wave takes a token
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

// Values i .. i + 7 of a head. FULL: all of them are in it, and they stay as they are in memory until they are used, so that
// loads follow each other without a wait; low .. m - 1 are stored. Otherwise the first m <= 8 are there.
template <uint32_t TYPE, bool FULL>
struct RoEight {
    gd_u32x4 raw[TYPE == ROW_F32 ? 2 : 1];
    float v[8];
    __device__ __forceinline__ void load(uint64_t head, uint32_t i, uint32_t m) {
        if constexpr (FULL) {
#pragma unroll
            for (uint32_t j = 0; j < sizeof(raw) / 16u; ++j) raw[j] = gd_at<const gd_u32x4_any>(head + ((uint64_t)i << row_shift(TYPE)))[j];
        } else if (m == 8u) {
            row_load8<TYPE>(head, i, v);
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) v[j] = j < m ? row_load(head, i + j, TYPE) : 0.f;
        }
    }
    __device__ __forceinline__ void unpack() {
        if constexpr (FULL) {
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) {
                if constexpr (TYPE == ROW_F32) v[j] = gd_bits_f32(raw[j >> 2][j & 3u]);
                else v[j] = row_value16(raw[0][j >> 1] >> (16u * (j & 1u)) & 0xffffu, TYPE);
            }
        }
    }
    __device__ __forceinline__ void store(uint64_t head, uint32_t i, uint32_t m, uint32_t low, uint32_t type) const {
        if (!FULL || (!low && m == 8u)) return row_store8(head, i, i + m, type, v);
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j)
            if (j >= low && j < m) row_store(head, i + j, type, v[j]);
    }
};

// Eight values from i on that are copied, as far as the head goes.
template <bool FULL>
__device__ __forceinline__ void ro_end(uint32_t D, uint32_t &i, uint32_t &m, uint32_t &low) {
    if (FULL) {
        const uint32_t at = min(i, D - 8u);
        low = min(8u, i - at);
        i = at;
    } else {
        m = i < D ? min(8u, D - i) : 0u;
    }
}

// (fused in one way, wherever it stands)
__device__ __forceinline__ void ro_pair(float &x, float &y, float c, float s) {
    const float x1 = x;
    x = fmaf(-y, s, x1 * c);
    y = fmaf(y, c, x1 * s);
}

#define RO_TABLE 512u  // pairs of a head at most

template <uint32_t TYPE, bool FULL>
__device__ __forceinline__ void rotary_rows(const GdArgs &a, float *cosines, float *sines) {
    const uint32_t D = a.c[32], pairs = a.c[33], QH = a.c[34], KVH = a.c[35], n = a.c[36], types = a.c[37], flags = a.c[38];
    const uint32_t sharers = a.c[42], units = a.c[43], turns = a.c[44], heads = QH + 2u * KVH;
    const uint64_t id = (uint64_t)blockIdx.y * gridDim.x + blockIdx.x, of = id / sharers;
    const bool narrow = a.c[45];  // a token a wave
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), width = narrow ? 64u : 256u, tid = threadIdx.x & (width - 1u);
    if (of * (narrow ? 4u : 1u) >= n) return;
    const uint32_t wanted = (uint32_t)of * (narrow ? 4u : 1u) + (narrow ? wave : 0u), t = min(wanted, n - 1u), table = narrow ? wave * (RO_TABLE / 4u) : 0u;
    // A thread takes one unit of every at_once-th head, two heads a turn; a group that shares a token its turns' heads.
    const uint32_t at_once = width / units, own = tid / units, u = tid - own * units;
    const uint32_t head0 = (uint32_t)(id - of * sharers) * turns * 2u * at_once + own;
    const uint32_t turning = (pairs + 7u) / 8u;  // units of pairs; the others' values are copied
    // The halves of a unit in a head that turns and in one that does not: their places, and how many values of each there are.
    // FULL: a half that would reach past the pairs or the head's end moves down to it, and begins to store at its own first
    // value; pairs that two units turn need no such care but in place, as both have the same values. Fewer than eight pairs are
    // one unit's, which reads on behind them.
    uint32_t f1, f2, n1 = 8, n2 = 8, low1 = 0, low2 = 0, pair0 = 8u * u;
    if (u < turning) {
        const uint32_t m = min(8u, pairs - pair0);
        const bool apart = !(flags & 1u);
        if (FULL && pairs >= 8u) {
            pair0 -= 8u - m;
            if (flags & 8u) {
                low1 = apart ? 8u - m : min(8u, 16u - 2u * m);
                low2 = apart ? 8u - m : max(8u, 16u - 2u * m) - 8u;
            }
        } else {
            n1 = apart ? m : min(8u, 2u * m);
            n2 = apart ? m : 2u * m - n1;
        }
        f1 = apart ? pair0 : 2u * pair0;
        f2 = apart ? pairs + pair0 : 2u * pair0 + 8u;
    } else {
        f1 = 2u * pairs + 16u * (u - turning);
        f2 = f1 + 8u;
        ro_end<FULL>(D, f1, n1, low1);
        ro_end<FULL>(D, f2, n2, low2);
    }
    uint32_t v1 = 16u * u, v2 = v1 + 8u, mv1 = 8, mv2 = 8, vlow1 = 0, vlow2 = 0;
    ro_end<FULL>(D, v1, mv1, vlow1);
    ro_end<FULL>(D, v2, mv2, vlow2);
    const uint32_t to_q = types & 15u, to_cache = types >> 4;

    // Where the token's rows begin, and its place in the cache.
    const uint64_t from_q = gd_addr(a, 0) + ((t * gd_addr(a, 2)) << row_shift(TYPE)), from_k = gd_addr(a, 8) + ((t * gd_addr(a, 10)) << row_shift(TYPE)),
                   from_v = gd_addr(a, 12) + ((t * gd_addr(a, 14)) << row_shift(TYPE)), out_q = gd_addr(a, 4) + ((t * gd_addr(a, 6)) << row_shift(to_q));
    uint64_t cache_k = gd_addr(a, 16), cache_v = gd_addr(a, 18);
    bool kept = false;
    if (KVH) {
        const int64_t slot = ro_index(gd_addr(a, 30), t, flags & 4u);
        kept = (uint64_t)slot < a.c[41];
        const uint32_t where = kept ? (uint32_t)slot : 0u, page = where / a.c[40];
        const uint64_t at = page * gd_addr(a, 20) + (where - page * a.c[40]) * gd_addr(a, 24);
        cache_k += at;
        cache_v += at;
    }
#pragma unroll 1
    for (uint32_t turn = 0; turn < turns; ++turn) {
        // Two heads at a time: the second's loads are on their way with the first's, the first turn's while the angles are
        // formed.
        RoEight<TYPE, FULL> first[2], second[2];
        uint64_t y[2];
        bool stays[2], query[2], value[2];
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
            const uint32_t head = head0 + (2u * turn + i) * at_once;
            const bool there = own < at_once && head < heads && wanted < n;
            const uint32_t h = there ? head : 0u;
            query[i] = h < QH;
            value[i] = h >= QH + KVH;
            const uint32_t in_row = query[i] ? h : value[i] ? h - QH - KVH : h - QH;
            const uint64_t x = (query[i] ? from_q : value[i] ? from_v : from_k) + ((uint64_t)(in_row * D) << row_shift(TYPE));
            y[i] = query[i] ? out_q + ((uint64_t)(in_row * D) << row_shift(to_q)) : (value[i] ? cache_v : cache_k) + in_row * gd_addr(a, 22);
            stays[i] = there && (query[i] || kept);
            first[i].load(x, value[i] ? v1 : f1, value[i] ? mv1 : n1);
            second[i].load(x, value[i] ? v2 : f2, value[i] ? mv2 : n2);
        }
        if (!turn) {
            for (uint32_t i = tid; i < pairs; i += width)
                ro_turn((uint64_t)ro_index(gd_addr(a, 28), t, flags & 2u) * gd_at<const uint64_t>(gd_addr(a, 26))[i], gd_bits_f32(a.c[39]), cosines[table + i], sines[table + i]);
            __syncthreads();
        }
        float c[8], s[8];  // of the thread's pairs (of a head's last ones the table's end is read again)
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            const uint32_t at = min(table + pair0 + j, RO_TABLE - 1u);
            c[j] = cosines[at];
            s[j] = sines[at];
        }
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
            if (!stays[i]) continue;
            first[i].unpack();
            second[i].unpack();
            auto &p = first[i].v, &q = second[i].v;
            if (u < turning && !value[i]) {
                if (flags & 1u) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        ro_pair(p[2 * j], p[2 * j + 1], c[j], s[j]);
                        ro_pair(q[2 * j], q[2 * j + 1], c[4 + j], s[4 + j]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) ro_pair(p[j], q[j], c[j], s[j]);
                }
            }
            const uint32_t to = query[i] ? to_q : to_cache;
            first[i].store(y[i], value[i] ? v1 : f1, value[i] ? mv1 : n1, value[i] ? vlow1 : low1, to);
            second[i].store(y[i], value[i] ? v2 : f2, value[i] ? mv2 : n2, value[i] ? vlow2 : low2, to);
        }
    }
}

// (smaller heads have no eight values to move down to, or to read on behind their pairs)
template <uint32_t TYPE>
__device__ __forceinline__ void rotary_body(const GdArgs &a) {
    __shared__ __align__(16) float cosines[RO_TABLE], sines[RO_TABLE];
    const uint32_t D = a.c[32], pairs = a.c[33];
    if (D >= 8u && (!pairs || pairs >= 8u || D >= (a.c[38] & 1u ? 16u : pairs + 8u))) rotary_rows<TYPE, true>(a, cosines, sines);
    else rotary_rows<TYPE, false>(a, cosines, sines);
}
