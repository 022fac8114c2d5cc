// Rows of logits to the log probabilities of given tokens, the entropy and the top alternatives, in one pass over the
// logits: with m = max x, d = scale (x - m) (the difference first: the scale may not take the type's lowest value out
// of range), S = sum exp(d), T = sum d exp(d):
//   logprob[j] = d[token j] - log S,   entropy = log S - T / S,   the `top` largest x, equal ones by id.
//
// A row goes in batches of 2048 values, 32 to a lane of one wave, held in registers for all uses: the lane's
// maximum, which rescales its running S and T once per batch, the exponentials, and the choice of the top.
// The top are kept as a superset, a list in LDS of 64-bit places in the order (lp_place). The first batch's list
// takes what is above a lower bound of its top-th value: the top-th largest of the wave's 256 maxima of 8 values,
// by its leading 16 bits (16 rounds of ballots). Later batches add what is above the bound, usually a few values or
// none: one comparison per lane. A list that would run over is cut to its top and the bound raised to the last of
// them; a batch that by itself runs over the list (ties, values in step with the lanes) goes through an exact
// selection. The result depends on none of this: places are unique, and the final order is by place.
//
// Rows shared by several groups (`parts`) leave their sums and lists in the workspace for logprobs_join.
// Constants: 0 x 2 x stride 4 type 5 V 6 scale (fp32 bits) 7 top 8 tokens 10 tokens' stride 12 given 13 token type
// (0 int32, 1 int64) 14 logprob 16 logprob stride 18 entropy (0: none) 20 ids 22 top logprobs 24 top stride 26 n
// 27 parts 28 workspace.
#pragma once
#include "rows.h"

#define LP_WAVES 4u
#define LP_BATCH 2048u
#define LP_LIST 512u
#define LP_TOP 64u

// Sums relative to the maximum m; s is 0 where there is no term (-infinity has none).
struct LpSums {
    float m, s, t;
};

// scale (a - b), at least -1e30 so that an exp of 0 times it is 0.
__device__ __forceinline__ float lp_diff(float a, float b, float scale) { return fmaxf(scale * (a - b), -1e30f); }

__device__ __forceinline__ LpSums lp_join(const LpSums &p, const LpSums &q, float scale) {
    LpSums o;
    o.m = fmaxf(p.m, q.m);
    const float m = o.m == -INFINITY ? 0.f : o.m;
    const float dp = lp_diff(p.m, m, scale), dq = lp_diff(q.m, m, scale), ep = __expf(dp), eq = __expf(dq);
    o.s = p.s * ep + q.s * eq;
    o.t = ep * (p.t + p.s * dp) + eq * (q.t + q.s * dq);
    return o;
}
__device__ __forceinline__ LpSums lp_wave_join(LpSums p, float scale) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        p = lp_join(p, LpSums{__shfl_xor(p.m, o, 64), __shfl_xor(p.s, o, 64), __shfl_xor(p.t, o, 64)}, scale);
    return p;
}

// Order of a value: falling with it, NaNs above all, both zeros alike; never 0 nor ~0.
__device__ __forceinline__ uint32_t lp_order(float x) {
    const uint32_t u = gd_f32_bits(x + 0.0f);
    return x != x ? 0xfffffffeu : u & 0x80000000u ? ~u : u | 0x80000000u;
}
// A value of the order u, -infinity's or above it; of a NaN's +infinity, so that only NaNs are not at or below it.
__device__ __forceinline__ float lp_value(uint32_t u) {
    if (u > 0xff800000u) return INFINITY;
    if (u == 0x7fffffffu) u = 0x7ffffffeu;  // between the smallest negative value and the zeros
    return gd_bits_f32(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ uint64_t lp_place(float x, uint32_t i) { return (uint64_t)lp_order(x) << 32 | (uint32_t)~i; }

__device__ __forceinline__ void lp_wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
__device__ __forceinline__ uint32_t lp_before(uint64_t mask) {  // set bits of the lanes before this one
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
}

// A place below every value's, for a list that is not full; no two alike (n < 2^31).
__device__ __forceinline__ uint64_t lp_nothing(uint32_t n) { return n + 1u; }

// Cuts list[0 .. c) (c <= LP_LIST, unique places) to its `top` largest, in no order; returns their count and, where
// something was cut, the order of the last in `bound`. One wave.
__device__ __forceinline__ uint32_t lp_cut(uint64_t *list, uint32_t c, uint32_t top, uint32_t &bound) {
    if (c <= top) return c;
    const uint32_t lane = threadIdx.x & 63u, steps = (c + 63u) >> 6;
    uint32_t hi[LP_LIST / 64], lo[LP_LIST / 64];
    lp_wave_sync();
#pragma unroll
    for (uint32_t r = 0; r < LP_LIST / 64; ++r) {
        const uint64_t p = lane + 64u * r < c ? list[lane + 64u * r] : 0ull;
        hi[r] = (uint32_t)(p >> 32);
        lo[r] = (uint32_t)p;
    }
    lp_wave_sync();
    // The largest value reached by `top` orders, then, of those that equal it, the largest reached by the rest.
    uint32_t at = 0, count = c;
    for (uint32_t bit = 0x80000000u; bit && count != top; bit >>= 1) {
        uint32_t n = 0;
#pragma unroll
        for (uint32_t r = 0; r < LP_LIST / 64; ++r)
            if (r < steps) n += __popcll(__ballot(hi[r] >= (at | bit)));
        if (n >= top) {
            at |= bit;
            count = n;
        }
    }
    uint32_t low = 0;
    if (count != top) {
        uint32_t above = 0;
#pragma unroll
        for (uint32_t r = 0; r < LP_LIST / 64; ++r)
            if (r < steps) above += __popcll(__ballot(hi[r] > at));
        for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
            uint32_t n = above;
#pragma unroll
            for (uint32_t r = 0; r < LP_LIST / 64; ++r)
                if (r < steps) n += __popcll(__ballot(hi[r] == at && lo[r] >= (low | bit)));
            if (n >= top) low |= bit;
        }
    }
    uint32_t out = 0;
#pragma unroll
    for (uint32_t r = 0; r < LP_LIST / 64; ++r) {
        if (r >= steps) break;
        const bool keep = count == top ? hi[r] >= at : hi[r] > at || (hi[r] == at && lo[r] >= low);
        const uint64_t mask = __ballot(keep);
        if (keep) list[out + lp_before(mask)] = (uint64_t)hi[r] << 32 | lo[r];
        out += __popcll(mask);
    }
    lp_wave_sync();
    bound = at;
    return out;
}

// One wave's share of a row's top: its list, the count and the bound (values at or below it are out). -infinity is
// never in a list: where the lists of a row hold less than `top`, all that is left are -infinity, and lp_finish finds
// the first of them.
struct LpTop {
    uint64_t *list;
    uint32_t c, top;
    float bound;
};

// The 32 values of a lane, x[8 j + e] being value first + 512 j + 8 lane + e of the row (-infinity outside it).
// gd_rounded: the compiler makes ballots and orders again where they are used again, instead of keeping 32 of them.
__device__ __forceinline__ void lp_add(LpTop &l, const float (&x)[32], uint32_t first, float most, bool nan) {
    if (!__any(nan || !(most <= l.bound))) return;
    const uint32_t at0 = first + 8u * (threadIdx.x & 63u);
    auto count = [&](float bound) {
        const float b = gd_rounded(bound);
        uint32_t n = 0;
#pragma unroll
        for (uint32_t i = 0; i < 32; ++i) n += __popcll(__ballot(!(x[i] <= b)));
        return n;
    };
    float bound = l.bound;
    uint32_t n = count(bound);
    if (l.c + n > LP_LIST && l.c > l.top) {
        uint32_t last = 0;
        l.c = lp_cut(l.list, l.c, l.top, last);
        bound = l.bound = lp_value(last);
        n = count(bound);
    }
    if (l.c + n > LP_LIST) {
        // A lower bound of the batch's top-th value from the maxima of 8, by their leading 16 bits.
        uint32_t group[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            float m = x[8 * j];
#pragma unroll
            for (uint32_t e = 1; e < 8; ++e) m = fmaxf(m, x[8 * j + e]);
            group[j] = lp_order(m);
        }
        uint32_t at = 0;
#pragma unroll 1
        for (uint32_t bit = 0x80000000u; bit >= 0x10000u; bit >>= 1) {
            uint32_t reached = 0;
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) reached += __popcll(__ballot(group[j] >= (at | bit)));
            if (reached >= l.top) at |= bit;
        }
        if (at > lp_order(-INFINITY)) {
            const float low = lp_value(at - 1u);
            if (!(low <= bound)) bound = low;
        }
        n = count(bound);
    }
    if (l.c + n <= LP_LIST) {
        const float b = gd_rounded(bound);
#pragma unroll
        for (uint32_t i = 0; i < 32; ++i) {
            const bool take = !(x[i] <= b);
            const uint64_t mask = __ballot(take);
            if (!mask) continue;
            if (take) l.list[l.c + lp_before(mask)] = lp_place(x[i], at0 + 512u * (i >> 3) + (i & 7u));
            l.c += __popcll(mask);
        }
    } else {
        // The batch's own top, exactly (more than LP_LIST of its values are above the bound): the largest order that
        // `top` of its values reach, what is above it, and of those that equal it the first.
        auto order = [&](float v) {
            const float w = gd_rounded(v);
            return w <= bound ? 0u : lp_order(w);
        };
        uint32_t at = 0;
#pragma unroll 1
        for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
            uint32_t reached = 0;
#pragma unroll
            for (uint32_t i = 0; i < 32; ++i) reached += __popcll(__ballot(order(x[i]) >= (at | bit)));
            if (reached >= l.top) at |= bit;
        }
        uint32_t left = l.top;
#pragma unroll
        for (uint32_t i = 0; i < 32; ++i) {
            const bool take = order(x[i]) > at;
            const uint64_t mask = __ballot(take);
            if (!mask) continue;
            if (take) l.list[l.c + lp_before(mask)] = lp_place(x[i], at0 + 512u * (i >> 3) + (i & 7u));
            l.c += __popcll(mask);
            left -= __popcll(mask);  // fewer than `top` are above
        }
        // 512 values of a step in order: by lane, then within its 8.
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            if (!left) break;
            uint32_t mine = 0;
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) mine += order(x[8 * j + e]) == at ? 1u : 0u;
            const uint32_t upto = gd_wave_scan_u32(mine), all = __shfl(upto, 63, 64);
            uint32_t pos = upto - mine;
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e)
                if (order(x[8 * j + e]) == at) {
                    if (pos < left) l.list[l.c + pos] = lp_place(x[8 * j + e], at0 + 512u * j + e);
                    ++pos;
                }
            const uint32_t took = min(all, left);
            l.c += took;
            left -= took;
        }
        bound = lp_value(at);
    }
    lp_wave_sync();
    if (l.c >= l.top && !(bound <= l.bound)) l.bound = bound;
}

// What a row's given tokens need, loaded before the sums are there.
struct LpGiven {
    float x;
    int kind;  // 0 a token, 1 none, 2 outside
};
__device__ __forceinline__ LpGiven lp_given(const GdArgs &a, uint64_t row, uint64_t X) {
    LpGiven g = {0.f, 1};
    if (threadIdx.x >= a.c[12]) return g;
    const uint64_t at = row * gd_addr(a, 10) + threadIdx.x;
    const int64_t token = a.c[13] ? gd_at<const int64_t>(gd_addr(a, 8))[at] : (int64_t)gd_at<const int32_t>(gd_addr(a, 8))[at];
    g.kind = token < 0 ? 1 : token >= (int64_t)a.c[5] ? 2 : 0;
    if (g.kind == 0) g.x = row_load(X, (uint64_t)token, a.c[4]);
    return g;
}

// The row's outputs from its sums and the list of `c` <= 4 LP_TOP places in LDS; the first wave.
__device__ __forceinline__ void lp_finish(const GdArgs &a, uint64_t row, uint64_t X, const LpSums &p, const LpGiven &g,
                                          uint64_t *list, uint32_t c) {
    const float scale = gd_bits_f32(a.c[6]);
    const bool none = p.s == 0.f;
    const float logs = none ? 0.f : logf(p.s);
    auto logprob = [&](float x) { return none ? -INFINITY : scale * (x - p.m) - logs; };
    const uint32_t lane = threadIdx.x, top = a.c[7];
    if (lane == 0 && gd_addr(a, 18)) gd_at<float>(gd_addr(a, 18))[row] = none ? 0.f : logs - p.t / p.s;
    if (lane < a.c[12])
        gd_at<float>(gd_addr(a, 14))[row * gd_addr(a, 16) + lane] =
            g.kind == 0 ? logprob(g.x) : g.kind == 1 ? 0.f : __builtin_nanf("");
    if (!top) return;
    uint32_t bound;
    lp_cut(list, c, top, bound);
    const uint64_t mine = lane < top ? list[lane] : 0ull;
    const bool real = (mine >> 32) != 0;
    const auto ids = gd_at<uint32_t>(gd_addr(a, 20)) + row * gd_addr(a, 24);
    const auto tops = gd_at<float>(gd_addr(a, 22)) + row * gd_addr(a, 24);
    uint32_t rank = 0;
    for (uint32_t k = 0; k < top; ++k) rank += list[k] > mine ? 1u : 0u;
    if (real) {
        const uint32_t id = ~(uint32_t)mine;
        ids[rank] = id;
        tops[rank] = logprob(row_load(X, id, a.c[4]));
    }
    // What is missing are the first logits of -infinity.
    for (uint32_t found = __popcll(__ballot(real)), i = 0; found < top && i < a.c[5]; i += 64u) {
        const bool hit = i + lane < a.c[5] && row_load(X, i + lane, a.c[4]) == -INFINITY;
        const uint64_t mask = __ballot(hit);
        const uint32_t at = found + lp_before(mask);
        if (hit && at < top) {
            ids[at] = i + lane;
            tops[at] = logprob(-INFINITY);
        }
        found += __popcll(mask);
    }
}

// Workspace of a row's part: the sums (4 words), then `top` places, in 16-byte units.
__device__ __forceinline__ uint64_t lp_part(const GdArgs &a, uint64_t row, uint32_t part) {
    return gd_addr(a, 28) + (row * a.c[27] + part) * (16u + 8ull * ((a.c[7] + 1u) & ~1u));
}
