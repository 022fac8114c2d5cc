// Rows of logits to the log probabilities of given tokens, the entropy and the top alternatives, in one pass over the
// logits: with m = max x, d = scale (x - m) (the difference first: the scale may not take the type's lowest value out
// of range), S = sum exp(d), T = sum d exp(d):
//   logprob[j] = d[token j] - log S,   entropy = log S - T / S,   the `top` largest x, equal ones by id.
//
// A row goes in batches of 1024 values, 16 to a lane of one wave, held in registers for all uses: the lane's
// maximum, which rescales its running S and T once per batch, the exponentials, and the choice of the top.
// The top are kept as a superset, a list in LDS of 64-bit places in the order (lp_place). The first batch's list
// takes what is above a lower bound of its top-th value: the top-th largest of the wave's 128 maxima of 8 values,
// by its leading bits. Later batches add what is above the bound, usually a few values or
// none: one comparison per lane. A list that grows is cut to its top and the bound raised to the last of them; a batch
// that by itself runs over the list (ties, values in step with the lanes) goes through an exact
// selection. The result depends on none of this: places are unique, and the final order is by place.
//
// What bounds it: of many rows the reads (1023 fp32 rows of 131072: 96 us in a loop, 5.6 TB/s, 99 with the top 20; median 102 of
// kernel); of few rows the launches and one batch's chain of dependent steps, the bit searches for the top among them (one such
// row: 5.5 us without a top, 14.6 with the top 20, of which the join's kernel, 7.8 by itself, is half; 64 bf16 rows of
// 100003 with the top 5 20). Batches of 2048 took 101 to 121 us for the first and 6.1 to 14.2 for the second: half
// the waves per SIMD, and 1023 rows in one round and a third instead of one.
//
// Rows shared by several groups (`parts`) leave their sums and lists in the workspace for logprobs_join.
// Constants: 0 x 2 x stride 4 type 5 V 6 scale (fp32 bits) 7 top 8 tokens 10 tokens' stride 12 given 13 token type
// (0 int32, 1 int64) 14 logprob 16 logprob stride 18 entropy (0: none) 20 ids 22 top logprobs 24 top stride 26 n
// 27 parts 28 workspace.
#pragma once
#include "rows.h"

#define LP_WAVES 4u
#define LP_VALUES 16u                 // a lane's of a batch
#define LP_EIGHTS (LP_VALUES / 8u)
#define LP_BATCH (64u * LP_VALUES)
#define LP_LIST 512u
#define LP_TOP 64u

// Sums relative to the maximum m; s is 0 where there is no term (-infinity has none).
struct LpSums {
    float m, s, t;
};

// A distance whose exp is 0, and that times a sum of up to 2^31 terms is within fp32's range, so that 0 times either is 0.
#define LP_FAR -1e28f

// scale (a - b), LP_FAR at least.
__device__ __forceinline__ float lp_diff(float a, float b, float scale) { return fmaxf(scale * (a - b), LP_FAR); }

// Moves p's sums to the maximum m >= p.m (-infinity: there is no term yet, and any reference will do).
__device__ __forceinline__ void lp_move(LpSums &p, float m, float scale) {
    const float d = lp_diff(p.m, m == -INFINITY ? 0.f : m, scale), e = __expf(d);
    p.t = e * (p.t + p.s * d);
    p.s *= e;
    p.m = m;
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float lp_dpp_max_step(float v) {
    return fmaxf(v, gd_bits_f32((uint32_t)__builtin_amdgcn_update_dpp((int)0xff800000, (int)gd_f32_bits(v), CTRL, ROWS, 0xf, false)));
}
// Sums of the wave's lanes, in every lane: one maximum by DPP, then two sums (gd_wave_sum_dpp's steps).
__device__ __forceinline__ LpSums lp_wave_join(LpSums p, float scale) {
    float m = p.m;
    m = lp_dpp_max_step<0x111, 0xf>(m);
    m = lp_dpp_max_step<0x112, 0xf>(m);
    m = lp_dpp_max_step<0x114, 0xf>(m);
    m = lp_dpp_max_step<0x118, 0xf>(m);
    m = lp_dpp_max_step<0x142, 0xa>(m);
    m = lp_dpp_max_step<0x143, 0xc>(m);
    lp_move(p, gd_bits_f32((uint32_t)__builtin_amdgcn_readlane((int)gd_f32_bits(m), 63)), scale);
    return {p.m, gd_wave_sum_dpp(p.s), gd_wave_sum_dpp(p.t)};
}

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t lp_dpp_max_step_u32(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false));
}
// The wave's largest, a scalar.
__device__ __forceinline__ uint32_t lp_wave_max_u32(uint32_t v) {
    v = lp_dpp_max_step_u32<0x111, 0xf>(v);
    v = lp_dpp_max_step_u32<0x112, 0xf>(v);
    v = lp_dpp_max_step_u32<0x114, 0xf>(v);
    v = lp_dpp_max_step_u32<0x118, 0xf>(v);
    v = lp_dpp_max_step_u32<0x142, 0xa>(v);
    v = lp_dpp_max_step_u32<0x143, 0xc>(v);
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// The largest order u with reached(u) >= top, by its bits from the highest down to `lowest`, until reached(u) <= enough;
// `count` becomes reached(u) (from `all`, of 0), and `above` what reaches more where the search went to the last bit.
// The top of a row mostly lie within a factor of two, so the search starts below the exponent of the largest, `most`,
// where `top` reach that.
template <typename F>
__device__ __forceinline__ uint32_t lp_search(F &&reached, uint32_t most, uint32_t top, uint32_t enough, uint32_t lowest,
                                              uint32_t all, uint32_t &count, uint32_t &above) {
    uint32_t at = most & 0xff800000u, bit = 0x00400000u;
    count = reached(at);
    above = 0;
    if (count < top) {
        above = count;
        at = 0;
        bit = 0x80000000u;
        count = all;
    }
#pragma unroll 1
    for (; bit >= lowest && count > enough; bit >>= 1) {
        const uint32_t n = reached(at | bit);
        if (n >= top) {
            at |= bit;
            count = n;
        } else {
            above = n;
        }
    }
    return at;
}

// Order of a value: falling with it, NaNs above all, both zeros alike; never 0 nor ~0.
__device__ __forceinline__ uint32_t lp_order(float x) {
    const uint32_t u = gd_f32_bits(x + 0.0f);
    return x != x ? 0xfffffffeu : u & 0x80000000u ? ~u : u | 0x80000000u;
}
// A value of the order u, -infinity's or above it.
__device__ __forceinline__ float lp_value(uint32_t u) { return gd_bits_f32(u & 0x80000000u ? u & 0x7fffffffu : ~u); }
// A bound that exactly the values of orders above u pass (of orders up to infinity's): no value lies between the
// smallest negative one and the zeros, and only NaNs are not at or below +infinity.
__device__ __forceinline__ float lp_bound(uint32_t u) {
    return u > 0xff800000u ? INFINITY : lp_value(u == 0x7fffffffu ? 0x7ffffffeu : u);
}
__device__ __forceinline__ uint64_t lp_place(float x, uint32_t i) { return (uint64_t)lp_order(x) << 32 | (uint32_t)~i; }
// A place below every value's, for a list that is not full; no two alike (n < 2^31).
__device__ __forceinline__ uint64_t lp_nothing(uint32_t n) { return n + 1u; }

__device__ __forceinline__ void lp_wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
__device__ __forceinline__ uint32_t lp_before(uint64_t mask) {  // set bits of the lanes before this one
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
}

// Moves the `top` largest of list[0 .. c) (top <= c <= LP_LIST, unique places) to out[0 .. top), in no order; out may
// be list. Returns the order of the last of them. One wave. Code is kept small: at one batch per wave, what an
// instruction costs is fetching it.
__device__ __forceinline__ uint32_t lp_cut(const uint64_t *list, uint32_t c, uint32_t top, uint64_t *out) {
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t hi[LP_LIST / 64], lo[LP_LIST / 64];
    lp_wave_sync();
#pragma unroll
    for (uint32_t r = 0; r < LP_LIST / 64; ++r) {
        hi[r] = lo[r] = 0u;
        if (64u * r < c) {
            const uint64_t p = list[min(lane + 64u * r, c - 1u)];
            if (lane + 64u * r < c) {
                hi[r] = (uint32_t)(p >> 32);
                lo[r] = (uint32_t)p;
            }
        }
    }
    lp_wave_sync();
    // The largest order that `top` reach, then, of those that equal it, the largest low word that the rest reach.
    uint32_t low = 0, count, above, most = 0;
#pragma unroll
    for (uint32_t r = 0; r < LP_LIST / 64; ++r) most = max(most, hi[r]);
    const uint32_t at = lp_search(
        [&](uint32_t probe) {
            uint32_t n = 0;
#pragma unroll
            for (uint32_t r = 0; r < LP_LIST / 64; ++r) {
                if (64u * r >= c) break;
                n += __popcll(__ballot(hi[r] >= probe));
            }
            return n;
        },
        lp_wave_max_u32(most), top, top, 1u, c, count, above);
    for (uint32_t bit = 0x80000000u; bit && count != top; bit >>= 1) {
        const uint32_t probe = low | bit;
        uint32_t n = above;
#pragma unroll
        for (uint32_t r = 0; r < LP_LIST / 64; ++r) {
            if (64u * r >= c) break;
            n += __popcll(__ballot(hi[r] == at && lo[r] >= probe));
        }
        if (n >= top) {
            low = probe;
            count = n;
        }
    }
    uint32_t o = 0;
#pragma unroll
    for (uint32_t r = 0; r < LP_LIST / 64; ++r) {
        if (64u * r >= c) break;
        const bool keep = hi[r] > at || (hi[r] == at && lo[r] >= low);
        const uint64_t mask = __ballot(keep);
        if (keep) out[o + lp_before(mask)] = (uint64_t)hi[r] << 32 | lo[r];
        o += __popcll(mask);
    }
    lp_wave_sync();
    return at;
}

// One wave's share of a row's top: its list, the count and the bound (values at or below it are out). -infinity is
// never in a list: where the lists of a row hold less than `top`, all that is left are -infinity, and lp_finish finds
// the first of them.
struct LpTop {
    uint64_t *list;
    uint32_t c, top;
    float bound;
};

// Adds to the list what may be among the top of the LP_VALUES values of a lane, x[8 j + e] being value at(j) + e of the row
// (-infinity outside it). gd_rounded: the compiler makes ballots and orders again where they are used again, instead
// of keeping all of them.
template <typename F>
__device__ __forceinline__ void lp_add(LpTop &l, const float (&x)[LP_VALUES], F &&at, bool nan) {
    float group[LP_EIGHTS];  // maxima of 8
#pragma unroll
    for (uint32_t j = 0; j < LP_EIGHTS; ++j) {
        group[j] = x[8 * j];
#pragma unroll
        for (uint32_t e = 1; e < 8; ++e) group[j] = fmaxf(group[j], x[8 * j + e]);
    }
    auto groups = [&](float bound) {
        uint32_t n = 0;
#pragma unroll
        for (uint32_t j = 0; j < LP_EIGHTS; ++j) n += __popcll(__ballot(!(group[j] <= bound)));
        return n;
    };
    float bound = l.bound;
    uint32_t n = nan ? 64u * LP_EIGHTS : groups(bound);  // a maximum leaves out NaNs
    if (!n) return;
    // Cut once a wave's worth more than the top have come, which keeps the bound near the top of what was read.
    if (l.c > l.top && (l.c >= l.top + 64u || l.c + 8u * n > LP_LIST)) {
        bound = l.bound = lp_bound(lp_cut(l.list, l.c, l.top, l.list));
        l.c = l.top;
        if (!nan) n = groups(bound);
        if (!n) return;
    }
    if (l.c + 8u * n > LP_LIST) {
        // A lower bound of the batch's top-th value from the maxima of 8, by their leading bits: up to 16, fewer where
        // no more than 8 maxima too many reach it.
        uint32_t order[LP_EIGHTS], count, above, top = 0;
#pragma unroll
        for (uint32_t j = 0; j < LP_EIGHTS; ++j) {
            order[j] = lp_order(group[j]);
            top = max(top, order[j]);
        }
        const uint32_t leading = lp_search(
            [&](uint32_t probe) {
                uint32_t reached = 0;
#pragma unroll
                for (uint32_t j = 0; j < LP_EIGHTS; ++j) reached += __popcll(__ballot(order[j] >= probe));
                return reached;
            },
            lp_wave_max_u32(top), l.top, l.top + 8u, 0x10000u, 64u * LP_EIGHTS, count, above);
        if (leading > lp_order(-INFINITY)) {
            const float low = lp_bound(leading - 1u);
            if (!(low <= bound)) bound = low;
        }
        n = nan ? 64u * LP_EIGHTS : groups(bound);
        if (l.c + 8u * n > LP_LIST) {
            n = 0;
            const float b = gd_rounded(bound);
#pragma unroll
            for (uint32_t i = 0; i < LP_VALUES; ++i) n += __popcll(__ballot(!(x[i] <= b)));
        } else {
            n = 0;  // fits, however many of them pass
        }
        if (l.c + n > LP_LIST) {
            // The batch's own top, exactly: the largest order that `top` of its values reach, what is above it, and of
            // those that equal it the first.
            auto exact = [&](float v) {
                const float w = gd_rounded(v);
                return w <= bound ? 0u : lp_order(w);
            };
            uint32_t last = 0, left = l.top;
#pragma unroll 1
            for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
                uint32_t reached = 0;
#pragma unroll
                for (uint32_t i = 0; i < LP_VALUES; ++i) reached += __popcll(__ballot(exact(x[i]) >= (last | bit)));
                if (reached >= l.top) last |= bit;
            }
#pragma unroll
            for (uint32_t i = 0; i < LP_VALUES; ++i) {
                const bool take = exact(x[i]) > last;
                const uint64_t mask = __ballot(take);
                if (!mask) continue;
                if (take) l.list[l.c + lp_before(mask)] = lp_place(x[i], at(i >> 3) + (i & 7u));
                l.c += __popcll(mask);
                left -= __popcll(mask);  // fewer than `top` are above
            }
            // The 512 values of a step in order: by lane, then within its 8.
#pragma unroll
            for (uint32_t j = 0; j < LP_EIGHTS; ++j) {
                if (!left) break;
                uint32_t mine = 0;
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) mine += exact(x[8 * j + e]) == last ? 1u : 0u;
                const uint32_t upto = gd_wave_scan_u32(mine), all = __shfl(upto, 63, 64);
                uint32_t pos = upto - mine;
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e)
                    if (exact(x[8 * j + e]) == last) {
                        if (pos < left) l.list[l.c + pos] = lp_place(x[8 * j + e], at(j) + e);
                        ++pos;
                    }
                const uint32_t took = min(all, left);
                l.c += took;
                left -= took;
            }
            lp_wave_sync();
            l.bound = lp_bound(last);
            return;
        }
    }
    // Few lanes have any: a bit for each value that passes, then a round of the wave for the first of each lane's.
    uint32_t passing = 0;
#pragma unroll
    for (uint32_t i = 0; i < LP_VALUES; ++i) {
        passing |= !(x[i] <= bound) ? 1u << i : 0u;
        asm("" : "+v"(passing));  // one comparison at a time, not all kept apart
    }
    for (uint64_t mask = __ballot(passing != 0u); mask; mask = __ballot(passing != 0u)) {
        const uint32_t i = (uint32_t)__builtin_ctz(passing | 0x80000000u);
        float v[LP_VALUES / 2];
        auto choose = [](bool upper, float hi, float lo) { return upper ? hi : lo; };
#pragma unroll
        for (uint32_t k = 0; k < LP_VALUES / 2; ++k) v[k] = choose(i & (LP_VALUES / 2), x[LP_VALUES / 2 + k], x[k]);
#pragma unroll
        for (uint32_t w = LP_VALUES / 4; w > 0; w >>= 1)
#pragma unroll
            for (uint32_t k = 0; k < w; ++k) v[k] = choose(i & w, v[w + k], v[k]);
        if (passing) l.list[l.c + lp_before(mask)] = lp_place(v[0], at(i >> 3) + (i & 7u));
        l.c += __popcll(mask);
        passing &= passing - 1u;
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

// The row's outputs from its sums and its `top` places (list, in LDS, in any order); the first wave.
__device__ __forceinline__ void lp_finish(const GdArgs &a, uint64_t row, uint64_t X, const LpSums &p, const LpGiven &g,
                                          const uint64_t *list) {
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
    const uint64_t mine = lane < top ? list[lane] : 0ull;
    const uint32_t hi = (uint32_t)(mine >> 32), lo = (uint32_t)mine;
    uint32_t rank = 0;
#pragma unroll 4
    for (uint32_t k = 0; k < top; ++k) {
        const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)hi, (int)k) << 32 |
                               (uint32_t)__builtin_amdgcn_readlane((int)lo, (int)k);
        rank += other > mine ? 1u : 0u;
    }
    const auto ids = gd_at<uint32_t>(gd_addr(a, 20)) + row * gd_addr(a, 24);
    const auto tops = gd_at<float>(gd_addr(a, 22)) + row * gd_addr(a, 24);
    if (hi) {
        ids[rank] = ~lo;
        tops[rank] = logprob(lp_value(hi));
    }
    // What is missing are the first logits of -infinity.
    for (uint32_t found = __popcll(__ballot(hi != 0u)), i = 0; found < top && i < a.c[5]; i += 64u) {
        const bool hit = i + lane < a.c[5] && row_load(X, i + lane, a.c[4]) == -INFINITY;
        const uint64_t mask = __ballot(hit);
        const uint32_t to = found + lp_before(mask);
        if (hit && to < top) {
            ids[to] = i + lane;
            tops[to] = logprob(-INFINITY);
        }
        found += __popcll(mask);
    }
}

// Workspace of a row's part: the sums (4 words), then `top` places, in 16-byte units.
__device__ __forceinline__ uint64_t lp_part(const GdArgs &a, uint64_t row, uint32_t part) {
    return gd_addr(a, 28) + (row * a.c[27] + part) * (16u + 8ull * ((a.c[7] + 1u) & ~1u));
}

// A group of four waves takes a row, or a part of one, wave w batches w, w + 4, ... of it. Grid: x rows (up to 65535),
// y = (rows / 65535) * parts + part.
template <uint32_t TYPE>
__device__ __forceinline__ void logprobs_body(const GdArgs &a) {
    __shared__ uint64_t lists[LP_WAVES * LP_LIST];
    __shared__ uint64_t merged[LP_LIST];
    __shared__ LpSums sums[LP_WAVES];
    __shared__ uint32_t counts[LP_WAVES];
    const uint32_t V = a.c[5], top = a.c[7], parts = a.c[27], lane = threadIdx.x & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // uniform: branches and loops by it are scalar
    const uint32_t part = blockIdx.y % parts;
    const uint64_t row = (uint64_t)(blockIdx.y / parts) * gridDim.x + blockIdx.x;
    if (row >= a.c[26]) return;
    const float scale = gd_bits_f32(a.c[6]);
    const uint64_t X = gd_addr(a, 0) + ((row * gd_addr(a, 2)) << row_shift(TYPE));
    LpGiven given = {0.f, 1};
    if (parts == 1u) given = lp_given(a, row, X);
    const uint32_t batches = (V + LP_BATCH - 1u) / LP_BATCH;
    const uint32_t b0 = (uint32_t)((uint64_t)batches * part / parts), b1 = (uint32_t)((uint64_t)batches * (part + 1u) / parts);
    LpTop l = {lists + wave * LP_LIST, 0u, top, -INFINITY};
    LpSums p = {-INFINITY, 0.f, 0.f};
    for (uint32_t b = b0 + wave; b < b1; b += LP_WAVES) {
        const uint32_t first = b * LP_BATCH + 8u * lane;
        float x[LP_VALUES];
        // Eight values at a time; a lane that reaches past the row reads the row's last eight and leaves out (as
        // -infinity) those before its own. A row of fewer than eight is one lane's.
        auto at = [&](uint32_t j) { return V < 8u ? first + 512u * j : min(first + 512u * j, V - 8u); };
        if (V >= 8u) {
#pragma unroll
            for (uint32_t j = 0; j < LP_EIGHTS; ++j) {
                float v[8];
                row_load8<TYPE>(X, at(j), v);
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) x[8 * j + e] = v[e];
            }
            if (b + 1u == batches) {
#pragma unroll
                for (uint32_t i = 0; i < LP_VALUES; ++i)
                    if (at(i >> 3) + (i & 7u) < first + 512u * (i >> 3)) x[i] = -INFINITY;
            }
        } else {
#pragma unroll
            for (uint32_t i = 0; i < LP_VALUES; ++i) x[i] = i < 8u && first + i < V ? row_load(X, first + i, TYPE) : -INFINITY;
        }
        float most = x[0];
#pragma unroll
        for (uint32_t i = 1; i < LP_VALUES; ++i) most = fmaxf(most, x[i]);
        lp_move(p, fmaxf(p.m, most), scale);
        const float ref = p.m == -INFINITY ? 0.f : p.m;
        float s = 0.f, t = 0.f;
#pragma unroll
        for (uint32_t i = 0; i < LP_VALUES; ++i) {
            const float d = scale * (x[i] - ref), e = __expf(d);
            s += e;
            t += e * fmaxf(d, LP_FAR);
        }
        p.s += s;
        p.t += t;
        if (top) lp_add(l, x, at, __any(p.s != p.s));
    }
    p = lp_wave_join(p, scale);
    if (lane == 0) {
        sums[wave] = p;
        counts[wave] = l.c;
    }
    __syncthreads();
    if (top) {
        // The waves' lists side by side, each cut to its top first where they are too long together; the first `top`
        // places of a short one are filled up.
        uint32_t c[LP_WAVES], total = 0;
#pragma unroll
        for (uint32_t w = 0; w < LP_WAVES; ++w) total += c[w] = counts[w];
        const bool cut = total > LP_LIST - top;
        uint32_t start = 0, mine = l.c;
#pragma unroll
        for (uint32_t w = 0; w < LP_WAVES; ++w)
            if (w < wave) start += cut ? min(c[w], top) : c[w];
        if (cut && l.c > top) {
            lp_cut(l.list, l.c, top, l.list);
            mine = top;
        }
        for (uint32_t i = lane; i < mine; i += 64u) merged[start + i] = l.list[i];
        if (wave == LP_WAVES - 1u && start + mine < top)
            for (uint32_t i = start + mine + lane; i < top; i += 64u) merged[i] = lp_nothing(part * LP_TOP + i);
        __syncthreads();
        if (wave) return;
        total = 0;
#pragma unroll
        for (uint32_t w = 0; w < LP_WAVES; ++w) total += cut ? min(c[w], top) : c[w];
        if (total > top) lp_cut(merged, total, top, merged);
    }
    if (wave) return;
    p = lp_wave_join(lane < LP_WAVES ? sums[lane] : LpSums{-INFINITY, 0.f, 0.f}, scale);
    if (parts == 1u) {
        lp_finish(a, row, X, p, given, merged);
        return;
    }
    const uint64_t out = lp_part(a, row, part);
    if (lane == 0) gd_at<gd_f32x4>(out)[0] = gd_f32x4{p.m, p.s, p.t, 0.f};
    if (lane < top) gd_at<uint64_t>(out + 16u)[lane] = merged[lane];
}
