// Log probabilities, entropy and top alternatives of rows of logits (logprobs.h): a group of four waves per row, or per
// part of one, wave w taking batches w, w + 4, ... of it. Grid: (row blocks of 65535, parts) as y = row block * parts + part.
#include "logprobs.h"

GD_PIPELINE_NAMED(logprobs, 256) {
    __shared__ uint64_t lists[LP_WAVES * LP_LIST];
    __shared__ uint64_t merged[LP_WAVES * LP_TOP];
    __shared__ LpSums sums[LP_WAVES];
    const uint32_t V = a.c[5], type = a.c[4], top = a.c[7], parts = a.c[27];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t part = blockIdx.y % parts;
    const uint64_t row = (uint64_t)(blockIdx.y / parts) * gridDim.x + blockIdx.x;
    if (row >= a.c[26]) return;
    const float scale = gd_bits_f32(a.c[6]);
    const uint64_t X = gd_addr(a, 0) + ((row * gd_addr(a, 2)) << row_shift(type));
    LpGiven given = {0.f, 1};
    if (parts == 1u) given = lp_given(a, row, X);

    // Values are counted from the 16-byte boundary at or before the row: the row is [from, to).
    const uint32_t from = (uint32_t)(X & 15u) >> row_shift(type), to = from + V;
    const uint64_t base = X & ~15ull;
    const uint32_t batches = (to + LP_BATCH - 1u) / LP_BATCH;
    const uint32_t b0 = (uint32_t)((uint64_t)batches * part / parts), b1 = (uint32_t)((uint64_t)batches * (part + 1u) / parts);
    LpTop l = {lists + wave * LP_LIST, 0u, top, -INFINITY};
    LpSums p = {-INFINITY, 0.f, 0.f};
    for (uint32_t b = b0 + wave; b < b1; b += LP_WAVES) {
        const uint32_t first = b * LP_BATCH;
        float x[32];
        const bool whole = first >= from && first + LP_BATCH <= to;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            const uint32_t i = first + 512u * j + 8u * lane;
            float v[8];
            if (whole) {
                row_load8(base, i, i + 8u, type, true, v);
            } else {
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e)
                    v[e] = i + e >= from && i + e < to ? row_load(base, i + e, type) : -INFINITY;
            }
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) x[8 * j + e] = v[e];
        }
        float most = x[0];
#pragma unroll
        for (uint32_t i = 1; i < 32; ++i) most = fmaxf(most, x[i]);
        // The lane's sums so far move to the new maximum; a maximum of -infinity counts as 0 (no term yet).
        const float m = fmaxf(p.m, most), ref = m == -INFINITY ? 0.f : m;
        const float back = lp_diff(p.m, ref, scale), shrink = __expf(back);
        p.t = shrink * (p.t + p.s * back);
        p.s *= shrink;
        p.m = m;
        float s = 0.f, t = 0.f;
#pragma unroll
        for (uint32_t i = 0; i < 32; ++i) {
            const float d = scale * (x[i] - ref), e = __expf(d);
            s += e;
            t += e * fmaxf(d, -1e30f);
        }
        p.s += s;
        p.t += t;
        if (top) lp_add(l, x, first - from, most, p.s != p.s);
    }
    p = lp_wave_join(p, scale);
    if (lane == 0) sums[wave] = p;
    if (top) {
        uint32_t bound;
        l.c = lp_cut(l.list, l.c, top, bound);
        lp_wave_sync();
        if (lane < top) merged[wave * top + lane] = lane < l.c ? l.list[lane] : lp_nothing(wave * LP_TOP + lane);
    }
    __syncthreads();
    if (wave) return;
    p = lp_join(lp_join(sums[0], sums[1], scale), lp_join(sums[2], sums[3], scale), scale);
    if (parts == 1u) {
        lp_finish(a, row, X, p, given, merged, LP_WAVES * top);
        return;
    }
    const uint64_t out = lp_part(a, row, part);
    if (lane == 0) gd_at<gd_f32x4>(out)[0] = gd_f32x4{p.m, p.s, p.t, 0.f};
    if (top) {
        uint32_t bound;
        lp_cut(merged, LP_WAVES * top, top, bound);
        if (lane < top) {
            const uint64_t p = merged[lane];
            gd_at<uint64_t>(out + 16u)[lane] = p >> 32 ? p : lp_nothing(part * LP_TOP + lane);
        }
    }
}
