// Joins the parts of rows that several groups of logprobs shared (logprobs.h): a group per row, a wave per quarter of
// the parts' places (at most 32 parts of at most 64), or the first wave alone where all of them fit its list.
#include "logprobs.h"

GD_PIPELINE_NAMED(logprobs_join, 256) {
    __shared__ uint64_t lists[LP_WAVES * LP_LIST];
    __shared__ uint64_t merged[LP_WAVES * LP_TOP];
    const uint32_t top = a.c[7], parts = a.c[27], lane = threadIdx.x & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // uniform: branches and loops by it are scalar
    const uint64_t row = (uint64_t)blockIdx.y * gridDim.x + blockIdx.x;
    if (row >= a.c[26]) return;
    const float scale = gd_bits_f32(a.c[6]);
    const uint64_t X = gd_addr(a, 0) + ((row * gd_addr(a, 2)) << row_shift(a.c[4]));
    const LpGiven given = lp_given(a, row, X);
    LpSums p = {-INFINITY, 0.f, 0.f};
    if (wave == 0 && lane < parts) {
        const gd_f32x4 v = gd_at<const gd_f32x4>(lp_part(a, row, lane))[0];
        p = LpSums{v[0], v[1], v[2]};
    }
    const bool alone = parts * top <= LP_LIST;
    if (top) {
        uint64_t *list = lists + wave * LP_LIST;
        const uint32_t step = alone ? 1u : LP_WAVES, total = parts * top;
        if (alone && wave == 0) {
            for (uint32_t i = lane; i < total; i += 64u) {
                const uint32_t part = i / top;
                list[i] = gd_at<const uint64_t>(lp_part(a, row, part) + 16u)[i - part * top];
            }
            lp_cut(list, total, top, merged);
        } else if (!alone) {
            // Wave w: parts w, w + 4, ..., up to 8 of them.
            uint32_t c = 0;
            for (uint32_t part = wave; part < parts; part += step, c += top)
                if (lane < top) list[c + lane] = gd_at<const uint64_t>(lp_part(a, row, part) + 16u)[lane];
            lp_cut(list, c, top, list);  // more than 512 places: every wave has a part
            if (lane < top) merged[wave * top + lane] = list[lane];
            __syncthreads();
            if (wave == 0) lp_cut(merged, LP_WAVES * top, top, merged);
        }
    }
    if (wave) return;
    lp_finish(a, row, X, lp_wave_join(p, scale), given, merged);
}
