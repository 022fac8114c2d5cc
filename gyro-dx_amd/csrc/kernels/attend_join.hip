// Joins the parts of rows whose keys several groups shared (attend.h): a wave a row, four channels a lane.
#include "attend.h"

GD_PIPELINE_NAMED(attend_join, 256) {
    constexpr uint32_t HELD = 4;  // parts of a lane, of at most 64 of them each
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t rows = a.c[44], id = (blockIdx.y * gridDim.x + blockIdx.x) * 4u + wave, item = id / rows, r = id - item * rows;
    const uint32_t D = a.c[30], group = a.c[29];
    AtItem o;
    if (!at_item(a, item, rows, o) || o.row0 + r >= o.rows) return;
    uint32_t tile0;
    const uint32_t shared = at_parts(a, at_tiles(o, a.c[45], tile0), a.c[46]);
    if (shared == 1u) return;  // its group has written the rows
    float top[HELD], most = AT_LOWEST, total = 0.f;
#pragma unroll
    for (uint32_t k = 0; k < HELD; ++k) {
        const uint32_t part = 64u * k + lane;
        top[k] = part < shared ? gd_at<const float>(at_part(a, item, part, rows))[r] : AT_LOWEST;
        most = fmaxf(most, top[k]);
    }
    most = gd_wave_max(most);
#pragma unroll
    for (uint32_t k = 0; k < HELD; ++k) {
        const uint32_t part = 64u * k + lane;
        top[k] = at_exp2(top[k] - most);
        if (part < shared) total += top[k] * gd_at<const float>(at_part(a, item, part, rows))[rows + r];
    }
    total = gd_wave_sum_dpp(total);
    gd_f32x4 x = {0.f, 0.f, 0.f, 0.f};
    const uint64_t from = at_part(a, item, 0, rows) + 8ull * rows + ((uint64_t)r * D + 4u * lane) * 4u, step = (uint64_t)(rows * 4u) * (D + 2u);
    if (4u * lane < D)
#pragma unroll
        for (uint32_t k = 0; k < HELD; ++k)
            for (uint32_t part = 64u * k; part < min(shared, 64u * k + 64u); ++part) {
                const float w = gd_bits_f32((uint32_t)__builtin_amdgcn_readlane((int)gd_f32_bits(top[k]), (int)(part & 63u)));
                const gd_f32x4 y = *gd_at<const gd_f32x4>(from + part * step);
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] += w * y[i];
            }
    if (4u * lane >= D) return;
    const uint32_t token = (o.row0 + r) / group, type = a.c[43];
    const uint64_t at = gd_addr(a, 4) + (((uint64_t)(o.token0 + token) * gd_addr(a, 6) + (uint64_t)(o.head * group + o.row0 + r - token * group) * D +
                                          4u * lane) << row_shift(type));
#pragma unroll
    for (int i = 0; i < 4; ++i) row_store(at, i, type, total == 0.f ? 0.f : x[i] / total);
}
