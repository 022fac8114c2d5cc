// Joins the parts of rows whose keys several groups shared (attend.h): a wave a row, four channels a lane. The first groups
// take the few rows' items, the others the plan's split tiles in turn.
#include "attend.h"

// A row's parts, `shared` of them and `step` bytes apart from `at` on, its row r of `rows`, into `out`.
__device__ __forceinline__ void aj_row(const GdArgs &a, uint64_t at, uint64_t step, uint32_t shared, uint32_t rows, uint32_t r, uint64_t out) {
    constexpr uint32_t HELD = 4;  // a lane's parts, of at most 64 of them each
    const uint32_t lane = threadIdx.x & 63u, D = a.c[30], type = a.c[43];
    float top[HELD], most = AT_LOWEST, total = 0.f;
#pragma unroll
    for (uint32_t k = 0; k < HELD; ++k) {
        const uint32_t part = 64u * k + lane;
        top[k] = part < shared ? gd_at<const float>(at + part * step)[r] : AT_LOWEST;
        most = fmaxf(most, top[k]);
    }
    most = gd_wave_max(most);
#pragma unroll
    for (uint32_t k = 0; k < HELD; ++k) {
        const uint32_t part = 64u * k + lane;
        top[k] = at_exp2(top[k] - most);
        if (part < shared) total += top[k] * gd_at<const float>(at + part * step)[rows + r];
    }
    total = gd_wave_sum_dpp(total);
    if (4u * lane >= D) return;
    gd_f32x4 x = {0.f, 0.f, 0.f, 0.f};
    const uint64_t from = at + 8ull * rows + ((uint64_t)r * D + 4u * lane) * 4u;
#pragma unroll
    for (uint32_t k = 0; k < HELD; ++k)
        for (uint32_t part = 64u * k; part < min(shared, 64u * k + 64u); ++part) {
            const float w = gd_bits_f32((uint32_t)__builtin_amdgcn_readlane((int)gd_f32_bits(top[k]), (int)(part & 63u)));
            const gd_f32x4 y = *gd_at<const gd_f32x4>(from + part * step);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] += w * y[i];
        }
    const float by = 1.f / total;
    if (type == ROW_F32) at_store4<ROW_F32>(out, 4u * lane, x, by, total == 0.f);
    else if (type == ROW_BF16) at_store4<ROW_BF16>(out, 4u * lane, x, by, total == 0.f);
    else at_store4<ROW_F16>(out, 4u * lane, x, by, total == 0.f);
}

// Row r of a sequence and head in out.
__device__ __forceinline__ uint64_t aj_out(const GdArgs &a, const AtItem &o, uint32_t r) {
    const uint32_t group = a.c[29], token = r / group;
    return gd_addr(a, 4) + (((uint64_t)(o.token0 + token) * gd_addr(a, 6) + (uint64_t)(o.head * group + r - token * group) * a.c[30]) << row_shift(a.c[43]));
}

GD_PIPELINE_NAMED(attend_join, 256) {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = blockIdx.y * gridDim.x + blockIdx.x, few = a.c[47];
    AtItem o;
    if (group < few) {
        const uint32_t id = group * 4u + wave, item = id / AF_ROWS, r = id - item * AF_ROWS;
        if (!af_item(a, item, o) || o.row0 + r >= o.rows) return;
        uint32_t tile0;
        const uint32_t shared = at_parts(a, at_tiles(o, a.c[44], tile0));
        if (shared == 1u) return;  // its group has written the rows
        aj_row(a, af_part(a, item, 0), at_part_bytes(a, AF_ROWS), shared, AF_ROWS, r, aj_out(a, o, o.row0 + r));
        return;
    }
    if (!gd_addr(a, 48)) return;
    const uint32_t KVH = a.c[31], groups = gridDim.x * gridDim.y - few;
    const uint64_t rows = (uint64_t)at_plan(a)->splits * KVH * AT_ROWS;
    for (uint64_t id = (uint64_t)(group - few) * 4u + wave; id < rows; id += groups * 4u) {
        const uint32_t rest = (uint32_t)(id / AT_ROWS), r = (uint32_t)id % AT_ROWS, index = rest / KVH;
        const uint32_t at = at_plan(a)->split[index];
        if (at == 0xffffffffu) continue;
        const AtUnit unit = at_units(a)[at];
        at_sequence(a, unit.seq, o);
        o.head = rest - index * KVH;
        if (unit.tile * AT_ROWS + r >= o.rows) continue;
        aj_row(a, at_slot(a, unit.slot, o.head), at_part_bytes(a, AT_ROWS) * KVH, unit.parts, AT_ROWS, r, aj_out(a, o, unit.tile * AT_ROWS + r));
    }
}
