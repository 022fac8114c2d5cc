// Joins the parts of rows whose keys several groups shared (attend.h). The first groups take the few rows' split entries, a
// group a row, as these may have hundreds of parts; the others the plan's split tiles, a wave a row, in turn.
#include "attend.h"

// Row r of a sequence and head in out.
__device__ __forceinline__ uint64_t aj_out(const GdArgs &a, const AtItem &o, uint32_t r) {
    const uint32_t group = a.c[29], token = r / group;
    return gd_addr(a, 4) + (((uint64_t)(o.token0 + token) * gd_addr(a, 6) + (uint64_t)(o.head * group + r - token * group) * a.c[30]) << row_shift(a.c[43]));
}
__device__ __forceinline__ void aj_store(const GdArgs &a, uint64_t out, uint32_t d, gd_f32x4 x, float total) {
    const float by = 1.f / total;
    if (a.c[43] == ROW_F32) at_store4<ROW_F32>(out, d, x, by, total == 0.f);
    else if (a.c[43] == ROW_BF16) at_store4<ROW_BF16>(out, d, x, by, total == 0.f);
    else at_store4<ROW_F16>(out, d, x, by, total == 0.f);
}

#define AJ_WAVES 4u
#define AJ_THREADS (64u * AJ_WAVES)

// The waves' values, as one.
template <typename F>
__device__ __forceinline__ float aj_group(float v, float *waves, F join) {
    if ((threadIdx.x & 63u) == 0u) waves[threadIdx.x >> 6] = v;
    __syncthreads();
    v = waves[0];
#pragma unroll
    for (uint32_t w = 1; w < AJ_WAVES; ++w) v = join(v, waves[w]);
    return v;
}

// A row of few rows' parts, `step` bytes apart from `at` on, by the group: slices of it take parts in turn, four channels a thread.
__device__ __forceinline__ void aj_by_group(const GdArgs &a, uint64_t at, uint64_t step, uint32_t parts, uint32_t r, uint64_t out) {
    constexpr uint32_t HELD = 5, MOST = HELD * AJ_THREADS;  // few rows' keys are split for 1024 groups at most, an entry in one part more
    __shared__ float weights[MOST], waves[2][AJ_WAVES];
    __shared__ __align__(16) float sums[4u * AJ_THREADS];
    const uint32_t tid = threadIdx.x, D = a.c[30], wide = D > 128u ? 64u : D > 64u ? 32u : 16u, slices = AJ_THREADS / wide;
    const uint32_t slice = tid / wide, d = 4u * (tid - slice * wide);
    const uint64_t from = at + 8u * AF_ROWS + ((uint64_t)r * D + (d < D ? d : 0u)) * 4u;
    gd_f32x4 y[4];  // asked for together with the statistics
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) y[i] = *gd_at<const gd_f32x4>(from + min(slice + i * slices, parts - 1u) * step);
    float top[HELD], sum[HELD], most = AT_LOWEST, total = 0.f;
#pragma unroll
    for (uint32_t i = 0; i < HELD; ++i) {
        const uint32_t p = tid + AJ_THREADS * i;
        top[i] = AT_LOWEST;
        sum[i] = 0.f;
        if (AJ_THREADS * i < parts) {
            const uint64_t own = at + min(p, parts - 1u) * step;
            const float t = gd_at<const float>(own)[r], s = gd_at<const float>(own)[AF_ROWS + r];
            top[i] = p < parts ? t : AT_LOWEST;
            sum[i] = p < parts ? s : 0.f;
        }
        most = fmaxf(most, top[i]);
    }
    most = aj_group(gd_wave_max(most), waves[0], [](float x, float y) { return fmaxf(x, y); });
#pragma unroll
    for (uint32_t i = 0; i < HELD; ++i) {
        const float w = at_exp2(top[i] - most);
        if (AJ_THREADS * i < parts) weights[tid + AJ_THREADS * i] = w;
        total += w * sum[i];
    }
    total = aj_group(gd_wave_sum_dpp(total), waves[1], [](float x, float y) { return x + y; });
    gd_f32x4 x = {0.f, 0.f, 0.f, 0.f};
    auto add = [&](gd_f32x4 v, uint32_t p) {
        const float w = weights[p];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] += w * v[i];
    };
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
        if (slice + i * slices < parts) add(y[i], slice + i * slices);
    for (uint32_t p = slice + 4u * slices; p < parts; p += 8u * slices) {
        gd_f32x4 v[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) v[i] = *gd_at<const gd_f32x4>(from + min(p + i * slices, parts - 1u) * step);
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
            if (p + i * slices < parts) add(v[i], p + i * slices);
    }
    *reinterpret_cast<gd_f32x4 *>(sums + 4u * tid) = x;
    __syncthreads();
    if (slice || d >= D) return;
    for (uint32_t k = 1; k < min(slices, parts); ++k) {
        const gd_f32x4 v = *reinterpret_cast<const gd_f32x4 *>(sums + 4u * (tid + k * wide));
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] += v[i];
    }
    aj_store(a, out, d, x, total);
}

// A row of many rows' parts, by a wave: four channels a lane.
__device__ __forceinline__ void aj_by_wave(const GdArgs &a, uint64_t at, uint64_t step, uint32_t parts, uint32_t r, uint64_t out) {
    constexpr uint32_t HELD = 8;  // a lane's parts, of 64 of them each: attend_plan splits a tile into 512 at most
    const uint32_t lane = threadIdx.x & 63u, D = a.c[30], d = 4u * lane < D ? 4u * lane : 0u;
    const uint64_t from = at + 8u * AT_ROWS + ((uint64_t)r * D + d) * 4u;
    gd_f32x4 first[4];  // asked for together with the statistics
#pragma unroll
    for (uint32_t p = 0; p < 4; ++p) first[p] = *gd_at<const gd_f32x4>(from + min(p, parts - 1u) * step);
    float top[HELD], sum[HELD], most = AT_LOWEST, total = 0.f;
#pragma unroll
    for (uint32_t k = 0; k < HELD; ++k) {
        top[k] = AT_LOWEST;
        sum[k] = 0.f;
        if (64u * k < parts) {
            const uint64_t own = at + min(64u * k + lane, parts - 1u) * step;
            const float t = gd_at<const float>(own)[r], s = gd_at<const float>(own)[AT_ROWS + r];
            top[k] = 64u * k + lane < parts ? t : AT_LOWEST;
            sum[k] = 64u * k + lane < parts ? s : 0.f;
        }
        most = fmaxf(most, top[k]);
    }
    most = gd_wave_max(most);
#pragma unroll
    for (uint32_t k = 0; k < HELD; ++k) {
        top[k] = at_exp2(top[k] - most);
        total += top[k] * sum[k];
    }
    total = gd_wave_sum_dpp(total);
    gd_f32x4 x = {0.f, 0.f, 0.f, 0.f};
    auto add = [&](gd_f32x4 y, float of, uint32_t p) {
        const float w = gd_bits_f32((uint32_t)__builtin_amdgcn_readlane((int)gd_f32_bits(of), (int)(p & 63u)));
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] += w * y[i];
    };
#pragma unroll
    for (uint32_t p = 0; p < 4; ++p)
        if (p < parts) add(first[p], top[0], p);
#pragma unroll
    for (uint32_t k = 0; k < HELD; ++k)
#pragma unroll 4
        for (uint32_t p = k ? 64u * k : 4u; p < min(parts, 64u * k + 64u); ++p) add(*gd_at<const gd_f32x4>(from + p * step), top[k], p);
    if (4u * lane < D) aj_store(a, out, d, x, total);
}

GD_PIPELINE_NAMED(attend_join, 256) {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = blockIdx.y * gridDim.x + blockIdx.x, few = a.c[47], KVH = a.c[31];
    AtItem o;
    if (group < few) {
        const uint32_t rest = group / a.c[56], r = group - rest * a.c[56], index = rest / KVH;
        uint32_t wanted = index, entry, parts, slot, tile0;
        if (!af_find<AF_SPLITS>(a, af_share(a), wanted, entry, parts, slot)) return;
        af_entry(a, entry, o, tile0);
        o.head = rest - index * KVH;
        if (o.row0 + r >= o.rows) return;
        aj_by_group(a, af_part(a, slot, o.head), at_part_bytes(a, AF_ROWS) * KVH, parts, r, aj_out(a, o, o.row0 + r));
        return;
    }
    if (!gd_addr(a, 48)) return;
    const uint32_t groups = gridDim.x * gridDim.y - few;
    const uint64_t rows = (uint64_t)at_plan(a)->splits * KVH * AT_ROWS;
    for (uint64_t id = (uint64_t)(group - few) * AJ_WAVES + wave; id < rows; id += groups * AJ_WAVES) {
        const uint32_t rest = (uint32_t)(id / AT_ROWS), r = (uint32_t)id % AT_ROWS, index = rest / KVH;
        const uint32_t at = at_plan(a)->split[index];
        if (at == 0xffffffffu) continue;
        const AtUnit unit = at_units(a)[at];
        at_sequence(a, unit.seq, o);
        o.head = rest - index * KVH;
        if (unit.tile * AT_ROWS + r >= o.rows) continue;
        aj_by_wave(a, at_slot(a, unit.slot, o.head), at_part_bytes(a, AT_ROWS) * KVH, unit.parts, r, aj_out(a, o, unit.tile * AT_ROWS + r));
    }
}
