// Joins the parts of rows whose keys several groups shared (attend.h). The first groups take the few rows' split entries, a
// group a row, as these may have hundreds of parts; the others the many rows' split tiles, in turn. Bound by latency (which
// were split, statistics, parts): 5 to 10 us, of which the launch is 2.
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

// A row of parts of ROWS rows, `step` bytes apart from `at` on, by the group: slices of it take parts in turn, four channels a
// thread.
template <uint32_t ROWS>
__device__ __forceinline__ void aj_by_group(const GdArgs &a, uint64_t at, uint64_t step, uint32_t parts, uint32_t r, uint64_t out) {
    constexpr uint32_t HELD = 5, MOST = HELD * AJ_THREADS;  // few rows' keys are split for 1024 groups at most, an entry in one part more
    __shared__ float weights[MOST], waves[2][AJ_WAVES];
    __shared__ __align__(16) float sums[4u * AJ_THREADS];
    const uint32_t tid = threadIdx.x, D = a.c[30], wide = D > 128u ? 64u : D > 64u ? 32u : 16u, slices = AJ_THREADS / wide;
    const uint32_t slice = tid / wide, d = 4u * (tid - slice * wide);
    const uint64_t from = at + 8u * ROWS + ((uint64_t)r * D + (d < D ? d : 0u)) * 4u;
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
            const float t = gd_at<const float>(own)[r], s = gd_at<const float>(own)[ROWS + r];
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

// A row of a few parts, by as many lanes as have four channels each; the others do nothing. Every lane reads all statistics.
__device__ __forceinline__ void aj_by_lanes(const GdArgs &a, uint64_t at, uint64_t step, uint32_t parts, uint32_t r, uint32_t d, uint64_t out) {
    const uint32_t D = a.c[30];
    const uint64_t from = at + 8u * AT_ROWS + ((uint64_t)r * D + (d < D ? d : 0u)) * 4u;
    gd_f32x4 x = {0.f, 0.f, 0.f, 0.f};
    float most = AT_LOWEST, total = 0.f;
    for (uint32_t p = 0; p < parts; p += 4u) {
        gd_f32x4 y[4];
        float top[4], sum[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const uint64_t off = min(p + i, parts - 1u) * step;
            y[i] = *gd_at<const gd_f32x4>(from + off);
            top[i] = gd_at<const float>(at + off)[r];
            sum[i] = gd_at<const float>(at + off)[AT_ROWS + r];
        }
        float next = most;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) next = fmaxf(next, top[i]);
        const float shrink = at_exp2(most - next);
        most = next;
        total *= shrink;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] *= shrink;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const float w = p + i < parts ? at_exp2(top[i] - most) : 0.f;
            if (p + i < parts) total += w * sum[i];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (p + i < parts) x[e] += w * y[i][e];
        }
    }
    if (d < D) aj_store(a, out, d, x, total);
}

// The rows of split tiles, `splits` of them, each of every head, among the groups from number `group` on. `entry` tells a
// split's sequence, tile of rows, first slot and parts.
template <typename F>
__device__ __forceinline__ void aj_tiles(const GdArgs &a, uint32_t group, uint32_t groups, uint32_t splits, F entry) {
    const uint32_t KVH = a.c[31], D = a.c[30], wide = D > 128u ? 64u : D > 64u ? 32u : 16u, at_once = AJ_THREADS / wide;
    const uint64_t step = at_part_bytes(a, AT_ROWS) * KVH;
    // A group's turn: at_once neighbouring rows of a split tile and head, which AT_ROWS is a multiple of, or fewer, down to one,
    // while that leaves every turn a group of its own (20 rows of 16000 keys and two heads: 40 us with
    // at_once rows a turn, 20 with one).
    uint32_t own = at_once;
    while (own > 1u && (uint64_t)splits * KVH * (AT_ROWS / own) * 2u <= groups) own >>= 1;
    const uint64_t turns = (uint64_t)splits * KVH * (AT_ROWS / own);
    for (uint64_t turn = group; turn < turns; turn += groups) {
        const uint32_t rest = (uint32_t)(turn / (AT_ROWS / own)), row0 = (uint32_t)(turn % (AT_ROWS / own)) * own, index = rest / KVH;
        AtItem o;
        uint32_t tile, slot, parts;
        if (!entry(index, o, tile, slot, parts)) continue;
        o.head = rest - index * KVH;
        const uint64_t at = at_slot(a, slot, o.head);
        if (parts <= 16u) {
            const uint32_t r = row0 + threadIdx.x / wide;
            if (r < row0 + own && tile * AT_ROWS + r < o.rows) aj_by_lanes(a, at, step, parts, r, 4u * (threadIdx.x % wide), aj_out(a, o, tile * AT_ROWS + r));
        } else {
            for (uint32_t r = row0; r < row0 + own && tile * AT_ROWS + r < o.rows; ++r) {
                aj_by_group<AT_ROWS>(a, at, step, parts, r, aj_out(a, o, tile * AT_ROWS + r));
                __syncthreads();
            }
        }
    }
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
        aj_by_group<AF_ROWS>(a, af_part(a, slot, o.head), at_part_bytes(a, AF_ROWS) * KVH, parts, r, aj_out(a, o, o.row0 + r));
        return;
    }
    const uint32_t groups = gridDim.x * gridDim.y - few;
    if (gd_addr(a, 48)) {
        aj_tiles(a, group - few, groups, at_plan(a)->splits, [&](uint32_t i, AtItem &o, uint32_t &tile, uint32_t &slot, uint32_t &parts) {
            const uint32_t at = at_plan(a)->split[i];
            if (at == 0xffffffffu) return false;
            const AtUnit unit = at_units(a)[at];
            at_sequence(a, unit.seq, o);
            tile = unit.tile;
            slot = unit.slot;
            parts = unit.parts;
            return true;
        });
    } else if (a.c[28]) {
        __shared__ AtShare s;
        at_share(a, s, 0u, true);
        const uint32_t share = at_fair(a, s.all);
        aj_tiles(a, group - few, groups, min(s.splits, AT_SPLITS), [&](uint32_t i, AtItem &o, uint32_t &tile, uint32_t &slot, uint32_t &parts) {
            const uint32_t entry = s.split[i] & 0xffffu, S = a.c[32], back = entry / S;
            uint32_t tile0;
            tile = a.c[28] - 1u - back;
            slot = s.split[i] >> 16;
            at_sequence(a, entry - back * S, o);
            at_keys(a, tile * AT_ROWS, AT_ROWS, o);
            parts = (at_tiles(o, a.c[55], tile0) + share - 1u) / share;
            return true;
        });
    }
}
