// Cuts the sequences of many rows into units for attend_tile (attend.h), one group for the launch: the tiles of 128 rows, whose
// keys are split where one has more tiles of them than its share (at_fair), the units of most tiles first. Units of one size
// come in any order, which changes no result.
#include "attend.h"

#define AP_CLASSES 32u

GD_PIPELINE_NAMED(attend_plan, 1024) {
    __shared__ uint32_t before[1025];  // tiles of rows of the chunk's sequences before each
    __shared__ uint32_t waves[16];
    __shared__ uint64_t total;
    __shared__ uint32_t cursor[AP_CLASSES], slots, splits;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, S = a.c[32], most = a.c[53], most_slots = a.c[54];
    const gd_gptr<AtPlan> plan = at_plan(a);
    const gd_gptr<AtUnit> units = at_units(a);
    if (tid < AP_CLASSES) cursor[tid] = 0u;
    if (tid == 0u) {
        total = 0;
        slots = splits = 0u;
    }
    // Calls f(sequence, tile of rows, tiles of keys, the first's number) for every tile of rows.
    auto each = [&](auto f) {
        for (uint32_t s0 = 0; s0 < S; s0 += 1024u) {
            AtItem o;
            uint32_t own = 0;
            if (s0 + tid < S) {
                at_sequence(a, s0 + tid, o);
                // (of a sequence of more than `longest` tokens those alone: the list has room for no more)
                if (o.rows >= a.c[46]) own = (min(o.rows, a.c[33] * a.c[29]) + AT_ROWS - 1u) / AT_ROWS;
            }
            const uint32_t upto = gd_wave_scan_u32(own);
            __syncthreads();  // the chunk before is done
            if (lane == 63u) waves[wave] = upto;
            __syncthreads();
            uint32_t base = 0;
            for (uint32_t w = 0; w < wave; ++w) base += waves[w];
            before[tid + 1u] = base + upto;
            if (tid == 0u) before[0] = 0u;
            __syncthreads();
            const uint32_t tiles = before[1024];
            for (uint32_t i = tid; i < tiles; i += 1024u) {
                uint32_t b = 0;
#pragma unroll
                for (uint32_t step = 512; step > 0; step >>= 1)
                    if (before[b + step] <= i) b += step;
                at_sequence(a, s0 + b, o);
                at_keys(a, (i - before[b]) * AT_ROWS, AT_ROWS, o);
                uint32_t tile0;
                const uint32_t keys = at_tiles(o, a.c[55], tile0);
                f(s0 + b, i - before[b], keys, tile0);
            }
        }
        __syncthreads();
    };
    uint64_t sum = 0;
    each([&](uint32_t, uint32_t, uint32_t keys, uint32_t) { sum += keys; });
    if (sum) atomicAdd((unsigned long long *)&total, (unsigned long long)sum);
    __syncthreads();
    const uint32_t share = at_fair(a, total);
    auto parts_of = [&](uint32_t keys) { return max(1u, (uint32_t)(((uint64_t)keys + share - 1u) / share)); };
    auto class_of = [&](uint32_t keys, uint32_t parts) {
        return AP_CLASSES - 1u - min(AP_CLASSES - 1u, (uint32_t)((uint64_t)(keys / parts) * AP_CLASSES / ((uint64_t)share + 1u)));
    };
    each([&](uint32_t, uint32_t, uint32_t keys, uint32_t) {
        const uint32_t parts = parts_of(keys);
        atomicAdd(&cursor[class_of(keys, parts)], parts);
    });
    if (tid == 0u) {
        uint32_t at = 0;
        for (uint32_t i = 0; i < AP_CLASSES; ++i) {
            const uint32_t count = cursor[i];
            cursor[i] = at;
            at += count;
        }
        plan->units = min(at, most);
    }
    __syncthreads();
    each([&](uint32_t seq, uint32_t tile, uint32_t keys, uint32_t tile0) {
        uint32_t parts = parts_of(keys), slot = 0;
        const uint32_t at = atomicAdd(&cursor[class_of(keys, parts)], parts);
        const uint32_t planned = parts;
        if (parts > 1u) {
            slot = atomicAdd(&slots, parts);
            const uint32_t split = atomicAdd(&splits, 1u);
            if (slot + parts > most_slots || split >= AT_SPLITS || at + parts > most) parts = 1u;  // starts that fall make too many
            if (split < AT_SPLITS) plan->split[split] = parts > 1u ? at : 0xffffffffu;
        }
        for (uint32_t part = 0; part < planned; ++part) {
            if (at + part >= most) break;
            const bool whole = parts == 1u;
            units[at + part] = AtUnit{seq, tile, tile0 + (whole ? (part ? keys : 0u) : (uint32_t)((uint64_t)keys * part / parts)),
                                      tile0 + (whole ? keys : (uint32_t)((uint64_t)keys * (part + 1u) / parts)),
                                      whole && part ? 0xffffffffu : slot, part, parts, 0u};
        }
    });
    if (tid == 0u) plan->splits = min(splits, AT_SPLITS);
}
