// Attention of many rows (attend.h), 16-bit types: a group of four waves takes 128 rows, 32 a wave, and a run of tiles of 64 or 32 keys
// (attend_plan says which), keys and values of a tile in LDS, the next one on its way in registers.
//
// Scores are K Q^T by v_mfma_f32_32x32x16: a lane holds half the keys of one row, the other half is lane ^ 32's, so the
// running maximum needs one exchange per tile, the sum none until the end, and the weights are the second product's operand
// as they lie: O^T += V^T P^T, contracted over keys in the order in which lanes hold them; values come out of LDS transposed
// (ds_read_b64_tr_b16). The maximum that weights are relative to follows the running one only when that has grown by
// more than 2^8, so that the sums are rarely rescaled; weights are at most 2^8 then, and as precise.
#pragma once
#include "attend16.h"

template <uint32_t TYPE>
__device__ __forceinline__ at_f32x16 at_mfma(gd_u32x4 a, gd_u32x4 b, at_f32x16 c) {
    if constexpr (TYPE == ROW_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(at_f16x8, a), __builtin_bit_cast(at_f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(gd_bf16x8, a), __builtin_bit_cast(gd_bf16x8, b), c, 0, 0, 0);
}

// Asks the scheduler for FIRST reads of LDS, then STEPS times MFMAS products and READS reads: operands come just ahead of their
// products, and few registers hold them.
template <int FIRST, int READS, int MFMAS, int STEPS>
__device__ __forceinline__ void at_feed() {
    __builtin_amdgcn_sched_group_barrier(0x100, FIRST, 0);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, MFMAS, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
}

template <uint32_t TYPE, uint32_t DT, uint32_t KEYS>
__device__ __forceinline__ void attend_tile_body(const GdArgs &a) {
    // Rows in LDS: keys' 16 bytes of 8 neighbouring keys, and values' 64 of 4, in all banks.
    constexpr uint32_t KROW = DT * 2u + 16u, VROW = DT * 2u + 64u, STEPS = DT / 16u, DIMS = DT / 32u, CHUNKS = DT / 8u;
    constexpr uint32_t PASS = 256u / CHUNKS, PASSES = KEYS / PASS, BLOCKS = KEYS / 32u;  // keys that 256 threads load at once
    __shared__ __align__(16) char lds_k[2][KEYS * KROW];
    __shared__ __align__(16) char lds_v[2][KEYS * VROW];
    // Keys of a tile whose values are not all finite: of the one read, the one stored, and the one before, being cleared.
    __shared__ uint32_t lds_bad[3][2];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, col = lane & 31u, h = lane >> 5, D = a.c[30], group = a.c[29], KVH = a.c[31];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t id = blockIdx.y * gridDim.x + blockIdx.x, index = id / KVH, head = id - index * KVH;
    if (index >= at_plan(a)->units) return;
    const gd_gptr<const AtUnit> unit = at_units(a) + index;
    const uint32_t seq = unit->seq, unit_from = unit->from, unit_to = unit->to, slot = unit->slot + unit->part;
    const bool alone = unit->parts == 1u;
    if (unit->slot == 0xffffffffu) return;
    AtItem o;
    at_sequence(a, seq, o);
    at_keys(a, unit->tile * AT_ROWS, AT_ROWS, o);
    const int32_t end = o.end, all_first = o.all_first, all_end = o.all_end;
    const gd_u32x4 empty = {0u, 0u, 0u, 0u};

    const uint32_t row = min(o.row0 + 32u * wave + col, o.rows - 1u), token = row / group;  // rows past the last are the last again
    const bool idle = o.row0 + 32u * wave >= o.rows;                                       // a wave with none but those
    const uint64_t at = (uint64_t)(head * group + row - token * group) * D;
    const int32_t p = o.kl - (int32_t)o.ql + (int32_t)token, window = (int32_t)a.c[39];
    const int32_t last = a.c[38] ? p : o.kl - 1, first = window ? p - window + 1 : 0;
    gd_u32x4 q[STEPS];
#pragma unroll
    for (uint32_t s = 0; s < STEPS; ++s) {
        q[s] = empty;
        if (16u * s + 8u * h < D)
            q[s] = *gd_at<const gd_u32x4_any>(gd_addr(a, 0) + ((uint64_t)(o.token0 + token) * gd_addr(a, 2) + at) * 2u + 32u * s + 16u * h);
    }
    const float scale = gd_bits_f32(a.c[40]);
    const uint64_t K = gd_addr(a, 8), V = gd_addr(a, 10);
    at_f32x16 acc[DIMS];
#pragma unroll
    for (uint32_t d = 0; d < DIMS; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
    float top = AT_LOWEST, sum = 0.f;

    // Tile t's keys: a lane knows one's place in the cache, a thread loads 16 bytes of each of PASSES.
    // (Where there is none, it loads the cache's first, and drops it when it stores.)
    const uint32_t chunk = tid % CHUNKS, mine = tid / CHUNKS, in_head = 8u * chunk < D ? chunk : 0u;
    gd_u32x4 k_next[PASSES], v_next[PASSES];
    uint64_t valid_next = 0, valid = 0;
    const uint32_t to_k = at_lds(lds_k) + mine * KROW + 16u * chunk, to_v = at_lds(lds_v) + mine * VROW + 16u * chunk;
    // Where a lane's operands begin: its key of 32 and 8 of its channels, its 4 of 16 keys and 4 of its 32 channels.
    const uint32_t from_k = at_lds(lds_k) + col * KROW + 16u * h;
    const uint32_t from_v = at_lds(lds_v) + (4u * h + ((lane & 15u) >> 2)) * VROW + 32u * (lane >> 4 & 1u) + 8u * (lane & 3u);
    auto key_of = [&](uint32_t t) { return (int32_t)(KEYS * t + lane % KEYS); };
    auto page = [&](uint32_t t) { return at_page(a, seq, key_of(t), t < unit_to ? end : 0); };
    auto load = [&](uint32_t t, uint32_t page) {
        const int64_t where = at_key(a, page, head, key_of(t), t < unit_to ? end : 0);
        valid_next = __ballot(where >= 0);  // (32 keys: twice)
        const uint64_t offset = where < 0 ? 0ull : (uint64_t)where;
#pragma unroll
        for (uint32_t i = 0; i < PASSES; ++i) {
            const uint32_t key = PASS * i + mine;
            const uint32_t lo = __shfl((uint32_t)offset, key, 64), hi = __shfl((uint32_t)(offset >> 32), key, 64);
            const uint64_t from = ((uint64_t)lo | (uint64_t)hi << 32) + 16u * in_head;
            k_next[i] = *gd_at<const gd_u32x4_any>(K + from);
            v_next[i] = *gd_at<const gd_u32x4_any>(V + from);
        }
    };
    // Tiles that not every row sees whole.
    auto mixed = [&](uint32_t t) { return (int32_t)(KEYS * t) < all_first || (int32_t)(KEYS * t + KEYS) > all_end; };
    auto store = [&](uint32_t t, uint32_t buffer, uint32_t marks) {
        if (valid_next != ~0ull || D != DT) {
#pragma unroll
            for (uint32_t i = 0; i < PASSES; ++i)
                if ((8u * chunk >= D) | !(valid_next >> (PASS * i + mine) & 1u)) k_next[i] = v_next[i] = empty;
        }
        if (mixed(t)) {
            // A value that is not finite must reach no row that does not see its key (0 times it is NaN): such keys are
            // taken out here and come back one by one below.
#pragma unroll
            for (uint32_t i = 0; i < PASSES; ++i) {
                float finite = 0.f;
#pragma unroll
                for (int e = 0; e < 4; ++e) finite = at_finite<TYPE>(v_next[i][e], finite);
                const uint64_t odd = __ballot(!(finite == 0.f));
                if (odd) {
                    const uint32_t key = PASS * i + mine;
                    if (!(finite == 0.f)) atomicOr(&lds_bad[marks][key >> 5], 1u << (key & 31u));
                    if (odd >> (lane - lane % CHUNKS) & ((1ull << CHUNKS) - 1u)) v_next[i] = empty;
                }
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < PASSES; ++i) {
            at_lds_store(to_k + buffer * (KEYS * KROW) + PASS * i * KROW, k_next[i]);
            at_lds_store(to_v + buffer * (KEYS * VROW) + PASS * i * VROW, v_next[i]);
        }
    };

    if (tid < 6u) lds_bad[tid >> 1][tid & 1u] = 0u;
    __syncthreads();
    uint32_t soon = page(unit_from + 1u);
    load(unit_from, page(unit_from));
    if (unit_from < unit_to) store(unit_from, 0u, 0u);
    valid = valid_next;
    __syncthreads();
    uint32_t marks = 0;
    for (uint32_t t = unit_from; t < unit_to; ++t) {
        const uint32_t buffer = (t - unit_from) & 1u, marks_next = marks == 2u ? 0u : marks + 1u;
        const uint32_t later = page(t + 2u);
        load(t + 1u, soon);  // behind the last as well: at_page says why
        soon = later;
        const uint32_t kl = from_k + buffer * (KEYS * KROW), vl = from_v + buffer * (KEYS * VROW);
        if (!idle) {
            at_f32x16 s[BLOCKS];
#pragma unroll
            for (uint32_t b = 0; b < BLOCKS; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[b][i] = 0.f;
#pragma unroll
            for (uint32_t e = 0; e < STEPS; ++e)
#pragma unroll
                for (uint32_t b = 0; b < BLOCKS; ++b)
                    s[b] = at_mfma<TYPE>(at_lds_load(kl + 32u * b * KROW + 32u * e), q[e], s[b]);
            at_feed<2 * BLOCKS, BLOCKS, BLOCKS, STEPS>();
            if (valid != ~0ull || mixed(t)) {
                const int32_t key0 = (int32_t)(KEYS * t + 4u * h), most_key = last - key0, least_key = first - key0;
#pragma unroll
                for (int b = 0; b < (int)BLOCKS; ++b) {
                    const uint32_t held = (uint32_t)(valid >> (32 * b)) >> (4u * h);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int key = 8 * (i >> 2) + (i & 3);
                        const bool hidden = !(held >> key & 1u) | (32 * b + key > most_key) | (32 * b + key < least_key);
                        s[b][i] = hidden ? -INFINITY : s[b][i];
                    }
                }
            }
            float most = s[0][0];
#pragma unroll
            for (int i = 1; i < 16 * (int)BLOCKS; ++i) most = fmaxf(most, s[i >> 4][i & 15]);
            most = at_max_halves(most) * scale;
            if (__ballot(most > top + 8.f)) {
                most = fmaxf(most, top);
                const float shrink = at_exp2(top - most);
                top = most;
                sum *= shrink;
#pragma unroll
                for (uint32_t d = 0; d < DIMS; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[d][i] *= shrink;
            }
            gd_u32x4 w[BLOCKS][2];
            float part = 0.f;
#pragma unroll
            for (uint32_t b = 0; b < BLOCKS; ++b)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float x = at_exp2(fmaf(s[b][2 * i], scale, -top)), y = at_exp2(fmaf(s[b][2 * i + 1], scale, -top));
                    part += x + y;
                    w[b][i >> 2][i & 3] = at_pair<TYPE>(x, y);
                }
            sum += part;
#pragma unroll
            for (uint32_t b = 0; b < BLOCKS; ++b)
#pragma unroll
                for (uint32_t e = 0; e < 2; ++e)
#pragma unroll
                    for (uint32_t d = 0; d < DIMS; ++d) {
                        const uint32_t from = vl + (32u * b + 16u * e) * VROW + 64u * d;
                        const gd_u32x2 x = at_transposed(from), y = at_transposed(from + 8u * VROW);
                        acc[d] = at_mfma<TYPE>(gd_u32x4{x[0], x[1], y[0], y[1]}, w[b][e], acc[d]);
                    }
            at_feed<8, 2, 1, 2 * BLOCKS * DIMS>();
            uint64_t bad = (uint64_t)lds_bad[marks][0] | (uint64_t)lds_bad[marks][1] << 32;
            while (bad) {
                const uint32_t key = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)__builtin_ctzll(bad));
                bad &= bad - 1u;
                const int32_t j = (int32_t)(KEYS * t + key);
                const int64_t where = at_key(a, at_page(a, seq, j, end), head, j, end);
                const bool seen = j <= last && j >= first;
                // The key's weight is in the lanes of half key / 4 % 2, one of a pair in a word.
                uint32_t pair = 0;
#pragma unroll
                for (uint32_t i = 0; i < 8u * BLOCKS; ++i)
                    if (((key >> 5) * 8u + (key >> 4 & 1u) * 4u + (key >> 3 & 1u) * 2u + (key >> 1 & 1u)) == i) pair = w[i >> 3][i >> 2 & 1][i & 3];
                pair = key & 1u ? pair >> 16 : pair & 0xffffu;
                pair = __shfl(pair, col + 32u * (key >> 2 & 1u), 64);
                const float weight = row_value16(pair, TYPE);
#pragma unroll
                for (uint32_t d = 0; d < DIMS; ++d)
#pragma unroll
                    for (uint32_t b = 0; b < 4; ++b) {
                        const uint32_t dim = 32u * d + 8u * b + 4u * h;
                        const gd_u32x2 x = *gd_at<const at_u32x2_any>(V + (uint64_t)where + 2u * (dim < D ? dim : 0u));
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            acc[d][4 * b + i] += seen ? weight * row_value16(x[i >> 1] >> (16 * (i & 1)) & 0xffffu, TYPE) : 0.f;
                    }
            }
        }
        if (t + 1u < unit_to) {
            store(t + 1u, buffer ^ 1u, marks_next);
            valid = valid_next;
        }
        if (tid < 2u) lds_bad[marks_next == 2u ? 0u : marks_next + 1u][tid] = 0u;  // read a tile ago, written after the barrier
        marks = marks_next;
        __syncthreads();
    }

    if (o.row0 + 32u * wave + col >= o.rows) return;
    sum = at_sum_halves(sum);
    // (The row's place is worked out anew rather than held through the loop, which has no registers to spare.)
    uint32_t r = 32u * wave + col;
    asm volatile("" : "+v"(r));
    const uint32_t out_token = (o.row0 + r) / group;
    const uint64_t out = gd_addr(a, 4) + ((uint64_t)(o.token0 + out_token) * gd_addr(a, 6) + (uint64_t)(head * group + o.row0 + r - out_token * group) * D) * 2u;
    const uint64_t part = at_slot(a, slot, head);
    if (!alone && h == 0u) {
        gd_at<float>(part)[r] = top;
        gd_at<float>(part)[AT_ROWS + r] = sum;
    }
    const float by = 1.f / sum;
#pragma unroll
    for (uint32_t d = 0; d < DIMS; ++d)
#pragma unroll
        for (uint32_t b = 0; b < 4; ++b) {
            const uint32_t dim = 32u * d + 8u * b + 4u * h;
            const gd_f32x4 x = {acc[d][4 * b], acc[d][4 * b + 1], acc[d][4 * b + 2], acc[d][4 * b + 3]};
            if (dim >= D) continue;
            if (!alone) *gd_at<gd_f32x4>(part + 8u * AT_ROWS + ((uint64_t)r * D + dim) * 4u) = x;
            else at_store4<TYPE>(out, dim, x, by, sum == 0.f);
        }
}
