// Attention of many rows (attend.h), 16-bit types: a group of four waves takes 128 rows, 32 a wave, and a run of tiles of 64 or
// 32 keys (its unit), which go from memory straight to LDS, two buffers of keys and of values in turn.
//
// Scores are K Q^T by v_mfma_f32_32x32x16: a lane holds half the keys of one row, the other half is lane ^ 32's, so the
// running maximum needs one exchange per tile, the sum none until the end, and the weights are the second product's operand
// as they lie: O^T += V^T P^T, contracted over keys in the order in which lanes hold them; values come out of LDS transposed
// (ds_read_b64_tr_b16). The next tile's scores are multiplied while this one's weights are worked out, which are independent: the
// matrix unit and the vector unit work side by side within a wave. Sums are rescaled only when the maximum has grown by more than
// 2^8, of binary16 2^4 (at_grown).
//
// LDS is filled 1 KB an instruction in the order of lanes, so rows cannot be padded; instead their 16-byte pieces are swapped
// by the row's number such that every read finds its lanes in different banks (at_tile_k, at_tile_v; no conflict was counted).
//
// Weights are rounded once to the type before they meet the values, at most half a step and both ways alike, and summed as
// rounded: a second product for what is lost, as attend_few.h has it, would be half of the second products' work again, and the
// matrix unit is what bounds this kernel. Against 64 bits a bf16 prompt is off by 0.0020, with its result's rounding alone by
// 0.0016.
//
// 4096 tokens of 32 heads over 8 of 128 values, causal: 158 us with the join (869 TFLOP/s; a large library product reaches
// 1131). Matrix instructions fill 40% of all cycles and vector instructions 45%, at two waves a SIMD, which 249 registers
// allow. More buffers and earlier reads of LDS gained nothing, a wave's higher priority around its products 6%, 32-bit offsets
// into the cache, groups that find their units without a list and even rounds 5%. 128 rows halve the reads of 64; 256 would
// leave one wave a SIMD.
#pragma once
#include "attend16.h"
#include <type_traits>

template <uint32_t TYPE>
__device__ __forceinline__ at_f32x16 at_mfma(gd_u32x4 a, gd_u32x4 b, at_f32x16 c) {
    if constexpr (TYPE == ROW_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(at_f16x8, a), __builtin_bit_cast(at_f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(gd_bf16x8, a), __builtin_bit_cast(gd_bf16x8, b), c, 0, 0, 0);
}

// 16 bytes at each lane's address to LDS, from `lds` (of the wave) on in the order of lanes. Counted by vmcnt; at_landed waits.
// (The load needs a wait state behind M0's write, which the compiler does not see to within a statement.)
__device__ __forceinline__ void at_to_lds(uint32_t lds, uint64_t from) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(__builtin_amdgcn_readfirstlane(lds)), "v"(from)
                 : "memory", "m0");
}
// The same at a 32-bit offset from a uniform address.
__device__ __forceinline__ void at_to_lds(uint32_t lds, uint64_t base, uint32_t offset) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)base), hi = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(base >> 32));
    const uint64_t uniform = (uint64_t)hi << 32 | (uint64_t)lo;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(lds)), "v"(offset),
                 "s"(uniform)
                 : "memory", "m0");
}
__device__ __forceinline__ void at_landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// What a 16-byte piece's number in its row is changed by (exclusive or). Keys: 8 neighbouring rows are read at once, one piece of
// each. Values: 4 neighbouring rows, 4 pieces of each.
template <uint32_t CHUNKS>
__device__ __forceinline__ uint32_t at_tile_k(uint32_t row) { return row & (CHUNKS < 16u ? CHUNKS - 1u : 15u); }
template <uint32_t CHUNKS>
__device__ __forceinline__ uint32_t at_tile_v(uint32_t row) { return (CHUNKS < 16u ? row >> 1 & 1u : row & 3u) << 2; }

template <uint32_t TYPE, uint32_t DT, uint32_t KEYS, bool SMALL>
__device__ __forceinline__ void attend_tile_of(const GdArgs &a, const AtUnit &unit, uint32_t head, char *lds_k, char *lds_v, uint32_t (*lds_bad)[2]) {
    constexpr uint32_t ROW = DT * 2u, STEPS = DT / 16u, DIMS = DT / 32u, CHUNKS = DT / 8u, BLOCKS = KEYS / 32u;
    constexpr uint32_t PER = 64u / CHUNKS, LOADS = KEYS / (4u * PER);  // keys of a wave's load, loads of a wave
    using Place = std::conditional_t<SMALL, uint32_t, uint64_t>;  // of a key in the cache (in a head of it, if 32 bits span it)
    const uint32_t tid = threadIdx.x, lane = tid & 63u, col = lane & 31u, h = lane >> 5, D = a.c[30], group = a.c[29];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t seq = unit.seq, unit_from = unit.from, unit_to = unit.to, slot = unit.slot + unit.part;
    const bool alone = unit.parts == 1u;
    AtItem o;
    at_sequence(a, seq, o);
    at_keys(a, unit.tile * AT_ROWS, AT_ROWS, o);
    const int32_t end = o.end, all_first = o.all_first, all_end = o.all_end;
    const gd_u32x4 empty = {0u, 0u, 0u, 0u};

    const uint32_t row = min(o.row0 + 32u * wave + col, o.rows - 1u), token = row / group;  // rows past the last are the last again
    const bool idle = o.row0 + 32u * wave >= o.rows;                                       // a wave with none but those
    const int32_t p = o.kl - (int32_t)o.ql + (int32_t)token, window = (int32_t)a.c[39];
    const int32_t last = a.c[38] & 1u ? p : o.kl - 1, first = window ? p - window + 1 : 0;
    gd_u32x4 q[STEPS];
    {
        const uint64_t at = (uint64_t)(o.token0 + token) * gd_addr(a, 2) + (uint64_t)(head * group + row - token * group) * D;
#pragma unroll
        for (uint32_t s = 0; s < STEPS; ++s) {
            q[s] = empty;
            if (16u * s + 8u * h < D) q[s] = *gd_at<const gd_u32x4_any>(gd_addr(a, 0) + at * 2u + 32u * s + 16u * h);
        }
    }
    const float scale = gd_bits_f32(a.c[40]);
    const uint64_t of_head = SMALL ? head * gd_addr(a, 14) : 0ull, K = gd_addr(a, 8) + of_head, V = gd_addr(a, 10) + of_head;
    at_f32x16 acc[DIMS];
#pragma unroll
    for (uint32_t d = 0; d < DIMS; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
    float top = AT_LOWEST, sum = 0.f;
    bool far = false;  // some row's top is (at_far)

    // Load i of a wave brings keys 4 PER i + PER wave .. of a tile; a lane piece lane % CHUNKS of key lane / CHUNKS, which is the
    // piece of the head that belongs there. (Of shorter heads the others stay zeros.)
    const uint32_t of_key = PER * wave + lane / CHUNKS;  // + 4 PER i: at_tile_k and at_tile_v are the same for each i
    const uint32_t piece_k = (lane % CHUNKS) ^ at_tile_k<CHUNKS>(of_key), piece_v = (lane % CHUNKS) ^ at_tile_v<CHUNKS>(of_key);
    static_assert(4u * PER % 16u == 0u || CHUNKS > 16u, "a load's rows");
    auto key_of = [&](uint32_t t) { return (int32_t)(KEYS * t + lane % KEYS); };
    auto page = [&](uint32_t t) { return at_page(a, seq, key_of(t), t < unit_to ? end : 0); };
    // Where a tile's keys are in the cache (those that are not: at its start), of each load; which there are.
    auto locate = [&](uint32_t t, uint32_t page, Place (&at)[LOADS]) {
        bool there;
        if constexpr (SMALL) {
            const uint32_t offset = at_key_small(a, page, key_of(t), t < unit_to ? end : 0, there);
#pragma unroll
            for (uint32_t i = 0; i < LOADS; ++i) at[i] = __shfl(offset, 4u * PER * i + of_key, 64);
        } else {
            const int64_t where = at_key(a, page, head, key_of(t), t < unit_to ? end : 0);
            there = where >= 0;
            const uint64_t offset = there ? (uint64_t)where : 0ull;
#pragma unroll
            for (uint32_t i = 0; i < LOADS; ++i) {
                const uint32_t key = 4u * PER * i + of_key;
                at[i] = (uint64_t)__shfl((uint32_t)offset, key, 64) | (uint64_t)__shfl((uint32_t)(offset >> 32), key, 64) << 32;
            }
        }
        return (uint64_t)__ballot(there);  // (32 keys: twice)
    };
    auto fetch = [&](uint32_t lds, uint32_t t, uint64_t cache, Place at, uint32_t i, uint32_t piece) {
        lds += (t & 1u) * (KEYS * ROW) + (4u * PER * i + PER * wave) * ROW;
        if (D != DT && 8u * piece >= D) return;
        if constexpr (SMALL) at_to_lds(lds, cache, at + 16u * piece);
        else at_to_lds(lds, cache + at + 16u * piece);
    };
    // Load i of tile t's keys, or values, in buffer t % 2. (Of 256 values the rows of a load number are not those of the first.)
    auto fetch_k = [&](uint32_t t, Place at, uint32_t i) {
        fetch(at_lds(lds_k), t, K, at, i, CHUNKS > 16u ? (lane % CHUNKS) ^ at_tile_k<CHUNKS>(4u * PER * i + of_key) : piece_k);
    };
    auto fetch_v = [&](uint32_t t, Place at, uint32_t i) { fetch(at_lds(lds_v), t, V, at, i, piece_v); };

    // Where a lane's operands begin: its key of 32 and 8 of its channels; its 4 of 16 keys and 4 of 32 channels.
    const uint32_t from_k = at_lds(lds_k) + col * ROW + ((h ^ at_tile_k<CHUNKS>(col)) * 16u);
    const uint32_t of_v = (lane & 15u) >> 2, from_v = at_lds(lds_v) + (4u * h + of_v) * ROW + 32u * (lane >> 4 & 1u) + 8u * (lane & 3u);
    auto keys = [&](uint32_t base, uint32_t b, uint32_t e) { return at_lds_load((base ^ (32u * e)) + 32u * b * ROW); };
    auto values = [&](uint32_t t, uint32_t j, uint32_t d) {
        const uint32_t at = from_v + (t & 1u) * (KEYS * ROW) + 16u * j * ROW + 16u * (4u * d ^ at_tile_v<CHUNKS>(of_v));
        const gd_u32x2 lower = at_transposed(at), upper = at_transposed(at + 8u * ROW);
        return gd_u32x4{lower[0], lower[1], upper[0], upper[1]};
    };
    // Tiles that not every row sees whole.
    auto mixed = [&](uint32_t t) { return (int32_t)(KEYS * t) < all_first || (int32_t)(KEYS * t + KEYS) > all_end; };

    if (D != DT)
        for (uint32_t i = tid; i < 2u * KEYS * CHUNKS; i += 256u) {
            at_lds_store(at_lds(lds_k) + 16u * i, empty);
            at_lds_store(at_lds(lds_v) + 16u * i, empty);
        }
    if (tid < 4u) lds_bad[tid >> 1][tid & 1u] = 0u;
    __syncthreads();
    Place place[LOADS], place_next[LOADS];  // of the next tile's values, of the keys of the one after it
    uint64_t valid = locate(unit_from, page(unit_from), place);
#pragma unroll
    for (uint32_t i = 0; i < LOADS; ++i) {
        fetch_k(unit_from, place[i], i);
        fetch_v(unit_from, place[i], i);
    }
    uint64_t valid_next = locate(unit_from + 1u, page(unit_from + 1u), place);
#pragma unroll
    for (uint32_t i = 0; i < LOADS; ++i) fetch_k(unit_from + 1u, place[i], i);
    uint32_t soon = page(unit_from + 2u);
    asm volatile("" : "+v"(soon));
    at_f32x16 s[BLOCKS];
    // A tile's scores, a product a step: its operand is read AHEAD steps before, `beside` is work to run beside it. The steps
    // stay in this order (the scheduler would put one kind of work after the other).
    constexpr uint32_t PRODUCTS = STEPS * BLOCKS, AHEAD = 3;
    gd_u32x4 operand[AHEAD];
    uint32_t base_k = 0;
    auto scores_begin = [&](uint32_t t) {
        base_k = from_k + (t & 1u) * (KEYS * ROW);
        asm volatile("" : "+v"(base_k));  // (what follows from it is not to be held through the loop)
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i) operand[i] = keys(base_k, i % BLOCKS, i / BLOCKS);
    };
    auto scores = [&](at_f32x16 (&s)[BLOCKS], auto beside) {
#pragma unroll
        for (uint32_t b = 0; b < BLOCKS; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[b][i] = 0.f;
#pragma unroll
        for (uint32_t i = 0; i < PRODUCTS; ++i) {
            s[i % BLOCKS] = at_mfma<TYPE>(operand[i % AHEAD], q[i / BLOCKS], s[i % BLOCKS]);
            __builtin_amdgcn_sched_barrier(0);
            if (i + AHEAD < PRODUCTS) operand[i % AHEAD] = keys(base_k, (i + AHEAD) % BLOCKS, (i + AHEAD) / BLOCKS);
            beside(i);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    at_landed();
    __syncthreads();
    if (!idle) {
        scores_begin(unit_from);
        scores(s, [](uint32_t) {});
    }
    __syncthreads();  // its buffer is filled again

    auto tile = [&](uint32_t t, at_f32x16 (&s)[BLOCKS], at_f32x16 (&s_next)[BLOCKS]) {
        const uint64_t valid_later = locate(t + 2u, soon, place_next);
        const uint32_t later = page(t + 3u);
        // To be on its way during this tile: the next one's values, the keys of the one after it (behind the last tile, the
        // cache's first). Loads one behind another wait for the address unit: 8 of them took 1300 cycles of a tile's 4200.
        auto fetch_next = [&](uint32_t i) {
            if (i < LOADS) fetch_v(t + 1u, place[i], i);
            else if (i < 2u * LOADS) fetch_k(t + 2u, place_next[i - LOADS], i - LOADS);
        };
        const bool partly = valid != ~0ull || mixed(t);
        if (partly) {
            // Values of keys that are not there become zeros. One that is not finite must reach no row that does not see its
            // key (0 times it is NaN): such keys are taken out here and come back one by one below. (The empty asm keeps the
            // addresses out of the loop's registers.)
            uint32_t key0 = of_key;
            asm volatile("" : "+v"(key0));
#pragma unroll
            for (uint32_t i = 0; i < LOADS; ++i) {
                const uint32_t key = 4u * PER * i + key0, at = at_lds(lds_v) + (t & 1u) * (KEYS * ROW) + key * ROW + 16u * (lane % CHUNKS);
                const gd_u32x4 x = at_lds_load(at);
                float finite = 0.f;
#pragma unroll
                for (int e = 0; e < 4; ++e) finite = at_finite<TYPE>(x[e], finite);
                const bool there = valid >> key & 1u, odd = there & !(finite == 0.f);
                const uint64_t lanes = __ballot(odd);
                if (odd) atomicOr(&lds_bad[t & 1u][key >> 5], 1u << (key & 31u));
                if (!there | ((lanes >> (lane - lane % CHUNKS) & ((1ull << CHUNKS) - 1u)) != 0ull)) at_lds_store(at, empty);
            }
            __syncthreads();
        }
        if (tid < 2u) lds_bad[(t + 1u) & 1u][tid] = 0u;  // read a tile ago, written after the next barrier
        if (!idle) {
            if (partly) {
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
            scores_begin(t + 1u);
            float most = s[0][0];
#pragma unroll
            for (int i = 1; i < 16 * (int)BLOCKS; ++i) most = fmaxf(most, s[i >> 4][i & 15]);
            most = at_max_halves(most) * scale;
            if (__ballot(at_grown<TYPE>(most, top))) {
                most = at_new_top<TYPE, 11>(most, top);
                const float shrink = at_exp2(top - most);
                top = most;
                far = __ballot(at_far(top));
                sum *= shrink;
#pragma unroll
                for (uint32_t d = 0; d < DIMS; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[d][i] *= shrink;
            }
            if (far)
#pragma unroll
                for (int i = 0; i < 16 * (int)BLOCKS; ++i) s[i >> 4][i & 15] = at_from_top(s[i >> 4][i & 15], scale, top);
            const float by = far ? 1.f : scale, from = far ? 0.f : top;
            // The weights beside the next tile's scores (of the last one's: of what is in the buffer), with the first of V^T,
            // whose 16 keys and 32 channels an operand has in the order of the weights, behind.
            constexpr uint32_t PAIRS = 8u * BLOCKS;
            constexpr uint32_t SUMS = 2u * BLOCKS * DIMS, RING = 4;
            gd_u32x4 w[BLOCKS][2], x[RING];
            __builtin_amdgcn_s_setprio(1);  // the wave that multiplies goes first: 6% (two share a unit)
            scores(s_next, [&](uint32_t step) {
#pragma unroll
                for (uint32_t i = step * PAIRS / PRODUCTS; i < (step + 1u) * PAIRS / PRODUCTS; ++i) {
                    const uint32_t b = i >> 3, e = i & 7u;
                    const float x = at_exp2(fmaf(s[b][2 * e], by, -from)), y = at_exp2(fmaf(s[b][2 * e + 1], by, -from));
                    w[b][e >> 2][e & 3u] = at_pair<TYPE>(x, y);
                    sum = at_add_pair<TYPE>(w[b][e >> 2][e & 3u], sum);  // the sum of what the values are weighed with
                }
                if (step % 2u == 0u) fetch_next(step / 2u);
                if (step + RING >= PRODUCTS) x[step + RING - PRODUCTS] = values(t, (step + RING - PRODUCTS) / DIMS, (step + RING - PRODUCTS) % DIMS);
            });
#pragma unroll
            for (uint32_t i = 0; i < SUMS; ++i) {
                const uint32_t d = i % DIMS, j = i / DIMS, ahead = i + RING;
                acc[d] = at_mfma<TYPE>(x[i % RING], w[j >> 1][j & 1u], acc[d]);
                __builtin_amdgcn_sched_barrier(0);
                if (ahead < SUMS) x[i % RING] = values(t, ahead / DIMS, ahead % DIMS);
                __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_s_setprio(0);
            if (partly) {
                uint64_t bad = (uint64_t)lds_bad[t & 1u][0] | (uint64_t)lds_bad[t & 1u][1] << 32;
                while (bad) {
                    const uint32_t key = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)__builtin_ctzll(bad));
                    bad &= bad - 1u;
                    const int32_t j = (int32_t)(KEYS * t + key);
                    const int64_t where = at_key(a, at_page(a, seq, j, end), SMALL ? 0u : head, j, end);
                    const bool seen = j <= last && j >= first;
                    // The key's weight is in the lanes of half key / 4 % 2, one of a pair in a word.
                    uint32_t pair = 0;
#pragma unroll
                    for (uint32_t i = 0; i < 8u * BLOCKS; ++i)
                        if (((key >> 5) * 8u + (key >> 4 & 1u) * 4u + (key >> 3 & 1u) * 2u + (key >> 1 & 1u)) == i) pair = w[i >> 3][i >> 2 & 1][i & 3];
                    pair = __shfl(key & 1u ? pair >> 16 : pair & 0xffffu, col + 32u * (key >> 2 & 1u), 64);
                    const float weight = row_value16(pair, TYPE);
                    uint32_t half = h;
                    asm volatile("" : "+v"(half));
#pragma unroll
                    for (uint32_t d = 0; d < DIMS; ++d) {
#pragma unroll
                        for (uint32_t b = 0; b < 4; ++b) {
                            const uint32_t dim = 32u * d + 8u * b + 4u * half;
                            const gd_u32x2 x = *gd_at<const at_u32x2_any>(V + (uint64_t)where + 2u * (dim < D ? dim : 0u));
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                acc[d][4 * b + i] += seen ? weight * row_value16(x[i >> 1] >> (16 * (i & 1)) & 0xffffu, TYPE) : 0.f;
                        }
                        if constexpr (DT > 128u) asm volatile("" : "+a"(acc[d]));  // not all of them beside the others at once
                    }
                }
            }
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 2u * LOADS; ++i) fetch_next(i);
        }
        valid = valid_next;
        valid_next = valid_later;
        soon = later;
#pragma unroll
        for (uint32_t i = 0; i < LOADS; ++i) place[i] = place_next[i];
        at_landed();
        asm volatile("" : "+v"(soon));  // (it has landed as well: the compiler, which counts its load alone, is not to wait for others)
        __syncthreads();
    };
    at_f32x16 s_next[BLOCKS];
    for (uint32_t t = unit_from; t < unit_to;) {  // the scores by turns: copying them would be a tenth of the work
        tile(t, s, s_next);
        if (++t == unit_to) break;
        tile(t++, s_next, s);
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

template <uint32_t TYPE, uint32_t DT, uint32_t KEYS>
__device__ __forceinline__ void attend_tile_body(const GdArgs &a) {
    __shared__ __align__(1024) char lds_k[2 * KEYS * DT * 2];
    __shared__ __align__(1024) char lds_v[2 * KEYS * DT * 2];
    __shared__ uint32_t lds_bad[2][2];  // keys of a tile whose values are not all finite, by turns
    const uint32_t id = blockIdx.y * gridDim.x + blockIdx.x, KVH = a.c[31], index = id / KVH, head = id - index * KVH;
    AtUnit unit;
    if (gd_addr(a, 48)) {
        if (index >= at_plan(a)->units) return;
        const gd_gptr<const AtUnit> listed = at_units(a) + index;
        unit = AtUnit{listed->seq, listed->tile, listed->from, listed->to, listed->slot, listed->part, listed->parts, 0u};
        if (unit.slot == 0xffffffffu) return;
    } else {
        static_assert(sizeof(AtShare) <= sizeof(lds_k), "what a group works out before its first keys");
        AtShare &s = *reinterpret_cast<AtShare *>(lds_k);
        at_share(a, s, index, false);
        if (!__builtin_amdgcn_readfirstlane(s.found)) return;
        const uint32_t entry = __builtin_amdgcn_readfirstlane(s.entry), S = a.c[32], back = entry / S;
        unit.part = __builtin_amdgcn_readfirstlane(s.part);
        unit.parts = __builtin_amdgcn_readfirstlane(s.parts);
        unit.seq = entry - back * S;
        unit.tile = a.c[28] - 1u - back;
        unit.slot = index - unit.part;
        AtItem o;
        uint32_t tile0;
        at_sequence(a, unit.seq, o);
        at_keys(a, unit.tile * AT_ROWS, AT_ROWS, o);
        const uint32_t keys = at_tiles(o, KEYS, tile0);
        unit.from = tile0 + (uint32_t)((uint64_t)keys * unit.part / unit.parts);
        unit.to = tile0 + (uint32_t)((uint64_t)keys * (unit.part + 1u) / unit.parts);
        __syncthreads();
    }
    if (a.c[38] & 2u) attend_tile_of<TYPE, DT, KEYS, true>(a, unit, head, lds_k, lds_v, lds_bad);
    else attend_tile_of<TYPE, DT, KEYS, false>(a, unit, head, lds_k, lds_v, lds_bad);
}
