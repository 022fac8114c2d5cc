// Attention of few rows (attend.h), 16-bit types: a group of four waves takes up to 16 rows and a part of the keys, its waves
// every fourth tile of 32 keys.
//
// A tile's scores are K Q^T by two v_mfma_f32_16x16x32 a step: a lane then holds 8 keys of one row, the others are 16, 32 and 48
// lanes away, so that the running maximum needs two exchanges per tile, the sum none until the end, and the weights are the
// second product's operand as they lie: O^T += V^T P^T, contracted over keys in the order in which lanes hold them. Keys go
// from memory straight to operands. Values go through LDS, a wave's tile its own, and come back transposed
// (ds_read_b64_tr_b16).
//
// The weights are the sum of two 16-bit parts, so that they lose nothing: these rows are bound by memory, and the second
// products run in its shadow.
#pragma once
#include "attend16.h"

#define AF_KEYS 32u

template <uint32_t TYPE>
__device__ __forceinline__ gd_f32x4 af_mfma(gd_u32x4 a, gd_u32x4 b, gd_f32x4 c) {
    if constexpr (TYPE == ROW_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(at_f16x8, a), __builtin_bit_cast(at_f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(gd_bf16x8, a), __builtin_bit_cast(gd_bf16x8, b), c, 0, 0, 0);
}
template <uint32_t TYPE, uint32_t DT>
__device__ __forceinline__ void attend_few_body(const GdArgs &a) {
    // VROW: 16 rows' neighbouring 32 bytes in all banks.
    constexpr uint32_t STEPS = DT / 32u, DIMS = DT / 16u, VROW = DT * 2u + 32u, CHUNKS = DT / 8u, PER = 64u / CHUNKS;
    constexpr uint32_t VTILE = AF_KEYS * VROW;
    __shared__ __align__(16) char lds[AF_WAVES * VTILE];
    const uint32_t lane = threadIdx.x & 63u, col = lane & 15u, h = lane >> 4, D = a.c[30];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    AfWork work;
    if (!af_work(a, work)) return;
    const AtItem &o = work.o;
    const gd_u32x4 empty = {0u, 0u, 0u, 0u};
    const gd_f32x4 none = {0.f, 0.f, 0.f, 0.f};
    gd_u32x4 q[STEPS];
#pragma unroll
    for (uint32_t s = 0; s < STEPS; ++s) {
        q[s] = empty;
        if (32u * s + 8u * h < D) q[s] = *gd_at<const gd_u32x4_any>(gd_addr(a, 0) + 2u * work.q + 64u * s + 16u * h);
    }
    const float scale = gd_bits_f32(a.c[40]);
    const uint64_t K = gd_addr(a, 8), V = gd_addr(a, 10);
    const uint32_t mine = at_lds(lds) + wave * VTILE;
    gd_f32x4 acc[DIMS];
#pragma unroll
    for (uint32_t d = 0; d < DIMS; ++d) acc[d] = none;
    float top = AT_LOWEST, sum = 0.f;

    for (uint32_t t = work.from + wave; t < work.to; t += AF_WAVES) {
        const int64_t at = at_key(a, o.seq, o.head, (int32_t)(32u * t + (lane & 31u)), o.end);
        const uint32_t valid = (uint32_t)__ballot(at >= 0);  // both halves of the wave hold the same keys
        const uint64_t offset = at < 0 ? 0ull : (uint64_t)at;
        gd_u32x4 k[2][STEPS], v[AF_KEYS / PER];
#pragma unroll
        for (uint32_t b = 0; b < 2; ++b) {
            const uint32_t lo = __shfl((uint32_t)offset, 16u * b + col, 64), hi = __shfl((uint32_t)(offset >> 32), 16u * b + col, 64);
#pragma unroll
            for (uint32_t s = 0; s < STEPS; ++s) {
                k[b][s] = empty;
                if (32u * s + 8u * h < D) k[b][s] = *gd_at<const gd_u32x4_any>(K + ((uint64_t)lo | (uint64_t)hi << 32) + 64u * s + 16u * h);
            }
        }
#pragma unroll
        for (uint32_t j = 0; j < AF_KEYS / PER; ++j) {
            const uint32_t key = PER * j + lane / CHUNKS, chunk = lane % CHUNKS;
            const uint32_t lo = __shfl((uint32_t)offset, key, 64), hi = __shfl((uint32_t)(offset >> 32), key, 64);
            v[j] = empty;
            if (8u * chunk < D && (valid >> key & 1u)) v[j] = *gd_at<const gd_u32x4_any>(V + ((uint64_t)lo | (uint64_t)hi << 32) + 16u * chunk);
        }
        gd_f32x4 s[2] = {none, none};
#pragma unroll
        for (uint32_t e = 0; e < STEPS; ++e)
#pragma unroll
            for (uint32_t b = 0; b < 2; ++b) s[b] = af_mfma<TYPE>(k[b][e], q[e], s[b]);
        // Tiles that not every row sees whole.
        if (valid != ~0u || (int32_t)(32u * t) < o.all_first || (int32_t)(32u * t + 32u) > o.all_end) {
#pragma unroll
            for (uint32_t b = 0; b < 2; ++b)
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const uint32_t key = 16u * b + 4u * h + i;
                    const int32_t j = (int32_t)(32u * t + key);
                    s[b][i] = !(valid >> key & 1u) | (j > work.last) | (j < work.first) ? -INFINITY : s[b][i];
                }
        }
        // Keys whose values are not all finite.
        uint32_t bad = 0, largest = 0;
#pragma unroll
        for (uint32_t j = 0; j < AF_KEYS / PER; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) largest = at_larger(largest, v[j][i]);
        if (__ballot(at_not_finite<TYPE>(largest))) {
#pragma unroll
            for (uint32_t j = 0; j < AF_KEYS / PER; ++j) {
                largest = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) largest = at_larger(largest, v[j][i]);
                const uint64_t lanes = __ballot(at_not_finite<TYPE>(largest));
#pragma unroll
                for (uint32_t e = 0; e < PER; ++e)
                    if (lanes >> (e * CHUNKS) & ((1ull << CHUNKS) - 1u)) bad |= 1u << (PER * j + e);
            }
        }
        float most = s[0][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) most = fmaxf(most, s[i >> 2][i & 3]);
        most = fmaxf(top, af_max(most) * scale);
        const float shrink = at_exp2(top - most);
        top = most;
        float of_tile = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            s[i >> 2][i & 3] = at_exp2(fmaf(s[i >> 2][i & 3], scale, -most));
            of_tile += s[i >> 2][i & 3];
        }
        sum = sum * shrink + of_tile;
#pragma unroll
        for (uint32_t d = 0; d < DIMS; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[d][i] *= shrink;
        gd_u32x4 large, small;  // the weights' parts
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = s[i >> 1][2 * (i & 1)], y = s[i >> 1][2 * (i & 1) + 1];
            large[i] = at_pair<TYPE>(x, y);
            small[i] = at_pair<TYPE>(x - row_value16(large[i] & 0xffffu, TYPE), y - row_value16(large[i] >> 16, TYPE));
        }
        auto stage = [&](uint32_t keys) {
            __builtin_amdgcn_wave_barrier();  // after the reads of what is there
#pragma unroll
            for (uint32_t j = 0; j < AF_KEYS / PER; ++j) {
                const uint32_t key = PER * j + lane / CHUNKS;
                at_lds_store(mine + key * VROW + (lane % CHUNKS) * 16u, keys >> key & 1u ? v[j] : empty);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        };
        // V^T of 16 channels and the keys 4 h .. and 16 + 4 h .., in the order of the weights.
        auto values = [&](uint32_t d) {
            const uint32_t p = mine + (4u * h + (col >> 2)) * VROW + 32u * d + 8u * (col & 3u);
            const gd_u32x2 x = at_transposed(p), y = at_transposed(p + 16u * VROW);
            return gd_u32x4{x[0], x[1], y[0], y[1]};
        };
        stage(~bad);
#pragma unroll
        for (uint32_t d = 0; d < DIMS; ++d) {
            const gd_u32x4 x = values(d);
            acc[d] = af_mfma<TYPE>(x, small, acc[d]);
            acc[d] = af_mfma<TYPE>(x, large, acc[d]);
        }
        // A value that is not finite reaches the rows that see its key, times the whole weight, and no other (0 times it is
        // NaN): one key after another.
        while (bad) {
            const uint32_t key = (uint32_t)__builtin_ctz(bad);
            bad &= bad - 1u;
            const int32_t j = (int32_t)(32u * t + key);
            const bool seen = j <= work.last && j >= work.first;
            stage(1u << key);
#pragma unroll
            for (uint32_t d = 0; d < DIMS; ++d) {
                const gd_f32x4 one = af_mfma<TYPE>(values(d), large, none);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    acc[d][i] += seen ? one[i] : 0.f;
            }
        }
    }
    af_finish<TYPE, DT, VTILE / 4u>(a, work, acc, top, sum, reinterpret_cast<float *>(lds));
}
