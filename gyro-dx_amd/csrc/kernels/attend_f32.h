// Attention of fp32 rows (attend.h): a group of four waves takes up to 16 rows and a part of the keys, its waves every
// fourth tile of 16 keys.
//
// As attend_few.h, by v_mfma_f32_16x16x4_f32: a lane holds 4 keys of one row, which are the second product's operand as they
// lie, and the values' operand is one value of a key, so that both cache arrays go from memory straight to operands.
#pragma once
#include "attend.h"

#define AS_KEYS 16u

template <uint32_t DT>
__device__ __forceinline__ void attend_f32_body(const GdArgs &a) {
    constexpr uint32_t STEPS = DT / 16u;
    __shared__ __align__(16) float lds[AF_WAVES * AF_ROWS * (DT + 4u)];
    const uint32_t lane = threadIdx.x & 63u, col = lane & 15u, h = lane >> 4, D = a.c[30];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    AfWork k;
    if (!af_work(a, k)) return;
    const AtItem &o = k.o;
    const gd_f32x4 none = {0.f, 0.f, 0.f, 0.f};
    gd_f32x4 q[STEPS], acc[STEPS];
#pragma unroll
    for (uint32_t s = 0; s < STEPS; ++s) {
        q[s] = acc[s] = none;
        if (16u * s + 4u * h < D) q[s] = *gd_at<const gd_f32x4_any>(gd_addr(a, 0) + 4u * k.q + 64u * s + 16u * h);
    }
    const float scale = gd_bits_f32(a.c[40]);
    const uint64_t K = gd_addr(a, 8), V = gd_addr(a, 10);
    float top = AT_LOWEST, sum = 0.f;

    for (uint32_t t = k.from + wave; t < k.to; t += AF_WAVES) {
        const int64_t at = at_key(a, o.seq, o.head, (int32_t)(16u * t + col), o.end);
        const uint32_t valid = (uint32_t)__ballot(at >= 0) & 0xffffu;  // the wave's quarters hold the same keys
        const uint64_t offset = at < 0 ? 0ull : (uint64_t)at;
        gd_f32x4 s = none;
#pragma unroll
        for (uint32_t e = 0; e < STEPS; ++e) {
            gd_f32x4 x = none;
            if (16u * e + 4u * h < D) x = *gd_at<const gd_f32x4_any>(K + offset + 64u * e + 16u * h);
#pragma unroll
            for (int i = 0; i < 4; ++i) s = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], q[e][i], s, 0, 0, 0);
        }
        float v[4][STEPS];
        bool odd = false;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t key = 4u * h + i;
            const uint32_t lo = __shfl((uint32_t)offset, key, 64), hi = __shfl((uint32_t)(offset >> 32), key, 64);
#pragma unroll
            for (uint32_t d = 0; d < STEPS; ++d) {
                v[i][d] = 0.f;
                if (16u * d + col < D && (valid >> key & 1u))
                    v[i][d] = *gd_at<const float>(V + ((uint64_t)lo | (uint64_t)hi << 32) + 64u * d + 4u * col);
                odd |= !(__builtin_fabsf(v[i][d]) < INFINITY);
            }
        }
        // Tiles that not every row sees whole.
        if (valid != 0xffffu || (int32_t)(16u * t) < o.all_first || (int32_t)(16u * t + 16u) > o.all_end) {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint32_t key = 4u * h + i;
                const int32_t j = (int32_t)(16u * t + key);
                if (!(valid >> key & 1u) || j > k.last || j < k.first) s[i] = -INFINITY;
            }
        }
        const float most = fmaxf(top, af_max(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]))) * scale);
        const float shrink = at_exp2(top - most);
        top = most;
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = at_exp2(fmaf(s[i], scale, -most));
        sum = sum * shrink + ((s[0] + s[1]) + (s[2] + s[3]));
#pragma unroll
        for (uint32_t d = 0; d < STEPS; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[d][i] *= shrink;
        if (__ballot(odd)) {
            // A value that is not finite reaches the rows that see its key, and no other (0 times it is NaN): one key
            // after another.
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
#pragma unroll 1
                for (uint32_t w = 0; w < 4; ++w) {
                    const int32_t j = (int32_t)(16u * t + 4u * w + i);
                    const bool seen = j <= k.last && j >= k.first;
#pragma unroll
                    for (uint32_t d = 0; d < STEPS; ++d) {
                        const gd_f32x4 one = __builtin_amdgcn_mfma_f32_16x16x4f32(h == w ? v[i][d] : 0.f, s[i], none, 0, 0, 0);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (seen) acc[d][e] += one[e];
                    }
                }
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
#pragma unroll
                for (uint32_t d = 0; d < STEPS; ++d) acc[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[i][d], s[i], acc[d], 0, 0, 0);
        }
    }
    af_finish<ROW_F32, DT, AF_ROWS * (DT + 4u)>(a, k, acc, top, sum, lds);
}
