// Attention of fp32 rows (attend.h): a group takes up to 16 rows and a part of the keys, its waves tiles of 16 or 32 keys in
// turn.
//
// As attend_few.h, by v_mfma_f32_16x16x4_f32: a lane holds 4 keys of one row, which are the second product's operand as they
// lie. Of the values a lane loads 4 neighbouring channels of a key, one for each of 4 products, whose rows are then channels 4
// apart: both cache arrays go from memory straight to operands, 16 bytes a lane.
//
// 37 tokens of 3 sequences over 1500 keys, 16 heads of 64 values, 144 groups: 26 us (38 MB, 1.4 TB/s; 26 TFLOP/s). The matrix
// unit's own time is 10 us of it on the compute units that have a group; the chain of scores, softmax and products in two waves
// a SIMD is the rest. Steps of 32 keys halve the chain's turns where registers hold them (heads of up to 64 values).
#pragma once
#include "attend.h"

template <uint32_t DT, uint32_t WAVES, uint32_t BLOCKS>
__device__ __forceinline__ void attend_f32_body(const GdArgs &a) {
    constexpr uint32_t KEYS = 16u * BLOCKS, STEPS = DT / 16u, WIDE = DT + 4u, EACH = AF_ROWS * WIDE;
    __shared__ __align__(16) float lds[WAVES * EACH];
    const uint32_t lane = threadIdx.x & 63u, col = lane & 15u, h = lane >> 4, D = a.c[30];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    AfWork work;
    if (!af_work(a, work)) return;
    const AtItem &o = work.o;
    const gd_f32x4 none = {0.f, 0.f, 0.f, 0.f};
    gd_f32x4 q[STEPS], acc[STEPS];
#pragma unroll
    for (uint32_t s = 0; s < STEPS; ++s) {
        q[s] = acc[s] = none;
        if (16u * s + 4u * h < D) q[s] = *gd_at<const gd_f32x4_any>(gd_addr(a, 0) + 4u * work.q + 64u * s + 16u * h);
    }
    const float scale = gd_bits_f32(a.c[40]);
    const uint64_t K = gd_addr(a, 8), V = gd_addr(a, 10);
    float top = AT_LOWEST, sum = 0.f;

    // A tile's keys, as in attend_few.h: lane l knows the place in the cache of key l % KEYS; k and v are on their way from when
    // their registers are free again.
    gd_f32x4 k[BLOCKS][STEPS], v[BLOCKS][4][STEPS / 4u];
    auto key_of = [&](uint32_t t) { return (int32_t)(KEYS * t + lane % KEYS); };
    auto page = [&](uint32_t t) { return at_page(a, o.seq, key_of(t), t < work.to ? o.end : 0); };
    auto locate = [&](uint32_t t, uint32_t page) { return at_key(a, page, o.head, key_of(t), t < work.to ? o.end : 0); };
    auto place = [&](int64_t at, uint32_t key) {
        const uint64_t offset = at < 0 ? 0ull : (uint64_t)at;
        return (uint64_t)__shfl((uint32_t)offset, key, 64) | (uint64_t)__shfl((uint32_t)(offset >> 32), key, 64) << 32;
    };
    auto head_end = [&] {
        uint32_t d = D;
        asm volatile("" : "+s"(d));
        return d;
    };
    auto load_k = [&](int64_t at) {
#pragma unroll
        for (uint32_t b = 0; b < BLOCKS; ++b) {
            const uint64_t from = K + place(at, 16u * b + col) + 16u * h;
            if (D == DT) {
#pragma unroll
                for (uint32_t s = 0; s < STEPS; ++s) k[b][s] = gd_at<const gd_f32x4_any>(from)[4u * s];
            } else {
                const uint32_t d = head_end();
#pragma unroll
                for (uint32_t s = 0; s < STEPS; ++s) k[b][s] = *gd_at<const gd_f32x4_any>(16u * s + 4u * h < d ? from + 64u * s : from - 16u * h);
            }
        }
    };
    auto load_v = [&](int64_t at) {
#pragma unroll
        for (uint32_t b = 0; b < BLOCKS; ++b)
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint64_t from = V + place(at, 16u * b + 4u * h + i) + 16u * col;
                if (D == DT) {
#pragma unroll
                    for (uint32_t g = 0; g < STEPS / 4u; ++g) v[b][i][g] = gd_at<const gd_f32x4_any>(from)[16u * g];
                } else {
                    const uint32_t d = head_end();
#pragma unroll
                    for (uint32_t g = 0; g < STEPS / 4u; ++g)
                        v[b][i][g] = *gd_at<const gd_f32x4_any>(64u * g + 4u * col < d ? from + 256u * g : from - 16u * col);
                }
            }
    };
    uint32_t soon = page(work.from + wave + WAVES);
    int64_t here = locate(work.from + wave, page(work.from + wave));
    load_k(here);
    __builtin_amdgcn_sched_barrier(0);  // keys first, as in the loop: the waits count what came after them
    load_v(here);
    for (uint32_t t = work.from + wave; t < work.to; t += WAVES) {
        const uint32_t later = page(t + 2u * WAVES);
        constexpr uint32_t ALL = BLOCKS == 2u ? ~0u : 0xffffu;
        const uint32_t valid = (uint32_t)__ballot(here >= 0) & ALL;  // the wave's other parts hold the same keys
        if (D != DT)
#pragma unroll
            for (uint32_t b = 0; b < BLOCKS; ++b)
#pragma unroll
                for (uint32_t e = 0; e < STEPS; ++e)
                    if (16u * e + 4u * h >= head_end()) k[b][e] = none;  // (q is zero there, but 0 times NaN is not)
        gd_f32x4 s[BLOCKS];
#pragma unroll
        for (uint32_t b = 0; b < BLOCKS; ++b) s[b] = none;
#pragma unroll
        for (uint32_t e = 0; e < STEPS; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (uint32_t b = 0; b < BLOCKS; ++b) s[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[b][e][i], q[e][i], s[b], 0, 0, 0);
        const int64_t next = locate(t + WAVES, soon);
        load_k(next);
        // Tiles that not every row sees whole.
        if (valid != ALL || (int32_t)(KEYS * t) < o.all_first || (int32_t)(KEYS * t + KEYS) > o.all_end) {
#pragma unroll
            for (uint32_t b = 0; b < BLOCKS; ++b)
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const uint32_t key = 16u * b + 4u * h + i;
                    const int32_t j = (int32_t)(KEYS * t + key);
                    s[b][i] = !(valid >> key & 1u) | (j > work.last) | (j < work.first) ? -INFINITY : s[b][i];
                }
        }
        float most = s[0][0];
#pragma unroll
        for (int i = 1; i < 4 * (int)BLOCKS; ++i) most = fmaxf(most, s[i >> 2][i & 3]);
        most = fmaxf(top, af_max(most) * scale);
        const float shrink = at_exp2(top - most);
        top = most;
        sum *= shrink;
        const bool far = __ballot(at_far(most));
        if (far)
#pragma unroll
            for (int i = 0; i < 4 * (int)BLOCKS; ++i) s[i >> 2][i & 3] = at_from_top(s[i >> 2][i & 3], scale, most);
        const float by = far ? 1.f : scale, from = far ? 0.f : most;
#pragma unroll
        for (uint32_t b = 0; b < BLOCKS; ++b) {
#pragma unroll
            for (int i = 0; i < 4; ++i) s[b][i] = at_exp2(fmaf(s[b][i], by, -from));
            sum += (s[b][0] + s[b][1]) + (s[b][2] + s[b][3]);
        }
#pragma unroll
        for (uint32_t d = 0; d < STEPS; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[d][i] *= shrink;
        if (valid != ALL || D != DT)
#pragma unroll
            for (uint32_t b = 0; b < BLOCKS; ++b)
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i)
#pragma unroll
                    for (uint32_t g = 0; g < STEPS / 4u; ++g)
                        if ((64u * g + 4u * col >= head_end()) | !(valid >> (16u * b + 4u * h + i) & 1u)) v[b][i][g] = none;
        float finite = 0.f;  // NaN from the first that is not on
#pragma unroll
        for (uint32_t b = 0; b < BLOCKS; ++b)
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
#pragma unroll
                for (uint32_t g = 0; g < STEPS / 4u; ++g)
#pragma unroll
                    for (int e = 0; e < 4; ++e) finite = fmaf(v[b][i][g][e], 0.f, finite);
        if (__ballot(!(finite == 0.f))) {
            // A value that is not finite reaches the rows that see its key, and no other (0 times it is NaN): one key
            // after another.
#pragma unroll
            for (uint32_t b = 0; b < BLOCKS; ++b)
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i)
#pragma unroll 1
                    for (uint32_t w = 0; w < 4; ++w) {
                        const int32_t j = (int32_t)(KEYS * t + 16u * b + 4u * w + i);
                        const bool seen = j <= work.last && j >= work.first;
#pragma unroll
                        for (uint32_t d = 0; d < STEPS; ++d) {
                            const gd_f32x4 one = __builtin_amdgcn_mfma_f32_16x16x4f32(h == w ? v[b][i][d >> 2][d & 3u] : 0.f, s[b][i], none, 0, 0, 0);
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[d][e] += seen ? one[e] : 0.f;
                        }
                    }
        } else {
#pragma unroll
            for (uint32_t b = 0; b < BLOCKS; ++b)
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i)
#pragma unroll
                    for (uint32_t d = 0; d < STEPS; ++d)
                        acc[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[b][i][d >> 2][d & 3u], s[b][i], acc[d], 0, 0, 0);
        }
        load_v(next);
        here = next;
        soon = later;
    }
    // Row 4 h + i of product 4 g + e is channel 64 g + 16 h + 4 i + e.
#pragma unroll
    for (uint32_t g = 0; g < STEPS / 4u; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<gd_f32x4 *>(lds + wave * EACH + col * WIDE + 64u * g + 16u * h + 4 * i) =
                gd_f32x4{acc[4 * g][i], acc[4 * g + 1][i], acc[4 * g + 2][i], acc[4 * g + 3][i]};
    af_finish<ROW_F32, DT, EACH, WAVES>(a, work, top, sum, lds);
}
