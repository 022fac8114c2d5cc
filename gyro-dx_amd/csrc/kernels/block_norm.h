// The residual step between two blocks, one launch (the stack's moe_stack_norm with a norm behind the block, a gate
// and other types):
//   a = h rsqrt(mean(h^2) + post_eps) post_w   (or h itself)
//   v = x + scale gate a;   out = v;   normed = v rsqrt(mean(v^2) + pre_eps) pre_w
// gate: none, one value per token, per channel or per value, as it is or through a sigmoid. v stays in fp32 from the
// sum to `normed`; out and normed are rounded once. A group of 256 threads takes a token's row, 8 neighbouring
// values per thread and step, all of them in registers between the two sums of squares, whose partial sums meet
// in fixed order. out may be x, and normed h, in place.
//
// What bounds it: of many rows the bytes (4096 rows of 2048, fp32 stream, bf16 in and out, 101 MB: median 26 us of kernel, 3.9
// TB/s, 24 in a loop; a large copy moves 5.1). Rows of 2560 take 28.5 us in a loop (4.4 TB/s), of 16384 192 (4.2), but of 8192
// 131 (3.1): half the steps of the longest build are empty, and its 221 registers leave two waves a SIMD. Of few rows, one
// row's chain of loads, two sums and stores: median 3.8 us at 2048 values, 5.3 at 2560. The chain waits for each input in turn:
// row_load8 converts inside the branch on the type, so the next input's load is asked for after the one before has come. 777
// rows with a gate per value, all binary16, take 9.3 us of kernel for 3.1 us of bytes, at odd addresses or not.
// One row to a group rather than to a wave: a wave would hold a row of 2048 in 100 registers and leave a single row to
// one unit's fourth part. The builds differ in the steps of 2048 values that registers hold (1, 2, 8): a shorter one
// has more waves in flight and less to skip (block_norm_s against the two-step build: one row of 2048 3.8 against 4.9 us, 4096
// rows 25.5 against 26.8).
// Constants: 0 h (0: none, v = x) 2 h stride 4 x 6 x stride 8 out (0: none) 10 out stride 12 normed (0: none)
// 14 normed stride 16 post weight (0: none) 18 pre weight (0: none) 20 gate (0: none) 22 gate's token stride
// 24 gate's channel step (0 or 1) 25 types (h | x << 4 | out << 8 | normed << 12 | gate << 16) 26 flags (1 post norm,
// 2 sigmoid) 27 E 28 post eps 29 pre eps 30 scale (fp32 bits) 31 tokens. Weights are fp32.
#pragma once
#include "rows.h"

// Sum over the group's four waves, in their order.
__device__ __forceinline__ float bn_group_sum(float v, float *part) {
    v = gd_wave_sum_dpp(v);
    if ((threadIdx.x & 63u) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    return (part[0] + part[1]) + (part[2] + part[3]);
}

template <int STEPS>
__device__ __forceinline__ void block_norm_body(const GdArgs &a) {
    __shared__ float part[2][4];
    const uint32_t E = a.c[27], types = a.c[25], flags = a.c[26];
    const uint32_t ht = types & 15u, xt = types >> 4 & 15u, ot = types >> 8 & 15u, nt = types >> 12 & 15u, gt = types >> 16 & 15u;
    const uint64_t H = gd_addr(a, 0), X = gd_addr(a, 4), O = gd_addr(a, 8), N = gd_addr(a, 12), PW = gd_addr(a, 16),
                   NW = gd_addr(a, 18), G = gd_addr(a, 20);
    const uint64_t hs = gd_addr(a, 2), xs = gd_addr(a, 6), os = gd_addr(a, 10), ns = gd_addr(a, 14), gs = gd_addr(a, 22);
    const bool channel = a.c[24] != 0u, post = flags & 1u, sigmoid = flags & 2u;
    const float scale = gd_bits_f32(a.c[30]);
    const uint64_t row = (uint64_t)blockIdx.y * gridDim.x + blockIdx.x;
    if (row >= a.c[31]) return;
    float v[STEPS][8], x[STEPS][8], w[STEPS][8];
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
        const uint32_t i = (k * 256u + threadIdx.x) * 8u;
        row_load8(X + ((row * xs) << row_shift(xt)), i, E, xt, x[k]);
        if (H) row_load8(H + ((row * hs) << row_shift(ht)), i, E, ht, v[k]);
        else
#pragma unroll
            for (int j = 0; j < 8; ++j) v[k][j] = 0.f;
    }
    // The factors of a beside its root: the post weight times the gate, while the sum of squares waits for h.
    float factor = scale;
    if (G && !channel) {
        const float g = row_load(G, row * gs, gt);
        factor *= sigmoid ? gd_sigmoid_accurate(g) : g;
    }
    auto factors = [&](int k) {
        const uint32_t i = (k * 256u + threadIdx.x) * 8u;
#pragma unroll
        for (int j = 0; j < 8; ++j) w[k][j] = 1.f;
        if (PW) row_load8(PW, i, E, ROW_F32, w[k]);
        if (G && channel) {
            float g[8];
            row_load8(G + ((row * gs) << row_shift(gt)), i, E, gt, g);
#pragma unroll
            for (int j = 0; j < 8; ++j) w[k][j] *= sigmoid ? gd_sigmoid_accurate(g[j]) : g[j];
        }
    };
    auto pre_weights = [&](int k) {
#pragma unroll
        for (int j = 0; j < 8; ++j) w[k][j] = 1.f;
        if (NW) row_load8(NW, (k * 256u + threadIdx.x) * 8u, E, ROW_F32, w[k]);
    };
    constexpr bool AHEAD = STEPS <= 2;  // weights asked for before the sums they wait for, where registers allow it
    if (H) {
        if (AHEAD)
#pragma unroll
            for (int k = 0; k < STEPS; ++k) factors(k);
        float r = factor;
        if (post) {
#pragma unroll
            for (int k = 0; k < STEPS; ++k)
#pragma unroll
                for (int j = 0; j < 8; ++j) ss += v[k][j] * v[k][j];
            r = factor / sqrtf(bn_group_sum(ss, part[0]) / (float)E + gd_bits_f32(a.c[28]));
        }
#pragma unroll
        for (int k = 0; k < STEPS; ++k) {
            if (!AHEAD) factors(k);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[k][j] += v[k][j] * r * w[k][j];
        }
    }
    if (AHEAD && N)
#pragma unroll
        for (int k = 0; k < STEPS; ++k) pre_weights(k);
    if (O)
#pragma unroll
        for (int k = 0; k < STEPS; ++k)
            row_store8(O + ((row * os) << row_shift(ot)), (k * 256u + threadIdx.x) * 8u, E, ot, x[k]);
    if (!N) return;
    ss = 0.f;
#pragma unroll
    for (int k = 0; k < STEPS; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) ss += x[k][j] * x[k][j];  // values past the row's end are zeros
    const float r = 1.0f / sqrtf(bn_group_sum(ss, part[1]) / (float)E + gd_bits_f32(a.c[29]));
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
        if (!AHEAD) pre_weights(k);
#pragma unroll
        for (int j = 0; j < 8; ++j) w[k][j] *= x[k][j] * r;
        row_store8(N + ((row * ns) << row_shift(nt)), (k * 256u + threadIdx.x) * 8u, E, nt, w[k]);
    }
}
