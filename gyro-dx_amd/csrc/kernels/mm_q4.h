// Products of many tokens with a 4-bit matrix in the layout of q4_repack (q4.h).
//
// A group of four waves takes 16 tiles (256 weight rows), four to a wave, and 16 T tokens. Chunks of 128 columns of the
// tokens go through LDS as operands, two buffers in turn, one being filled while the other is multiplied;
// weights go from memory to registers, a chunk ahead. Per group of 32 columns a wave unpacks 4 operands, each used for T
// products, and scales 4 T sums: 28 + 16 T vector instructions beside 5 T matrix ones. bf16 and binary16 tokens are
// operands as they are; fp32 ones go through the products three times, a part each (PARTS).
#pragma once
#include "q4.h"

#define MM_WAVES 4u
#define MM_R 4

typedef _Float16 gd_f16x8 __attribute__((ext_vector_type(8)));

// c + a b of token operand a and weight operand b, both of the operand type.
template <bool HALF>
__device__ __forceinline__ gd_f32x4 mm_mfma(gd_u32x4 a, gd_u32x4 b, gd_f32x4 c) {
    if constexpr (HALF)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(gd_f16x8, a), __builtin_bit_cast(gd_f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(gd_bf16x8, a), __builtin_bit_cast(gd_bf16x8, b), c, 0, 0, 0);
}
template <uint32_t TYPE, bool MINIMA, int T>
__device__ __forceinline__ void mm_q4_tile(const GdArgs &a, gd_u32x4 *lds) {
    constexpr bool HALF = TYPE == ROW_F16;
    constexpr int PARTS = TYPE == ROW_F32 ? 3 : 1;
    constexpr uint32_t ROWS = 16u * T, UNITS = ROWS * 16u, PER = UNITS / 256u;  // 16-byte units of a chunk, of a thread
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, col = lane & 15u, h = lane >> 4;
    const uint64_t quants = gd_addr(a, 0), scales = gd_addr(a, 2), minima = gd_addr(a, 4);
    const uint32_t tiles = a.c[6], chunks = a.c[7], lg = a.c[8], cols = a.c[9], outputs = a.c[10], n = a.c[17];
    const uint64_t X = gd_addr(a, 12), xs = gd_addr(a, 14);
    // The groups of an XCD (i % 8) take neighbouring rows, all tokens of some before the next, so that its L2 holds
    // their weights.
    uint32_t rb = blockIdx.x, tb = blockIdx.y;
    if ((gridDim.x & 7u) == 0u) {
        const uint32_t i = blockIdx.y * gridDim.x + blockIdx.x, own = gridDim.x >> 3, s = i >> 3;
        tb = s % gridDim.y;
        rb = (i & 7u) * own + s / gridDim.y;
    }
    const uint32_t t0 = tb * ROWS, tile0 = (rb * MM_WAVES + wave) * MM_R;
    const MqSpread spread = mq_spread(lg);
    const MqBits bits = mq_bits<HALF>();
    const uint32_t b16 = HALF ? (MINIMA ? 0xcc00u : 0xce00u) : (MINIMA ? 0xc180u : 0xc1c0u), b32 = b16 | b16 << 16;  // -16, -24
    const gd_u32x4 unbias = {b32, b32, b32, b32};
    const gd_f32x4 zero = {0.f, 0.f, 0.f, 0.f};

    MqChunk cur[MM_R], next[MM_R];
    auto load = [&](uint32_t c, MqChunk (&o)[MM_R]) {
#pragma unroll
        for (int r = 0; r < MM_R; ++r) {
            // Tiles past the last read the last again; their sums are dropped.
            const uint64_t unit = (uint64_t)min(tile0 + r, tiles - 1u) * chunks + c;
            o[r].w = gd_at<const gd_u32x4>(quants)[unit * 64u + lane];
            o[r].s = mq_scales(scales, unit * 16u + col, lg);
            if constexpr (MINIMA) o[r].m = mq_scales(minima, unit * 16u + col, lg);
        }
    };
    // Unit i = tid + 256 k of a chunk of the tokens: row i / 16, values 8 (i % 16) ..; rows past the last token read the
    // last again. Held as loaded, made operands when they are stored.
    constexpr int RAW = TYPE == ROW_F32 ? 2 : 1;
    gd_u32x4 raw[PER][RAW];
    auto fetch = [&](uint32_t c) {
#pragma unroll
        for (uint32_t k = 0; k < PER; ++k) {
            const uint32_t i = tid + 256u * k, row = min(t0 + (i >> 4), n - 1u), at = c * 128u + 8u * (i & 15u);
            const uint64_t p = X + (((uint64_t)row * xs + at) << row_shift(TYPE));
#pragma unroll
            for (int q = 0; q < RAW; ++q) raw[k][q] = gd_u32x4{0u, 0u, 0u, 0u};
            if (at < cols)  // cols is a multiple of 32
#pragma unroll
                for (int q = 0; q < RAW; ++q) raw[k][q] = gd_at<const gd_u32x4_any>(p)[q];
        }
    };
    auto store = [&](uint32_t buffer) {
#pragma unroll
        for (uint32_t k = 0; k < PER; ++k) {
            const uint32_t i = tid + 256u * k, row = i >> 4, at = row * 16u + ((i & 15u) ^ (row & 15u));
            gd_u32x4 *const out = lds + buffer * (UNITS * PARTS) + at;
            if constexpr (TYPE == ROW_F32) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = gd_bits_f32(raw[k][e >> 2][e & 3]);
                mq_planes(v, PARTS, [&](uint32_t p, gd_u32x4 w) { out[p * UNITS] = w; });
            } else {
                out[0] = raw[k][0];
            }
        }
    };

    gd_f32x4 acc[MM_R][T];
#pragma unroll
    for (int r = 0; r < MM_R; ++r)
#pragma unroll
        for (int t = 0; t < T; ++t) acc[r][t] = zero;
    load(0, cur);
    fetch(0);
    store(0);
    for (uint32_t c = 0; c < chunks; ++c) {
        __syncthreads();
        const bool more = c + 1u < chunks;
        if (more) {
            fetch(c + 1u);
            load(c + 1u, next);
        }
#pragma unroll
        for (int r = 0; r < MM_R; ++r) {
            cur[r].s = mq_spread(cur[r].s, spread);
            if constexpr (MINIMA) cur[r].m = mq_spread(cur[r].m, spread);
        }
        const gd_u32x4 *const xl = lds + (c & 1u) * (UNITS * PARTS);
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            __builtin_amdgcn_sched_barrier(0);  // one group at a time: four at once take more registers than there are
            gd_u32x4 x[T][PARTS];
            gd_f32x4 corr[T];
#pragma unroll
            for (int t = 0; t < T; ++t) {
                corr[t] = zero;
#pragma unroll
                for (int p = PARTS - 1; p >= 0; --p) {  // the smallest part first
                    x[t][p] = xl[p * UNITS + (t * 16u + col) * 16u + ((4u * j + h) ^ col)];
                    corr[t] = mm_mfma<HALF>(x[t][p], unbias, corr[t]);
                }
            }
            // A tile's sums are scaled while the next tile's products run.
            gd_f32x4 d[2][T];
            auto scale = [&](int r) {
                const float s = mq_half(cur[r].s, j);
#pragma unroll
                for (int t = 0; t < T; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[r][t][i] += s * d[r & 1][t][i];
                if constexpr (MINIMA) {  // m sum x, corr being -16 sum x
                    const float m = mq_half(cur[r].m, j) * -0.0625f;
#pragma unroll
                    for (int t = 0; t < T; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[r][t][i] += m * corr[t][i];
                }
                // Now, not at the end of the chunk, which would keep the products of all its groups.
#pragma unroll
                for (int t = 0; t < T; ++t) asm volatile("" : "+v"(acc[r][t]));
            };
#pragma unroll
            for (int r = 0; r < MM_R; ++r) {
                uint32_t word = cur[r].w[j];
                asm volatile("" : "+v"(word));  // unpacked here and not all of a chunk ahead
                const gd_u32x4 w = mq_weights<HALF>(word, bits);
#pragma unroll
                for (int t = 0; t < T; ++t) {
                    d[r & 1][t] = corr[t];
#pragma unroll
                    for (int p = PARTS - 1; p >= 0; --p) d[r & 1][t] = mm_mfma<HALF>(x[t][p], w, d[r & 1][t]);
                }
                if (r) scale(r - 1);
                __builtin_amdgcn_sched_barrier(0);
            }
            scale(MM_R - 1);
        }
        if (more) {
            store((c + 1u) & 1u);  // its readers passed the barrier above
#pragma unroll
            for (int r = 0; r < MM_R; ++r) cur[r] = next[r];
        }
    }
    // Sums go out through LDS, 16 tokens at a time, as runs of 64 neighbouring outputs (32 of a gated pair): row r of
    // token k at k * 68 + r (the four tokens of a lane's quarter write to different banks).
    __syncthreads();
    const MqOut y = mq_out(a);
    float *const out = reinterpret_cast<float *>(lds) + wave * (16u * 68u);
    const uint32_t width = y.gated ? 32u : 64u, orow = lane & (width - 1u);
    const uint64_t first = (uint64_t)tile0 * 16u / (64u / width);
#pragma unroll
    for (int t = 0; t < T; ++t) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int r = 0; r < MM_R; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) out[(4u * h + i) * 68u + 16u * r + col] = acc[r][t][i];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (uint32_t k = lane / width; k < 16u; k += 64u / width) {
            const uint32_t token = t0 + 16u * t + k;
            if (token >= n) break;
            if (first + orow >= outputs) continue;
            // A gated pair's rows: 16 of gate, then 16 of up, and so on.
            const float *const at = out + k * 68u + (y.gated ? (orow & 15u) + 32u * (orow >> 4) : orow);
            mq_store(y, token, first + orow, at[0], at[y.gated ? 16 : 0]);
        }
    }
}

template <uint32_t TYPE, bool MINIMA>
__device__ __forceinline__ void mm_q4_body(const GdArgs &a) {
    constexpr int MOST = TYPE == ROW_F32 ? 3 : 4;  // two groups share a CU's LDS and registers
    __shared__ __align__(16) gd_u32x4 lds[2 * 16 * MOST * 16 * (TYPE == ROW_F32 ? 3 : 1)];
    switch (a.c[26]) {
        case 1: return mm_q4_tile<TYPE, MINIMA, 1>(a, lds);
        case 2: return mm_q4_tile<TYPE, MINIMA, 2>(a, lds);
        case 3: return mm_q4_tile<TYPE, MINIMA, 3>(a, lds);
        default: return mm_q4_tile<TYPE, MINIMA, MOST>(a, lds);
    }
}
