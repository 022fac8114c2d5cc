// Products of many tokens with a 4-bit matrix in the layout of q4_repack (q4.h).
//
// A group of four waves takes 16 tiles (256 weight rows), four to a wave, and 16 T tokens. Chunks of 128 columns of the
// tokens go through LDS as operands, two buffers in turn, one being filled while the other is multiplied; weights
// go from memory to registers, one or two chunks ahead. Of 32 columns a wave unpacks 4 operands, each used for T products
// of 16 + q; where two groups of 32 share a scale their products add up in the matrix unit before they are scaled into
// the sums, 16 T (or 8 T) vector instructions per 32 columns beside 28 for unpacking. What the 16 is too much starts
// each sum, as in mv_q4, so that sums are rounded at their own size. Minima times the chunk's four sums of 32 activations,
// which come with the staging, are a product of their own, in fp32 on v_mfma_f32_16x16x4_f32. bf16 and binary16 tokens
// are operands as they are; fp32 ones go through the products three times, a part each.
//
// What bounds it: dependent results at two waves a SIMD, which is what registers (208 to 256) and LDS hold. 8192 x 2048 on
// 1023 bf16 tokens takes 56 to 60 us with groups of 32 (570 TFLOP/s) and 51 with groups of 128 (670), half of a large matrix
// product's 1200; in fp32 111 to 118 us (300), of which three products of each operand explain 86. Of a gated 4096 x 2048
// in groups of 64 with minima on 1023 binary16 tokens (58 to 66 us, box to box) neither unit is full: the matrix unit is busy
// 36% of the cycles (two fifths of that corrections and minima), the vector unit 41%. Fewer tokens are bound by the chain
// of a chunk (load, store to LDS, barrier, products: 1.1 us), which one group goes through for all columns however few
// tokens there are: 8192 x 2048 on 64 bf16 tokens 18 us, 2048 x 2048 on 512 19, five to eight times their floors.
// 391 groups that do not divide among 256 units add a quarter at most (100003 x 2560 on 37 tokens: 49 to 55 us, 2.8 TB/s).
// Groups that start at different chunks gained nothing, nor did minima as exact bf16 parts in one 16x16x32 product, half
// the matrix cycles.
#pragma once
#include "q4.h"

#define MM_WAVES 4u
#define MM_R 4

typedef _Float16 gd_f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 gd_f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 gd_bf16x2 __attribute__((ext_vector_type(2)));

// c + a b of token operand a and weight operand b, both of the operand type.
template <bool HALF>
__device__ __forceinline__ gd_f32x4 mm_mfma(gd_u32x4 a, gd_u32x4 b, gd_f32x4 c) {
    if constexpr (HALF)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(gd_f16x8, a), __builtin_bit_cast(gd_f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(gd_bf16x8, a), __builtin_bit_cast(gd_bf16x8, b), c, 0, 0, 0);
}
// c + both values of a word of 16-bit tokens.
template <bool HALF>
__device__ __forceinline__ float mm_pair(uint32_t w, float c) {
    if constexpr (HALF)
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(gd_f16x2, w), gd_f16x2{(_Float16)1.f, (_Float16)1.f}, c, false);
    else
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(gd_bf16x2, w), gd_bf16x2{(__bf16)1.f, (__bf16)1.f}, c, false);
}
template <int CTRL>
__device__ __forceinline__ float mm_dpp(float v) {
    return gd_bits_f32((uint32_t)__builtin_amdgcn_update_dpp(0, (int)gd_f32_bits(v), CTRL, 0xf, 0xf, true));
}

// A chunk of a tile as a lane holds it: its 16 bytes, its row's 4 / SPAN scales, binary16 in order, and the minimum of
// group lane / 16 of 32 (where there are minima).
template <int SPAN>
struct MmChunk {
    gd_u32x4 w;
    uint32_t s[SPAN == 1 ? 2 : 1], m;
};
template <int SPAN>
__device__ __forceinline__ void mm_scales(uint64_t base, uint32_t row, uint32_t (&o)[SPAN == 1 ? 2 : 1]) {
    if constexpr (SPAN == 1) {
        const gd_u32x2 v = gd_load<gd_u32x2>(base, row * 8u);
        o[0] = v[0];
        o[1] = v[1];
    } else if constexpr (SPAN == 2) {
        o[0] = gd_load<uint32_t>(base, row * 4u);
    } else {
        o[0] = gd_load<uint16_t>(base, row * 2u);
    }
}

// Asks the scheduler for `others` vector instructions spread between `products` matrix ones.
template <int PRODUCTS, int OTHERS>
__device__ __forceinline__ void mm_interleave() {
#pragma unroll
    for (int t = 0; t < PRODUCTS; ++t) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, (OTHERS + PRODUCTS - 1) / PRODUCTS, 0);
    }
}

template <uint32_t TYPE, int SPAN, int T>
__device__ __forceinline__ void mm_q4_tile(const GdArgs &a, gd_u32x4 *lds, float *sums) {
    constexpr bool HALF = TYPE == ROW_F16;
    constexpr int PARTS = TYPE == ROW_F32 ? 3 : 1;
    // Groups of 32 that are scaled together (fp32 tokens' operands leave no registers for a second one's).
    constexpr uint32_t PAIR = SPAN == 1 || PARTS > 1 ? 1u : 2u;
    constexpr uint32_t ROWS = 16u * T, UNITS = ROWS * 16u, PER = UNITS / 256u;  // 16-byte units of a chunk, of a thread
    constexpr uint32_t SUMS = ROWS + 16u;  // a group's row of sums, the four groups' in different banks
    const uint32_t tid = threadIdx.x, lane = tid & 63u, col = lane & 15u, h = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint64_t quants = gd_addr(a, 0), scales = gd_addr(a, 2), minima = gd_addr(a, 4);
    const uint32_t tiles = a.c[6], chunks = a.c[7], cols = a.c[9], outputs = a.c[10], n = a.c[17];
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
    const MqBits bits = mq_bits<HALF>();
    // What the products' 16 is too much, and the 8 of weights without a minimum, as an operand of its own.
    const uint32_t bias = HALF ? (minima ? 0xcc00u : 0xce00u) : (minima ? 0xc180u : 0xc1c0u), bias2 = bias | bias << 16;  // -16, -24
    const gd_u32x4 unbias = {bias2, bias2, bias2, bias2};
    const gd_f32x4 zero = {0.f, 0.f, 0.f, 0.f};

    // Chunks asked for ahead: two where few tokens leave the registers and a chunk's products are shorter than a load takes (us
    // with one / two: 32768 x 2048 on 32 tokens 22.4 / 18.2, 131072 x 2048 on 12 fp32 tokens 48.5 / 43.2 and on 48 bf16 ones
    // 54.2 / 51.5, but 51.7 / 54.8 for 48 tokens a group of 100003 x 2560 in groups of 64).
    constexpr int AHEAD = T <= (PARTS > 1 ? 1 : SPAN == 4 ? 3 : 2) ? 2 : 1;
    MmChunk<SPAN> held[AHEAD + 1][MM_R];
    auto load = [&](uint32_t c, MmChunk<SPAN> (&o)[MM_R]) {
#pragma unroll
        for (int r = 0; r < MM_R; ++r) {
            // Tiles past the last read the last again; their sums are dropped.
            const uint64_t unit = (uint64_t)min(tile0 + r, tiles - 1u) * chunks + c;
            o[r].w = gd_load<gd_u32x4>(quants + unit * 1024u, lane * 16u);
            mm_scales<SPAN>(scales + unit * (128u / SPAN), col, o[r].s);
            if (minima) o[r].m = gd_load<uint16_t>(minima + unit * (128u / SPAN), (col * (4u / SPAN) + h / SPAN) * 2u);
        }
    };
    // Unit i = tid + 256 k of a chunk of the tokens: row i / 16, values 8 (i % 16) ..; rows past the last token read the
    // last again, columns past the last are zeros. Held as loaded, made operands when they are stored. A row is at most
    // 2^24 values after the one before, so that a tile's 64 are within 32 bits of its first.
    constexpr int RAW = TYPE == ROW_F32 ? 2 : 1;
    gd_u32x4 raws[AHEAD == 1 ? 1 : 3][PER][RAW];
    uint32_t from[PER];
#pragma unroll
    for (uint32_t k = 0; k < PER; ++k) {
        const uint32_t i = tid + 256u * k, row = min(i >> 4, n - 1u - t0);
        from[k] = (row * (uint32_t)xs + 8u * (i & 15u)) << row_shift(TYPE);
    }
    const uint64_t X0 = X + (((uint64_t)t0 * xs) << row_shift(TYPE));
    auto fetch = [&](uint32_t c, gd_u32x4 (&raw)[PER][RAW]) {
        const uint64_t base = X0 + ((uint64_t)(c * 128u) << row_shift(TYPE));
        const uint32_t left = cols - c * 128u;
        // (Where chunks are asked for two ahead, no branch may make their number uncertain: the last one's missing columns
        // read its first, and store() drops them.)
        const uint32_t back = AHEAD > 1 && 8u * (tid & 15u) >= left ? (8u * (tid & 15u)) << row_shift(TYPE) : 0u;
        if (AHEAD > 1 || left >= 128u) {
#pragma unroll
            for (uint32_t k = 0; k < PER; ++k)
#pragma unroll
                for (int q = 0; q < RAW; ++q) raw[k][q] = gd_load<gd_u32x4_any>(base, from[k] - back + 16u * q);
        } else {
#pragma unroll
            for (uint32_t k = 0; k < PER; ++k)
#pragma unroll
                for (int q = 0; q < RAW; ++q) {
                    raw[k][q] = gd_u32x4{0u, 0u, 0u, 0u};
                    if (8u * (tid & 15u) < left) raw[k][q] = gd_load<gd_u32x4_any>(base, from[k] + 16u * q);
                }
        }
    };
    auto store = [&](uint32_t c, gd_u32x4 (&raw)[PER][RAW]) {
        const uint32_t buffer = c & 1u;
        if (AHEAD > 1 && 8u * (tid & 15u) >= cols - c * 128u) {
#pragma unroll
            for (uint32_t k = 0; k < PER; ++k)
#pragma unroll
                for (int q = 0; q < RAW; ++q) raw[k][q] = gd_u32x4{0u, 0u, 0u, 0u};
        }
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
        if (!minima) return;
#pragma unroll
        for (uint32_t k = 0; k < PER; ++k) {
            const uint32_t i = tid + 256u * k;
            float sum = 0.f;
            if constexpr (TYPE == ROW_F32) {
#pragma unroll
                for (int e = 0; e < 8; ++e) sum += gd_bits_f32(raw[k][e >> 2][e & 3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) sum = mm_pair<HALF>(raw[k][0][e], sum);
            }
            sum += mm_dpp<0xb1>(sum);  // lanes ^ 1
            sum += mm_dpp<0x4e>(sum);  // lanes ^ 2: the group's four units
            if ((i & 3u) == 0u) sums[(buffer * 4u + ((i & 15u) >> 2)) * SUMS + (i >> 4)] = sum;
        }
    };

    gd_f32x4 acc[MM_R][T];
#pragma unroll
    for (int r = 0; r < MM_R; ++r)
#pragma unroll
        for (int t = 0; t < T; ++t) acc[r][t] = zero;
    load(0, held[0]);
    fetch(0, raws[0]);
    store(0, raws[0]);
    const uint32_t last = chunks - 1u;
    if constexpr (AHEAD > 1) {
        fetch(min(1u, last), raws[1]);
        load(min(1u, last), held[1]);
    }
    // The products of chunk c.
    auto multiply = [&](uint32_t c, MmChunk<SPAN> (&cur)[MM_R]) {
        const uint32_t buffer = c & 1u;
        const gd_u32x4 *const xl = lds + buffer * (UNITS * PARTS);
        gd_u32x4 x[PAIR][T][PARTS];
        auto operand = [&](uint32_t j, int t) {
#pragma unroll
            for (int p = 0; p < PARTS; ++p) x[j % PAIR][t][p] = xl[p * UNITS + (t * 16u + col) * 16u + ((4u * j + h) ^ col)];
        };
#pragma unroll
        for (uint32_t j = 0; j < PAIR; ++j)
#pragma unroll
            for (int t = 0; t < T; ++t) operand(j, t);
        if (minima) {
#pragma unroll
            for (int t = 0; t < T; ++t) {
                const float sum = sums[(buffer * 4u + h) * SUMS + t * 16u + col];
#pragma unroll
                for (int r = 0; r < MM_R; ++r)
                    acc[r][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(sum, gd_half(cur[r].m), acc[r][t], 0, 0, 0);
            }
        }
        gd_f32x4 corr[T];
        auto correct = [&](int t) {
            corr[t] = zero;
#pragma unroll
            for (uint32_t e = 0; e < PAIR; ++e)
#pragma unroll
                for (int p = PARTS - 1; p >= 0; --p) corr[t] = mm_mfma<HALF>(x[e][t][p], unbias, corr[t]);
        };
        // A step is a tile's products with 32 columns; a tile takes PAIR of them, whose sums are scaled together, before
        // the next tile. Beside a step run the unpacking of the next one's weights, the scaling of the tile before and,
        // in the last tile's, the reads of the next operands; the empty asm statements and the barriers keep each where
        // it is written, the group barriers between the products.
        gd_f32x4 d[2][T];
        auto scale = [&](int r, uint32_t j) {
            const uint32_t g = j / SPAN;
            const float s = gd_half(cur[r].s[g >> 1] >> (16u * (g & 1u)) & 0xffffu);
#pragma unroll
            for (int t = 0; t < T; ++t) {
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[r][t][i] += s * d[r & 1][t][i];
                asm volatile("" : "+v"(acc[r][t]));
            }
        };
        gd_u32x4 w = mq_weights<HALF>(cur[0].w[0], bits);
#pragma unroll
        for (uint32_t k = 0; k < 4u * MM_R; ++k) {
            const uint32_t g = k / (PAIR * MM_R), r = k / PAIR % MM_R, e = k % PAIR, j = g * PAIR + e;
            const uint32_t gn = (k + 1u) / (PAIR * MM_R), rn = (k + 1u) / PAIR % MM_R, jn = gn * PAIR + (k + 1u) % PAIR;
            gd_u32x4 wn = w;
            if (r == 0 && e == 0)
#pragma unroll
                for (int t = 0; t < T; ++t) correct(t);
            if (jn < 4u) {
                asm volatile("" : "+v"(cur[rn].w));
                wn = mq_weights<HALF>(cur[rn].w[jn], bits);
            }
#pragma unroll
            for (int t = 0; t < T; ++t) {
                gd_f32x4 v = e ? d[r & 1][t] : corr[t];
#pragma unroll
                for (int p = 0; p < PARTS; ++p) v = mm_mfma<HALF>(x[e][t][p], w, v);  // the largest part first: it takes the correction away
                d[r & 1][t] = v;
                if (r == MM_R - 1 && j + PAIR < 4u) operand(j + PAIR, t);
            }
            if (jn < 4u) asm volatile("" : "+v"(wn));
            const bool scales_one = e == 0 && k;
            if (scales_one) scale(r ? r - 1 : MM_R - 1, r ? j : j - 1u);
            w = wn;
            if (scales_one) mm_interleave<T * PARTS, 8 + 4 * T>();
            else mm_interleave<T * PARTS, 8>();
            __builtin_amdgcn_sched_barrier(0);
        }
        scale(MM_R - 1, 3u);
    };
    if constexpr (AHEAD > 1) {
        // Three sets of registers in turn: a copy of what is on its way would wait for it.
        auto step = [&](uint32_t c, MmChunk<SPAN> (&cur)[MM_R], MmChunk<SPAN> (&second)[MM_R], gd_u32x4 (&raw)[PER][RAW],
                        gd_u32x4 (&raw2)[PER][RAW]) {
            __syncthreads();
            fetch(min(c + 2u, last), raw2);
            load(min(c + 2u, last), second);
            multiply(c, cur);
            if (c < last) store(c + 1u, raw);  // its buffer's readers passed the barrier above
        };
#pragma unroll 1
        for (uint32_t c = 0;; c += 3u) {
            step(c, held[0], held[2], raws[1], raws[2]);
            if (c + 1u > last) break;
            step(c + 1u, held[1], held[0], raws[2], raws[0]);
            if (c + 2u > last) break;
            step(c + 2u, held[2], held[1], raws[0], raws[1]);
            if (c + 3u > last) break;
        }
    } else {
        for (uint32_t c = 0; c < chunks; ++c) {
            __syncthreads();
            if (c < last) {
                fetch(c + 1u, raws[0]);
                load(c + 1u, held[1]);
            }
            multiply(c, held[0]);
            if (c < last) {
                store(c + 1u, raws[0]);  // its buffer's readers passed the barrier above
#pragma unroll
                for (int r = 0; r < MM_R; ++r) held[0][r] = held[1][r];
            }
        }
    }
    // Sums go out through LDS as runs of 64 neighbouring outputs (32 of a gated pair), four to a lane: row r of token k at
    // k * 68 + r (the four tokens of a lane's quarter write to different banks).
    __syncthreads();
    float *const out = reinterpret_cast<float *>(lds) + wave * (ROWS * 68u);
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
        for (int r = 0; r < MM_R; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) out[(16u * t + 4u * h + i) * 68u + 16u * r + col] = acc[r][t][i];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const MqOut y = mq_out(a);
    const uint32_t lanes = y.gated ? 8u : 16u, o4 = (lane & (lanes - 1u)) * 4u;  // lanes of a token's run
    const uint64_t first = (uint64_t)tile0 * 16u / (y.gated ? 2u : 1u) + o4;
    if (first >= outputs) return;
    const uint32_t count = (uint32_t)min((uint64_t)outputs - first, (uint64_t)4u);
    // A gated pair's rows: 16 of gate, then 16 of up, and so on.
    const float *const mine = out + (y.gated ? (o4 & 15u) + 32u * (o4 >> 4) : o4);
#pragma unroll 1
    for (uint32_t k = lane / lanes; k < min(ROWS, n - t0); k += 64u / lanes) {
        const gd_f32x4 v = *reinterpret_cast<const gd_f32x4 *>(mine + k * 68u);
        const gd_f32x4 up = *reinterpret_cast<const gd_f32x4 *>(mine + k * 68u + (y.gated ? 16 : 0));
        mq_store4(y, t0 + k, first, count, v, up);
    }
}

template <uint32_t TYPE, int SPAN>
__device__ __forceinline__ void mm_q4_body(const GdArgs &a) {
    // Two groups share a CU's registers and LDS: two buffers of a chunk's operands, then the sums of four waves.
    constexpr int MOST = TYPE == ROW_F32 ? (SPAN == 1 ? 2 : 3) : 4;
    constexpr uint32_t OPERANDS = 2 * 16 * MOST * 16 * (TYPE == ROW_F32 ? 3 : 1), OUT = MM_WAVES * 16 * MOST * 68 / 4;
    __shared__ __align__(16) gd_u32x4 lds[OPERANDS > OUT ? OPERANDS : OUT];
    __shared__ float sums[2 * 4 * (16 * MOST + 16)];
    switch (a.c[26]) {
        case 1: return mm_q4_tile<TYPE, SPAN, 1>(a, lds, sums);
        case 2: return mm_q4_tile<TYPE, SPAN, 2>(a, lds, sums);
        case 3: return mm_q4_tile<TYPE, SPAN, MOST < 3 ? MOST : 3>(a, lds, sums);
        default: return mm_q4_tile<TYPE, SPAN, MOST>(a, lds, sums);
    }
}
