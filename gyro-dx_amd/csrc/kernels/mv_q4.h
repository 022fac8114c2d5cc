// Products of up to 16 operand rows with a 4-bit matrix in the layout of q4_repack:
//   y[t][r] = act(scale sum_k W[r][k] x[t][k]) (+ y[t][r]),  W = s (q - 8)  or  s q + m  per group of 32, 64, 128
// or, of a gated pair, y[t][r] = scale silu(G[r] . x[t]) (U[r] . x[t]) (+ y[t][r]).
//
// The products run on v_mfma_f32_16x16x32_bf16 with the token rows as the A operand and 16 weight rows as B. A
// 4-bit value becomes a bf16 in half an instruction: its bits are or-ed into the top of the mantissa of 16, which
// gives 16 + q exactly. Those extra 16 (24 where W = s (q - 8)) times the group's sum of activations
// go in as the product's C operand, itself the product of the activations with a constant matrix, so nothing of the
// group's sum is kept apart, and it is at most five times what the group's own product rounds at. Group sums are
// scaled and added in fp32. Activations are exact: an fp32 value is the sum of three bf16 values (its 24 bits cut in
// eights), a binary16 one of two, each an operand row of its own, so 5 fp32, 8 binary16 or 16 bf16 tokens share a
// pass over the weights (blockIdx.y: the next tokens). A token with an infinity or NaN gets NaN in every output.
//
// A group of 8 waves takes WR = 8 / WK runs of R 16-row tiles, WK waves each a share of the columns; the
// waves' sums meet in LDS. It keeps its tokens' operand rows in LDS and goes on to the next run of rows.
// Constants: 0 quants 2 scales 4 minima (0: none) 6 tiles 7 chunks 8 log2(group) 9 cols 10 outputs per token
// 11 gated pair 12 x 14 x stride 16 x type 17 tokens 18 y 20 y stride 22 y type 23 act (0 none, 1 silu, 2
// sigmoid) 24 add to y 25 scale (fp32 bits) 26 WK. Addresses and strides have 64 bits; strides count values.
#pragma once
#include "rows.h"

#define MQ_POOL 81920u
#define MQ_WAVES 8u

// Values 0 .. 7 of a word (q4_repack) as 16 + q in bf16.
__device__ __forceinline__ gd_bf16x8 mq_weights(uint32_t w) {
    const uint32_t mask = 0x00780078u, one = 0x41804180u;
    gd_u32x4 v;
    v[0] = (w & mask) | one;
    v[1] = ((w >> 4) & mask) | one;
    v[2] = ((w >> 8) & mask) | one;
    v[3] = (__builtin_amdgcn_alignbit(w, w, 12) & mask) | one;
    return __builtin_bit_cast(gd_bf16x8, v);
}

// The bf16 rows that sum to the 8 values v, planes 0 .. P - 1, by truncation (each remainder is exact).
template <typename F>
__device__ __forceinline__ void mq_planes(const float (&v)[8], uint32_t P, F &&put) {
    float rest[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) rest[j] = v[j];
    for (uint32_t p = 0; p < P; ++p) {
        gd_u32x4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t lo = gd_f32_bits(rest[2 * j]) & 0xffff0000u, hi = gd_f32_bits(rest[2 * j + 1]) & 0xffff0000u;
            rest[2 * j] -= gd_bits_f32(lo);
            rest[2 * j + 1] -= gd_bits_f32(hi);
            w[j] = (lo >> 16) | hi;
        }
        put(p, w);
    }
}

template <int R>
__device__ __forceinline__ void mv_q4_body(const GdArgs &a) {
    __shared__ __align__(16) uint8_t pool[MQ_POOL];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, col = lane & 15u, h = lane >> 4;
    const uint64_t quants = gd_addr(a, 0), scales = gd_addr(a, 2), minima = gd_addr(a, 4);
    const uint32_t tiles = a.c[6], chunks = a.c[7], lg = a.c[8], cols = a.c[9], outputs = a.c[10], gated = a.c[11];
    const uint64_t X = gd_addr(a, 12), xs = gd_addr(a, 14), Y = gd_addr(a, 18), ys = gd_addr(a, 20);
    const uint32_t xt = a.c[16], yt = a.c[22], act = a.c[23], add = a.c[24], WK = a.c[26], WR = MQ_WAVES / WK;
    const float scale = gd_bits_f32(a.c[25]);
    const uint32_t P = xt == ROW_F32 ? 3u : xt == ROW_F16 ? 2u : 1u, per = 16u / P;
    const uint32_t t0 = blockIdx.y * per, nt = min(per, a.c[17] - t0), rows = nt * P;
    const uint32_t ks = wave & (WK - 1u), rg = wave / WK;

    // LDS: the waves' sums [wave][tile][operand row][16], then the operand rows of one segment of columns, row r's
    // 16-byte unit u at u ^ (r % 16) (the 16 rows of a read spread over the banks).
    float *red = reinterpret_cast<float *>(pool);
    const uint32_t red_bytes = MQ_WAVES * R * rows * 64u;
    gd_u32x4 *xl = reinterpret_cast<gd_u32x4 *>(pool + red_bytes);
    const uint32_t seg = min(chunks, (MQ_POOL - red_bytes) / (rows * 256u));  // chunks per segment
    const uint32_t units = seg * 16u;                                          // 16-byte units per operand row
    const uint32_t arow = min(col, rows - 1u);

    const float bias = minima ? -16.f : -24.f;
    const uint32_t b16 = gd_f32_bits(bias) >> 16, b32 = b16 | b16 << 16;
    const gd_bf16x8 unbias = __builtin_bit_cast(gd_bf16x8, gd_u32x4{b32, b32, b32, b32});
    const uint32_t runs = (tiles + R * WR - 1u) / (R * WR), gps = 128u >> lg;
    bool staged = false;

    for (uint32_t run = blockIdx.x; run < runs; run += gridDim.x) {
        const uint32_t tile0 = (run * WR + rg) * R;
        gd_f32x4 acc[R];
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r] = gd_f32x4{0.f, 0.f, 0.f, 0.f};
        for (uint32_t c0 = 0; c0 < chunks; c0 += seg) {
            if (!staged || seg < chunks) {
                __syncthreads();
                for (uint32_t i = tid; i < nt * units; i += 64u * MQ_WAVES) {
                    const uint32_t t = i / units, u = i - t * units;
                    float v[8];
                    row_load8(X + (((uint64_t)(t0 + t) * xs) << row_shift(xt)), c0 * 128u + u * 8u, cols, xt, v);
                    mq_planes(v, P, [&](uint32_t p, gd_u32x4 w) {
                        const uint32_t r = t * P + p;
                        xl[r * units + (u ^ (r & 15u))] = w;
                    });
                }
                __syncthreads();
                staged = true;
            }
            const uint32_t c1 = min(c0 + seg, chunks);
            for (uint32_t c = c0 + ks; c < c1; c += WK) {
                gd_u32x4 w[R];
                uint32_t s2[R][2], m2[R][2];
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    // Tiles past the last read the last again; their sums are dropped.
                    const uint64_t unit = (uint64_t)min(tile0 + r, tiles - 1u) * chunks + c;
                    w[r] = gd_at<const gd_u32x4>(quants)[unit * 64u + lane];
                    const uint64_t so = (unit * 16u + col) * gps;
                    s2[r][0] = s2[r][1] = m2[r][0] = m2[r][1] = 0;
                    if (lg == 5u) {
                        s2[r][0] = gd_at<const uint32_t>(scales + 2u * so)[0];
                        s2[r][1] = gd_at<const uint32_t>(scales + 2u * so)[1];
                        if (minima) {
                            m2[r][0] = gd_at<const uint32_t>(minima + 2u * so)[0];
                            m2[r][1] = gd_at<const uint32_t>(minima + 2u * so)[1];
                        }
                    } else if (lg == 6u) {
                        s2[r][0] = gd_at<const uint32_t>(scales + 2u * so)[0];
                        if (minima) m2[r][0] = gd_at<const uint32_t>(minima + 2u * so)[0];
                    } else {
                        s2[r][0] = gd_at<const uint16_t>(scales + 2u * so)[0];
                        if (minima) m2[r][0] = gd_at<const uint16_t>(minima + 2u * so)[0];
                    }
                }
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) {
                    const uint32_t u = (c - c0) * 16u + 4u * j + h;
                    const gd_bf16x8 x = __builtin_bit_cast(gd_bf16x8, xl[arow * units + (u ^ (arow & 15u))]);
                    const gd_f32x4 corr =
                        __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, unbias, gd_f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
                    const uint32_t g = j >> (lg - 5u);
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const gd_f32x4 d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, mq_weights(w[r][j]), corr, 0, 0, 0);
                        const float s = gd_half((g & 2u ? s2[r][1] : s2[r][0]) >> (g & 1u ? 16 : 0) & 0xffffu);
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[r][i] += s * d[i];
                        if (minima) {  // m sum x, corr being -16 sum x
                            const float m = gd_half((g & 2u ? m2[r][1] : m2[r][0]) >> (g & 1u ? 16 : 0) & 0xffffu) * -0.0625f;
#pragma unroll
                            for (int i = 0; i < 4; ++i) acc[r][i] += m * corr[i];
                        }
                    }
                }
            }
        }
        __syncthreads();  // the sums of the run before are read
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
                if (4u * h + i < rows) red[((wave * R + r) * rows + 4u * h + i) * 16u + col] = acc[r][i];
        __syncthreads();
        const uint32_t halves = gated ? 2u : 1u, width = WR * R * 16u / halves;  // outputs per token of this run
        for (uint32_t i = tid; i < nt * width; i += 64u * MQ_WAVES) {
            const uint32_t t = i / width, o = i - t * width;
            const uint64_t out = (uint64_t)run * width + o;
            if (out >= outputs) continue;
            const uint32_t tile = (o >> 4) * halves, orow = o & 15u;
            float sum[2] = {0.f, 0.f};
#pragma unroll
            for (uint32_t half = 0; half < 2; ++half) {
                if (half >= halves) break;
                const uint32_t g = (tile + half) / R, r = (tile + half) - g * R;
                for (uint32_t p = P; p-- > 0;)  // the smallest part first
                    for (uint32_t k = 0; k < WK; ++k)
                        sum[half] += red[(((g * WK + k) * R + r) * rows + t * P + p) * 16u + orow];
            }
            float v;
            if (gated) {
                v = scale * (gd_silu_accurate(sum[0]) * sum[1]);
            } else {
                v = scale * sum[0];
                if (act == 1u) v = gd_silu_accurate(v);
                else if (act == 2u) v = gd_sigmoid_accurate(v);
            }
            const uint64_t at = (uint64_t)(t0 + t) * ys + out;
            if (add) v += row_load(Y, at, yt);
            row_store(Y, at, yt, v);
        }
    }
}
