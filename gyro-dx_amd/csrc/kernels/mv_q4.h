// Products of up to 16 operand rows with a 4-bit matrix in the layout of q4_repack (q4.h):
//   y[t][r] = act(scale sum_k W[r][k] x[t][k]) (+ y[t][r]),  W = s (q - 8)  or  s q + m  per group of 32, 64, 128
// or, of a gated pair, y[t][r] = scale silu(G[r] . x[t]) (U[r] . x[t]) (+ y[t][r]).
//
// Each bf16 part of a token is an operand row of its own (three of an fp32 token, two of a binary16 one), so 5 fp32, 8
// binary16 or 16 bf16 tokens share a pass over the weights (blockIdx.y: the next tokens). A group of 8 waves takes
// WR = 8 / WK runs of R 16-row tiles, WK waves each a share of the columns; the waves' sums meet in LDS. It keeps
// its tokens' operand rows in LDS and goes on to the next run of rows.
//
// What bounds it: of a large matrix and one pass the weights' bytes (131072 x 2048 Q4_0, one fp32 token: median 34.6 us of
// kernel, 32.1 in a loop, 4.7 TB/s of 151 MB; a large copy moves 5.1). Of a small one the chain of a launch, staging, one
// chunk's loads and the join: 2048 x 512 median 5.2 us, a gated 1024 x 2048 with minima on 3 tokens 8.2. binary16 tokens go as
// two rows each, so that 9 to 16 of them read the weights twice (8192 x 2048 on 32 18.4 us, bf16 12.2). Every
// pass reads and unpacks all weights again: 2048 x 8192 on 128 bf16 tokens, 8 passes, 35 us for a floor of 3.6. The matrix
// unit is busy an eighth of the output head's time, so that fp32 activations as three planes cost nothing; vector
// instructions would need a product and a conversion per value beside the unpacking. Two tiles a wave (R) share its
// reads of the operand rows.
#pragma once
#include "q4.h"

#define MQ_POOL 81920u
#define MQ_WAVES 8u

template <int R, bool MINIMA>
__device__ __forceinline__ void mv_q4_body(const GdArgs &a) {
    __shared__ __align__(16) uint8_t pool[MQ_POOL];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, col = lane & 15u, h = lane >> 4;
    const uint64_t quants = gd_addr(a, 0), scales = gd_addr(a, 2), minima = gd_addr(a, 4);
    const uint32_t tiles = a.c[6], chunks = a.c[7], lg = a.c[8], cols = a.c[9], outputs = a.c[10], gated = a.c[11];
    const uint64_t X = gd_addr(a, 12), xs = gd_addr(a, 14);
    const uint32_t xt = a.c[16], WK = a.c[26], WR = MQ_WAVES / WK;
    const MqOut y = mq_out(a);
    const uint32_t P = xt == ROW_F32 ? 3u : xt == ROW_F16 ? 2u : 1u, per = 16u / P;
    const uint32_t t0 = blockIdx.y * per, nt = min(per, a.c[17] - t0), rows = nt * P;
    const uint32_t ks = __builtin_amdgcn_readfirstlane(wave & (WK - 1u)), rg = __builtin_amdgcn_readfirstlane(wave / WK);

    // LDS: the waves' sums [wave][tile][operand row][16], then the operand rows of one segment of columns, row r's
    // 16-byte unit u at u ^ (r % 16) (the 16 rows of a read spread over the banks).
    float *red = reinterpret_cast<float *>(pool);
    const uint32_t red_bytes = MQ_WAVES * R * rows * 64u;
    gd_u32x4 *xl = reinterpret_cast<gd_u32x4 *>(pool + red_bytes);
    const uint32_t most = (MQ_POOL - red_bytes) / (rows * 256u);               // chunks that LDS holds
    const uint32_t seg = most >= chunks ? chunks : most & ~(MQ_WAVES - 1u);    // chunks per segment, in whole rounds
    const uint32_t units = seg * 16u;                                          // 16-byte units per operand row
    const uint32_t arow = min(col, rows - 1u);

    const MqSpread spread = mq_spread(lg);
    const MqBits bits = mq_bits<false>();
    const float bias = MINIMA ? -16.f : -24.f;
    const uint32_t b16 = gd_f32_bits(bias) >> 16, b32 = b16 | b16 << 16;
    const gd_bf16x8 unbias = __builtin_bit_cast(gd_bf16x8, gd_u32x4{b32, b32, b32, b32});
    const uint32_t runs = (tiles + R * WR - 1u) / (R * WR);

    // Chunk c of the tiles of a run; tiles past the last read the last again, and their sums are dropped.
    auto load = [&](uint32_t run, uint32_t c, MqChunk (&o)[R]) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const uint64_t unit = (uint64_t)min((run * WR + rg) * R + r, tiles - 1u) * chunks + c;
            o[r].w = gd_load<gd_u32x4>(quants + unit * 1024u, lane * 16u);
            o[r].s = mq_scales(scales + (unit << (12u - lg)), col, lg);
            if constexpr (MINIMA) o[r].m = mq_scales(minima + (unit << (12u - lg)), col, lg);
        }
    };
    // The next chunk of this wave, of this run or the next, is in flight while one is multiplied; the first while
    // the tokens are staged.
    MqChunk cur[R];
    load(blockIdx.x, ks, cur);
    bool staged = false;
    for (uint32_t run = blockIdx.x; run < runs; run += gridDim.x) {
        gd_f32x4 acc[R];
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r] = gd_f32x4{0.f, 0.f, 0.f, 0.f};
        uint32_t c = ks;
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
            for (; c < c1; c += WK) {
                MqChunk next[R];
                if (c + WK < chunks) load(run, c + WK, next);
                else if (run + gridDim.x < runs) load(run + gridDim.x, ks, next);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    cur[r].s = mq_spread(cur[r].s, spread);
                    if constexpr (MINIMA) cur[r].m = mq_spread(cur[r].m, spread);
                }
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) {
                    const uint32_t u = (c - c0) * 16u + 4u * j + h;
                    const gd_bf16x8 x = __builtin_bit_cast(gd_bf16x8, xl[arow * units + (u ^ (arow & 15u))]);
                    const gd_f32x4 corr =
                        __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, unbias, gd_f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const gd_f32x4 d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            x, __builtin_bit_cast(gd_bf16x8, mq_weights<false>(cur[r].w[j], bits)), corr, 0, 0, 0);
                        const float s = mq_half(cur[r].s, j);
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[r][i] += s * d[i];
                        if constexpr (MINIMA) {  // m sum x, corr being -16 sum x
                            const float m = mq_half(cur[r].m, j) * -0.0625f;
#pragma unroll
                            for (int i = 0; i < 4; ++i) acc[r][i] += m * corr[i];
                        }
                    }
                }
#pragma unroll
                for (int r = 0; r < R; ++r) cur[r] = next[r];
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
            mq_store(y, t0 + t, out, sum[0], sum[1]);
        }
    }
}
