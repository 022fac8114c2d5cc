// 4-bit rows into the order that mv_q4 reads: 16-row tiles by 128-column chunks of 1024 bytes, chunk c of
// tile t at (t chunks + c) 1024. Lane l of a wave reads 16 bytes of a chunk: the values of row l % 16 in
// columns 32 j + 8 (l / 16) + 0 .. 7 as word j (0 .. 3), its operand of one 16x16x32 product with group j.
// In a word, value 2 p is at bit 3 + 4 p and value 2 p + 1 sixteen bits on (mod 32), so that
// rotate(word, 4 p) & 0x00780078 holds values 2 p and 2 p + 1 as the top mantissa bits of two bf16. The
// scales follow, [tile][chunk][row][128 / group] binary16, then the minima in the same order. Rows past
// the last and columns past the last (a chunk that is not full) are zeros with scale zero.
//
// A gated pair interleaves its matrices by tiles: gate rows 16 t .. in tile 2 t, up rows in tile 2 t + 1.
//
// Source (kind): 0 GGUF Q4_0 (18-byte blocks: binary16 scale, 16 bytes whose low bits hold values 0 .. 15
// and high bits 16 .. 31), 1 Q4_1 (20 bytes: scale, minimum, as before), 2 arrays: quants [rows][cols / 2]
// with value 2 i in byte i's low bits, scales and minima [rows][cols / group] binary16.
// One thread per 16 output bytes, which reads its bytes one by one: 0.5 ms for 131072 x 2048 Q4_0 (151 MB in, as much out),
// beside 4 ms for the upload before it. Constants: 0 kind 1 rows 2 cols 3 chunks 4 log2(group) 5 tiles 6 tile step
// (2 in a gated pair) 7 first tile 8 quants 10 scales 12 minima (0: none) 14 output quants 16 output scales
// 18 output minima (64-bit addresses). 32-bit thread index: tiles * chunks * 64 < 2^32.
#include "rows.h"

GD_PIPELINE_NAMED(q4_repack, 256) {
    const uint32_t kind = a.c[0], rows = a.c[1], cols = a.c[2], chunks = a.c[3], lg = a.c[4], tiles = a.c[5];
    const uint64_t index = ((uint64_t)blockIdx.y * gridDim.x + blockIdx.x) * 256u + threadIdx.x;
    if (index >= (uint64_t)tiles * chunks * 64u) return;
    const uint32_t lane = (uint32_t)(index & 63u);
    const uint32_t unit = (uint32_t)(index >> 6), t = unit / chunks, c = unit - t * chunks;
    const uint32_t row = t * 16u + (lane & 15u), h = lane >> 4;
    const uint64_t out = (uint64_t)(t * a.c[6] + a.c[7]) * chunks + c;
    const auto quants = gd_at<const uint8_t>(gd_addr(a, 8));
    const uint32_t block = kind == 0u ? 18u : 20u, head = kind == 0u ? 2u : 4u;
    gd_u32x4 w;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
        uint32_t word = 0;
        const uint32_t k = c * 128u + 32u * j + 8u * h;
        if (row < rows && k < cols) {
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) {
                uint32_t q;
                if (kind == 2u) {
                    const uint32_t b = quants[(uint64_t)row * (cols / 2u) + (k + e) / 2u];
                    q = e & 1u ? b >> 4 : b & 15u;
                } else {
                    const uint32_t i = (8u * h + e) & 15u;
                    const uint32_t b = quants[((uint64_t)row * (cols / 32u) + k / 32u) * block + head + i];
                    q = h >= 2u ? b >> 4 : b & 15u;
                }
                const uint32_t at = (3u + 4u * (e >> 1) + 16u * (e & 1u)) & 31u;
                word |= at == 31u ? (q << 31) | (q >> 1) : q << at;
            }
        }
        w[j] = word;
    }
    gd_at<gd_u32x4>(gd_addr(a, 14))[out * 64u + lane] = w;
    if (h != 0) return;
    const uint32_t per = 128u >> lg;
    for (uint32_t g = 0; g < per; ++g) {
        const uint32_t k = c * 128u + (g << lg);
        uint32_t s = 0, m = 0;
        if (row < rows && k < cols) {
            if (kind == 2u) {
                const uint64_t i = (uint64_t)row * (cols >> lg) + (k >> lg);
                s = gd_at<const uint16_t>(gd_addr(a, 10))[i];
                if (gd_addr(a, 12)) m = gd_at<const uint16_t>(gd_addr(a, 12))[i];
            } else {
                const uint64_t i = (((uint64_t)row * (cols / 32u) + k / 32u) * block) / 2u;
                s = gd_at<const uint16_t>(gd_addr(a, 8))[i];
                if (kind == 1u) m = gd_at<const uint16_t>(gd_addr(a, 8))[i + 1u];
            }
        }
        const uint64_t o = (out * 16u + lane) * per + g;
        gd_at<uint16_t>(gd_addr(a, 16))[o] = (uint16_t)s;
        if (gd_addr(a, 18)) gd_at<uint16_t>(gd_addr(a, 18))[o] = (uint16_t)m;
    }
}
