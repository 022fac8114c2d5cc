// What the 4-bit products share (mv_q4.h, mm_q4.h): weights and scales of q4_repack's layout as operands.
//
// They run on v_mfma_f32_16x16x32 with token rows as the A operand and 16 weight rows as B. A 4-bit value becomes a
// bf16 or binary16 in half an instruction: its bits are or-ed into the top of the mantissa of 16, which gives 16 + q
// exactly. Those extra 16 (24 where W = s (q - 8)) times the group's sum of activations go in as the product's C
// operand, itself the product of the activations with a constant matrix, so nothing of the group's sum is kept
// apart, and it is at most five times what the group's own product rounds at. Group sums are scaled and added
// in fp32. Activations are exact: an fp32 value is the sum of three bf16 values (its 24 bits cut in eights). The matrix unit
// takes bf16 values below 2^-126 as zero, so from 2^-103 on an activation keeps all its bits.
// Of a token with an infinity or NaN no output is finite: every group's product and sum with it are not, and no scale
// makes them so.
//
// Constants: 0 quants 2 scales 4 minima (0: none) 6 tiles 7 chunks 8 log2(group) 9 cols 10 outputs per token
// 11 gated pair 12 x 14 x stride 16 x type 17 tokens 18 y 20 y stride 22 y type 23 act (0 none, 1 silu, 2
// sigmoid) 24 add to y 25 scale (fp32 bits) 26 WK (mv_q4.h), T (mm_q4.h). Addresses and strides have 64 bits; strides
// count values.
#pragma once
#include "rows.h"

// Mask and exponent of the unpacking as a vector and a scalar register: v_and_or_b32 takes both in one instruction, and
// no constants.
struct MqBits {
    uint32_t mask, one;
};
template <bool HALF>
__device__ __forceinline__ MqBits mq_bits() {
    MqBits b = {HALF ? 0x03c003c0u : 0x00780078u, HALF ? 0x4c004c00u : 0x41804180u};
    asm("" : "+v"(b.mask));
    asm("" : "+s"(b.one));
    return b;
}
// Values 0 .. 7 of a word (q4_repack) as 16 + q, in bf16 or binary16.
template <bool HALF>
__device__ __forceinline__ gd_u32x4 mq_weights(uint32_t w, MqBits b) {
    if constexpr (HALF)
        return {((w << 3) & b.mask) | b.one, ((w >> 1) & b.mask) | b.one, ((w >> 5) & b.mask) | b.one,
                (__builtin_amdgcn_alignbit(w, w, 9) & b.mask) | b.one};
    else
        return {(w & b.mask) | b.one, ((w >> 4) & b.mask) | b.one, ((w >> 8) & b.mask) | b.one,
                (__builtin_amdgcn_alignbit(w, w, 12) & b.mask) | b.one};
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

// One chunk of a tile as a lane holds it: its 16 bytes and the scales (minima) of its row, four binary16 in order.
struct MqChunk {
    gd_u32x4 w;
    gd_u32x2 s, m;
};
typedef gd_u32x2 gd_u32x2_any __attribute__((aligned(2)));
// The 8 bytes at a row's scales of a chunk: 4, 2 or 1 of them are its own (128 / group), the buffer has room for the rest.
__device__ __forceinline__ gd_u32x2 mq_scales(uint64_t base, uint32_t row, uint32_t lg) {
    return gd_load<gd_u32x2_any>(base, row << (8u - lg));
}
// Of those, the scale of each group of 32, by the bytes that `even` and `odd` choose.
struct MqSpread {
    uint32_t even, odd;
};
__device__ __forceinline__ MqSpread mq_spread(uint32_t lg) {
    return {lg == 5u ? 0x03020100u : 0x01000100u, lg == 5u ? 0x07060504u : lg == 6u ? 0x03020302u : 0x01000100u};
}
__device__ __forceinline__ gd_u32x2 mq_spread(gd_u32x2 s, MqSpread by) {
    return {__builtin_amdgcn_perm(s[1], s[0], by.even), __builtin_amdgcn_perm(s[1], s[0], by.odd)};
}
__device__ __forceinline__ float mq_half(gd_u32x2 o, uint32_t j) { return gd_half(o[j >> 1] >> (16u * (j & 1u)) & 0xffffu); }

// scale act(v) and what the output held, stored: y[t][out] = v.
struct MqOut {
    uint64_t y, stride;
    uint32_t type, act, add, gated;
    float scale;
};
__device__ __forceinline__ MqOut mq_out(const GdArgs &a) {
    return {gd_addr(a, 18), gd_addr(a, 20), a.c[22], a.c[23], a.c[24], a.c[11], gd_bits_f32(a.c[25])};
}
__device__ __forceinline__ float mq_value(const MqOut &o, float sum, float up) {
    // x rcp(1 + e^-x): within two units of the last place of the division's result. expf's own relative error grows with |x|
    // to |x| 2^-24 (its argument times log2 e is rounded); e^-x counts in the result where x is negative.
    if (o.gated) return o.scale * (sum * __builtin_amdgcn_rcpf(1.0f + expf(-sum)) * up);
    float v = o.scale * sum;
    if (o.act == 1u) v = v * __builtin_amdgcn_rcpf(1.0f + expf(-v));
    else if (o.act == 2u) v = __builtin_amdgcn_rcpf(1.0f + expf(-v));
    return v;
}
__device__ __forceinline__ void mq_store(const MqOut &o, uint32_t t, uint64_t out, float sum, float up) {
    float v = mq_value(o, sum, up);
    const uint64_t at = (uint64_t)t * o.stride + out;
    if (o.add) v += row_load(o.y, at, o.type);
    row_store(o.y, at, o.type, v);
}
// Four neighbouring outputs, the first `count` of them.
__device__ __forceinline__ void mq_store4(const MqOut &o, uint32_t t, uint64_t out, uint32_t count, gd_f32x4 sum, gd_f32x4 up) {
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = mq_value(o, sum[i], up[i]);
    const uint64_t at = (uint64_t)t * o.stride + out;
    if (o.add)
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) v[i] += i < count ? row_load(o.y, at + i, o.type) : 0.f;
    if (count < 4u) {
#pragma unroll
        for (uint32_t i = 0; i < 3; ++i)
            if (i < count) row_store(o.y, at + i, o.type, v[i]);
    } else if (o.type == ROW_F32) {
        gd_at<gd_f32x4_any>(o.y + 4u * at)[0] = gd_f32x4{v[0], v[1], v[2], v[3]};
    } else {
        gd_at<gd_u32x2_any>(o.y + 2u * at)[0] = gd_u32x2{row_bits16(v[0], o.type) | row_bits16(v[1], o.type) << 16,
                                                         row_bits16(v[2], o.type) | row_bits16(v[3], o.type) << 16};
    }
}
