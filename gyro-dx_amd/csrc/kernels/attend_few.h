// Attention of few rows (attend.h), 16-bit types: a group takes up to 16 rows and a part of the keys, its waves tiles of 32 keys
// in turn.
//
// A tile's scores are K Q^T by two v_mfma_f32_16x16x32 a step: a lane then holds 8 keys of one row, the others are 16, 32 and 48
// lanes away, so that the running maximum needs two exchanges per tile, the sum none until the end, and the weights are the
// second product's operand as they lie: O^T += V^T P^T, contracted over keys in the order in which lanes hold them. Keys go
// from memory straight to operands. Values go through LDS, a wave's tile its own, and come back transposed
// (ds_read_b64_tr_b16).
//
// Weights are at most 2^8 in bf16, where the sums are rescaled only when the maximum has grown by as much; in binary16 they reach
// 2^15 and every growth is followed, so that small ones lose least (at_grown).
//
// The weights are the sum of two 16-bit parts, 16 bits of them in bf16 and 22 in binary16: these rows are bound by memory, and
// the second products run in its shadow.
//
// Bound by the cache's bytes: a token each of 64 sequences of 91 to 8192 keys, 8 heads of 128 values, 560 MB, 108 us (5.2 TB/s;
// vector unit 16% of cycles, matrix unit 5%); one token over 131072 keys, 2 heads of 256, 268 MB, 52 us (5.1 TB/s). A wave has a
// tile of keys and one of values on their way at any time. Of short contexts the chain of dependent loads is the time: 777
// keys by eight waves 12 us, 300 keys 8.5.
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
template <uint32_t TYPE, uint32_t DT, uint32_t WAVES>
__device__ __forceinline__ void attend_few_body(const GdArgs &a) {
    // VROW: 16 rows' neighbouring 32 bytes in all banks.
    constexpr uint32_t STEPS = DT / 32u, DIMS = DT / 16u, VROW = DT * 2u + 32u, CHUNKS = DT / 8u, PER = 64u / CHUNKS;
    constexpr uint32_t VTILE = AF_KEYS * VROW;
    __shared__ __align__(16) char lds[WAVES * VTILE];
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
    bool far = false;  // some row's top is (at_far)

    // A tile's keys: a lane knows the place in the cache of key l % 32; k and v are on their way from when their registers are
    // free again, a tile ahead of their use. (Where there is none, the cache's first are loaded, and dropped later: at_key says
    // why.)
    gd_u32x4 k[2][STEPS], v[AF_KEYS / PER];
    const uint32_t chunk = lane % CHUNKS, of_key = lane / CHUNKS;
    const bool beyond = 8u * chunk >= D;
    auto key_of = [&](uint32_t t) { return (int32_t)(32u * t + (lane & 31u)); };
    auto page = [&](uint32_t t) { return at_page(a, o.seq, key_of(t), t < work.to ? o.end : 0); };
    auto locate = [&](uint32_t t, uint32_t page) { return at_key(a, page, o.head, key_of(t), t < work.to ? o.end : 0); };
    auto place = [&](int64_t at, uint32_t key) {
        const uint64_t offset = at < 0 ? 0ull : (uint64_t)at;
        return (uint64_t)__shfl((uint32_t)offset, key, 64) | (uint64_t)__shfl((uint32_t)(offset >> 32), key, 64) << 32;
    };
    // (D as the compiler sees it anew in each tile: it would hold the clamped offsets in registers through the loop.)
    auto head_end = [&] {
        uint32_t d = D;
        asm volatile("" : "+s"(d));
        return d;
    };
    auto load_k = [&](int64_t at) {
        const uint64_t from[2] = {K + place(at, col) + 16u * h, K + place(at, 16u + col) + 16u * h};
        if (D == DT) {
#pragma unroll
            for (uint32_t b = 0; b < 2; ++b)
#pragma unroll
                for (uint32_t s = 0; s < STEPS; ++s) k[b][s] = gd_at<const gd_u32x4_any>(from[b])[4u * s];
        } else {
            const uint32_t d = head_end();
#pragma unroll
            for (uint32_t b = 0; b < 2; ++b)
#pragma unroll
                for (uint32_t s = 0; s < STEPS; ++s) k[b][s] = *gd_at<const gd_u32x4_any>(32u * s + 8u * h < d ? from[b] + 64u * s : from[b] - 16u * h);
        }
    };
    auto load_v = [&](int64_t at) {
#pragma unroll
        for (uint32_t j = 0; j < AF_KEYS / PER; ++j) v[j] = *gd_at<const gd_u32x4_any>(V + place(at, PER * j + of_key) + (beyond ? 0u : 16u * chunk));
    };
    uint32_t soon = page(work.from + wave + WAVES);
    int64_t here = locate(work.from + wave, page(work.from + wave));
    load_k(here);
    __builtin_amdgcn_sched_barrier(0);  // keys first, as in the loop: the waits count what came after them
    load_v(here);
    for (uint32_t t = work.from + wave; t < work.to; t += WAVES) {
        const uint32_t later = page(t + 2u * WAVES);
        const uint32_t valid = (uint32_t)__ballot(here >= 0);  // both halves of the wave hold the same keys
        if (D != DT)
#pragma unroll
            for (uint32_t b = 0; b < 2; ++b)
#pragma unroll
                for (uint32_t s = 0; s < STEPS; ++s)
                    if (32u * s + 8u * h >= head_end()) k[b][s] = empty;  // (q is zero there, but 0 times NaN is not)
        gd_f32x4 s[2] = {none, none};
#pragma unroll
        for (uint32_t e = 0; e < STEPS; ++e)
#pragma unroll
            for (uint32_t b = 0; b < 2; ++b) s[b] = af_mfma<TYPE>(k[b][e], q[e], s[b]);
        const int64_t next = locate(t + WAVES, soon);
        load_k(next);
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
        if (valid != ~0u || D != DT)
#pragma unroll
            for (uint32_t j = 0; j < AF_KEYS / PER; ++j)
                if (beyond | !(valid >> (PER * j + of_key) & 1u)) v[j] = empty;
        // Keys whose values are not all finite: taken out here, they come back one by one below.
        uint32_t bad = 0;
        float finite[2] = {0.f, 0.f};
#pragma unroll
        for (uint32_t j = 0; j < AF_KEYS / PER; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) finite[i & 1] = at_finite<TYPE>(v[j][i], finite[i & 1]);
        if (__ballot(!(finite[0] + finite[1] == 0.f))) {
#pragma unroll
            for (uint32_t j = 0; j < AF_KEYS / PER; ++j) {
                float c = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) c = at_finite<TYPE>(v[j][i], c);
                const uint64_t lanes = __ballot(!(c == 0.f));
#pragma unroll
                for (uint32_t e = 0; e < PER; ++e)
                    if (lanes >> (e * CHUNKS) & ((1ull << CHUNKS) - 1u)) bad |= 1u << (PER * j + e);
                if (bad >> (PER * j + of_key) & 1u) v[j] = empty;
            }
        }
        float most = s[0][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) most = fmaxf(most, s[i >> 2][i & 3]);
        most = af_max(most) * scale;
        if (__ballot(at_grown<TYPE>(most, top))) {
            most = at_new_top<TYPE, 15>(most, top);
            const float shrink = at_exp2(top - most);
            top = most;
            far = __ballot(at_far(top));
            sum *= shrink;
#pragma unroll
            for (uint32_t d = 0; d < DIMS; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[d][i] *= shrink;
        }
        if (far)
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i >> 2][i & 3] = at_from_top(s[i >> 2][i & 3], scale, top);
        const float by = far ? 1.f : scale, from = far ? 0.f : top;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            s[i >> 2][i & 3] = at_exp2(fmaf(s[i >> 2][i & 3], by, -from));
            sum += s[i >> 2][i & 3];
        }
        gd_u32x4 large, small;  // the weights' parts
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = s[i >> 1][2 * (i & 1)], y = s[i >> 1][2 * (i & 1) + 1];
            large[i] = at_pair<TYPE>(x, y);
            small[i] = at_pair<TYPE>(x - row_value16(large[i] & 0xffffu, TYPE), y - row_value16(large[i] >> 16, TYPE));
        }
        __builtin_amdgcn_wave_barrier();  // after the reads of what is there
#pragma unroll
        for (uint32_t j = 0; j < AF_KEYS / PER; ++j) {
            const uint32_t key = PER * j + of_key;
            at_lds_store(mine + key * VROW + chunk * 16u, v[j]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        load_v(next);
        // V^T of 16 channels and the keys 4 h .. and 16 + 4 h .., in the order of the weights.
        auto values = [&](uint32_t d) {
            const uint32_t p = mine + (4u * h + (col >> 2)) * VROW + 32u * d + 8u * (col & 3u);
            const gd_u32x2 x = at_transposed(p), y = at_transposed(p + 16u * VROW);
            return gd_u32x4{x[0], x[1], y[0], y[1]};
        };
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
            const uint64_t from = V + place(here, key);
            // The key's weight is in the lanes of quarter key / 4 % 4.
            float weight = 0.f;
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i)
                if ((key >> 4) * 4u + (key & 3u) == i) weight = s[i >> 2][i & 3];
            weight = __shfl(weight, col + 16u * (key >> 2 & 3u), 64);
#pragma unroll
            for (uint32_t d = 0; d < DIMS; ++d) {
                const uint32_t dim = 16u * d + 4u * h;
                const gd_u32x2 x = *gd_at<const at_u32x2_any>(from + 2u * (dim < D ? dim : 0u));
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[d][i] += seen ? weight * row_value16(x[i >> 1] >> (16 * (i & 1)) & 0xffffu, TYPE) : 0.f;
            }
        }
        here = next;
        soon = later;
    }
    float *const rows = reinterpret_cast<float *>(lds);
#pragma unroll
    for (uint32_t d = 0; d < DIMS; ++d) *reinterpret_cast<gd_f32x4 *>(rows + wave * (VTILE / 4u) + col * (DT + 4u) + 16u * d + 4u * h) = acc[d];
    af_finish<TYPE, DT, VTILE / 4u, WAVES>(a, work, top, sum, rows);
}
