// Rows of fp32, bf16 or binary16 values in the caller's memory: element and 8-value loads and stores, the
// type known when the work is queued. Addresses travel in the constants (64 bits in two words).
#pragma once
#include "gd_kernel.h"

enum { ROW_F32 = 0, ROW_BF16 = 1, ROW_F16 = 2 };

typedef __bf16 gd_bf16x8 __attribute__((ext_vector_type(8)));
typedef float gd_f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t gd_u32x2 __attribute__((ext_vector_type(2)));

// The address in constants W and W + 1, in global address space (global loads, not flat ones).
template <typename T>
using gd_gptr = __attribute__((address_space(1))) T *;
__device__ __forceinline__ uint64_t gd_addr(const GdArgs &a, int w) { return (uint64_t)a.c[w] | ((uint64_t)a.c[w + 1] << 32); }
template <typename T>
__device__ __forceinline__ gd_gptr<T> gd_at(uint64_t address) { return (gd_gptr<T>)(uintptr_t)address; }

// The T at `offset` bytes past a wave-uniform address: scalar base, 32-bit vector offset.
template <typename T>
__device__ __forceinline__ T gd_load(uint64_t base, uint32_t offset) {
    return *(gd_gptr<const T>)(gd_at<const char>(base) + offset);
}

__device__ __forceinline__ uint32_t row_shift(uint32_t type) { return type == ROW_F32 ? 2u : 1u; }

// fp32 bits of the 16-bit value h of type bf16 or binary16.
__device__ __forceinline__ float row_value16(uint32_t h, uint32_t type) {
    return type == ROW_BF16 ? gd_bits_f32(h << 16) : gd_half(h);
}
// v rounded to nearest even in a 16-bit type.
__device__ __forceinline__ uint32_t row_bits16(float v, uint32_t type) {
    return type == ROW_BF16 ? (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v)
                            : (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v);
}

__device__ __forceinline__ float row_load(uint64_t base, uint64_t i, uint32_t type) {
    if (type == ROW_F32) return gd_at<const float>(base)[i];
    return row_value16(gd_at<const uint16_t>(base)[i], type);
}
__device__ __forceinline__ void row_store(uint64_t base, uint64_t i, uint32_t type, float v) {
    if (type == ROW_F32) gd_at<float>(base)[i] = v;
    else gd_at<uint16_t>(base)[i] = (uint16_t)row_bits16(v, type);
}

// 16-byte accesses at any address of the type's alignment (a row starts where the caller's stride puts it).
typedef gd_u32x4 gd_u32x4_any __attribute__((aligned(2)));
typedef gd_f32x4 gd_f32x4_any __attribute__((aligned(4)));

// Values i .. i + 7 of a row.
template <uint32_t TYPE>
__device__ __forceinline__ void row_load8(uint64_t row, uint32_t i, float (&v)[8]) {
    if constexpr (TYPE == ROW_F32) {
        const gd_f32x4 a = gd_at<const gd_f32x4_any>(row + 4ull * i)[0], b = gd_at<const gd_f32x4_any>(row + 4ull * i)[1];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = a[j];
            v[4 + j] = b[j];
        }
    } else {
        const gd_u32x4 w = gd_at<const gd_u32x4_any>(row + 2ull * i)[0];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[2 * j] = row_value16(w[j] & 0xffffu, TYPE);
            v[2 * j + 1] = row_value16(w[j] >> 16, TYPE);
        }
    }
}
// As before, of a type known at run time, those from `n` on as zeros: a lane that reaches past the end reads the row's
// last eight and moves them down.
__device__ __forceinline__ void row_load8(uint64_t row, uint32_t i, uint32_t n, uint32_t type, float (&v)[8]) {
    if (n >= 8u) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.f;
        if (i >= n) return;
        const uint32_t at = min(i, n - 8u), past = i - at;
        if (type == ROW_F32) row_load8<ROW_F32>(row, at, v);
        else if (type == ROW_BF16) row_load8<ROW_BF16>(row, at, v);
        else row_load8<ROW_F16>(row, at, v);
        if (past) {
#pragma unroll
            for (uint32_t step = 4; step > 0; step >>= 1)
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j)
                    if (past & step) v[j] = j + step < 8u ? v[(j + step) & 7u] : 0.f;
        }
        return;
    }
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) v[j] = i + j < n ? row_load(row, i + j, type) : 0.f;
}
__device__ __forceinline__ void row_store8(uint64_t row, uint32_t i, uint32_t n, uint32_t type, const float (&v)[8]) {
    if (i + 8u <= n) {
        if (type == ROW_F32) {
            gd_f32x4 a, b;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                a[j] = v[j];
                b[j] = v[4 + j];
            }
            gd_at<gd_f32x4_any>(row + 4ull * i)[0] = a;
            gd_at<gd_f32x4_any>(row + 4ull * i)[1] = b;
        } else {
            gd_u32x4 w;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = row_bits16(v[2 * j], type) | row_bits16(v[2 * j + 1], type) << 16;
            gd_at<gd_u32x4_any>(row + 2ull * i)[0] = w;
        }
        return;
    }
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j)
        if (i + j < n) row_store(row, i + j, type, v[j]);
}
