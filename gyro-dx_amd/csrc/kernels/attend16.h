// What the 16-bit builds of attention share beside attend.h.
#pragma once
#include "attend.h"

typedef _Float16 at_f16x8 __attribute__((ext_vector_type(8)));
typedef float at_f32x16 __attribute__((ext_vector_type(16)));
typedef short at_s16x4 __attribute__((ext_vector_type(4)));

// Two values rounded to the type, to nearest even, as a word.
typedef __bf16 at_bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 at_f16x2 __attribute__((ext_vector_type(2)));
typedef float at_f32x2 __attribute__((ext_vector_type(2)));
template <uint32_t TYPE>
__device__ __forceinline__ uint32_t at_pair(float lo, float hi) {
    if constexpr (TYPE == ROW_BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector((at_f32x2{lo, hi}), at_bf16x2));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector((at_f32x2{lo, hi}), at_f16x2));
}
// c and both values of a word.
template <uint32_t TYPE>
__device__ __forceinline__ float at_add_pair(uint32_t w, float c) {
    if constexpr (TYPE == ROW_BF16)
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(at_bf16x2, w), at_bf16x2{(__bf16)1.f, (__bf16)1.f}, c, false);
    else
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(at_f16x2, w), at_f16x2{(_Float16)1.f, (_Float16)1.f}, c, false);
}
// c while a word's values are finite, from then on NaN (0 times the others is).
template <uint32_t TYPE>
__device__ __forceinline__ float at_finite(uint32_t w, float c) {
    if constexpr (TYPE == ROW_BF16)
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(at_bf16x2, w), at_bf16x2{(__bf16)0.f, (__bf16)0.f}, c, false);
    else
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(at_f16x2, w), at_f16x2{(_Float16)0.f, (_Float16)0.f}, c, false);
}

// Weights are relative to a top that follows the running maximum only when that has grown by more than 2^GROWN, so that the
// sums are rarely rescaled. bf16 has fp32's exponents, and GROWN 8. Binary16 ends at 2^-24: its weights are 2^LIFT larger,
// which the sums share, as far as 2^16 allows. A weight is then rounded by half a unit of its last place or by 2^-25-LIFT of
// the largest. (131,071 keys 19 nats below one whose value is zero: off by 67% with LIFT 0 and GROWN 8.) Rows bound by memory
// have LIFT 15, many rows 11: 4096 tokens of 32 heads of 128 over 8, us: LIFT 7 170, 11 172, 13 175, heads of 256, 2048 tokens
// 171, 183, 195. A top that is far has no room for LIFT in its last places, and needs none.
template <uint32_t TYPE>
__device__ __forceinline__ bool at_grown(float most, float top) { return most > top + (TYPE == ROW_F16 ? 15.f : 8.f); }
template <uint32_t TYPE, uint32_t LIFT>
__device__ __forceinline__ float at_new_top(float most, float top) {
    static_assert(LIFT <= 15u, "GROWN is what LIFT leaves of 15");
    if (TYPE == ROW_F16) most -= fabsf(most) >= AT_FAR ? 0.f : (float)LIFT;
    return fmaxf(most, top);
}

// LDS by its 32-bit addresses.
template <typename T>
using at_lptr = __attribute__((address_space(3))) T *;
__device__ __forceinline__ uint32_t at_lds(const void *p) { return (uint32_t)(uintptr_t)(at_lptr<const char>)p; }
__device__ __forceinline__ gd_u32x4 at_lds_load(uint32_t at) { return *(at_lptr<const gd_u32x4>)(uintptr_t)at; }
__device__ __forceinline__ void at_lds_store(uint32_t at, gd_u32x4 v) { *(at_lptr<gd_u32x4>)(uintptr_t)at = v; }
// Of 4 rows of 16 neighbouring 16-bit values in LDS, lane l of 16 names values 4 (l % 4) .. of row l / 4 and gets column l.
__device__ __forceinline__ gd_u32x2 at_transposed(uint32_t at) {
    return __builtin_bit_cast(gd_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_lptr<at_s16x4>)(uintptr_t)at));
}
