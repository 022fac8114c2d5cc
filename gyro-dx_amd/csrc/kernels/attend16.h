// What the 16-bit builds of attention share beside attend.h.
#pragma once
#include "attend.h"

typedef _Float16 at_f16x8 __attribute__((ext_vector_type(8)));
typedef float at_f32x16 __attribute__((ext_vector_type(16)));
typedef short at_s16x4 __attribute__((ext_vector_type(4)));

template <uint32_t TYPE>
__device__ __forceinline__ uint32_t at_pair(float lo, float hi) {
    return row_bits16(lo, TYPE) | row_bits16(hi, TYPE) << 16;
}
// The larger magnitudes of two words' values, as bits; and whether one of them is not finite.
typedef uint16_t at_u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t at_larger(uint32_t a, uint32_t w) {
    const at_u16x2 r = __builtin_elementwise_max(__builtin_bit_cast(at_u16x2, a), __builtin_bit_cast(at_u16x2, w & 0x7fff7fffu));
    return __builtin_bit_cast(uint32_t, r);
}
template <uint32_t TYPE>
__device__ __forceinline__ bool at_not_finite(uint32_t a) {
    constexpr uint32_t e = TYPE == ROW_BF16 ? 0x7f80u : 0x7c00u;
    return (a & 0xffffu) >= e || a >> 16 >= e;
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
