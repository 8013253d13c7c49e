// Element types of the head operators: loads, stores and roundings (to nearest, ties to even).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/azamd.h"

namespace az {

typedef float f32x4 __attribute__((ext_vector_type(4)));

enum { DT_F32 = AZ_DT_F32, DT_BF16 = AZ_DT_BF16, DT_F16 = AZ_DT_F16 };

__device__ __forceinline__ uint16_t bf16_bits(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
__device__ __forceinline__ float bf16_value(uint16_t b) { return __builtin_bit_cast(float, (uint32_t)b << 16); }

template <int DT> __device__ __forceinline__ uint16_t to_bits(float v) {
    if constexpr (DT == DT_BF16) return bf16_bits(v);
    else return __builtin_bit_cast(uint16_t, (_Float16)v);
}
template <int DT> __device__ __forceinline__ float from_bits(uint16_t b) {
    if constexpr (DT == DT_BF16) return bf16_value(b);
    else return (float)__builtin_bit_cast(_Float16, b);
}
template <int DT> __device__ __forceinline__ uint2 pack4(float a, float b, float c, float d) {
    return make_uint2((uint32_t)to_bits<DT>(a) | (uint32_t)to_bits<DT>(b) << 16, (uint32_t)to_bits<DT>(c) | (uint32_t)to_bits<DT>(d) << 16);
}
template <int DT> __device__ __forceinline__ float load_scalar(const void* p, int64_t i) {
    if constexpr (DT == DT_F32) return ((const float*)p)[i];
    else return from_bits<DT>(((const uint16_t*)p)[i]);
}
template <int DT> __device__ __forceinline__ void store_scalar(void* p, int64_t i, float v) {
    if constexpr (DT == DT_F32) ((float*)p)[i] = v;
    else ((uint16_t*)p)[i] = to_bits<DT>(v);
}
// Four neighbours at i, a multiple of 4 elements from a 16-byte aligned p.
template <int DT> __device__ __forceinline__ void store4(void* p, int64_t i, float a, float b, float c, float d) {
    if constexpr (DT == DT_F32) {
        *(float4*)((float*)p + i) = make_float4(a, b, c, d);
    } else {
        const uint16_t h[4] = {to_bits<DT>(a), to_bits<DT>(b), to_bits<DT>(c), to_bits<DT>(d)};
        *(uint2*)((uint16_t*)p + i) = *(const uint2*)h;
    }
}
// A vector along a tile's p axis, read through a buffer descriptor: a short offset per lane instead of an address, and zeros
// behind the last element.
#ifdef __HIP_DEVICE_COMPILE__
struct AxisView {
    __amdgpu_buffer_rsrc_t r;
    template <class E> __device__ __forceinline__ AxisView(const E* p, int64_t count)
        : r(__builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)((count < 0 ? 0 : count < 65536 ? count : 65536) * sizeof(E)), 0x00020000)) {}
    __device__ __forceinline__ f32x4 four(int i) const { return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, i * 4, 0, 0)); }
    template <int DT> __device__ __forceinline__ float one(int i) const {
        if constexpr (DT == DT_F32) return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, i * 4, 0, 0));
        else return from_bits<DT>((uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, i * 2, 0, 0));
    }
};
#endif

// v = h + m / 2048 in float16, both differences exact: 22 bits and a sign come through where |v| is within 2^14 and above 2^-13
// (below that the smallest step of m, 2^-35, is what is left). Infinities are all in h.
__device__ __forceinline__ void split2(float v, uint16_t& h, uint16_t& m) {
    const _Float16 a = (_Float16)v;
    h = __builtin_bit_cast(uint16_t, a);
    m = (h & 0x7fff) == 0x7c00 ? (uint16_t)0 : __builtin_bit_cast(uint16_t, (_Float16)((v - (float)a) * 2048.0f));
}
// The power of two that takes values of at most `top` to at most 2^14, as its reciprocal: 1 for an infinity or NaN, next to nothing
// for zero (its values stay zero, and it never is the largest of several).
__device__ __forceinline__ float unscale_of(float top) {
    if (!(top < INFINITY)) return 1.0f;
    if (top == 0.0f) return 0x1p-120f;
    const int e = ilogbf(top) - 13;
    return ldexpf(1.0f, e < -120 ? -120 : e > 120 ? 120 : e);
}

}  // namespace az
