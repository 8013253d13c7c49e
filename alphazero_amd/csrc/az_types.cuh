// Element types of the head operators: loads, stores and roundings (to nearest, ties to even).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/azamd.h"

namespace az {

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
// v = h + m + l with 8 significant bits each: the two differences are exact, so 24 bits come through.
__device__ __forceinline__ void split3(float v, uint16_t& h, uint16_t& m, uint16_t& l) {
    h = bf16_bits(v);
    const float a = (h & 0x7fff) == 0x7f80 ? 0.0f : v - bf16_value(h);   // an infinity is all in h
    m = bf16_bits(a);
    l = bf16_bits(a - bf16_value(m));
}

}  // namespace az
