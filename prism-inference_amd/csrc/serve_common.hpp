// serve_common.hpp -- element types and 8-bit codes shared by the kernels between and behind the projections of many requests.
#pragma once

#include "device_common.hpp"
#include "kernels.hpp"
#include "serving.hpp"

namespace prism {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

// N consecutive elements aligned to one element; global memory takes such accesses whole.
template <typename V, typename T>
__device__ __forceinline__ V load_any(const T *p) {
    V v;
    __builtin_memcpy(&v, p, sizeof(V));
    return v;
}
template <typename V, typename T>
__device__ __forceinline__ void store_any(T *p, V v) {
    __builtin_memcpy(p, &v, sizeof(V));
}
template <typename T>
struct Four;
template <>
struct Four<float> {
    typedef f32x4 type;
};
template <>
struct Four<_Float16> {
    typedef f16x4 type;
};
template <>
struct Four<__bf16> {
    typedef bf16x4 type;
};
template <typename T>
__device__ __forceinline__ f32x4 load4(const T *p) {
    return __builtin_convertvector(load_any<typename Four<T>::type>(p), f32x4);
}
template <typename T>
__device__ __forceinline__ void store4(T *p, f32x4 v) {  // ties to even
    store_any(p, __builtin_convertvector(v, typename Four<T>::type));
}
// Whether four values are finite once they are rounded to the type.
template <typename T>
__device__ __forceinline__ bool fits(f32x4 v) {
    const f32x4 r = __builtin_convertvector(__builtin_convertvector(v, typename Four<T>::type), f32x4);
    return finite(r[0]) && finite(r[1]) && finite(r[2]) && finite(r[3]);
}

// What a wavefront's lanes wrote to LDS is there for the others.
__device__ __forceinline__ void settle() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

constexpr int kInt8 = PRISM_CACHE_INT8, kE4m3 = PRISM_CACHE_E4M3;

// The codes of four values, ties to even, magnitudes past the format's largest at it.  Not for NaN.
template <int FMT>
__device__ __forceinline__ uint32_t code4(f32x4 v) {
    constexpr float top = FMT == kInt8 ? 127.0f : 448.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __builtin_amdgcn_fmed3f(v[i], -top, top);
    if constexpr (FMT == kInt8) {
        // 1.5 * 2^23 + v rounds v to an integer, whose two's complement the sum's low byte is.
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += 12582912.0f;
        const uint32_t low = perm(__float_as_uint(v[1]), __float_as_uint(v[0]), 0x0c0c0400u);
        const uint32_t high = perm(__float_as_uint(v[3]), __float_as_uint(v[2]), 0x04000c0cu);
        return low | high;
    } else {
        const int r = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
        return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], r, true));
    }
}
template <int FMT>
__device__ __forceinline__ f32x4 value4(uint32_t c) {
    if constexpr (FMT == kInt8)
        return f32x4{static_cast<float>(static_cast<int8_t>(c)), static_cast<float>(static_cast<int8_t>(c >> 8)),
                     static_cast<float>(static_cast<int8_t>(c >> 16)), static_cast<float>(static_cast<int8_t>(c >> 24))};
    else
        return f32x4{__builtin_amdgcn_cvt_f32_fp8(static_cast<int>(c), 0), __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(c), 1),
                     __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(c), 2), __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(c), 3)};
}

}  // namespace prism
