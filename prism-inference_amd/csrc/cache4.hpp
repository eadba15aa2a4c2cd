// cache4.hpp -- codes and scales of the cache of 4 bits a value: e2m1 with a power of two for each 32 dimensions.
#pragma once

#include "serve_common.hpp"

namespace prism {

namespace {

constexpr int kE2m1 = PRISM_CACHE_E2M1;
constexpr int kLeastExp = -23, kMostExp = 13;
constexpr uint32_t kGroup = 32;  // dimensions of a scale

// The least e with most <= 6 * 2^e (6 is 1.5 * 2^2), within the format's exponents.
__device__ __forceinline__ int exponent_of(uint32_t most) {
    const int e = static_cast<int>(most >> 23) - 127 - 2 + ((most & 0x7fffffu) > 0x400000u ? 1 : 0);
    return min(max(e, kLeastExp), kMostExp);
}

// Tokens of k and v and their slots.
struct Append4Args {
    prism_kv_cache c;
    const void *k, *v;
    uint64_t k_stride, v_stride;
    const int32_t *slots;
    uint32_t tokens;
};
struct NoAppend {};
__device__ __forceinline__ uint32_t rows_of(const Append4Args &a) { return a.c.kv_heads; }
__device__ __forceinline__ uint32_t rows_of(const NoAppend &) { return 0; }

// The slot of token t, -1 where there is none; there: it is a slot or -1.
__device__ __forceinline__ int32_t slot_of(const Append4Args &a, uint32_t t, bool *there) {
    const int32_t slot = a.slots[t];
    const bool in = slot >= 0 && static_cast<uint32_t>(slot) < a.c.pages * a.c.page_size;
    *there = in || slot == -1;
    return in ? slot : -1;
}
__device__ __forceinline__ int32_t slot_of(const NoAppend &, uint32_t, bool *there) { return *there = true, -1; }

template <typename T>
__device__ __forceinline__ f32x4 rounded(f32x4 v) {
    return __builtin_convertvector(__builtin_convertvector(v, typename Four<T>::type), f32x4);
}

// Dimensions 8 li .. + 7 (w0, w1) of one head's row into a slot; four neighbouring lanes share a scale.
// bad: a value is not finite; over: a magnitude is past the format.
template <int D>
__device__ __forceinline__ void write_codes4(const prism_kv_cache &c, bool is_v, uint32_t head, uint32_t slot, uint32_t li, f32x4 w0, f32x4 w1,
                                             bool *bad, bool *over) {
    float w[8] = {w0[0], w0[1], w0[2], w0[3], w1[0], w1[1], w1[2], w1[3]};
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const bool fine = finite(w[i]);
        *bad |= !fine;
        if (w[i] != w[i]) w[i] = 0.0f;
        if (fine) most = max(most, __float_as_uint(w[i]) & 0x7fffffffu);
    }
    most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 1)));
    most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 2)));
    *over |= most > 0x47400000u;  // 49152
    const int e = exponent_of(most);
    const float scale = __uint_as_float(static_cast<uint32_t>(e + 127) << 23), top = 6.0f * scale;
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = __builtin_amdgcn_fmed3f(w[i], -top, top);
    uint32_t code = 0;
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, w[0], w[1], scale, 0);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, w[2], w[3], scale, 1);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, w[4], w[5], scale, 2);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, w[6], w[7], scale, 3);
    const uint32_t ps = c.page_size, place = slot % ps;
    const uint64_t unit = static_cast<uint64_t>(slot / ps) * c.kv_heads + head;
    reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(is_v ? c.v : c.k) + (unit * ps + place) * (D / 2))[li] = code;
    if (li % 4 == 0) (is_v ? c.v_exponent : c.k_exponent)[(unit * (D / kGroup) + li / 4) * ps + place] = static_cast<uint8_t>(e + 127);
}

}  // namespace

}  // namespace prism
