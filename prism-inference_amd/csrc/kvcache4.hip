// kvcache4.hip -- tokens into the paged cache of 4 bits a value, and slots of a cache of any format back (gfx950).
//
// A value of the 4-bit cache is an e2m1 code times 2^e, with one e for each 32 consecutive dimensions of a token and head.  The
// scales are powers of two from 2^-23 to 2^13, so every value is one of binary16 and a token's bytes depend on nothing
// else in the page: no page is rescaled, slots come in any order, and a step's tokens need no common writer.
#include "rope_rows.hpp"

namespace prism {

namespace {

// A lane has eight consecutive dimensions of one token and head, four lanes a scale.
template <typename T, int D>
__global__ __launch_bounds__(256) void k_append4(Append4Args a, int *err) {
    constexpr uint32_t kLanes = D / 8, kRows = 256 / kLanes;
    const uint32_t li = threadIdx.x % kLanes, t = blockIdx.x * kRows + threadIdx.x / kLanes;
    const bool is_v = blockIdx.y >= a.c.kv_heads;
    const uint32_t head = is_v ? blockIdx.y - a.c.kv_heads : blockIdx.y;
    if (t >= a.tokens) return;
    bool there, bad = false, over = false;
    const int32_t slot = slot_of(a, t, &there);
    if (!there && blockIdx.y + li == 0) raise_error(err, kErrIndex);
    if (slot < 0) return;  // whole rows leave, so the lanes of a scale stay together
    const T *x = static_cast<const T *>(is_v ? a.v : a.k) + t * (is_v ? a.v_stride : a.k_stride) + static_cast<uint64_t>(head) * D + 8 * li;
    write_codes4<D>(a.c, is_v, head, static_cast<uint32_t>(slot), li, load4(x), load4(x + 4), &bad, &over);
    if (bad) raise_error(err, kErrInput);
    if (over) raise_error(err, kErrNonfinite);
}

struct ReadArgs {
    prism_kv_cache c;
    const int32_t *slots;
    uint32_t tokens;
    void *k, *v;
    uint64_t k_stride, v_stride;
};

template <typename T, int FMT, int D>
__global__ __launch_bounds__(256) void k_read(ReadArgs a, int *err) {
    constexpr uint32_t kLanes = D / 8, kRows = 256 / kLanes;
    const uint32_t li = threadIdx.x % kLanes, t = blockIdx.x * kRows + threadIdx.x / kLanes;
    const uint32_t task = blockIdx.y + (a.k ? 0 : a.c.kv_heads);
    const bool is_v = task >= a.c.kv_heads;
    const uint32_t head = is_v ? task - a.c.kv_heads : task, ps = a.c.page_size;
    const int32_t slot = t < a.tokens ? a.slots[t] : -1;
    const bool there = slot >= 0 && static_cast<uint32_t>(slot) < a.c.pages * ps;
    if (slot != -1 && !there && blockIdx.y + li == 0) raise_error(err, kErrIndex);
    if (!there) return;
    const uint32_t place = static_cast<uint32_t>(slot) % ps;
    const uint64_t unit = static_cast<uint64_t>(static_cast<uint32_t>(slot) / ps) * a.c.kv_heads + head;
    const uint8_t *codes = static_cast<const uint8_t *>(is_v ? a.c.v : a.c.k);
    f32x4 w[2];
    if constexpr (FMT == kE2m1) {
        const uint32_t code = reinterpret_cast<const uint32_t *>(codes + (unit * ps + place) * (D / 2))[li];
        const uint32_t e = (is_v ? a.c.v_exponent : a.c.k_exponent)[(unit * (D / kGroup) + li / 4) * ps + place];
        // 2^(e - 127) of any byte; 255 is no number.
        const float scale = e == 0 ? 0x1p-127f : __uint_as_float(e == 255 ? 0x7fc00000u : e << 23);
        const f32x2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 1),
                            __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 3)};
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i / 4][i % 4] = p[i / 2][i % 2] * scale;
    } else {
        const float scale = (is_v ? a.c.v_scale : a.c.k_scale)[unit];
        uint32_t code[2];
        if (!is_v) {
            __builtin_memcpy(code, codes + (unit * ps + place) * D + 8 * li, 8);
        } else {
            const uint8_t *p = codes + (unit * D + 8 * li) * ps + place;
            code[0] = p[0] | p[ps] << 8 | p[2 * ps] << 16 | static_cast<uint32_t>(p[3 * ps]) << 24;
            code[1] = p[4 * ps] | p[5 * ps] << 8 | p[6 * ps] << 16 | static_cast<uint32_t>(p[7 * ps]) << 24;
        }
        w[0] = value4<FMT>(code[0]) * scale;
        w[1] = value4<FMT>(code[1]) * scale;
    }
    if (!fits<T>(w[0]) || !fits<T>(w[1])) raise_error(err, kErrNonfinite);
    T *out = static_cast<T *>(is_v ? a.v : a.k) + t * (is_v ? a.v_stride : a.k_stride) + static_cast<uint64_t>(head) * D + 8 * li;
    store4(out, w[0]);
    store4(out + 4, w[1]);
}

template <typename T>
int append4_typed(const Append4Args &a, int *err, hipStream_t s) {
    const uint32_t rows = 256 / (a.c.head_dim / 8);
    const dim3 grid((a.tokens + rows - 1) / rows, 2 * a.c.kv_heads);
    switch (a.c.head_dim) {
    case 64: k_append4<T, 64><<<grid, 256, 0, s>>>(a, err); break;
    case 128: k_append4<T, 128><<<grid, 256, 0, s>>>(a, err); break;
    case 256: k_append4<T, 256><<<grid, 256, 0, s>>>(a, err); break;
    default: return kLaunchUnsupported;
    }
    return launch_status();
}

template <typename T, int D>
int qkv4_typed(const Rotation &rot, const RopeRows &q, const RopeRows &k, const int32_t *positions, float eps, const Append4Args &a, int *err,
               hipStream_t s) {
    const uint32_t tiles = (a.tokens + kRopeTokens - 1) / kRopeTokens, heads = q.heads + 2 * k.heads;
    // Heads are split over workgroups until some 1024 of them share the rows, whole row groups each.
    constexpr uint32_t least = 64 / (D / 8);
    uint32_t parts = (1024 + tiles - 1) / tiles;
    if (parts > (heads + least - 1) / least) parts = (heads + least - 1) / least;
    const uint32_t each = ((heads + parts - 1) / parts + least - 1) / least * least;
    const dim3 grid(tiles, (heads + each - 1) / each);
    if (rot.interleaved) k_rope<T, D, true><<<grid, 256, 0, s>>>(q, k, rot, positions, a.tokens, each, eps, a, err);
    else k_rope<T, D, false><<<grid, 256, 0, s>>>(q, k, rot, positions, a.tokens, each, eps, a, err);
    return launch_status();
}
template <typename T>
int qkv4_headed(const Rotation &rot, const RopeRows &q, const RopeRows &k, const int32_t *positions, float eps, const Append4Args &a, int *err,
                hipStream_t s) {
    switch (a.c.head_dim) {
    case 64: return qkv4_typed<T, 64>(rot, q, k, positions, eps, a, err, s);
    case 128: return qkv4_typed<T, 128>(rot, q, k, positions, eps, a, err, s);
    case 256: return qkv4_typed<T, 256>(rot, q, k, positions, eps, a, err, s);
    default: return kLaunchUnsupported;
    }
}

template <typename T, int FMT>
int read_headed(const ReadArgs &a, int *err, hipStream_t s) {
    const uint32_t rows = 256 / (a.c.head_dim / 8);
    const dim3 grid((a.tokens + rows - 1) / rows, (a.k ? a.c.kv_heads : 0) + (a.v ? a.c.kv_heads : 0));
    switch (a.c.head_dim) {
    case 64: k_read<T, FMT, 64><<<grid, 256, 0, s>>>(a, err); break;
    case 128: k_read<T, FMT, 128><<<grid, 256, 0, s>>>(a, err); break;
    case 256: k_read<T, FMT, 256><<<grid, 256, 0, s>>>(a, err); break;
    default: return kLaunchUnsupported;
    }
    return launch_status();
}
template <typename T>
int read_typed(const ReadArgs &a, int *err, hipStream_t s) {
    if (a.c.format == PRISM_CACHE_INT8) return read_headed<T, kInt8>(a, err, s);
    if (a.c.format == PRISM_CACHE_E4M3) return read_headed<T, kE4m3>(a, err, s);
    return read_headed<T, kE2m1>(a, err, s);
}

}  // namespace

int launch_kv_append4(const prism_kv_cache &cache, int dtype, const void *k, uint64_t k_stride, const void *v, uint64_t v_stride,
                      const int32_t *slots, uint32_t tokens, int *err, hipStream_t s) {
    const Append4Args a{cache, k, v, k_stride, v_stride, slots, tokens};
    if (dtype == PRISM_DTYPE_F32) return append4_typed<float>(a, err, s);
    if (dtype == PRISM_DTYPE_F16) return append4_typed<_Float16>(a, err, s);
    return append4_typed<__bf16>(a, err, s);
}

int launch_qkv_append4(const prism_kv_cache &cache, int dtype, const Rotation &rot, const RopeRows &q, const RopeRows &k, const void *v,
                       uint64_t v_stride, const int32_t *positions, const int32_t *slots, uint32_t tokens, float eps, int *err, hipStream_t s) {
    const Append4Args a{cache, nullptr, v, 0, v_stride, slots, tokens};
    if (dtype == PRISM_DTYPE_F32) return qkv4_headed<float>(rot, q, k, positions, eps, a, err, s);
    if (dtype == PRISM_DTYPE_F16) return qkv4_headed<_Float16>(rot, q, k, positions, eps, a, err, s);
    return qkv4_headed<__bf16>(rot, q, k, positions, eps, a, err, s);
}

int launch_kv_read(const prism_kv_cache &cache, int dtype, const int32_t *slots, uint32_t tokens, void *k, uint64_t k_stride, void *v,
                   uint64_t v_stride, int *err, hipStream_t s) {
    const ReadArgs a{cache, slots, tokens, k, v, k_stride, v_stride};
    if (dtype == PRISM_DTYPE_F32) return read_typed<float>(a, err, s);
    if (dtype == PRISM_DTYPE_F16) return read_typed<_Float16>(a, err, s);
    return read_typed<__bf16>(a, err, s);
}

}  // namespace prism
