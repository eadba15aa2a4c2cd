// kvcache4.hip -- tokens into the paged cache of 4 bits a value, and slots of a cache of any format back (gfx950).
//
// A value of the 4-bit cache is an e2m1 code times 2^e, with one e for each 32 consecutive dimensions of a token and head.  The
// scales are powers of two from 2^-23 to 2^13, so every value is one of binary16 and a token's bytes depend on nothing
// else in the page: no page is rescaled, slots come in any order, and a step's tokens need no common writer.
#include "rope_rows.hpp"

namespace prism {

namespace {

// A lane has eight consecutive dimensions of one token and head, four lanes a scale; one instruction makes two codes, so memory
// bounds it: 7314 tokens of 48 requests, 4 heads of 256 in binary16, take 10.4 us, 3.7 TB/s.
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

// The slot of a token to read: -1 where there is none, which is an error but for -1 itself.
__device__ __forceinline__ int32_t slot_read(const ReadArgs &a, uint32_t t, bool tells, int *err) {
    if (t >= a.tokens) return -1;
    const int32_t slot = a.slots[t];
    const bool in = slot >= 0 && static_cast<uint32_t>(slot) < a.c.pages * a.c.page_size;
    if (!in && slot != -1 && tells) raise_error(err, kErrIndex);
    return in ? slot : -1;
}
template <typename T>
__device__ __forceinline__ T *row_read(const ReadArgs &a, bool is_v, uint32_t t, uint32_t head, uint32_t dim) {
    return static_cast<T *>(is_v ? a.v : a.k) + t * (is_v ? a.v_stride : a.k_stride) + static_cast<uint64_t>(head) * a.c.head_dim + dim;
}

// 4 bits: a lane has eight consecutive dimensions of one token and head.  8192 tokens of 8 heads of 128 take 10 us as bf16, 4.2 TB/s.
template <typename T, int D>
__global__ __launch_bounds__(256) void k_read4(ReadArgs a, int *err) {
    constexpr uint32_t kLanes = D / 8, kRows = 256 / kLanes;
    const uint32_t li = threadIdx.x % kLanes, t = blockIdx.x * kRows + threadIdx.x / kLanes;
    const uint32_t task = blockIdx.y + (a.k ? 0 : a.c.kv_heads);
    const bool is_v = task >= a.c.kv_heads;
    const uint32_t head = is_v ? task - a.c.kv_heads : task, ps = a.c.page_size;
    const int32_t slot = slot_read(a, t, blockIdx.y + li == 0, err);
    if (slot < 0) return;
    const uint32_t place = static_cast<uint32_t>(slot) % ps;
    const uint64_t unit = static_cast<uint64_t>(static_cast<uint32_t>(slot) / ps) * a.c.kv_heads + head;
    const uint32_t code = reinterpret_cast<const uint32_t *>(static_cast<const uint8_t *>(is_v ? a.c.v : a.c.k) + (unit * ps + place) * (D / 2))[li];
    const uint32_t e = (is_v ? a.c.v_exponent : a.c.k_exponent)[(unit * (D / kGroup) + li / 4) * ps + place];
    // 2^(e - 127) of any byte; 255 is no number.
    const float scale = e == 0 ? 0x1p-127f : __uint_as_float(e == 255 ? 0x7fc00000u : e << 23);
    const f32x2 x[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 1),
                        __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 3)};
    const f32x4 w0 = f32x4{x[0][0], x[0][1], x[1][0], x[1][1]} * scale, w1 = f32x4{x[2][0], x[2][1], x[3][0], x[3][1]} * scale;
    if (!fits<T>(w0) || !fits<T>(w1)) raise_error(err, kErrNonfinite);
    T *out = row_read<T>(a, is_v, t, head, 8 * li);
    store4(out, w0);
    store4(out + 4, w1);
}

// 8 bits, keys: the same.
template <typename T, int FMT, int D>
__device__ __forceinline__ void read_keys(const ReadArgs &a, uint32_t block, uint32_t head, int *err) {
    constexpr uint32_t kLanes = D / 8, kRows = 256 / kLanes;
    const uint32_t li = threadIdx.x % kLanes, t = block * kRows + threadIdx.x / kLanes, ps = a.c.page_size;
    const int32_t slot = slot_read(a, t, head + li == 0, err);
    if (slot < 0) return;
    const uint64_t unit = static_cast<uint64_t>(static_cast<uint32_t>(slot) / ps) * a.c.kv_heads + head;
    const float scale = a.c.k_scale[unit];
    const u32x2 code = *reinterpret_cast<const u32x2 *>(static_cast<const uint8_t *>(a.c.k) + (unit * ps + static_cast<uint32_t>(slot) % ps) * D + 8 * li);
    const f32x4 w0 = value4<FMT>(code[0]) * scale, w1 = value4<FMT>(code[1]) * scale;
    if (!fits<T>(w0) || !fits<T>(w1)) raise_error(err, kErrNonfinite);
    T *out = row_read<T>(a, false, t, head, 8 * li);
    store4(out, w0);
    store4(out + 4, w1);
}
// 8 bits, values, which a page holds by dimension: D / 4 lanes take eight tokens, a lane four dimensions.  Tokens that follow each
// other stand in one or two runs of sixteen places, which a lane loads whole, sixteen bytes a dimension, before it writes
// any token; others load a byte a value.  Each run is loaded by both windows of its sixteen places, and a window within one run loads it twice.  The values of 8192 tokens of 8 heads of 128 take 10.9 us this way, a byte a value 19.5, runs
// loaded in the loop over the tokens 22 (a load's wait is one for every store before it too); windows of 16 tokens are as fast
// there and slower where requests end inside them (40 of 1 to 333 tokens: 11.7 and 7.9), windows of 4 take 13.8 and 7.3.
constexpr uint32_t kWindow = 8;
template <typename T, int FMT, int D>
__device__ __forceinline__ void read_values(const ReadArgs &a, uint32_t block, uint32_t head, int *err) {
    constexpr uint32_t kLanes = D / 4, kUnits = 256 / kLanes;
    __shared__ int32_t slots[kWindow * kUnits];
    const uint32_t li = threadIdx.x % kLanes, mine = threadIdx.x / kLanes, ps = a.c.page_size, t0 = block * kWindow * kUnits;
    if (threadIdx.x < kWindow * kUnits) slots[threadIdx.x] = slot_read(a, t0 + threadIdx.x, head == 0 && !a.k, err);
    __syncthreads();
    int32_t slot[kWindow], first = -1, last = -1;  // first, last: runs
    bool two = true;
#pragma unroll
    for (int i = 0; i < static_cast<int>(kWindow); ++i) {
        slot[i] = slots[kWindow * mine + i];
        if (slot[i] >= 0) last = slot[i] / 16;
    }
#pragma unroll
    for (int i = kWindow - 1; i >= 0; --i)
        if (slot[i] >= 0) first = slot[i] / 16;
    if (first < 0) return;
#pragma unroll
    for (int i = 0; i < static_cast<int>(kWindow); ++i) two &= slot[i] < 0 || slot[i] / 16 == first || slot[i] / 16 == last;
    auto unit_of = [&](int32_t run) { return static_cast<uint64_t>(static_cast<uint32_t>(run) / (ps / 16)) * a.c.kv_heads + head; };
    auto codes_of = [&](int32_t run) {
        return static_cast<const uint8_t *>(a.c.v) + (unit_of(run) * D + 4 * li) * ps + static_cast<uint32_t>(run) % (ps / 16) * 16;
    };
    bool bad = false;
    auto write = [&](int i, uint32_t code, float scale) {
        const f32x4 v = value4<FMT>(code) * scale;
        bad |= !fits<T>(v);
        store4(row_read<T>(a, true, t0 + kWindow * mine + i, head, 4 * li), v);
    };
    if (two) {
        u32x4 code[2][4];
        const uint8_t *p = codes_of(first), *q = codes_of(last);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            code[0][j] = *reinterpret_cast<const u32x4 *>(p + j * ps);
            code[1][j] = *reinterpret_cast<const u32x4 *>(q + j * ps);
        }
        const float scale[2] = {a.c.v_scale[unit_of(first)], a.c.v_scale[unit_of(last)]};
#pragma unroll
        for (int i = 0; i < static_cast<int>(kWindow); ++i) {
            if (slot[i] < 0) continue;
            const bool far = slot[i] / 16 != first;
            const uint32_t place = static_cast<uint32_t>(slot[i]) % 16, byte = place % 4;
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const u32x4 c = far ? code[1][j] : code[0][j];
                const uint32_t low = place & 4 ? c[1] : c[0], high = place & 4 ? c[3] : c[2];
                w[j] = place & 8 ? high : low;
            }
            const uint32_t pick = byte | (byte + 4) << 8 | 0x0c0c0000u;
            write(i, perm(w[1], w[0], pick) | perm(w[3], w[2], pick) << 16, far ? scale[1] : scale[0]);
        }
    } else {
        uint32_t code[kWindow];
        float scale[kWindow];
#pragma unroll
        for (int i = 0; i < static_cast<int>(kWindow); ++i) {
            const int32_t at = slot[i] < 0 ? 16 * first : slot[i];
            const uint8_t *p = codes_of(at / 16) + at % 16;
            code[i] = p[0] | p[ps] << 8 | p[2 * ps] << 16 | static_cast<uint32_t>(p[3 * ps]) << 24;
            scale[i] = a.c.v_scale[unit_of(at / 16)];
        }
#pragma unroll
        for (int i = 0; i < static_cast<int>(kWindow); ++i)
            if (slot[i] >= 0) write(i, code[i], scale[i]);
    }
    if (bad) raise_error(err, kErrNonfinite);
}
// The blocks of the values, then those of the keys.
template <typename T, int FMT, int D>
__global__ __launch_bounds__(256) void k_read8(ReadArgs a, uint32_t value_blocks, uint32_t key_blocks, int *err) {
    const uint32_t values = value_blocks * a.c.kv_heads;
    if (blockIdx.x < values) read_values<T, FMT, D>(a, blockIdx.x % value_blocks, blockIdx.x / value_blocks, err);
    else read_keys<T, FMT, D>(a, (blockIdx.x - values) % key_blocks, (blockIdx.x - values) / key_blocks, err);
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

// A step's rotation and both appends in one launch: rotated keys go into codes without a pass through memory, and a step of 32
// requests takes 4.4 us (two launches 8.1).  6030 tokens of 32 + 2 x 8 heads of 128, bf16, take 42 us from and to HBM, 130 MB, 3.1 TB/s (33
// where the last-level cache has them), and without norms 36 (27): between them stand the norms' sums and products in binary64, whose issue
// is the bound.  In binary32 55 us, 4.6 TB/s.
// More workgroups to a token's heads are slower (twice as many 45 us: each makes the cosines again).
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

template <typename T, int D>
int read_typed(const ReadArgs &a, int *err, hipStream_t s) {
    const uint32_t heads = a.c.kv_heads;
    if (a.c.format == PRISM_CACHE_E2M1) {
        const uint32_t rows = 256 / (D / 8);
        const dim3 grid((a.tokens + rows - 1) / rows, (a.k ? heads : 0) + (a.v ? heads : 0));
        k_read4<T, D><<<grid, 256, 0, s>>>(a, err);
        return launch_status();
    }
    constexpr uint32_t key_tokens = 256 / (D / 8), value_tokens = kWindow * 256 / (D / 4);
    const uint32_t keys = a.k ? (a.tokens + key_tokens - 1) / key_tokens : 0, values = a.v ? (a.tokens + value_tokens - 1) / value_tokens : 0;
    const uint32_t grid = (keys + values) * heads;
    if (a.c.format == PRISM_CACHE_INT8) k_read8<T, kInt8, D><<<grid, 256, 0, s>>>(a, values, keys, err);
    else k_read8<T, kE4m3, D><<<grid, 256, 0, s>>>(a, values, keys, err);
    return launch_status();
}
template <typename T>
int read_headed(const ReadArgs &a, int *err, hipStream_t s) {
    switch (a.c.head_dim) {
    case 64: return read_typed<T, 64>(a, err, s);
    case 128: return read_typed<T, 128>(a, err, s);
    case 256: return read_typed<T, 256>(a, err, s);
    default: return kLaunchUnsupported;
    }
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
    if (dtype == PRISM_DTYPE_F32) return read_headed<float>(a, err, s);
    if (dtype == PRISM_DTYPE_F16) return read_headed<_Float16>(a, err, s);
    return read_headed<__bf16>(a, err, s);
}

}  // namespace prism
