// paged_attention4.hip -- grouped-query attention over the paged cache of 4 bits a value (gfx950).
//
// Codes are e2m1 with a power of two for each 32 dimensions of a key, so keys and values are exact in binary16.
#include "attend_common.hpp"

namespace prism {

namespace {

__device__ __forceinline__ float level(uint32_t code) {
    const float v[8] = {0.0f, 0.5f, 1.0f, 1.5f, 2.0f, 3.0f, 4.0f, 6.0f};
    return code & 8 ? -v[code & 7] : v[code & 7];
}

// A wavefront has one row: its lanes the keys for the scores, the dimensions for the sums.
template <typename T, int D>
__global__ __launch_bounds__(64) void k_attend4_row(AttendArgs p, int *err) {
    __shared__ float q[D], prob[64];
    __shared__ int32_t where[64];
    const uint32_t lane = threadIdx.x, token = blockIdx.x, head = blockIdx.y, kvh = head / p.group;
    if (token + head == 0)
        for (uint32_t i = lane; i < p.a.requests; i += 64)
            if (request_of(p, i).bad) raise_error(err, kErrIndex);
    uint32_t r = 0;
    Request rq{};
    for (; r < p.a.requests; ++r) {
        rq = request_of(p, r);
        if (!rq.bad && token >= rq.first && token < rq.first + rq.n) break;
    }
    if (r == p.a.requests) return;
    int32_t lo, hi;
    visible(p, rq, token - rq.first, &lo, &hi);
    const uint32_t ps = p.c.page_size;
    const int32_t *table = p.a.block_table + static_cast<uint64_t>(r) * p.a.max_pages;
    const T *src = static_cast<const T *>(p.a.q) + token * p.a.q_stride + static_cast<uint64_t>(head) * D;
    for (uint32_t i = lane; i < D; i += 64) q[i] = static_cast<float>(src[i]);
    __syncthreads();
    float m = kNone, l = 0.0f, acc[D / 64] = {};
    for (int32_t base = lo; base < hi; base += 64) {
        const int32_t key = base + static_cast<int32_t>(lane);
        int32_t slot = -1;
        float z = kNone;
        if (key < hi) {
            const int32_t page = table[key >> p.page_log2];
            if (static_cast<uint32_t>(page) >= p.c.pages) raise_error(err, kErrIndex);
            else slot = page * static_cast<int32_t>(ps) + (key & static_cast<int32_t>(ps - 1));
        }
        if (slot >= 0) {
            const uint32_t place = slot % ps;
            const uint64_t unit = static_cast<uint64_t>(slot / ps) * p.c.kv_heads + kvh;
            const uint8_t *codes = static_cast<const uint8_t *>(p.c.k) + (unit * ps + place) * (D / 2);
            float sum = 0.0f;
            for (uint32_t g = 0; g < D / 32; ++g) {
                float part = 0.0f;
                for (uint32_t i = 0; i < 16; ++i) {
                    const uint32_t c = codes[16 * g + i];
                    part += q[32 * g + 2 * i] * level(c & 15) + q[32 * g + 2 * i + 1] * level(c >> 4);
                }
                sum += part * __uint_as_float(static_cast<uint32_t>(p.c.k_exponent[(unit * (D / 32) + g) * ps + place]) << 23);
            }
            z = sum * p.a.scale * kLog2e;
        }
        float top = z;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
        const float next = fmaxf(m, top), ref = next == kNone ? 0.0f : next;
        const float alpha = __builtin_amdgcn_exp2f(m - ref), e = __builtin_amdgcn_exp2f(z - ref);
        m = next;
        l = l * alpha + e;
        __syncthreads();
        prob[lane] = e;
        where[lane] = slot;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < D / 64; ++i) acc[i] *= alpha;
        for (int j = 0; j < 64; ++j) {
            const int32_t at = where[j];
            if (at < 0) continue;
            const uint32_t place = at % ps;
            const uint64_t unit = static_cast<uint64_t>(at / ps) * p.c.kv_heads + kvh;
#pragma unroll
            for (int i = 0; i < D / 64; ++i) {
                const uint32_t d = lane + 64 * i;
                const uint32_t c = static_cast<const uint8_t *>(p.c.v)[(unit * ps + place) * (D / 2) + d / 2];
                const uint32_t x = p.c.v_exponent[(unit * (D / 32) + d / 32) * ps + place];
                acc[i] += prob[j] * (level(d & 1 ? c >> 4 : c & 15) * __uint_as_float(x << 23));
            }
        }
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) l += __shfl_xor(l, d);
    T *out = static_cast<T *>(p.a.out) + token * p.a.out_stride + static_cast<uint64_t>(head) * D;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
        const T v = static_cast<T>(l == 0.0f ? 0.0f : acc[i] / l);
        bad |= !finite(static_cast<float>(v));
        out[lane + 64 * i] = v;
    }
    if (bad) raise_error(err, kErrNonfinite);
}

template <typename T>
int attend4_headed(const AttendArgs &p, int *err, hipStream_t s) {
    const dim3 grid(p.a.tokens, p.a.heads);
    switch (p.c.head_dim) {
    case 64: k_attend4_row<T, 64><<<grid, 64, 0, s>>>(p, err); break;
    case 128: k_attend4_row<T, 128><<<grid, 64, 0, s>>>(p, err); break;
    case 256: k_attend4_row<T, 256><<<grid, 64, 0, s>>>(p, err); break;
    default: return kLaunchUnsupported;
    }
    return launch_status();
}

}  // namespace

size_t attention4_scratch_bytes(const prism_kv_cache &, const prism_attention &, uint32_t) { return 0; }

int launch_attention4_paged(const prism_kv_cache &c, const prism_attention &a, void *, uint32_t, int *err, hipStream_t s) {
    AttendArgs p{c, a, a.heads / c.kv_heads, static_cast<uint32_t>(__builtin_ctz(c.page_size)), 0, 0, 1, nullptr, nullptr};
    if (a.dtype == PRISM_DTYPE_F32) return attend4_headed<float>(p, err, s);
    if (a.dtype == PRISM_DTYPE_F16) return attend4_headed<_Float16>(p, err, s);
    return attend4_headed<__bf16>(p, err, s);
}

}  // namespace prism
