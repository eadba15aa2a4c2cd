// rope_rows.hpp -- rotary positions of rows, into memory (kvcache.hip) or on into the 4-bit cache (kvcache4.hip).
#pragma once

#include <type_traits>

#include "cache4.hpp"

namespace prism {

namespace {

// A workgroup rotates kRopeTokens tokens of some heads, a wavefront one token: the workgroup makes
// their cosines and sines in binary64 first (one pair of them serves every head), then each lane
// keeps those of its four pairs and takes the heads, several rows in flight.  binary64 FMAs
// run at the binary32 rate here, so the exact rotation costs no more than a rounded one.  Memory
// bounds it without norms: from and to HBM 4099 tokens x 24 heads of 256 bf16, interleaved, take 26 us, 3.9 TB/s, 8192 x 40 of
// 128 37 us, 4.5 TB/s (a lane with four elements that looked their partners up, one row in flight: 56 and 137).  Norms, whose
// sums, roots and products are binary64 too, make them 29 and 41 us.

constexpr uint32_t kRopeTokens = 4;

__device__ __forceinline__ void rope_table(double (*cs)[128], double (*sn)[128], const Rotation &rot, const int32_t *positions,
                                           uint32_t nt) {
    const uint32_t half = rot.dims / 2;
    for (uint32_t i = threadIdx.x; i < nt * half; i += 256) {
        const uint32_t t = i / half, k = i % half;
        double s, c;
        sincos(static_cast<double>(positions[t]) * rot.freq[k], &s, &c);
        cs[t][k] = c * rot.magnitude;
        sn[t][k] = s * rot.magnitude;
    }
    __syncthreads();
}

// A lane's value of another lane of its 16, without LDS.
template <int CTRL>
__device__ __forceinline__ double of_lane(double v) {
    const u32x2 w = __builtin_bit_cast(u32x2, v);
    return __builtin_bit_cast(double, u32x2{static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(w[0]), CTRL, 15, 15, true)),
                                            static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(w[1]), CTRL, 15, 15, true))});
}
constexpr int quad(int a, int b, int c, int d) { return a | b << 2 | c << 4 | d << 6; }
// The sum over LANES neighbours, the same in all of them: those of a pair, of a quad, mirrored quads, mirrored eights.
template <uint32_t LANES>
__device__ __forceinline__ double row_sum(double q) {
    q += of_lane<quad(1, 0, 3, 2)>(q);
    q += of_lane<quad(2, 3, 0, 1)>(q);
    q += of_lane<0x141>(q);
    if constexpr (LANES > 8) q += of_lane<0x140>(q);
    if constexpr (LANES > 16) q += __shfl_xor(q, 16);
    return q;
}

// The largest magnitude of eight values, NaN if one is.
__device__ __forceinline__ float most_of(f32x4 a, f32x4 b) {
    f32x4 m = __builtin_elementwise_maximum(__builtin_elementwise_abs(a), __builtin_elementwise_abs(b));
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(m[0], m[1]), __builtin_elementwise_maximum(m[2], m[3]));
}
// The least magnitude that rounds to an infinity of the type.
template <typename T>
constexpr float kPast = sizeof(T) == 4 ? __builtin_inff() : std::is_same_v<T, _Float16> ? 65520.0f : 0x1.ffp127f;

// dims a multiple of 8: a lane has four pairs of a row (four elements of each half, or eight
// neighbours where interleaved), or eight elements behind the rotated ones.
// APPEND: where b's rows and a third tensor's go instead of memory: nowhere else (NoAppend), or into the cache of 4 bits a value
// (Append4Args, whose v are the third, as they are): a row's values pass through LDS, so that eight neighbours are a lane's.
template <typename T, int D, bool INTERLEAVED, typename APPEND>
__global__ __launch_bounds__(256) void k_rope(RopeRows a, RopeRows b, Rotation rot, const int32_t *positions, uint32_t tokens,
                                              uint32_t heads_each, double eps, APPEND into, int *err) {
    constexpr bool kAppends = !std::is_same_v<APPEND, NoAppend>;
    constexpr uint32_t kLanes = D / 8, kRows = 64 / kLanes;  // lanes of a row, rows of a wavefront
    constexpr uint32_t kFlight = 4;                          // row groups whose loads are in flight together
    __shared__ double cs[kRopeTokens][128], sn[kRopeTokens][128];
    __shared__ float row[kAppends ? 4 : 1][64 * 8];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64, half = rot.dims / 2;
    const uint32_t t0 = blockIdx.x * kRopeTokens, nt = min(kRopeTokens, tokens - t0);
    rope_table(cs, sn, rot, positions + t0, nt);
    if (wave >= nt) return;
    const uint32_t li = lane % kLanes, t = t0 + wave;
    const bool turns = 8 * li < rot.dims;
    // This lane's two runs of four elements.
    const uint32_t e0 = INTERLEAVED || !turns ? 8 * li : 4 * li, e1 = INTERLEAVED || !turns ? e0 + 4 : e0 + half;
    double c[4], s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        c[j] = turns ? cs[wave][4 * li + j] : 1.0;
        s[j] = turns ? sn[wave][4 * li + j] : 0.0;
    }
    const uint32_t h0 = blockIdx.y * heads_each, h1 = min(a.heads + b.heads + rows_of(into), h0 + heads_each);
    bool bad = false, over = false;
    int32_t slot = -1;
    if constexpr (kAppends) {
        bool there;
        slot = slot_of(into, t, &there);
        if (!there && lane + h0 == 0) raise_error(err, kErrIndex);
    }
    // The heads of a, then those of b.
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const RopeRows &m = which ? b : a;
        const uint32_t from = which ? max(h0, a.heads) - a.heads : h0;
        const uint32_t to = which ? (h1 > a.heads ? min(h1 - a.heads, b.heads) : 0) : min(h1, a.heads);
        if (from >= to) continue;
        f32x4 w0{1, 1, 1, 1}, w1{1, 1, 1, 1};
        if (m.norm) w0 = load4(m.norm + e0), w1 = load4(m.norm + e1);
        const T *x = static_cast<const T *>(m.x) + t * m.x_stride;
        T *out = static_cast<T *>(m.out) + t * m.out_stride;
        // Row groups whose heads are all there run without a condition; the rest of them (all, where a token has
        // few heads) leave out the missing ones.  Conditions everywhere cost 24 -> 29 us for 24 heads of
        // 256, none 64 us instead of 34 for 3 + 1 heads of 64.
        auto rows = [&](uint32_t base, auto whole) {
            const uint32_t h = base + lane / kLanes;
            typedef uint32_t Raw __attribute__((ext_vector_type(sizeof(T))));  // four elements as they are
            Raw r0[kFlight], r1[kFlight];
#pragma unroll
            for (uint32_t u = 0; u < kFlight; ++u) {
                if (!whole && base + u * kRows >= to) break;
                const uint32_t hh = min(h + u * kRows, to - 1);
                r0[u] = load_any<Raw>(x + hh * D + e0);
                r1[u] = load_any<Raw>(x + hh * D + e1);
            }
            auto four = [](Raw r) { return __builtin_convertvector(__builtin_bit_cast(typename Four<T>::type, r), f32x4); };
            // The rows' norms: a quad's lanes take a root and a quotient each, of one row group, and hand them round (each lane
            // with all four, and sums by way of LDS: 42 -> 37 us for 6030 tokens of 48 heads of 128 into the 4-bit cache).
            static_assert(kFlight == 4);
            double root = 0.0;
            if (m.norm) {
                double mine = 0.0;
#pragma unroll
                for (uint32_t u = 0; u < kFlight; ++u) {
                    if (!whole && base + u * kRows >= to) break;
                    double q = 0.0;
                    const f32x4 v0 = four(r0[u]), v1 = four(r1[u]);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const double y = j < 4 ? v0[j] : v1[j - 4];
                        q = __builtin_fma(y, y, q);
                    }
                    q = row_sum<kLanes>(q);
                    if (u == 0 || li % 4 == u) mine = q;
                }
                root = 1.0 / sqrt(mine / D + eps);
            }
#pragma unroll
            for (uint32_t u = 0; u < kFlight; ++u) {
                if (!whole && base + u * kRows >= to) break;
                asm volatile("" : "+v"(r0[u]), "+v"(r1[u]));  // their binary64 forms are made again: kept, they would take 64 registers
                const f32x4 v0 = four(r0[u]), v1 = four(r1[u]);
                bad |= !(most_of(v0, v1) < __builtin_inff());
                double y[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    y[j] = v0[j];
                    y[4 + j] = v1[j];
                }
                if (m.norm) {
                    const double scale = u == 0   ? of_lane<quad(0, 0, 0, 0)>(root)
                                         : u == 1 ? of_lane<quad(1, 1, 1, 1)>(root)
                                         : u == 2 ? of_lane<quad(2, 2, 2, 2)>(root)
                                                  : of_lane<quad(3, 3, 3, 3)>(root);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        y[j] = y[j] * scale * static_cast<double>(w0[j]);
                        y[4 + j] = y[4 + j] * scale * static_cast<double>(w1[j]);
                    }
                }
                f32x4 o0, o1;
                if (turns) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const double p = INTERLEAVED ? y[2 * j] : y[j], q = INTERLEAVED ? y[2 * j + 1] : y[4 + j];
                        const float f = static_cast<float>(__builtin_fma(p, c[j], -(q * s[j])));
                        const float g = static_cast<float>(__builtin_fma(q, c[j], p * s[j]));
                        if constexpr (INTERLEAVED) (j < 2 ? o0 : o1)[2 * (j & 1)] = f, (j < 2 ? o0 : o1)[2 * (j & 1) + 1] = g;
                        else o0[j] = f, o1[j] = g;
                    }
                } else {  // as they are: a turn by nothing would lose a zero's sign, and an infinity's neighbours
#pragma unroll
                    for (int j = 0; j < 4; ++j) o0[j] = static_cast<float>(y[j]), o1[j] = static_cast<float>(y[4 + j]);
                }
                over |= !(most_of(o0, o1) < kPast<T>);
                if constexpr (kAppends) {
                    if (which) {
                        if (slot < 0 || h + u * kRows >= to) continue;  // whole rows
                        float *mine = row[wave] + lane / kLanes * D;
                        o0 = rounded<T>(o0), o1 = rounded<T>(o1);
                        *reinterpret_cast<f32x4 *>(mine + e0) = o0;
                        *reinterpret_cast<f32x4 *>(mine + e1) = o1;
                        settle();
                        o0 = *reinterpret_cast<const f32x4 *>(mine + 8 * li), o1 = *reinterpret_cast<const f32x4 *>(mine + 8 * li + 4);
                        settle();
                        write_codes4<D>(into.c, false, h + u * kRows, static_cast<uint32_t>(slot), li, o0, o1, &bad, &over);
                        continue;
                    }
                }
                if (h + u * kRows < to) {
                    store4(out + (h + u * kRows) * D + e0, o0);
                    store4(out + (h + u * kRows) * D + e1, o1);
                }
            }
        };
        uint32_t base = from;
        for (; base + (kFlight - 1) * kRows < to; base += kRows * kFlight) rows(base, std::true_type());
        if (base < to) rows(base, std::false_type());
    }
    if constexpr (kAppends) {
        const uint32_t from = max(h0, a.heads + b.heads) - a.heads - b.heads, to = h1 > a.heads + b.heads ? h1 - a.heads - b.heads : 0;
        const T *x = static_cast<const T *>(into.v) + t * into.v_stride + 8 * li;
        if (slot >= 0)
            for (uint32_t base = from; base < to; base += kFlight * kRows) {
                f32x4 v0[kFlight], v1[kFlight];
#pragma unroll
                for (uint32_t u = 0; u < kFlight; ++u) {
                    const uint32_t h = min(base + u * kRows + lane / kLanes, to - 1);
                    v0[u] = load4(x + h * D);
                    v1[u] = load4(x + h * D + 4);
                }
#pragma unroll
                for (uint32_t u = 0; u < kFlight; ++u) {
                    const uint32_t h = base + u * kRows + lane / kLanes;
                    if (h < to) write_codes4<D>(into.c, true, h, static_cast<uint32_t>(slot), li, v0[u], v1[u], &bad, &over);
                }
            }
    }
    if (bad) raise_error(err, kErrInput);
    if (over) raise_error(err, kErrNonfinite);
}

}  // namespace

}  // namespace prism
