// paged_attention.hip -- grouped-query attention over the paged 8-bit cache (gfx950), for
// single tokens, chunks and prompts of many requests in one call.
//
// A request's queries of one kv head form rows (token, head of the group); a wavefront takes
// 16 * NT of them through blocks of 64 keys with the running maximum and sum of the softmax:
//   S^T = K Q^T   K codes (exact in binary16) as the A operand, 16 keys a matrix instruction
//   z = S * (scale * k_scale) + log2 v_scale, p = 2^(z - m), l = sum p / v_scale
//   O^T += V^T P^T
// so a page's two scales cost nothing per key: the keys' joins the softmax scale, the values'
// the exponent, and p stays within the operand's range however the pages' scales differ.
//
// Keys are assigned to the rows of K's matrix instructions so that a lane's 16 scores of a
// block are 16 consecutive keys, all of one page: they are the B operand of the second product
// as they stand (no exchange between lanes), and one 16-byte load of the transposed values
// is the A operand that meets them.
#include <type_traits>

#include "serve_common.hpp"

namespace prism {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
// Probabilities enter the second product as 2^11 2^(z - m), with m at most kSlack below the largest z
// (rows are rescaled only where it grew by more): at most 2^15.  One binary16 part has its full precision, half a step of
// 2^-11, for contributions down to 2^-25 of the largest, two have theirs, 2^-22, down to 2^-14; below, and in all, the
// error is at most 2^-36 of the largest.  One part rounds a 16-bit result's terms no more than the result is rounded.
constexpr float kHeadroom = 11.0f, kSlack = 4.0f;
constexpr float kNone = -__builtin_inff();
// The denominator l is held times 2^-12 relative to the numerator.  A key's term of it is 2^(S - m + 11 - 12): with value
// scales of 2^-100 to 2^122, as the append makes them, S - m of the largest term is between -122 and 104, so
// neither the smallest sum leaves binary32's normal numbers nor that of 2^24 keys its range.
constexpr float kSumShift = 12.0f, kSumUnit = 0x1p-12f;
// While every value scale met is within 2^+-40, the largest p of a row and those of keys that matter to l are less than
// 2^100 apart, and l takes a key's p over the scale.  Past that p may vanish where the key's weight does not (a page of
// zeros, scale 2^-100, beside one of 2^38): from there on l's terms are exponentials of their own, relative to the largest
// S the lane has met (a reference of its own, in LDS: no register is left for it) until the keys are done.  Looking for
// such scales costs a prompt 1.4 % (627 -> 636 us); a second copy of the loop for them cost long caches and chunks 3 to 8 %.
constexpr float kWide = 40.0f;

struct AttendArgs {
    prism_kv_cache c;
    prism_attention a;
    uint32_t group, page_log2;
    uint32_t slots;     // row tiles, at most (tile_request)
    uint32_t each;      // key blocks of 64 a part of a tile's keys has, at least
    uint32_t splits;    // parts, at most
    float *part;        // [splits][tokens * heads][head_dim] unnormalised rows
    float *part_ml;     // [splits][tokens * heads][2]: maximum (base 2), sum
};

struct Request {
    uint32_t first, n;      // its tokens
    uint32_t length;        // its keys
    bool bad;
};
__device__ __forceinline__ Request request_of(const AttendArgs &p, uint32_t r) {
    const int32_t o0 = p.a.offsets[r], o1 = p.a.offsets[r + 1];
    const int32_t len = p.a.lengths[r];
    const int64_t room = static_cast<int64_t>(p.a.max_pages) << p.page_log2;
    Request q;
    q.bad = o0 < 0 || o1 < o0 || static_cast<uint32_t>(o1) > p.a.tokens || len < 0 || len > room;
    q.first = q.bad ? 0 : o0;
    q.n = q.bad ? 0 : o1 - o0;
    q.length = q.bad ? 0 : len;
    return q;
}
// Keys [lo, hi) that token i of the request sees.
__device__ __forceinline__ void visible(const AttendArgs &p, const Request &q, uint32_t i, int32_t *lo, int32_t *hi) {
    *lo = 0;
    *hi = static_cast<int32_t>(q.length);
    if (!p.a.causal) return;
    const int32_t at = static_cast<int32_t>(q.length) - static_cast<int32_t>(q.n) + static_cast<int32_t>(i);
    *hi = at + 1 > 0 ? at + 1 : 0;
    if (p.a.window && at + 1 > static_cast<int64_t>(p.a.window)) *lo = at + 1 - static_cast<int32_t>(p.a.window);
}
// The 64-key blocks [b0, b1) any of the request's tokens i0 .. i1 sees, and the parts they are split into.
__device__ __forceinline__ void blocks_of(const AttendArgs &p, const Request &q, uint32_t i0, uint32_t i1, uint32_t *b0,
                                          uint32_t *b1) {
    int32_t lo, hi, x;
    visible(p, q, i0, &lo, &x);
    visible(p, q, i1, &x, &hi);
    *b0 = static_cast<uint32_t>(lo) / 64;
    *b1 = hi > lo ? (static_cast<uint32_t>(hi) + 63) / 64 : *b0;
}
__device__ __forceinline__ uint32_t part_blocks(const AttendArgs &p, uint32_t blocks) {
    return max(p.each, (blocks + p.splits - 1) / p.splits);
}
__device__ __forceinline__ uint32_t parts_of(const AttendArgs &p, uint32_t blocks) {
    const uint32_t each = part_blocks(p, blocks);
    return blocks <= each ? 1 : (blocks + each - 1) / each;
}

// Tiles of M rows: request r has the slots from offsets[r] * group / M + r on, at least as
// many as it needs and in ascending order, so no sums over the requests are needed first.
__device__ __forceinline__ uint32_t tile_start(const AttendArgs &p, uint32_t r, uint32_t M) {
    const int32_t o = p.a.offsets[r];
    const uint64_t tokens = o < 0 ? 0 : static_cast<uint32_t>(o) > p.a.tokens ? p.a.tokens : static_cast<uint32_t>(o);
    return static_cast<uint32_t>(tokens * p.group / M) + r;
}
__device__ __forceinline__ uint32_t tile_request(const AttendArgs &p, uint32_t slot, uint32_t M) {
    // The last r with tile_start(r) <= slot, 64 candidates at a time.
    uint32_t lo = 0, n = p.a.requests;
    const uint32_t lane = threadIdx.x & 63;
    while (n > 1) {
        const uint32_t step = (n + 63) / 64, k = lane * step;
        const bool at = k < n && tile_start(p, lo + k, M) <= slot;
        const uint64_t on = __ballot(at);
        const uint32_t j = on ? 63 - __builtin_clzll(on) : 0;
        n = min(step, n - j * step);
        lo += j * step;
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

// Eight codes of two dwords as binary16.
template <int FMT>
__device__ __forceinline__ f16x8 halves(uint32_t a, uint32_t b) {
    union {
        uint32_t u[4];
        f16x2 h[4];
        f16x8 v;
    } r;
    if constexpr (FMT == kInt8) {
        // 0x6400 | (code + 128) is 1024 + code + 128.
        a ^= 0x80808080u;
        b ^= 0x80808080u;
        r.u[0] = perm(0x64646464u, a, 0x04010400u);
        r.u[1] = perm(0x64646464u, a, 0x04030402u);
        r.u[2] = perm(0x64646464u, b, 0x04010400u);
        r.u[3] = perm(0x64646464u, b, 0x04030402u);
        const f16x2 off = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
#pragma unroll
        for (int i = 0; i < 4; ++i) r.h[i] += off;
    } else {
        r.h[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(a), 1.0f, false);
        r.h[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(a), 1.0f, true);
        r.h[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(b), 1.0f, false);
        r.h[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(b), 1.0f, true);
    }
    return r.v;
}

__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// Over the four lanes of a row: lane groups 0 and 1, 2 and 3 exchange, then the halves of the wavefront.
__device__ __forceinline__ float across_max(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float across_sum(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int32_t uniform(int32_t v) { return __builtin_amdgcn_readfirstlane(v); }

template <typename T>
__device__ __forceinline__ void write_row(const AttendArgs &p, uint32_t token, uint32_t head, uint32_t dim, f32x4 v, bool *bad) {
    *bad |= !fits<T>(v);
    store4(static_cast<T *>(p.a.out) + token * p.a.out_stride + static_cast<uint64_t>(head) * p.c.head_dim + dim, v);
}

// The lane, made where it is used (the mask is opaque, so it is not made ahead): no register holds it meanwhile.
__device__ __forceinline__ uint32_t this_lane() {
    uint32_t all = ~0u;
    asm volatile("" : "+s"(all));
    return __builtin_amdgcn_mbcnt_hi(all, __builtin_amdgcn_mbcnt_lo(all, 0u));
}
// The sum l of a row whose reference goes up by -by: by 2^by, as its numerator, so that the rounding of 2^by cancels, and in
// two steps where 2^by nears the smallest normal number and the sum need not.
__device__ __forceinline__ float scaled_sum(float l, float by) {
    const bool deep = by < -100.0f;
    const float f = __builtin_amdgcn_exp2f(deep ? 0.5f * by : by);
    return l * f * (deep ? f : 1.0f);
}
// What takes the numerator to the row (past 2^114, tens of thousands of keys with values below 2^-93, with fewer bits).
__device__ __forceinline__ float inverse(float l) { return l == 0.0f ? 0.0f : kSumUnit / l; }

// What both kernels below share: a wavefront's 16 * NT rows, their queries, statistics and sums.
// T: type of q and out; LIMBS: binary16 parts of q and of the probabilities (2 for binary32).
template <typename T, int D, int FMT, int NT>
struct Rows {
    static constexpr int LIMBS = sizeof(T) == 4 ? 2 : 1;
    static constexpr int KS = D / 32, DT = D / 16;
    uint32_t token[NT], head[NT];  // of this lane's rows
    bool live[NT];
    int32_t lo[NT], hi[NT];        // the keys they see
    int32_t all_lo, all_hi;        // keys every row of the wavefront sees
    int32_t any_lo, any_hi;        // keys any row sees
    float kf[NT];                  // base-2 softmax scale of the row's integer-like queries, not negative
    f16x8 qv[LIMBS][NT][KS];
    float m[NT], l[NT];
    bool wide = false;             // a value scale past kWide has been met (the same in all lanes)
    f32x4 acc[NT][DT];

    __device__ __forceinline__ void load(const AttendArgs &p, const Request &q, uint32_t base_row, uint32_t last, uint32_t kvh) {
        const uint32_t lane = threadIdx.x & 63, n = lane & 15, g = lane / 16;
        all_lo = 0, all_hi = 0x7fffffff, any_lo = 0x7fffffff, any_hi = 0;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const uint32_t row = base_row + 16 * t + n;
            live[t] = row <= last;
            const uint32_t rr = live[t] ? row : last, i = rr / p.group;
            token[t] = q.first + i;
            head[t] = kvh * p.group + rr % p.group;
            visible(p, q, i, &lo[t], &hi[t]);
            all_lo = max(all_lo, lo[t]);
            all_hi = min(all_hi, hi[t]);
            any_lo = min(any_lo, lo[t]);
            any_hi = max(any_hi, hi[t]);
            // Lane group g has the dimensions [g D/4, (g + 1) D/4) of the row.
            const T *src = static_cast<const T *>(p.a.q) + token[t] * p.a.q_stride + static_cast<uint64_t>(head[t]) * D + g * (D / 4);
            f32x4 x[D / 16];
            float most = 0.0f;
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
                x[j] = load4(src + 4 * j);
#pragma unroll
                for (int k = 0; k < 4; ++k) most = fmaxf(most, fabsf(x[j][k]));
            }
            most = across_max(most);
            // A power of two, at most 2^113, takes the row's largest value to [2^13, 2^14); the sign of the scale goes along.
            int e = static_cast<int>(__float_as_uint(most) >> 23 & 255) - 127;
            e = !finite(most) ? 0 : max(e, -100);
            float up = __uint_as_float(static_cast<uint32_t>(127 + 13 - e) << 23);
            if (p.a.scale < 0.0f) up = -up;
            kf[t] = fabsf(p.a.scale) * kLog2e * __uint_as_float(static_cast<uint32_t>(127 - 13 + e) << 23);
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float v = x[2 * s + j / 4][j % 4] * up;
                    const _Float16 h = static_cast<_Float16>(v);
                    qv[0][t][s][j] = h;
                    if constexpr (LIMBS == 2) qv[LIMBS - 1][t][s][j] = static_cast<_Float16>(v - static_cast<float>(h));
                }
            m[t] = kNone;
            l[t] = 0.0f;
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[t][d] = f32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int d = 1; d < 16; d *= 2) {
            all_lo = max(all_lo, __shfl_xor(all_lo, d));
            all_hi = min(all_hi, __shfl_xor(all_hi, d));
            any_lo = min(any_lo, __shfl_xor(any_lo, d));
            any_hi = max(any_hi, __shfl_xor(any_hi, d));
        }
        all_lo = uniform(all_lo), all_hi = uniform(all_hi), any_lo = uniform(any_lo), any_hi = uniform(any_hi);
    }

    // Scores s of the lane's 16 keys from `key` on are masked and the statistics follow their maximum; p = 2^(s ff + off).
    // ks, vs: the scales of their page; edge: some row does not see some key of the block; ref: the lanes' references of l.
    __device__ __forceinline__ void scores(f32x4 (&s)[NT][4], float ks, float vs, bool there, bool edge, int32_t key, float (&ff)[NT],
                                           float (&off)[NT], float (*ref)[64]) {
        const float lv = __builtin_amdgcn_logf(vs);
        float f[NT], top[NT];
        bool grows = false;
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            if (edge)
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int32_t k = key + 4 * t + i;
                        s[u][t][i] = there && k >= lo[u] && k < hi[u] ? s[u][t][i] : kNone;
                    }
            f[u] = kf[u] * ks;
            // z = s f + lv rises with s, so the largest s gives the largest z.
            float most = kNone;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) most = fmaxf(most, s[u][t][i]);
            top[u] = across_max(most == kNone ? kNone : __builtin_fmaf(most, f[u], lv));
            grows |= top[u] > m[u] + kSlack || m[u] == kNone;
        }
        if (__ballot(grows)) {
#pragma unroll
            for (int u = 0; u < NT; ++u) {
                const float next = fmaxf(m[u], top[u]);
                const float by = next == kNone ? 0.0f : m[u] - next, alpha = __builtin_amdgcn_exp2f(by);
                m[u] = next;
                l[u] = wide ? l[u] : scaled_sum(l[u], by);  // wide: l has its own reference
#pragma unroll
                for (int d = 0; d < DT; ++d) acc[u][d] *= alpha;
            }
        }
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            // A row that has seen no key yet has m = -inf, and scores of -inf.
            off[u] = lv + kHeadroom - (m[u] == kNone ? 0.0f : m[u]);
            // 0 * -inf would be NaN where a page's keys are all zero and a key is masked.
            ff[u] = f[u] < 0x1p-120f ? 0x1p-120f : f[u];
        }
        if (__builtin_expect(__ballot(fabsf(lv) > kWide) != 0 && !wide, 0)) {
            wide = true;
#pragma unroll
            for (int u = 0; u < NT; ++u) {  // l 2^(m + 1) = mantissa 2^(exponent + m + 1)
                ref[u][this_lane()] = l[u] == 0.0f ? kNone : m[u] + (kSumShift - kHeadroom) + static_cast<float>(__builtin_amdgcn_frexp_expf(l[u]));
                l[u] = __builtin_amdgcn_frexp_mantf(l[u]);
            }
        }
        if (__builtin_expect(wide, 0)) {
#pragma unroll
            for (int u = 0; u < NT; ++u) {
                const float before = ref[u][this_lane()];
                float next = before, sum = 0.0f;
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) next = fmaxf(next, s[u][t][i] * ff[u]);
                ref[u][this_lane()] = next;
                next = next == kNone ? 0.0f : next;
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum += __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][t][i], ff[u], -next));
                l[u] = __builtin_fmaf(l[u], __builtin_amdgcn_exp2f(before - next), sum);
            }
        }
    }
    // Probabilities of half `c` of the keys: an operand of the second product.
    template <int c>
    __device__ __forceinline__ void probabilities(const f32x4 (&s)[NT][4], f16x8 (&pv)[LIMBS][NT], const float (&ff)[NT],
                                                  const float (&off)[NT], float (&sum)[NT]) {
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][2 * c + j / 4][j % 4], ff[u], off[u]));
                sum[u] += e;
                const _Float16 h = static_cast<_Float16>(e);
                pv[0][u][j] = h;
                if constexpr (LIMBS == 2) pv[LIMBS - 1][u][j] = static_cast<_Float16>(e - static_cast<float>(h));
            }
    }
    __device__ __forceinline__ void add(const float (&sum)[NT], float vs) {
        const float iv = wide ? 0.0f : kSumUnit / vs;  // wide: l has the terms already
#pragma unroll
        for (int u = 0; u < NT; ++u) l[u] += sum[u] == 0.0f ? 0.0f : sum[u] * iv;
    }

    // l once the keys are done: the row's, of all four lanes, relative to m.
    __device__ __forceinline__ void total(const float (*ref)[64]) {
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            if (wide && l[u] != 0.0f) {
                const float half = __builtin_amdgcn_exp2f(0.5f * (ref[u][this_lane()] - m[u] + (kHeadroom - kSumShift)));
                l[u] = l[u] * half * half;
            }
            l[u] = across_sum(l[u]);
        }
    }

    // The rows, or with more than one part their unnormalised sums: lane (n, g) has the dimensions
    // 16 d + 4 g .. + 3 of row n.
    __device__ __forceinline__ void write(const AttendArgs &p, uint32_t parts, uint32_t split, int *err) const {
        const uint32_t g = (threadIdx.x & 63) / 16;
        bool bad = false;
        const uint64_t all_rows = static_cast<uint64_t>(p.a.tokens) * p.a.heads;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if (!live[t]) continue;
            if (parts == 1) {
                const float inv = inverse(l[t]);
#pragma unroll
                for (int d = 0; d < DT; ++d) write_row<T>(p, token[t], head[t], 16 * d + 4 * g, acc[t][d] * inv, &bad);
            } else {
                const uint64_t row = split * all_rows + static_cast<uint64_t>(token[t]) * p.a.heads + head[t];
#pragma unroll
                for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4 *>(p.part + row * D + 16 * d + 4 * g) = acc[t][d];
                if (g == 0) {
                    p.part_ml[2 * row] = m[t];
                    p.part_ml[2 * row + 1] = l[t];
                }
            }
        }
        if (bad) raise_error(err, kErrNonfinite);
    }
};

// A workgroup's tile: its request, rows and part of the key blocks; false: nothing to do.
struct Tile {
    Request q;
    uint32_t kvh, r, row0, last, b0, b1, parts;
    int32_t seen_lo, seen_hi;  // keys some row sees
};
__device__ __forceinline__ bool tile_of(const AttendArgs &p, uint32_t M, uint32_t split, int *err, Tile *t) {
    // Heavy tiles first (a prompt's last rows see the most keys), all heads' of them: the other order left the last
    // head's longest tiles for the end.  With eight kv heads each XCD's L2 also has one head's keys.
    t->kvh = uniform(blockIdx.x % p.c.kv_heads);
    const uint32_t slot = uniform(p.slots - 1 - blockIdx.x / p.c.kv_heads);
    t->r = tile_request(p, slot, M);
    t->q = request_of(p, t->r);
    t->q.first = uniform(t->q.first), t->q.n = uniform(t->q.n), t->q.length = uniform(t->q.length);
    if (blockIdx.x + blockIdx.z == 0)  // offsets out of order may leave a request without a tile
        for (uint32_t i = threadIdx.x; i < p.a.requests; i += blockDim.x)
            if (request_of(p, i).bad) raise_error(err, kErrIndex);
    const uint32_t rows = t->q.n * p.group, start = tile_start(p, t->r, M);
    t->row0 = (slot - start) * M;
    if (slot < start || t->row0 >= rows) return false;
    t->last = min(rows, t->row0 + M) - 1;
    int32_t x;
    visible(p, t->q, t->row0 / p.group, &t->seen_lo, &x);
    visible(p, t->q, t->last / p.group, &x, &t->seen_hi);
    t->seen_lo = uniform(t->seen_lo), t->seen_hi = uniform(t->seen_hi);
    uint32_t b0, b1;
    blocks_of(p, t->q, t->row0 / p.group, t->last / p.group, &b0, &b1);
    const uint32_t each = part_blocks(p, b1 - b0);
    t->parts = uniform(parts_of(p, b1 - b0));
    t->b0 = uniform(b0 + split * each);
    t->b1 = uniform(min(b1, b0 + (split + 1) * each));
    return split < t->parts;
}

// Some row of the tile sees one of the 16 keys from `key` on.  The first block of a window and the last of the
// keys also cover pages that none sees, whose columns, scales and codes may be anything.
__device__ __forceinline__ bool seen(const Tile &t, int32_t key) { return key < t.seen_hi && key > t.seen_lo - 16; }
// The table's entry for 16 keys from `key` on (the nearest seen column's where none is seen): their page, where
// they are seen and the entry is a page; else page 0 stands in and they count as masked.  Entries and scales
// are taken as loaded and looked at where they are used, blocks later.
__device__ __forceinline__ int32_t entry_at(const AttendArgs &p, const Tile &t, const int32_t *table, int32_t key) {
    return table[min(max(key, t.seen_lo), t.seen_hi - 1) >> p.page_log2];
}
__device__ __forceinline__ bool is_page(const AttendArgs &p, const Tile &t, int32_t id, int32_t key) {
    return seen(t, key) && static_cast<uint32_t>(id) < p.c.pages;
}
__device__ __forceinline__ float value_scale(float v, bool there) {  // log2 and 1 / v stay finite; NaN stays NaN
    return !there ? 1.0f : v < 0x1p-100f ? 0x1p-100f : v;
}
// Bytes behind the keys, and stand-ins, may hold NaN codes, which zero probabilities do not silence: the first `keep` of 16 stay.
__device__ __forceinline__ void keep_bytes(u32x4 &v, int32_t keep) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const int32_t left = keep - 4 * w;
        v[w] &= left >= 4 ? ~0u : left <= 0 ? 0u : (1u << (8 * left)) - 1;
    }
}

// Few rows (single tokens, drafts): the workgroup's four wavefronts share 16 * NT rows and split the
// keys.  Every code is used once, so they go from memory to registers; the cache's bytes bound it:
// 64 requests of 1 to 8192 keys (8 kv heads of 128) take 108 us, 5.0 TB/s, eight of 20001 to 65536 (4 of 256) 144.
// WIDE: byte offsets into the keys or values pass 32 bits; else a lane's address is one register
// beside a scalar base.
template <typename T, int D, int FMT, int NT, bool WIDE>
__global__ __launch_bounds__(256, D == 256 && sizeof(T) == 4 ? 1 : 2) void k_attend_rows(AttendArgs p, int *err) {
    typedef Rows<T, D, FMT, NT> R;
    constexpr int LIMBS = R::LIMBS, KS = R::KS, DT = R::DT;
    __shared__ float join_ml[4][16 * NT][2];
    __shared__ f32x4 join_acc[3][NT * DT][64];
    __shared__ float sum_ref[4][NT][64];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t n = lane & 15, g = lane / 16;
    Tile tile;
    if (!tile_of(p, 16 * NT, blockIdx.z, err, &tile)) return;
    const uint32_t kvh = tile.kvh;
    const uint32_t page_mask = p.c.page_size - 1;
    const int32_t *table = p.a.block_table + static_cast<uint64_t>(tile.r) * p.a.max_pages;
    const uint8_t *kc = static_cast<const uint8_t *>(p.c.k), *vc = static_cast<const uint8_t *>(p.c.v);
    const uint32_t kgroup = (lane >> 2) & 3;  // 16-key group whose keys this lane loads for the first product
    // Registers of codes are filled again as soon as a product has used them, the next block's keys behind the
    // first product and its values behind the second; its table entries are a block further ahead.
    // Heads of 256, and two row tiles of binary32 at 128, have no registers for that (spilled: 205 us instead of 153
    // for eight long requests, 206 instead of 91 for 24 rows a request): their codes are loaded at the
    // block's start, two wavefronts a SIMD covering each other; binary32 with heads of 256 has registers for one
    // wavefront only, and four values spilled to accumulation registers (171 us where the 16-bit types take 151).
    constexpr bool kAhead = D < 256 && !(D == 128 && NT == 2 && LIMBS == 2);
    int32_t id_k = 0, id_v = 0;
    u32x4 kraw[4][D / 64], vraw[DT];
    typedef std::conditional_t<WIDE, uint64_t, uint32_t> Offset;
    Offset v_at = 0;
    float ks_next = 0.0f, vs_next = 1.0f;
    bool there_next = false, missing = false;
    auto look = [&](uint32_t b) {
        const int32_t base = static_cast<int32_t>(64 * b);
        id_k = entry_at(p, tile, table, base + 16 * static_cast<int32_t>(kgroup));
        id_v = entry_at(p, tile, table, base + 16 * static_cast<int32_t>(g));
    };
    auto fetch_keys = [&](uint32_t b) {
        const int32_t base = static_cast<int32_t>(64 * b);
        const int32_t key_k = base + 16 * static_cast<int32_t>(kgroup), key_v = base + 16 * static_cast<int32_t>(g);
        there_next = is_page(p, tile, id_v, key_v);
        missing |= !there_next && seen(tile, key_v);
        const Offset unit_k = static_cast<Offset>(is_page(p, tile, id_k, key_k) ? id_k : 0) * p.c.kv_heads + kvh;
        const Offset unit_v = static_cast<Offset>(there_next ? id_v : 0) * p.c.kv_heads + kvh;
        ks_next = p.c.k_scale[unit_v];
        vs_next = p.c.v_scale[unit_v];
        const Offset k_at = ((unit_k << p.page_log2) + (static_cast<uint32_t>(key_k) & page_mask) + (lane & 3)) * D + g * (D / 4);
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int j = 0; j < D / 64; ++j) kraw[t][j] = *reinterpret_cast<const u32x4 *>(kc + k_at + (4 * t * D + 16 * j));
        v_at = ((unit_v * D + n) << p.page_log2) + (static_cast<uint32_t>(key_v) & page_mask);
    };
    auto fetch_values = [&] {
#pragma unroll
        for (int d = 0; d < DT; ++d)
            vraw[d] = *reinterpret_cast<const u32x4 *>(vc + (static_cast<uint64_t>(16 * d) << p.page_log2) + v_at);
    };
    const uint32_t first = tile.b0 + wave;
    if (first < tile.b1) look(first);
    R rows;
    rows.load(p, tile.q, tile.row0, tile.last, kvh);
    if (kAhead && first < tile.b1) {
        fetch_keys(first);
        fetch_values();
        if (first + 4 < tile.b1) look(first + 4);
    }
    for (uint32_t b = first; b < tile.b1; b += 4) {
        if constexpr (!kAhead) {
            fetch_keys(b);
            fetch_values();
            if (b + 4 < tile.b1) look(b + 4);
        }
        const int32_t base = static_cast<int32_t>(64 * b), key = base + 16 * static_cast<int32_t>(g);
        const bool there = there_next;
        const float ks = there ? ks_next : 0.0f, vs = value_scale(vs_next, there);
        const bool edge = base < rows.all_lo || base > rows.all_hi - 64 || __ballot(there) != ~0ull;
        f32x4 s[NT][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int u = 0; u < NT; ++u) s[u][t] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const f16x8 kv = halves<FMT>(kraw[t][k / 2][2 * (k % 2)], kraw[t][k / 2][2 * (k % 2) + 1]);
#pragma unroll
                for (int u = 0; u < NT; ++u)
#pragma unroll
                    for (int i = 0; i < LIMBS; ++i) s[u][t] = mfma(kv, rows.qv[i][u][k], s[u][t]);
            }
        }
        const bool more = kAhead && b + 4 < tile.b1;
        if (more) fetch_keys(b + 4);
        f16x8 pv[2][LIMBS][NT];
        float ff[NT], off[NT], sum[NT] = {};
        rows.scores(s, ks, vs, there, edge, key, ff, off, sum_ref[wave]);
        rows.template probabilities<0>(s, pv[0], ff, off, sum);
        rows.template probabilities<1>(s, pv[1], ff, off, sum);
        rows.add(sum, vs);
        if (edge && FMT == kE4m3)
#pragma unroll
            for (int d = 0; d < DT; ++d) keep_bytes(vraw[d], there ? tile.seen_hi - key : 0);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const f16x8 vv = halves<FMT>(vraw[d][2 * c], vraw[d][2 * c + 1]);
#pragma unroll
                for (int u = 0; u < NT; ++u)
#pragma unroll
                    for (int i = 0; i < LIMBS; ++i) rows.acc[u][d] = mfma(vv, pv[c][i][u], rows.acc[u][d]);
            }
        if (more) {
            fetch_values();
            if (b + 8 < tile.b1) look(b + 8);
        }
    }
    if (missing) raise_error(err, kErrIndex);

    // The four wavefronts' rows join in the first.
    rows.total(sum_ref[wave]);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        if (g == 0) {
            join_ml[wave][16 * t + n][0] = rows.m[t];
            join_ml[wave][16 * t + n][1] = rows.l[t];
        }
        if (wave)
#pragma unroll
            for (int d = 0; d < DT; ++d) join_acc[wave - 1][t * DT + d][lane] = rows.acc[t][d];
    }
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        float top = rows.m[t];
#pragma unroll
        for (int w = 1; w < 4; ++w) top = fmaxf(top, join_ml[w][16 * t + n][0]);
        const float ref = top == kNone ? 0.0f : top;
        const float mine = __builtin_amdgcn_exp2f(rows.m[t] - ref);
        rows.l[t] = scaled_sum(rows.l[t], rows.m[t] - ref);
#pragma unroll
        for (int d = 0; d < DT; ++d) rows.acc[t][d] *= mine;
#pragma unroll
        for (int w = 1; w < 4; ++w) {
            const float other = __builtin_amdgcn_exp2f(join_ml[w][16 * t + n][0] - ref);
            rows.l[t] += scaled_sum(join_ml[w][16 * t + n][1], join_ml[w][16 * t + n][0] - ref);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const f32x4 v = join_acc[w - 1][t * DT + d][lane];
#pragma unroll
                for (int i = 0; i < 4; ++i) rows.acc[t][d][i] = __builtin_fmaf(v[i], other, rows.acc[t][d][i]);
            }
        }
        rows.m[t] = top;
    }
    rows.write(p, tile.parts, blockIdx.z, err);
}

// Many rows (prompts, chunks): each wavefront has 16 * NT rows of its own and all keys.  A block's codes are
// converted to binary16 once by the workgroup, a quarter by each wavefront, into LDS in the order of the
// operands (a fragment is 16 consecutive bytes a lane: no bank conflicts); the next block's codes
// come from memory meanwhile and are converted behind the products, so a block costs one barrier.
// A prompt of 8192 tokens (32 heads of 128 on 8) takes 617 to 672 us, card by card, 820 to 890 TFLOP/s: VALU issue fills 55 % of the cycles (some 390
// instructions a block and wavefront, 80 of them conversions), the matrix cores 37 %; 246 registers leave two wavefronts a
// SIMD.  Binary32 at 128 takes 976 us (both products twice; four registers spilled), heads of 64 477 us,
// heads of 256 2040 us (one wavefront a SIMD).  Converting in every
// wavefront took 1240 us, eight wavefronts a workgroup 827 where four took 755.
template <typename T, int D, int FMT, int NT>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void k_attend_tile(AttendArgs p, int *err) {
    typedef Rows<T, D, FMT, NT> R;
    constexpr int LIMBS = R::LIMBS, KS = R::KS, DT = R::DT;
    __shared__ f16x8 kf[2][4][KS][64], vf[2][DT][2][64];
    __shared__ float sum_ref[4][NT][64];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t n = lane & 15, g = lane / 16;
    Tile tile;
    if (!tile_of(p, 64 * NT, blockIdx.z, err, &tile)) return;
    const uint32_t kvh = tile.kvh;
    R rows;
    rows.load(p, tile.q, min(tile.row0 + wave * 16 * NT, tile.last), tile.last, kvh);
    const bool idle = tile.row0 + wave * 16 * NT > tile.last;  // converts only

    const uint32_t page_mask = p.c.page_size - 1;
    const int32_t *table = p.a.block_table + static_cast<uint64_t>(tile.r) * p.a.max_pages;
    const uint8_t *kc = static_cast<const uint8_t *>(p.c.k), *vc = static_cast<const uint8_t *>(p.c.v);
    const uint32_t kgroup = (lane >> 2) & 3;
    bool missing = false;

    // Codes of block b: K's 16-key tile `wave`, and V's dimension tiles wave DT/4 ...
    u32x4 kraw[D / 64], vraw[DT / 4];
    float ks_next = 0.0f, vs_next = 1.0f;
    bool there_next = false;
    int32_t id_k = 0, id_v = 0;
    auto look = [&](uint32_t b) {  // the table's entries of block b
        const int32_t base = static_cast<int32_t>(64 * b);
        id_k = entry_at(p, tile, table, base + 16 * static_cast<int32_t>(kgroup));
        id_v = entry_at(p, tile, table, base + 16 * static_cast<int32_t>(g));
    };
    auto fetch = [&](uint32_t b) {  // its codes and scales, from the pages that look found
        const int32_t base = static_cast<int32_t>(64 * b);
        const int32_t key_k = base + 16 * static_cast<int32_t>(kgroup), key_v = base + 16 * static_cast<int32_t>(g);
        there_next = is_page(p, tile, id_v, key_v);
        missing |= !there_next && seen(tile, key_v);
        const uint64_t unit_k = static_cast<uint64_t>(is_page(p, tile, id_k, key_k) ? id_k : 0) * p.c.kv_heads + kvh;
        const uint64_t unit_v = static_cast<uint64_t>(there_next ? id_v : 0) * p.c.kv_heads + kvh;
        ks_next = p.c.k_scale[unit_v];
        vs_next = p.c.v_scale[unit_v];
        const uint8_t *kp = kc + ((unit_k << p.page_log2) + (static_cast<uint32_t>(key_k) & page_mask) + 4 * wave + (lane & 3)) * D + g * (D / 4);
#pragma unroll
        for (int j = 0; j < D / 64; ++j) kraw[j] = *reinterpret_cast<const u32x4 *>(kp + 16 * j);
        const uint8_t *vp = vc + ((unit_v * D + 16 * (DT / 4) * wave + n) << p.page_log2) + (static_cast<uint32_t>(key_v) & page_mask);
#pragma unroll
        for (int d = 0; d < DT / 4; ++d) vraw[d] = *reinterpret_cast<const u32x4 *>(vp + (static_cast<uint64_t>(16 * d) << p.page_log2));
    };
    auto convert = [&](uint32_t b) {  // into buffer b & 1
        const uint32_t at = b & 1;
#pragma unroll
        for (int k = 0; k < KS; ++k) kf[at][wave][k][lane] = halves<FMT>(kraw[k / 2][2 * (k % 2)], kraw[k / 2][2 * (k % 2) + 1]);
        if (FMT == kE4m3) {
            const int32_t left = tile.seen_hi - static_cast<int32_t>(64 * b + 16 * g);
            if (__ballot(!there_next || left < 16))
#pragma unroll
                for (int d = 0; d < DT / 4; ++d) keep_bytes(vraw[d], there_next ? left : 0);
        }
#pragma unroll
        for (int d = 0; d < DT / 4; ++d)
#pragma unroll
            for (int c = 0; c < 2; ++c) vf[at][DT / 4 * wave + d][c][lane] = halves<FMT>(vraw[d][2 * c], vraw[d][2 * c + 1]);
    };

    if (tile.b0 < tile.b1) {
        look(tile.b0);
        fetch(tile.b0);
        if (tile.b0 + 1 < tile.b1) look(tile.b0 + 1);
        convert(tile.b0);
    }
    for (uint32_t b = tile.b0; b < tile.b1; ++b) {
        __syncthreads();  // block b is in LDS, and every wavefront is done with block b - 1
        const bool there = there_next;
        const float ks = there ? ks_next : 0.0f, vs = value_scale(vs_next, there);
        if (b + 1 < tile.b1) {
            fetch(b + 1);
            if (b + 2 < tile.b1) look(b + 2);
        }
        const int32_t base = static_cast<int32_t>(64 * b);
        if (!idle && base < rows.any_hi && base > rows.any_lo - 64) {  // base + 64 may be 2^31
            const bool edge = base < rows.all_lo || base > rows.all_hi - 64 || __ballot(there) != ~0ull;
            // Products of one step of dimensions, four key tiles by NT row tiles, do not wait for each other.
            f32x4 s[NT][4];
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const f16x8 kv = kf[b & 1][t][k][lane];
#pragma unroll
                    for (int i = 0; i < LIMBS; ++i)
#pragma unroll
                        for (int u = 0; u < NT; ++u) s[u][t] = mfma(kv, rows.qv[i][u][k], k || i ? s[u][t] : f32x4{0, 0, 0, 0});
                }
            float ff[NT], off[NT], sum[NT] = {};
            rows.scores(s, ks, vs, there, edge, base + 16 * static_cast<int32_t>(g), ff, off, sum_ref[wave]);
            f16x8 pv[2][LIMBS][NT];
            rows.template probabilities<0>(s, pv[0], ff, off, sum);
            rows.template probabilities<1>(s, pv[1], ff, off, sum);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const f16x8 vv = vf[b & 1][d][0][lane];
#pragma unroll
                for (int i = 0; i < LIMBS; ++i)
#pragma unroll
                    for (int u = 0; u < NT; ++u) rows.acc[u][d] = mfma(vv, pv[0][i][u], rows.acc[u][d]);
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const f16x8 vv = vf[b & 1][d][1][lane];
#pragma unroll
                for (int i = 0; i < LIMBS; ++i)
#pragma unroll
                    for (int u = 0; u < NT; ++u) rows.acc[u][d] = mfma(vv, pv[1][i][u], rows.acc[u][d]);
            }
            rows.add(sum, vs);
        }
        if (b + 1 < tile.b1) convert(b + 1);
    }
    if (missing) raise_error(err, kErrIndex);
    if (idle) return;
    rows.total(sum_ref[wave]);
    rows.write(p, tile.parts, blockIdx.z, err);
}

// Joins the parts of the rows that have more than one: WAVES wavefronts a row, which share its parts, a lane
// with D / 64 dimensions; four parts in flight each.
template <typename T, int D, int WAVES>
__global__ __launch_bounds__(256) void k_attend_join(AttendArgs p, uint32_t M, int *err) {
    constexpr int E = D / 64;
    __shared__ float join[WAVES > 1 ? 4 : 1][D + 1];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64, mine = wave % WAVES;
    const uint64_t row = uniform(blockIdx.x * (4 / WAVES) + wave / WAVES), all_rows = static_cast<uint64_t>(p.a.tokens) * p.a.heads;
    if (row >= all_rows) return;
    const uint32_t token = static_cast<uint32_t>(row / p.a.heads), head = static_cast<uint32_t>(row % p.a.heads);
    // The request of the token, 64 candidates at a time.
    uint32_t lo = 0, n = p.a.requests;
    while (n > 1) {
        const uint32_t step = (n + 63) / 64, k = lane * step;
        const uint64_t on = __ballot(k < n && p.a.offsets[lo + k] <= static_cast<int32_t>(token));
        const uint32_t j = on ? 63 - __builtin_clzll(on) : 0;
        n = min(step, n - j * step);
        lo += j * step;
    }
    const uint32_t r = uniform(lo);
    const Request q = request_of(p, r);
    if (token < q.first || token >= q.first + q.n) return;
    const uint32_t rows = q.n * p.group, row0 = ((token - q.first) * p.group + head % p.group) / M * M, last = min(rows, row0 + M) - 1;
    uint32_t b0, b1;
    blocks_of(p, q, row0 / p.group, last / p.group, &b0, &b1);
    const uint32_t parts = uniform(parts_of(p, b1 - b0));
    if (parts <= 1) return;
    float top = kNone;
    for (uint32_t s = lane; s < parts; s += 64) top = fmaxf(top, p.part_ml[2 * (s * all_rows + row)]);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
    const float ref = top == kNone ? 0.0f : top;
    float l = 0.0f, acc[E] = {};
    for (uint32_t s0 = 4 * mine; s0 < parts; s0 += 4 * WAVES) {
        float f[4], pl[4], v[4][E];
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u) {
            const uint64_t at = min(s0 + u, parts - 1) * all_rows + row;
            f[u] = p.part_ml[2 * at];
            pl[u] = p.part_ml[2 * at + 1];
            __builtin_memcpy(v[u], p.part + at * D + E * lane, sizeof v[u]);
        }
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u) {
            const float w = s0 + u < parts ? __builtin_amdgcn_exp2f(f[u] - ref) : 0.0f;
            // A part no key of which the row sees has sums of zero; those of a duplicate count for nothing.
            if (s0 + u < parts) {
                l += scaled_sum(pl[u], f[u] - ref);
#pragma unroll
                for (int i = 0; i < E; ++i) acc[i] = __builtin_fmaf(v[u][i], w, acc[i]);
            }
        }
    }
    if constexpr (WAVES > 1) {
#pragma unroll
        for (int i = 0; i < E; ++i) join[wave][E * lane + i] = acc[i];
        if (lane == 0) join[wave][D] = l;
        __syncthreads();
        if (mine) return;
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i) acc[i] = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            l += join[w][D];
#pragma unroll
            for (int i = 0; i < E; ++i) acc[i] += join[w][E * lane + i];
        }
    }
    const float inv = inverse(l);
    bool bad = false;
    T *out = static_cast<T *>(p.a.out) + token * p.a.out_stride + static_cast<uint64_t>(head) * D + E * lane;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const T v = static_cast<T>(acc[i] * inv);
        bad |= !finite(static_cast<float>(v));
        out[i] = v;
    }
    if (bad) raise_error(err, kErrNonfinite);
}

// How a call runs: rows a workgroup takes, whether its wavefronts share them, and the most splits.
struct Plan {
    uint32_t nt, M, slots, each, splits;
    bool shared;
};
Plan attend_plan(const prism_kv_cache &c, const prism_attention &a, uint32_t cus) {
    const uint32_t group = a.heads / c.kv_heads;
    const uint64_t typical = (static_cast<uint64_t>(a.tokens) * group + a.requests - 1) / a.requests;  // rows of a request
    Plan p;
    // 16 requests of 4000 keys, heads of 128 in binary16, whole tiles against shared rows: 8 rows a request 52 / 34 us, 24
    // 51 / 41, 32 51 / 55, 48 87 / 54, 96 93 / 79; 64 requests of 1000 keys 39 / 34, 40 / 45, 39 / 61, 68 / 43, 74 / 72.
    // Times rise where rows begin another tile, so no one line fits all; binary32 (24 rows 75 / 50, 48 rows 128 / 69) and
    // heads of 256 (174 / 75, 250 / 120) are for shared rows further up.
    p.shared = typical <= 32;
    p.nt = p.shared && (c.head_dim == 256 || typical <= 16) ? 1 : 2;
    p.M = p.shared ? 16 * p.nt : 64 * p.nt;
    p.slots = static_cast<uint32_t>(static_cast<uint64_t>(a.tokens) * group / p.M) + a.requests;
    uint64_t longest = a.max_length;
    if (a.window && longest > a.window + p.M / group) longest = a.window + p.M / group;  // what a tile sees of it
    const uint64_t tiles = static_cast<uint64_t>(p.slots) * c.kv_heads, blocks = longest / 64 + 1;
    uint64_t parts;
    if (p.shared) {
        // Some eight workgroups a CU were every request as long as max_length, so that long requests among
        // short ones do not finish last; eight blocks a part at least, two for each wavefront.  A batch of 64
        // requests up to 8192 keys took 171 us unsplit, with 4 / 8 / 16 / 32 workgroups 140 / 135 / 134 / 140;
        // eight requests up to 65536 keys 168 / 153 / 163 / 173.
        parts = (blocks + 7) / 8;
        if (parts > 8ull * cus / tiles) parts = 8ull * cus / tiles;
    } else {
        // A part writes and reads its rows' sums, as long as five blocks take, so parts have 24 blocks or more
        // (32 blocks a tile: 89 us whole, 111 in parts of 16) until the chip is full, and then up to eight
        // workgroups a CU (79 blocks on 480 tiles: 267 / 241 / 210 us in parts of 76 / 40 / 20), eight
        // blocks where the tiles leave CUs idle.
        parts = blocks / 24;
        if (parts > 8ull * cus / tiles) parts = 8ull * cus / tiles;
        uint64_t fill = 2ull * cus / tiles;
        if (fill > blocks / 8) fill = blocks / 8;
        if (parts < fill) parts = fill;
    }
    if (parts < 1) parts = 1;
    p.each = static_cast<uint32_t>((blocks + parts - 1) / parts);
    p.splits = static_cast<uint32_t>((blocks + p.each - 1) / p.each);
    return p;
}

template <typename T, int D, int FMT>
int attend_launch(const AttendArgs &p, const Plan &plan, int *err, hipStream_t s) {
    const dim3 grid(p.slots * p.c.kv_heads, 1, p.splits);
    constexpr int most = D == 256 ? 1 : 2;  // row tiles of the kernel for few rows
    const bool wide = static_cast<uint64_t>(p.c.pages) * p.c.page_size * p.c.kv_heads * D > 0xffffffffull;
    if (!plan.shared) k_attend_tile<T, D, FMT, 2><<<grid, 256, 0, s>>>(p, err);
    else if (wide && plan.nt == 1) k_attend_rows<T, D, FMT, 1, true><<<grid, 256, 0, s>>>(p, err);
    else if (wide) k_attend_rows<T, D, FMT, most, true><<<grid, 256, 0, s>>>(p, err);
    else if (plan.nt == 1) k_attend_rows<T, D, FMT, 1, false><<<grid, 256, 0, s>>>(p, err);
    else k_attend_rows<T, D, FMT, most, false><<<grid, 256, 0, s>>>(p, err);
    int rc = launch_status();
    if (rc || p.splits == 1) return rc;
    const uint64_t rows = static_cast<uint64_t>(p.a.tokens) * p.a.heads;
    if (p.splits > 8) k_attend_join<T, D, 4><<<static_cast<uint32_t>(rows), 256, 0, s>>>(p, plan.M, err);
    else k_attend_join<T, D, 1><<<static_cast<uint32_t>((rows + 3) / 4), 256, 0, s>>>(p, plan.M, err);
    return launch_status();
}
template <typename T, int D>
int attend_format(const AttendArgs &p, const Plan &plan, int *err, hipStream_t s) {
    return p.c.format == PRISM_CACHE_INT8 ? attend_launch<T, D, kInt8>(p, plan, err, s) : attend_launch<T, D, kE4m3>(p, plan, err, s);
}
template <typename T>
int attend_headed(const AttendArgs &p, const Plan &plan, int *err, hipStream_t s) {
    switch (p.c.head_dim) {
    case 64: return attend_format<T, 64>(p, plan, err, s);
    case 128: return attend_format<T, 128>(p, plan, err, s);
    case 256: return attend_format<T, 256>(p, plan, err, s);
    default: return kLaunchUnsupported;
    }
}

}  // namespace

size_t attention_scratch_bytes(const prism_kv_cache &c, const prism_attention &a, uint32_t cus) {
    const Plan p = attend_plan(c, a, cus);
    return p.splits == 1 ? 0 : sizeof(float) * p.splits * (static_cast<size_t>(a.tokens) * a.heads) * (c.head_dim + 2);
}

int launch_attention_paged(const prism_kv_cache &c, const prism_attention &a, void *scratch, uint32_t cus, int *err, hipStream_t s) {
    const Plan plan = attend_plan(c, a, cus);
    AttendArgs p{c, a, a.heads / c.kv_heads, 0, plan.slots, plan.each, plan.splits, static_cast<float *>(scratch), nullptr};
    p.page_log2 = static_cast<uint32_t>(__builtin_ctz(c.page_size));
    p.part_ml = p.part + static_cast<size_t>(plan.splits) * a.tokens * a.heads * c.head_dim;
    if (a.dtype == PRISM_DTYPE_F32) return attend_headed<float>(p, plan, err, s);
    if (a.dtype == PRISM_DTYPE_F16) return attend_headed<_Float16>(p, plan, err, s);
    return attend_headed<__bf16>(p, plan, err, s);
}

}  // namespace prism
