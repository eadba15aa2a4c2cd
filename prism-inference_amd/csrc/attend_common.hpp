// attend_common.hpp -- what the attention kernels over paged caches share (paged_attention.hip for 8 bits a
// value, paged_attention4.hip for 4): requests, row tiles, the parts of their keys and the join of those parts.
#pragma once

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
// Bytes behind the keys, and stand-ins, may hold NaN codes, which zero probabilities do not silence: the first `keep` of 16 stay.
__device__ __forceinline__ void keep_bytes(u32x4 &v, int32_t keep) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const int32_t left = keep - 4 * w;
        v[w] &= left >= 4 ? ~0u : left <= 0 ? 0u : (1u << (8 * left)) - 1;
    }
}

// Joins the parts of the rows that have more than one: WAVES wavefronts a row, which share its parts, a lane
// with D / 64 dimensions; four parts in flight each.  EARLY (single tokens, where most rows have parts and a load's latency
// counts): the first four are loaded before it is known how many the row has.
template <typename T, int D, int WAVES, bool EARLY = false>
__global__ __launch_bounds__(256) void k_attend_join(AttendArgs p, uint32_t M, int *err) {
    constexpr int E = D / 64;
    __shared__ float join[WAVES > 1 ? 4 : 1][D + 1];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64, mine = wave % WAVES;
    const uint64_t row = uniform(blockIdx.x * (4 / WAVES) + wave / WAVES), all_rows = static_cast<uint64_t>(p.a.tokens) * p.a.heads;
    if (row >= all_rows) return;
    const uint32_t token = static_cast<uint32_t>(row / p.a.heads), head = static_cast<uint32_t>(row % p.a.heads);
    float f[4], pl[4], v[4][E];
    auto load = [&](uint32_t s0, uint32_t n) {
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u) {
            const uint64_t at = min(s0 + u, n - 1) * all_rows + row;
            f[u] = p.part_ml[2 * at];
            pl[u] = p.part_ml[2 * at + 1];
            __builtin_memcpy(v[u], p.part + at * D + E * lane, sizeof v[u]);
        }
    };
    if constexpr (EARLY) load(4 * mine, p.splits);
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
        if (!EARLY || s0 != 4 * mine) load(s0, parts);
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

}  // namespace

}  // namespace prism
