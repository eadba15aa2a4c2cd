// kvcache.hip -- what keeps the paged 8-bit cache of many requests (gfx950): pages and slots
// of a step's new tokens, rotary positions, and the append that quantizes keys and values.
#include <type_traits>

#include "rope_rows.hpp"

namespace prism {

namespace {

// ---- plan -------------------------------------------------------------------------------
// Exclusive sums over the requests of their new tokens, of the pages they need and of those
// they give back; every token's position, page and slot follows from these by itself.  A workgroup
// makes the sums of a few thousand requests in its LDS (a few loads a thread) and fills tokens; many
// tokens take several workgroups, each with sums of its own (2048 requests, 88000 tokens: 13.7 us where sums and
// tokens in two launches took 9.2 and 7.0 and the gap between).  Where the step writes over its own lengths or count they would
// race, and more requests do not fit: there one workgroup makes the sums and a grid fills, whose wavefronts look
// the request of their first token up 64 offsets at a time and the others' in the 64 offsets behind it.

constexpr uint32_t kPlanThreads = 1024;
constexpr uint32_t kPlanOwnTokens = 4096, kPlanOwnRequests = 4096;

struct PlanScratch {
    int32_t *need_base, *back_base;  // [requests + 1]
    int32_t *head;                   // {tokens, free pages, pages given back}
};
PlanScratch plan_scratch(void *p, uint32_t requests) {
    int32_t *i = static_cast<int32_t *>(p);
    return PlanScratch{i, i + requests + 1, i + 2 * (static_cast<size_t>(requests) + 1)};
}

__device__ __forceinline__ int64_t pages_of(int64_t tokens, uint32_t page) { return (tokens + page - 1) / page; }

// The last r in [0, n) with base[r] <= x, for base ascending with base[0] <= x.
__device__ __forceinline__ uint32_t last_at_most(const int32_t *base, uint32_t n, int32_t x) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (base[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}
// The same for a wavefront whose lanes have ascending x.
__device__ __forceinline__ uint32_t last_at_most_wave(const int32_t *base, uint32_t n, int32_t x) {
    const uint32_t lane = threadIdx.x & 63;
    const int32_t x0 = __shfl(x, 0);
    uint32_t lo = 0, left = n;
    while (left > 1) {
        const uint32_t step = (left + 63) / 64, k = lane * step;
        const uint64_t on = __ballot(k < left && base[lo + k] <= x0);
        const uint32_t j = on ? 63 - __builtin_clzll(on) : 0;
        left = min(step, left - j * step);
        lo += j * step;
    }
    const int32_t next = lo + 1 + lane < n ? base[lo + 1 + lane] : 0x7fffffff;
    uint32_t c = 0;  // of the 64 entries behind lo, those at most x
#pragma unroll
    for (uint32_t d = 32; d; d /= 2)
        if (__shfl(next, c + d - 1) <= x) c += d;
    if (c == 63 && __shfl(next, 63) <= x) c = 64;
    return c < 64 ? lo + c : lo + 64 + last_at_most(base + lo + 64, n - lo - 64, x);
}

// Pages given back, on top of the stack: the b-th of them.
__device__ __forceinline__ int32_t page_given_back(const prism_kv_plan &p, const int32_t *back_base, int32_t b) {
    const uint32_t r = last_at_most(back_base, p.requests, b);
    return p.block_table[static_cast<uint64_t>(r) * p.max_pages + (b - back_base[r])];
}

__device__ __forceinline__ void plan_token(const prism_kv_plan &p, const int32_t *back_base, uint32_t t, uint32_t r, int32_t old,
                                           int32_t offset, int32_t need_base, int32_t count, int32_t back, int *err) {
    const int32_t page = static_cast<int32_t>(p.page_size);
    const int32_t position = old + static_cast<int32_t>(t) - offset;
    const int32_t held = static_cast<int32_t>(pages_of(old, p.page_size)), j = position / page, place = position % page;
    int32_t *entry = p.block_table + static_cast<uint64_t>(r) * p.max_pages + j;
    int32_t id;
    if (j < held) {
        id = *entry;
    } else {
        const int32_t k = count + back - 1 - (need_base + j - held);
        id = k < count ? p.free_pages[k] : page_given_back(p, back_base, k - count);
        if (place == 0) *entry = id;  // a new page begins with a new token
    }
    const int64_t s = static_cast<int64_t>(id) * page + place;
    p.positions[t] = position;
    const bool page_ok = id >= 0 && s <= 0x7fffffff;
    if (!page_ok) raise_error(err, kErrIndex);
    p.slots[t] = page_ok ? static_cast<int32_t>(s) : -1;
    p.owners[t] = static_cast<int32_t>(r);
}
__device__ __forceinline__ void plan_no_token(const prism_kv_plan &p, uint32_t t) {
    p.positions[t] = 0;
    p.slots[t] = -1;
    p.owners[t] = -1;
}

__device__ __forceinline__ int64_t wave_inclusive(int64_t v) {
    const uint32_t lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int64_t o = __shfl_up(v, d);
        if (lane >= static_cast<uint32_t>(d)) v += o;
    }
    return v;
}

template <bool OWN>
__global__ __launch_bounds__(kPlanThreads) void k_plan(prism_kv_plan p, PlanScratch sc, int *err) {
    __shared__ int64_t part[3][kPlanThreads / 64];
    __shared__ int bad_any;
    constexpr uint32_t kOwn = OWN ? kPlanOwnRequests : 1;
    __shared__ int32_t own_offset[kOwn], own_old[kOwn], own_need[kOwn], own_back[kOwn];
    const uint32_t tid = threadIdx.x, wave = tid / 64, waves = blockDim.x / 64;
    const bool lead = blockIdx.x == 0;
    if (tid == 0) bad_any = 0;
    __syncthreads();
    const uint32_t each = (p.requests + blockDim.x - 1) / blockDim.x;
    const uint32_t r0 = min(p.requests, tid * each), r1 = min(p.requests, r0 + each);
    int64_t sum[3] = {0, 0, 0};  // tokens, pages needed, pages given back
    bool bad = false;
    for (uint32_t r = r0; r < r1; ++r) {
        const int64_t n = p.lengths[r], a = p.added[r];
        const bool ended = a == -1;
        bad |= n < 0 || a < -1 || pages_of(n + (ended ? 0 : a), p.page_size) > p.max_pages;
        const int64_t held = pages_of(n, p.page_size);
        sum[0] += ended ? 0 : a;
        sum[1] += ended ? 0 : pages_of(n + a, p.page_size) - held;
        sum[2] += ended ? held : 0;
    }
    if (bad) bad_any = 1;
    const int32_t count = *p.free_count;
    int64_t before[3], total[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const int64_t inc = wave_inclusive(sum[i]);
        before[i] = inc - sum[i];
        if ((tid & 63) == 63) part[i][wave] = inc;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        total[i] = 0;
        for (uint32_t w = 0; w < waves; ++w) {
            if (w < wave) before[i] += part[i][w];
            total[i] += part[i][w];
        }
    }
    const bool wrong = bad_any || count < 0 || static_cast<uint32_t>(count) > p.free_capacity ||
                       total[2] > static_cast<int64_t>(p.free_capacity) - count || total[0] > p.max_tokens;
    const int64_t height = count + total[2];
    const int64_t missing = wrong || total[1] <= height ? 0 : total[1] - height;
    const bool refused = wrong || missing > 0;
    for (uint32_t r = r0; r < r1; ++r) {
        const int32_t n = p.lengths[r], a = p.added[r];
        const int32_t offset = refused ? 0 : static_cast<int32_t>(before[0]);
        if (lead) p.offsets[r] = offset;
        if (refused) {
            if (lead) p.new_lengths[r] = n;
            continue;
        }
        if constexpr (OWN) {
            own_offset[r] = offset;
            own_old[r] = n;
            own_need[r] = static_cast<int32_t>(before[1]);
            own_back[r] = static_cast<int32_t>(before[2]);
        } else {
            sc.need_base[r] = static_cast<int32_t>(before[1]);
            sc.back_base[r] = static_cast<int32_t>(before[2]);
        }
        if (lead) p.new_lengths[r] = a == -1 ? 0 : n + a;
        const int64_t held = pages_of(n, p.page_size);
        before[0] += a == -1 ? 0 : a;
        before[1] += a == -1 ? 0 : pages_of(static_cast<int64_t>(n) + a, p.page_size) - held;
        before[2] += a == -1 ? held : 0;
    }
    const int32_t tokens = refused ? 0 : static_cast<int32_t>(total[0]), back = refused ? 0 : static_cast<int32_t>(total[2]);
    if (tid == 0 && lead) {
        p.offsets[p.requests] = tokens;
        p.counts[0] = static_cast<int32_t>(refused ? count : height - total[1]);
        p.counts[1] = tokens;
        p.counts[2] = static_cast<int32_t>(refused ? 0 : total[1]);
        p.counts[3] = static_cast<int32_t>(missing < 0x7fffffff ? missing : 0x7fffffff);
        if constexpr (!OWN) {
            sc.head[0] = tokens;
            sc.head[1] = count;
            sc.head[2] = back;
        }
        if (wrong) raise_error(err, kErrIndex);
        if (missing) raise_error(err, kErrPages);
    }
    if constexpr (OWN) {
        __syncthreads();
        const uint32_t at = blockIdx.x * blockDim.x + tid, step = gridDim.x * blockDim.x;
        for (uint32_t b = at; b < static_cast<uint32_t>(back); b += step)
            p.free_pages[count + b] = page_given_back(p, own_back, static_cast<int32_t>(b));
        for (uint32_t t = at; t < p.max_tokens; t += step) {
            if (static_cast<int32_t>(t) >= tokens) {
                plan_no_token(p, t);
                continue;
            }
            const uint32_t r = last_at_most(own_offset, p.requests, static_cast<int32_t>(t));
            plan_token(p, own_back, t, r, own_old[r], own_offset[r], own_need[r], count, back, err);
        }
    }
}

__global__ __launch_bounds__(256) void k_plan_fill(prism_kv_plan p, PlanScratch sc, int *err) {
    const uint32_t t = blockIdx.x * 256 + threadIdx.x;
    const int32_t tokens = sc.head[0], count = sc.head[1], back = sc.head[2];
    for (int32_t b = static_cast<int32_t>(t); b < back; b += static_cast<int32_t>(gridDim.x * 256))
        p.free_pages[count + b] = page_given_back(p, sc.back_base, b);
    if (static_cast<int32_t>(t & ~63u) < tokens) {
        const uint32_t r = last_at_most_wave(p.offsets, p.requests, static_cast<int32_t>(t));
        if (static_cast<int32_t>(t) < tokens) {
            plan_token(p, sc.back_base, t, r, p.new_lengths[r] - p.added[r], p.offsets[r], sc.need_base[r], count, back, err);
            return;
        }
    }
    if (t < p.max_tokens) plan_no_token(p, t);
}

// ---- rotary positions -------------------------------------------------------------------
// Dims that are multiples of 8 take k_rope (rope_rows.hpp).

// Any dims: a lane has four consecutive elements and looks their partners up, one row in flight (4099 tokens x 24 heads of
// 256 bf16 with 66 dims take 64 us where k_rope takes 26 with 64; 6030 x 40 of 128 with norms 181 where it takes 33).
template <typename T, int D>
__global__ __launch_bounds__(256) void k_rope_any(RopeRows a, RopeRows b, Rotation rot, const int32_t *positions, uint32_t tokens,
                                                  uint32_t heads_each, double eps, int *err) {
    constexpr uint32_t kLanes = D / 4, kRows = 64 / kLanes;
    __shared__ double cs[kRopeTokens][128], sn[kRopeTokens][128];
    const uint32_t lane = threadIdx.x & 63, half = rot.dims / 2;
    const uint32_t t0 = blockIdx.x * kRopeTokens, nt = min(kRopeTokens, tokens - t0);
    rope_table(cs, sn, rot, positions + t0, nt);
    const uint32_t h0 = blockIdx.y * heads_each, h1 = min(a.heads + b.heads, h0 + heads_each);
    const uint32_t groups = (h1 - h0 + kRows - 1) / kRows;
    const uint32_t e0 = 4 * (lane % kLanes);
    bool bad = false, over = false;
    for (uint32_t it = threadIdx.x / 64; it < nt * groups; it += 4) {
        const uint32_t t = it / groups, h = h0 + it % groups * kRows + lane / kLanes;
        const uint32_t hc = min(h, h1 - 1);
        const RopeRows &m = hc < a.heads ? a : b;
        const uint64_t row = static_cast<uint64_t>(hc < a.heads ? hc : hc - a.heads) * D;
        const T *x = static_cast<const T *>(m.x) + (t0 + t) * m.x_stride + row;
        const f32x4 v = load4(x + e0);
        f32x4 partner;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            const uint32_t e = e0 + j;
            const uint32_t o = e >= rot.dims ? e : rot.interleaved ? e ^ 1 : e < half ? e + half : e - half;
            partner[j] = static_cast<float>(x[o]);
        }
        double scale = 1.0;
        if (m.norm) {
            double q = 0.0;
#pragma unroll
            for (int j = 0; j < 4; ++j) q = __builtin_fma(static_cast<double>(v[j]), static_cast<double>(v[j]), q);
#pragma unroll
            for (uint32_t d = 1; d < kLanes; d *= 2) q += __shfl_xor(q, d);
            scale = 1.0 / sqrt(q / D + eps);
        }
        f32x4 out;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            const uint32_t e = e0 + j;
            bad |= !finite(v[j]);
            double y = v[j], z = partner[j];
            if (m.norm) y = y * scale * m.norm[e];
            if (e < rot.dims) {
                const bool first = rot.interleaved ? !(e & 1) : e < half;
                const uint32_t o = rot.interleaved ? e ^ 1 : first ? e + half : e - half;
                const uint32_t k = rot.interleaved ? e / 2 : first ? e : o;
                if (m.norm) z = z * scale * m.norm[o];
                y = first ? __builtin_fma(y, cs[t][k], -(z * sn[t][k])) : __builtin_fma(y, cs[t][k], z * sn[t][k]);
            }
            out[j] = static_cast<float>(y);
        }
        over |= !fits<T>(out);
        if (h < h1) store4(static_cast<T *>(m.out) + (t0 + t) * m.out_stride + row + e0, out);
    }
    if (bad) raise_error(err, kErrInput);
    if (over) raise_error(err, kErrNonfinite);
}

// ---- append -----------------------------------------------------------------------------
// A run is the new tokens of one page: consecutive tokens on consecutive slots.  One workgroup
// takes the keys or values of one head of the runs that begin among its tokens, so a page's
// scale and codes have one writer and no result depends on timing.  Runs that a wavefront's
// registers hold (single tokens above all) go to one wavefront each, longer ones to all four, which
// exchange their magnitudes.  Earlier codes of the page are rewritten only where the scale grew.
// 6030 bf16 tokens of 8 heads of 128 into e4m3 pages of 64 take 17.5 us (37 MB, 2.1 TB/s), 48 ragged f16 chunks of 4 heads of
// 256 20 us, 32 single f32 tokens 4 us: a few chains of loads per wavefront and its VALU work, not yet memory.

template <int FMT>
__device__ __forceinline__ float least_scale(float most) {  // 2^e, most <= qmax 2^e
    const uint32_t u = __float_as_uint(most);
    // qmax is 0.9921875 * 2^7, or 0.875 * 2^9: compare the significand with its.
    constexpr uint32_t significand = FMT == kInt8 ? 0x7e0000u : 0x600000u;
    int e = static_cast<int>(u >> 23) - 126 - (FMT == kInt8 ? 7 : 9) + ((u & 0x7fffffu) > significand ? 1 : 0);
    if (e < -100) e = -100;
    return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

template <int FMT>
__device__ __forceinline__ uint32_t rescale4(uint32_t c, float by) {
    f32x4 v = value4<FMT>(c);
    if constexpr (FMT == kE4m3)  // memory never written may hold NaN codes
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = v[i] == v[i] ? v[i] : 0.0f;
    return code4<FMT>(v * by);
}

struct AppendArgs {
    prism_kv_cache c;
    const void *k, *v;
    uint64_t k_stride, v_stride;
    const int32_t *slots;
    uint32_t tokens;
};

// The bytes of places below `end` among the four from `place` on.
__device__ __forceinline__ uint32_t bytes_below(uint32_t place, uint32_t end) {
    return end >= place + 4 ? ~0u : end <= place ? 0u : (1u << (8 * (end - place))) - 1;
}

// A lane has four dimensions of sixteen places (an aligned group of the page), their loads in
// flight together (places beside the run load its nearest token: no branches, and the same largest
// magnitude); a step is as many groups as the lanes of a wavefront, or of all four, cover.  The
// last step stays in registers; only runs of more than one are read twice.
template <typename T, int FMT, int D>
__device__ __forceinline__ void append_run(const prism_kv_cache &c, const T *x, uint64_t stride, bool is_v, uint32_t head, uint32_t page,
                                           uint32_t first, uint32_t n, bool all, float *shared, int *err) {
    constexpr uint32_t kLanes = D / 4;
    const uint32_t lanes = all ? 256 : 64, lane = threadIdx.x & (lanes - 1), groups = lanes / kLanes;
    const uint32_t e0 = 4 * (lane % kLanes), ps = c.page_size, end = first + n;
    const uint32_t g0 = first / 16, steps = ((end + 15) / 16 - g0 + groups - 1) / groups;
    const uint64_t unit = static_cast<uint64_t>(page) * c.kv_heads + head;
    float *scale = (is_v ? c.v_scale : c.k_scale) + unit;
    uint8_t *codes = static_cast<uint8_t *>(is_v ? c.v : c.k) + unit * ps * D;
    const float before = *scale;
    typename Four<T>::type held[16];
    uint32_t at = 0;  // the lane's group in the step that is held
    auto load = [&](uint32_t step) {
        at = 16 * (g0 + step * groups + lane / kLanes);
#pragma unroll
        for (uint32_t j = 0; j < 16; ++j)
            held[j] = load_any<typename Four<T>::type>(x + (min(max(at + j, first), end - 1) - first) * stride + e0);
    };
    uint32_t most = 0;  // magnitudes compare as integers, NaN and infinities above all others
    for (uint32_t step = 0; step < steps; ++step) {
        load(step);
#pragma unroll
        for (int j = 0; j < 16; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) most = max(most, __float_as_uint(static_cast<float>(held[j][i])) & 0x7fffffffu);
    }
    // What a group of values holds beside the run's places.
    u32x4 had[4];
    const bool whole = at >= first && at + 16 <= end, partial = is_v && !whole && at < end;
    if (partial)
#pragma unroll
        for (int i = 0; i < 4; ++i) had[i] = *reinterpret_cast<const u32x4 *>(codes + (e0 + i) * ps + at);
#pragma unroll
    for (uint32_t d = 1; d < 64; d *= 2) most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), d)));
    if (all) {  // also: every wavefront has read the scale before it is written
        if ((threadIdx.x & 63) == 0) shared[threadIdx.x / 64] = __uint_as_float(most);
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 4; ++w) most = max(most, __float_as_uint(shared[w]));
        __syncthreads();
    }
    const bool bad = most >= 0x7f800000u;
    if (bad) {  // the largest finite magnitude; each wavefront for itself
        raise_error(err, kErrInput);
        most = 0;
        const uint32_t l = threadIdx.x & 63;
        for (uint32_t i = l / kLanes; i < n; i += 64 / kLanes) {
            const f32x4 v = load4(x + i * stride + 4 * (l % kLanes));
#pragma unroll
            for (int k = 0; k < 4; ++k) most = finite(v[k]) ? max(most, __float_as_uint(v[k]) & 0x7fffffffu) : most;
        }
#pragma unroll
        for (uint32_t d = 1; d < 64; d *= 2) most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), d)));
    }
    const float old = first ? before : 0.0f, s = fmaxf(old, least_scale<FMT>(__uint_as_float(most)));
    const float inv = 1.0f / s, by = old * inv;
    const bool grew = first && s != old;
    if (lane == 0) *scale = s;
    if (grew) {  // the codes before the run, at the new scale; a group of values the run shares is done below
        const uint32_t pieces = is_v ? g0 * D : first * D / 16;  // of sixteen bytes
        for (uint32_t i = lane; i < pieces; i += 4 * lanes) {    // four in flight
            u32x4 r[4];
            u32x4 *w[4];
#pragma unroll
            for (uint32_t u = 0; u < 4; ++u) {
                const uint32_t k = min(i + lanes * u, pieces - 1);
                w[u] = reinterpret_cast<u32x4 *>(codes + (is_v ? k % D * ps + 16 * (k / D) : 16 * k));
                r[u] = *w[u];
            }
#pragma unroll
            for (uint32_t u = 0; u < 4; ++u) {
#pragma unroll
                for (int k = 0; k < 4; ++k) r[u][k] = rescale4<FMT>(r[u][k], by);
                if (i + lanes * u < pieces) *w[u] = r[u];
            }
        }
    }
    for (uint32_t step = steps; step-- > 0;) {
        if (step + 1 < steps) load(step);
        if (bad)
#pragma unroll
            for (int j = 0; j < 16; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) held[j][i] = held[j][i] == held[j][i] ? held[j][i] : static_cast<T>(0.0f);
        if (at >= end) continue;
        if (!is_v) {
#pragma unroll
            for (uint32_t j = 0; j < 16; ++j)
                if (at + j >= first && at + j < end)
                    *reinterpret_cast<uint32_t *>(codes + (at + j) * D + e0) = code4<FMT>(__builtin_convertvector(held[j], f32x4) * inv);
            continue;
        }
        const bool kept = at < first || at + 16 > end;  // the group has places beside the run
        if (kept && step + 1 < steps)
#pragma unroll
            for (int i = 0; i < 4; ++i) had[i] = *reinterpret_cast<const u32x4 *>(codes + (e0 + i) * ps + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u32x4 r;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                r[k] = code4<FMT>(f32x4{static_cast<float>(held[4 * k][i]), static_cast<float>(held[4 * k + 1][i]),
                                        static_cast<float>(held[4 * k + 2][i]), static_cast<float>(held[4 * k + 3][i])} * inv);
            if (kept)
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) {
                    const uint32_t low = bytes_below(at + 4 * k, first), below = bytes_below(at + 4 * k, end);
                    const uint32_t again = grew ? rescale4<FMT>(had[i][k], by) : had[i][k];
                    r[k] = (again & low) | (r[k] & below & ~low) | (had[i][k] & ~below);
                }
            *reinterpret_cast<u32x4 *>(codes + (e0 + i) * ps + at) = r;
        }
    }
}

// A run of one token whose page's scale holds it (most tokens of a decode step): nothing else of the page
// changes.  False: not such a run, nothing written.  A batch of 1000 single tokens on 8 heads of 128 spent
// sixteen places' instructions on one: 43 us with their rotation, 29 this way.
template <typename T, int FMT, int D>
__device__ __forceinline__ bool append_token(const prism_kv_cache &c, const T *x, bool is_v, uint32_t head, uint32_t page, uint32_t first) {
    constexpr uint32_t kLanes = D / 4;
    const uint32_t lane = threadIdx.x & 63, e0 = 4 * (lane % kLanes);
    const uint64_t unit = static_cast<uint64_t>(page) * c.kv_heads + head;
    float *scale = (is_v ? c.v_scale : c.k_scale) + unit;
    const float before = *scale;
    const f32x4 v = load4(x + e0);
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) most = max(most, __float_as_uint(v[i]) & 0x7fffffffu);
#pragma unroll
    for (uint32_t d = 1; d < kLanes; d *= 2) most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), d)));
    if (most >= 0x7f800000u) return false;
    const float least = least_scale<FMT>(__uint_as_float(most));
    if (first && !(before >= least)) return false;
    const float s = first ? before : least;
    const uint32_t code = code4<FMT>(v * (1.0f / s));
    uint8_t *codes = static_cast<uint8_t *>(is_v ? c.v : c.k) + unit * c.page_size * D;
    if (lane < kLanes) {
        if (!is_v) {
            *reinterpret_cast<uint32_t *>(codes + first * D + e0) = code;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) codes[(e0 + i) * c.page_size + first] = static_cast<uint8_t>(code >> (8 * i));
        }
    }
    if (lane == 0 && !first) *scale = s;
    return true;
}

// The runs that begin among `each` (at most 32) tokens.
template <typename T, int FMT, int D>
__global__ __launch_bounds__(256) void k_append(AppendArgs a, uint32_t each, int *err) {
    __shared__ float shared[4];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), task = blockIdx.y;
    const uint32_t t0 = blockIdx.x * each, ps = a.c.page_size;
    const int32_t slots = static_cast<int32_t>(a.c.pages * ps);
    // Lane l holds the slot of token t0 - 1 + l.
    const int64_t mine = static_cast<int64_t>(t0) + lane - 1;
    int32_t s = -1;
    if (mine >= 0 && mine < a.tokens) s = a.slots[mine];
    const bool here = lane >= 1 && lane <= each;
    bool bad = here && (s < -1 || s >= slots);
    if (s < 0 || s >= slots) s = -1;
    const int32_t prev = __shfl_up(s, 1);
    const bool follows = prev >= 0 && s == prev + 1 && s % static_cast<int32_t>(ps) != 0;
    bool leads = here && s >= 0 && !follows;
    if (leads && prev >= 0 && prev / static_cast<int32_t>(ps) == s / static_cast<int32_t>(ps)) {
        bad = true;  // a second run in the page
        leads = false;
    }
    if (bad && task == 0 && wave == 0) raise_error(err, kErrIndex);
    const bool is_v = task >= a.c.kv_heads;
    const uint32_t head = is_v ? task - a.c.kv_heads : task;
    const uint64_t stride = is_v ? a.v_stride : a.k_stride;
    // All four wavefronts see the same runs.
    uint32_t turn = 0;
    for (uint64_t left = __ballot(leads); left; left &= left - 1) {
        const int l = __builtin_ctzll(left);
        const uint32_t t = t0 + l - 1, slot = static_cast<uint32_t>(__shfl(s, l));
        const uint32_t page = slot / ps, first = slot % ps, most = min(ps - first, a.tokens - t);
        // How many tokens follow: among the lanes', and further on.
        const uint64_t off = __ballot(static_cast<int>(lane) >= l && static_cast<uint32_t>(s) != slot + lane - l) >> l;
        uint32_t n = off ? __builtin_ctzll(off) : 64 - l;
        if (n == 64u - l)
            for (uint32_t i0 = n; i0 < most; i0 += 64) {
                const uint32_t i = i0 + lane;
                const uint64_t no = ~__ballot(i < most && static_cast<uint32_t>(a.slots[t + i]) == slot + i);
                const uint32_t more = no ? __builtin_ctzll(no) : 64;
                n += more;
                if (more < 64) break;
            }
        n = min(n, most);
        const T *x = static_cast<const T *>(is_v ? a.v : a.k) + t * stride + static_cast<uint64_t>(head) * D;
        constexpr uint32_t kWaveGroups = 64 / (D / 4);
        const bool all = (first + n + 15) / 16 - first / 16 > kWaveGroups;
        if (!all && turn++ % 4 != wave) continue;
        if (n == 1 && append_token<T, FMT, D>(a.c, x, is_v, head, page, first)) continue;
        append_run<T, FMT, D>(a.c, x, stride, is_v, head, page, first, n, all, shared, err);
    }
}

template <typename T, int D>
int rope_typed(const Rotation &rot, const RopeRows &a, const RopeRows &b, const int32_t *positions, uint32_t tokens, float eps,
               int *err, hipStream_t s) {
    const uint32_t tiles = (tokens + kRopeTokens - 1) / kRopeTokens, heads = a.heads + b.heads;
    const bool eights = rot.dims % 8 == 0;
    // Heads are split over workgroups until some 1024 of them share the rows, whole row groups each.
    const uint32_t least = eights ? 64 / (D / 8) : 4 * 64 / (D / 4);
    uint32_t parts = (1024 + tiles - 1) / tiles;
    if (parts > (heads + least - 1) / least) parts = (heads + least - 1) / least;
    const uint32_t each = ((heads + parts - 1) / parts + least - 1) / least * least;
    const dim3 grid(tiles, (heads + each - 1) / each);
    if (!eights) k_rope_any<T, D><<<grid, 256, 0, s>>>(a, b, rot, positions, tokens, each, eps, err);
    else if (rot.interleaved) k_rope<T, D, true, NoAppend><<<grid, 256, 0, s>>>(a, b, rot, positions, tokens, each, eps, NoAppend{}, err);
    else k_rope<T, D, false, NoAppend><<<grid, 256, 0, s>>>(a, b, rot, positions, tokens, each, eps, NoAppend{}, err);
    return launch_status();
}
template <typename T>
int rope_headed(const Rotation &rot, const RopeRows &a, const RopeRows &b, const int32_t *positions, uint32_t tokens,
                uint32_t head_dim, float eps, int *err, hipStream_t s) {
    switch (head_dim) {
    case 64: return rope_typed<T, 64>(rot, a, b, positions, tokens, eps, err, s);
    case 128: return rope_typed<T, 128>(rot, a, b, positions, tokens, eps, err, s);
    case 256: return rope_typed<T, 256>(rot, a, b, positions, tokens, eps, err, s);
    default: return kLaunchUnsupported;
    }
}

template <typename T, int FMT>
int append_headed(const AppendArgs &a, uint32_t each, dim3 grid, int *err, hipStream_t s) {
    switch (a.c.head_dim) {
    case 64: k_append<T, FMT, 64><<<grid, 256, 0, s>>>(a, each, err); break;
    case 128: k_append<T, FMT, 128><<<grid, 256, 0, s>>>(a, each, err); break;
    case 256: k_append<T, FMT, 256><<<grid, 256, 0, s>>>(a, each, err); break;
    default: return kLaunchUnsupported;
    }
    return launch_status();
}
template <typename T>
int append_typed(const AppendArgs &a, uint32_t each, dim3 grid, int *err, hipStream_t s) {
    return a.c.format == PRISM_CACHE_INT8 ? append_headed<T, kInt8>(a, each, grid, err, s)
                                          : append_headed<T, kE4m3>(a, each, grid, err, s);
}

}  // namespace

static bool overlap(const int32_t *a, uint64_t n, const int32_t *b, uint64_t m) { return a < b + m && b < a + n; }

size_t plan_scratch_bytes(uint32_t requests) { return sizeof(int32_t) * (2 * (static_cast<size_t>(requests) + 1) + 4); }

int launch_kv_plan(const prism_kv_plan &p, void *scratch, int *err, hipStream_t s) {
    const PlanScratch sc = plan_scratch(scratch, p.requests);
    const uint32_t wide = p.requests > p.max_tokens ? p.requests : p.max_tokens;
    const uint32_t threads = wide >= kPlanThreads ? kPlanThreads : (wide + 63) / 64 * 64;
    const bool apart = !overlap(p.lengths, p.requests, p.new_lengths, p.requests) && !overlap(p.free_count, 1, p.counts, 4);
    if (p.requests <= kPlanOwnRequests && (apart || p.max_tokens <= kPlanOwnTokens)) {
        uint32_t blocks = p.max_tokens <= kPlanOwnTokens ? 1 : (p.max_tokens + threads - 1) / threads;
        if (blocks > 256) blocks = 256;
        k_plan<true><<<blocks, threads, 0, s>>>(p, sc, err);
        return launch_status();
    }
    k_plan<false><<<1, threads, 0, s>>>(p, sc, err);
    const int rc = launch_status();
    if (rc) return rc;
    k_plan_fill<<<(p.max_tokens + 255) / 256, 256, 0, s>>>(p, sc, err);
    return launch_status();
}

int launch_rope(int dtype, const Rotation &rot, const RopeRows &a, const RopeRows &b, const int32_t *positions,
                uint32_t tokens, uint32_t head_dim, float eps, int *err, hipStream_t s) {
    if (dtype == PRISM_DTYPE_F32) return rope_headed<float>(rot, a, b, positions, tokens, head_dim, eps, err, s);
    if (dtype == PRISM_DTYPE_F16) return rope_headed<_Float16>(rot, a, b, positions, tokens, head_dim, eps, err, s);
    return rope_headed<__bf16>(rot, a, b, positions, tokens, head_dim, eps, err, s);
}

int launch_kv_append(const prism_kv_cache &cache, int dtype, const void *k, uint64_t k_stride, const void *v,
                     uint64_t v_stride, const int32_t *slots, uint32_t tokens, int *err, hipStream_t s) {
    const AppendArgs a{cache, k, v, k_stride, v_stride, slots, tokens};
    const uint32_t each = tokens <= 1024 ? 4 : tokens <= 4096 ? 16 : 32;
    // Tasks of one window far apart: with them side by side a prompt's append took 25 us instead of 17.
    const dim3 grid((tokens + each - 1) / each, 2 * cache.kv_heads);
    if (dtype == PRISM_DTYPE_F32) return append_typed<float>(a, each, grid, err, s);
    if (dtype == PRISM_DTYPE_F16) return append_typed<_Float16>(a, each, grid, err, s);
    return append_typed<__bf16>(a, each, grid, err, s);
}

}  // namespace prism
